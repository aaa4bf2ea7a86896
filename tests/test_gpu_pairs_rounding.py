"""What gradients of pair log probabilities may lose to rounding: no more for one image because of what another's unused upstream
gradient holds."""
import pytest
import torch

from tests.test_gpu_pairs import BF16, DEV, F16, F32, NAN, check, gen, m, near, problem, run, want  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("M", [5, 20, 1100])
@pytest.mark.parametrize("unused", ["none given", "not finite"])
def test_unused_upstream_gradients(m, M, unused, dtype):  # noqa: F811
    """An image without a given reference, and one whose results are not finite, change nothing of the others' gradients, however large
    their upstream gradients are."""
    p = problem(M, 60, 40, dtype, seed=51)
    p["given"] = p["given"].clamp_min(0)
    if unused == "none given":
        p["given"][1], p["d_given"][1] = -1, -1e30
        check(m, p)
    else:
        p["images"][1, 3], p["d_given"][1], p["d_log_sum"][1] = NAN, 1e30, -1e30
        got = run(m, p)["d_images"]
        others = torch.arange(M, device=DEV) != 1
        alone = {k: v[others] if k in ("images", "given", "d_given", "d_log_sum") else v for k, v in p.items()}
        w = want(alone)
        near(got[others], w["d_images"], w["tol_d_images"], "d_images")
        assert got[1].isnan().all()


# tiles of each size, straight to LDS and staged (rows of an odd size), whole and in ranges
ROUNDED = [(70, 90, 136), (70, 90, 131), (300, 700, 264), (333, 1999, 2064), (333, 1999, 2070), (500, 4000, 1030), (4096, 4200, 4224), (4096, 4200, 4225),
           (4000, 100, 8192), (128, 4096, 8192), (2048, 17000, 64)]


def half_step(value, dtype):
    """Half the distance of the type's numbers next to a magnitude."""
    bits, least = (7, -133) if dtype == BF16 else (10, -24)
    e = torch.floor(torch.log2(value.clamp_min(2.0 ** -140)))
    return 0.5 * torch.exp2((e - bits).clamp_min(least))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("M,N,K", ROUNDED)
def test_gradients_of_half_rows_are_rounded_once(m, M, N, K, dtype):  # noqa: F811
    """From 16-bit rows the gradients are those of float32 rows of the same values, rounded at the end: within half a step of the type, and
    what sums in 32 bits lose.

    The scores' gradient G goes through 16-bit units in two pieces, which leave at most 2^-16 of it (bfloat16; 2^-22 in half
    precision, and 2^-25 of 2^-13 of the largest upstream gradient); sums of 2 n products lose (2 n + 16) 2^-24 of the magnitudes.
    The bound for float32 rows has (6 n + 16) 2^-24 for that: enough for n of at least 64, as here."""
    assert min(M, N) >= 64
    p = problem(M, N, K, dtype, seed=52)
    got = run(m, p)
    w = want({**p, "images": p["images"].float(), "references": p["references"].float()})
    tiny = 0.0
    if dtype == F16:
        tiny = 2.0 ** -37 * float((p["d_given"].abs() + p["d_log_sum"].abs()).max()) / p["temperature"]
    for k, other in (("d_images", "references"), ("d_references", "images")):
        tol = w["tol_" + k] + tiny * p[other].double().abs().sum(0)
        near(got[k], w[k], tol + half_step(w[k].abs() + tol, dtype), k)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("M,N,K", [(9, 1, 8), (65, 63, 72), (333, 129, 264), (333, 129, 131), (4097, 4095, 72)])
def test_last_image_and_last_reference(m, M, N, K, dtype):  # noqa: F811
    """Odd numbers of both: the last value of the scores' gradient is read where its operand ends."""
    p = problem(M, N, K, dtype, seed=53)
    p["mask"][:] = False
    p["mask"][N - 1] = True
    p["given"][:] = -1
    p["given"][::2] = N - 1
    got, w = run(m, p), want(p)
    assert (w["d_images"][M - 1].abs().max() > 0) and (w["d_references"][N - 1].abs().max() > 0)
    for k, v in got.items():
        near(v, w[k], w["tol_" + k], k)
