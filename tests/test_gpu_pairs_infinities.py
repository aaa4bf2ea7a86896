"""Pair log probabilities whose scores are not finite: the same for all types and numbers of images.  An allowed reference's score
that is NaN or an infinity of either sign makes its image's results NaN, and no other image's."""
import pytest
import torch

from tests.test_gpu_pairs import BF16, DEV, F16, F32, INF, gen, m, problem, run  # noqa: F401

pytestmark = pytest.mark.gpu
SIZES = [(1, 140, 72), (8, 140, 72), (9, 140, 72), (9, 40, 5000), (300, 700, 136), (300, 700, 131), (1100, 1300, 72)]


def no_results(got, p, rows):
    """NaN for these images, and in what references and biases get from them; nothing else changes."""
    none = p["given"] == -1
    assert got["log_sum"][rows].isnan().all()
    assert got["given"][rows & ~none].isnan().all() and (got["given"][none] == 0).all()
    assert got["d_images"][rows].isnan().all()
    allowed = p["mask"]
    assert got["d_references"][allowed].isnan().all() and (got["d_references"][~allowed] == 0).all()
    assert got["d_bias"][allowed].isnan().all() and (got["d_bias"][~allowed] == 0).all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("held", [INF, -INF])
@pytest.mark.parametrize("M,N,K", SIZES)
def test_infinite_value_of_a_reference(m, M, N, K, held, dtype):  # noqa: F811
    p = problem(M, N, K, dtype, seed=41)
    at = int(p["mask"].nonzero()[-1])
    p["references"][at, 5] = held
    no_results(run(m, p), p, torch.ones(M, dtype=torch.bool, device=DEV))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("held", [INF, -INF])
@pytest.mark.parametrize("M,N,K", SIZES)
def test_infinite_value_of_an_image(m, M, N, K, held, dtype):  # noqa: F811
    p = problem(M, N, K, dtype, seed=42)
    clean = run(m, p)
    p["images"][M - 1, K - 1] = held
    got = run(m, p)
    rows = torch.arange(M, device=DEV) == M - 1
    no_results(got, p, rows)
    for k in ("log_sum", "given", "d_images"):
        assert torch.equal(got[k][~rows], clean[k][~rows]), k


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("M,N,K", SIZES[1:])
def test_scores_past_the_largest_number(m, M, N, K, sign, dtype):  # noqa: F811
    """Finite values whose product is 1e60 or -1e60: one image's score alone."""
    p = problem(M, N, K, dtype, seed=43)
    p["images"][:, 0] = 0
    p["references"][:, 0] = 0
    clean = run(m, p)
    at = int(p["mask"].nonzero()[0])
    p["images"][2, 0], p["references"][at, 0] = sign * 1e30, 1e30
    got = run(m, p)
    rows = torch.arange(M, device=DEV) == 2
    no_results(got, p, rows)
    for k in ("log_sum", "given"):
        assert torch.equal(got[k][~rows], clean[k][~rows]), k
    assert torch.equal(got["d_images"][~rows, 1:], clean["d_images"][~rows, 1:])
    assert torch.isfinite(got["d_images"][~rows]).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("M", [3, 20])
@pytest.mark.parametrize("held", [float("nan"), INF])
def test_bias_that_is_not_finite(m, M, held, dtype):  # noqa: F811
    p = problem(M, 90, 64, dtype, seed=44)
    p["bias"][int(p["mask"].nonzero()[3])] = held
    no_results(run(m, p), p, torch.ones(M, dtype=torch.bool, device=DEV))
