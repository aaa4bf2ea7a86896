"""What references that are ruled out hold, and scores that are not finite, in the largest tiles and in several pieces: the masked loads of
every stage, masks and biases from a piece's first reference on, and a flag that outlives the piece which raised it."""
import pytest
import torch

from tests.test_gpu_pairs import BF16, DEV, F16, F32, INF, NAN, m, problem, run  # noqa: F401

pytestmark = pytest.mark.gpu
# images' gradients in 256 x 256 tiles (float32: 256 x 128) of one piece and of two
MASKED = [(F32, 8192, 8192, 1024), (F16, 8192, 8192, 4096), (BF16, 8192, 8192, 4096), (BF16, 4000, 100, 8192)]


@pytest.mark.parametrize("dtype,M,N,K", MASKED)
def test_what_ruled_out_references_hold(m, dtype, M, N, K):  # noqa: F811
    p = problem(M, N, K, dtype, seed=71)
    clean = run(m, p)
    assert not any(v.isnan().any() for v in clean.values())
    out = ~p["mask"]
    for which in (out & (torch.arange(N, device=DEV) >= N // 2), out & (torch.arange(N, device=DEV) == out.nonzero()[0]), out):
        bad = {**p, "references": p["references"].clone(), "bias": p["bias"].clone()}
        bad["references"][which] = NAN
        bad["references"][which, ::3] = INF
        bad["bias"][which] = NAN
        got = run(m, bad)
        for k in got:
            assert torch.equal(got[k], clean[k]), (k, int(which.sum()))


# scores in 256 x 256 tiles (float32: 256 x 128), whole and in ranges
LARGE = [(F32, 4096, 4096, 520), (F32, 1100, 1500, 16640), (F16, 4096, 4096, 520), (BF16, 2048, 4100, 264)]


@pytest.mark.parametrize("held", [INF, -INF, NAN])
@pytest.mark.parametrize("dtype,M,N,K", LARGE)
def test_scores_that_are_not_finite(m, dtype, M, N, K, held):  # noqa: F811
    p = problem(M, N, K, dtype, seed=72)
    p["given"] = p["given"].clamp_min(0)
    clean = run(m, p)
    rows = torch.zeros(M, dtype=torch.bool, device=DEV)
    rows[[3, M // 2 + 1, M - 1]] = True
    p["images"][rows, 7] = held
    got = run(m, p)
    for k in ("log_sum", "given", "d_images"):
        assert torch.equal(got[k][~rows], clean[k][~rows]) and got[k][rows].isnan().all(), k
    for k in ("d_references", "d_bias"):
        assert got[k][p["mask"]].isnan().all() and (got[k][~p["mask"]] == 0).all(), k
