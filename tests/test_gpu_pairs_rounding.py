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
