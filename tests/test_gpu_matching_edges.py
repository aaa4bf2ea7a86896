"""The matching operators where their definitions have ends: rows that are not finite, candidates out of range, many
given candidates, blocks at the ends of fp32's range, orders from elsewhere."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def m(gpu):
    from torch_projectors import matching
    return matching


def gen(seed):
    return torch.Generator().manual_seed(seed)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("V", [50, 3001])
def test_masked_places_have_no_gradient_in_rows_that_are_not_finite(m, V, dtype):
    """A NaN or +inf among the allowed scores, or an upstream gradient that is not finite: NaN or infinite gradients
    where scores are allowed, 0 where they are masked or -inf."""
    x = torch.randn(5, V, generator=gen(1)).to(dtype)
    x[1, 4], x[2, V - 1] = math.nan, math.inf
    x[:, 7] = -math.inf
    mask = torch.ones(V, dtype=torch.bool)
    mask[10:20] = False
    mask[V // 2:V - 3] = False
    s = x.to(DEV).requires_grad_()
    out = m.log_probs(s, mask=mask.to(DEV))
    up = torch.tensor([1.0, 1.0, 1.0, math.nan, math.inf])
    (d,) = torch.autograd.grad([out.log_sum, out.entropy], [s], [up.to(DEV), torch.full((5,), 0.1, device=DEV)])
    d = d.cpu()
    assert (d[:, ~mask] == 0).all() and (d[:, 7] == 0).all()
    allowed = mask.clone()
    allowed[7] = False
    assert torch.isfinite(d[0]).all() and d[1:4, allowed].isnan().all()
    assert not torch.isfinite(d[4, allowed]).any()


@pytest.mark.parametrize("G", [1, 3, 90])
@pytest.mark.parametrize("index", [300, 10 ** 12, -2, -(2 ** 63)])
def test_gradient_of_given_candidates_out_of_range(m, index, G):
    """Their log probability is NaN, and so is the gradient of their row, but for masked places; of a result that has no
    share in the loss (an upstream gradient of 0) there is none."""
    V = 300
    x = torch.randn(4, V, generator=gen(2))
    mask = torch.rand(V, generator=gen(3)) < 0.8
    given = torch.randint(0, V, (4, G), generator=gen(4))
    mask[given.flatten()] = True
    mask[5] = False
    given[given == 5] = -1
    fine = given.clone()
    given[1:, G // 2] = index
    fine[1:, G // 2] = -1
    up = torch.randn(4, G, generator=gen(5))
    up[2, G // 2] = 0.0

    def gradient(which):
        s = x.to(DEV).requires_grad_()
        out = m.log_probs(s, which.to(DEV), mask=mask.to(DEV))
        return out.given.detach().cpu(), torch.autograd.grad(out.given, s, up.to(DEV))[0].cpu()

    got, d = gradient(given)
    want, d_fine = gradient(fine)
    assert got[1:, G // 2].isnan().all() and int(got.isnan().sum()) == 3
    assert torch.equal(d[[0, 2]], d_fine[[0, 2]]) and torch.isfinite(d[[0, 2]]).all()
    assert d[[1, 3]][:, mask].isnan().all() and (d[:, ~mask] == 0).all()
