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
