"""Which 8-bit format is closer to the scores, against 64 bits: integers with a scale a row (row_scores) or blocks of floating
point (block_scores)."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def errors(K, image_fall, reference_fall):
    """Root mean square errors of both formats' scores in units of |image| |reference|; standard deviations of the values fall (or rise) by e^fall
    from a row's first to its last."""
    from torch_projectors import matching as m
    g = torch.Generator(device=DEV).manual_seed(int(K + 10 * image_fall + reference_fall))
    k = torch.linspace(0.0, 1.0, K, device=DEV)
    signal = torch.randn(700, K, generator=g, device=DEV)
    r = signal * torch.exp(-reference_fall * k)
    of = torch.randint(0, 700, (500,), generator=g, device=DEV)
    x = (signal[of] + torch.randn(500, K, generator=g, device=DEV)) * torch.exp(-image_fall * k)
    want = x.double() @ r.double().t()
    size = x.double().norm(dim=1)[:, None] * r.double().norm(dim=1)
    out = [float(((f(x, r).double() - want) / size).square().mean().sqrt()) for f in (m.row_scores, m.block_scores)]
    print(f"K {K} falls {image_fall} {reference_fall}: rows {out[0]:.2e} blocks {out[1]:.2e}", flush=True)
    return out


@pytest.mark.parametrize("K", [4224, 16640])
@pytest.mark.parametrize("fall", [0.0, 4.6, 9.2])
def test_integers_are_closer_where_large_values_meet(gpu, K, fall):
    """Whitened rows, and rows that fall alike on both sides.  A row's largest of K values is some 4 standard deviations, so that a code is off by
    4 / 127 / sqrt(12) = 0.9 % of one; three bits of a mantissa are off by 2.6 % of each value."""
    rows, blocks = errors(K, fall, fall)
    assert rows < 0.5 * blocks


@pytest.mark.parametrize("K", [4224, 16640])
def test_blocks_are_closer_where_small_values_meet_large_ones(gpu, K):
    """Images that rise by four orders of magnitude where the references fall: what counts is below an integer's step on either side."""
    rows, blocks = errors(K, -9.2, 9.2)
    assert blocks < 0.5 * rows
