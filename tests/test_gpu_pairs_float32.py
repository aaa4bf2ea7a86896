"""What float32 products as products of bfloat16 pieces lose, measured against 64 bits: tolerances that a lost piece, a sum without its
second set of registers or an error that all products have the sign of do not meet."""
import pytest
import torch

from tests.test_gpu_pairs import DEV, F32, gen, m  # noqa: F401

pytestmark = pytest.mark.gpu


def off(got, want):
    return (got.double() - want) / want


@pytest.mark.parametrize("M", [9, 300, 5000])
def test_values_whose_pieces_are_largest(m, M):  # noqa: F811
    """1 + 2^-7 - 2^-23: cut off, not rounded, its pieces are 1, 2^-7 and 2^-15, almost, and what the six products leave out is 2^-21.
    Rounded they leave nothing out, and the sum of six loses a rounding or two of float32: below 2^-22."""
    x = torch.full((M, 1), 1 + 2.0 ** -7 - 2.0 ** -23, device=DEV)
    for r in (x[:1], -x[:1]):
        s = m.pair_log_probs(x, r).log_sum
        assert (off(s, x[:, 0].double() * r[0, 0].double()).abs() < 2.0 ** -22).all()


def test_what_is_left_out_has_no_sign(m):  # noqa: F811
    """Sums of 16 products of random mantissas, one sign: the mean of 65536 errors of either sign, 6e-8 each, is below
    5e-9 or so; products that are all pulled by 2^-25 of themselves (the mean of two pieces' products that are cut off) make it 4e-8."""
    g = gen(61)
    x, r = 1 + torch.rand(65536, 16, generator=g, device=DEV), 1 + torch.rand(1, 16, generator=g, device=DEV)
    error = off(m.pair_log_probs(x, r).log_sum, (x.double() @ r.double().t())[:, 0])
    assert float(error.mean().abs()) < 1.5e-8 and float(error.abs().max()) < 3e-7


# (images, references, values): 64 x 64 and 128 x 128 tiles of the images' gradient, in ranges and whole, and of the references'
LONG_SUMS = [(64, 100000, 64), (9, 1000000, 16), (640, 30000, 640), (30000, 20, 32), (20000, 600, 520)]


@pytest.mark.parametrize("M,N,K", LONG_SUMS)
def test_long_sums_of_gradients(m, M, N, K):  # noqa: F811
    """Terms of one sign: what sums over all references or images lose adds up.  With a second set of registers 1.5e-7 on average and 5e-7 at
    most; without, 2.8e-6 over 3125 terms and 1e-5 over 31250."""
    g = gen(62)
    x = (0.01 * torch.rand(M, K, generator=g, device=DEV)).requires_grad_()
    r = (1 + torch.rand(N, K, generator=g, device=DEV)).requires_grad_()
    dx, dr = torch.autograd.grad(m.pair_log_probs(x, r).log_sum.sum(), (x, r))
    x64, r64 = x.detach().double(), r.detach().double()
    p = torch.softmax(x64 @ r64.t(), 1)
    for name, error in (("d_images", off(dx, p @ r64)), ("d_references", off(dr, p.t() @ x64))):
        print(name, float(error.mean()), float(error.square().mean().sqrt()), float(error.abs().max()))
        assert float(error.mean().abs()) < 3e-7 and float(error.abs().max()) < 2e-6, name


# 128 x 128 and 256 x 128 tiles of the scores, in ranges and whole
LONG_ROWS = [(100, 5000, 8280), (500, 1000, 16640), (1100, 1500, 16640), (2048, 4096, 16640)]


@pytest.mark.parametrize("M,N,K", LONG_ROWS)
def test_long_rows_of_large_tiles(m, M, N, K):  # noqa: F811
    """Scores of 16640 positive products: 7e-8 off on average.  One of the six products of pieces is 7e-6 of them or more, and one set
    of registers loses 4.8e-6."""
    g = gen(63)
    x, r = torch.rand(M, K, generator=g, device=DEV), 1 + torch.rand(N, K, generator=g, device=DEV)
    out = m.pair_log_probs(x, r, bias=-(torch.arange(N, device=DEV) % 7 * 100.0), temperature=40.0)
    z = (x.double() @ r.double().t() - (torch.arange(N, device=DEV) % 7 * 100.0).double()) / 40.0
    error = off(out.log_sum, torch.logsumexp(z, 1))
    print(float(error.square().mean().sqrt()), float(error.abs().max()))
    assert float(error.abs().max()) < 1e-6


@pytest.mark.parametrize("power", [108, 116, 124, 132, 140])
@pytest.mark.parametrize("M", [8, 64])
def test_values_next_to_the_smallest(m, M, power):  # noqa: F811
    """The pieces' last bits end at 2^-133: of more than 8 images a value is off by less than that."""
    g = gen(64)
    x = (1 + torch.rand(M, 16, generator=g, device=DEV)) * 2.0 ** min(power - 6, 120)
    r = ((1 + torch.rand(1, 16, generator=g, device=DEV, dtype=torch.float64)) * 2.0 ** -power).float()
    z = (x.double() @ r.double().t())[:, 0]
    error = (m.pair_log_probs(x, r).log_sum.double() - z).abs()
    assert (error <= 5e-7 * z + (2.0 ** -133 * x.double().sum(1) if M > 8 else 0.0)).all()
