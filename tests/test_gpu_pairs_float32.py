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
