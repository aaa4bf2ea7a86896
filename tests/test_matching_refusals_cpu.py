"""Refusals of the matching operators that need sizes of their own (no GPU)."""
import pytest
import torch

from torch_projectors import matching


@pytest.mark.parametrize("images,references", [
    ((2, 100), (3, 120)), ((2, 1), (3, 128)), ((1, 129), (4, 256)), ((2, 5, 20), (3, 10, 12))])
def test_rows_of_different_sizes_are_not_scored(images, references):
    with pytest.raises(ValueError, match="do not fit"):
        matching.block_scores(torch.zeros(images), torch.zeros(references))


def test_complex_rows_count_as_pairs():
    with pytest.raises(ValueError, match="Images of 120 values do not fit references of 100"):
        matching.block_scores(torch.zeros(2, 60, dtype=torch.complex64), torch.zeros(3, 100))
    with pytest.raises(NotImplementedError):  # (these fit: there is no CPU path)
        matching.block_scores(torch.zeros(2, 60, dtype=torch.complex64), torch.zeros(3, 120))
