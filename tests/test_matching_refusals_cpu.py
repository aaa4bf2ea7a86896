"""Refusals of the matching operators that need sizes of their own (no GPU)."""
import ctypes

import pytest
import torch

from torch_projectors import capi, matching


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


A, NULL = ctypes.c_void_p(256), ctypes.c_void_p(None)


@pytest.mark.parametrize("M,N,nb", [(333, 1999, 65), (2050, 200, 130), (500, 4099, 130)])
def test_small_workspaces_of_products_in_ranges_are_refused(M, N, nb):
    """Products that add up ranges of the blocks need their sums' room."""
    lib = capi.lib()
    need = lib.tp_block_scores_work(M, N, nb)
    assert need > 0 and need % (4 * M * N) == 0

    def call(work, size):
        return lib.tp_block_scores(A, A, M, A, A, N, nb, NULL, capi.TP_F32, A, work, size, NULL)

    assert call(A, need - 1) == capi.TP_ERR_INVALID and "work is smaller" in lib.tp_last_error().decode()
    assert call(A, 0) == capi.TP_ERR_INVALID and "work is smaller" in lib.tp_last_error().decode()
    assert call(NULL, need) == capi.TP_ERR_INVALID and "work must not be NULL" in lib.tp_last_error().decode()


@pytest.mark.parametrize("T,V,top", [(1, 1 << 20, 8), (8, 294912, 16), (300, 70001, 0)])
def test_small_workspaces_of_rows_in_parts_are_refused(T, V, top):
    lib = capi.lib()
    need = lib.tp_log_probs_work(T, V, top)
    assert need > 0
    outs = [A, A, A, A, A, A]

    def call(work, size):
        return lib.tp_log_probs(capi.TP_F32, A, T, V, V, NULL, 0, NULL, 0, top, 1.0, *outs, work, size, NULL)

    assert call(A, need - 1) == capi.TP_ERR_INVALID and "work is smaller" in lib.tp_last_error().decode()
    assert call(NULL, need) == capi.TP_ERR_INVALID and "work must not be NULL" in lib.tp_last_error().decode()


@pytest.mark.parametrize("n,E", [(4097, 16), (1 << 20, 64), (2049, 4096)])
def test_small_workspaces_of_sorts_in_stretches_are_refused(n, E):
    lib = capi.lib()
    need = lib.tp_sort_by_class_work(n, E)
    assert need > 0

    def call(work, size):
        return lib.tp_sort_by_class(8, A, n, E, A, A, A, work, size, NULL)

    assert call(A, need - 1) == capi.TP_ERR_INVALID and "work is smaller" in lib.tp_last_error().decode()
    assert call(NULL, need) == capi.TP_ERR_INVALID and "work must not be NULL" in lib.tp_last_error().decode()
