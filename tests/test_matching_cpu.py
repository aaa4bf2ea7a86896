"""The matching operators' boundary without a GPU: registrations, refusals of both the Python functions
and the C ABI, no CPU path, and the 64-bit definitions that the GPU tests compare with, checked against
torch's own functions."""
import ctypes
import math

import pytest
import torch

from tests import matching_reference as R
from torch_projectors import capi, matching

_P = ctypes.c_void_p
OPS = ("quantize_blocks", "block_scores", "log_probs", "log_probs_back", "sort_by_class", "spread_rows", "gather_rows")


@pytest.mark.parametrize("name", OPS)
def test_gpu_kernel_registered_and_no_cpu_kernel(name):
    op = f"torch_projectors::{name}"
    assert torch._C._dispatch_has_kernel_for_dispatch_key(op, "CUDA")
    assert not torch._C._dispatch_has_kernel_for_dispatch_key(op, "CPU")


ORDER = matching.ClassOrder(torch.zeros(6, dtype=torch.int32), torch.zeros(3, 2, dtype=torch.int32),
                            torch.zeros(4, dtype=torch.int32))


@pytest.mark.parametrize("call", [
    lambda: matching.quantize_blocks(torch.zeros(2, 3)),
    lambda: matching.block_scores(torch.zeros(2, 3), torch.zeros(2, 3)),
    lambda: matching.log_probs(torch.zeros(2, 3)),
    lambda: matching.log_probs(torch.zeros(2, 3, requires_grad=True)),
    lambda: matching.sort_by_class(torch.zeros(2, dtype=torch.int64), 3),
    lambda: matching.dispatch(torch.zeros(3, 4), ORDER),
    lambda: matching.combine(torch.zeros(6, 4), ORDER, torch.zeros(3, 2)),
])
def test_cpu_tensors_fail_loudly(call):
    with pytest.raises(NotImplementedError):
        call()


@pytest.mark.parametrize("call,msg", [
    (lambda: matching.quantize_blocks(torch.zeros(())), "at least 1 dimension"),
    (lambda: matching.log_probs(torch.zeros(())), "at least 1 dimension"),
    (lambda: matching.log_probs(torch.zeros(3, 4), torch.zeros(2, dtype=torch.int64)), "leading dimensions"),
    (lambda: matching.log_probs(torch.zeros(3, 4), torch.zeros(3, 2, 1, dtype=torch.int64)), "leading dimensions"),
    (lambda: matching.log_probs(torch.zeros(3, 4), mask=torch.ones(3, dtype=torch.bool)), "Mask"),
    (lambda: matching.log_probs(torch.zeros(3, 4), mask=torch.ones(1, 4, dtype=torch.bool)), "Mask"),
    (lambda: matching.sort_by_class(torch.zeros((), dtype=torch.int64), 3), "rows, choices"),
    (lambda: matching.sort_by_class(torch.zeros(2, 2, 2, dtype=torch.int64), 3), "rows, choices"),
    (lambda: matching.dispatch(torch.zeros(4, 5), ORDER), "must have 3 rows"),
    (lambda: matching.combine(torch.zeros(3, 5), ORDER), "must have 6 rows"),
    (lambda: matching.combine(torch.zeros(6, 5), ORDER, torch.zeros(2, 3)), "Weights"),
    (lambda: matching.combine(torch.zeros(6, 5), ORDER, torch.zeros(3)), "Weights"),
])
def test_python_argument_checks(call, msg):
    with pytest.raises(ValueError, match=msg):
        call()


def _refused(name, args, msg):
    assert getattr(capi.lib(), name)(*args) == capi.TP_ERR_INVALID
    assert msg in capi.lib().tp_last_error().decode()


A, NULL = _P(256), _P(None)


@pytest.mark.parametrize("name,good,bad", [
    ("tp_quantize_blocks", dict(dt=0, x=A, rows=2, cols=3, stride=3, codes=A, scales=A, stream=NULL), [
        (dict(dt=1), "dtype"), (dict(dt=9), "dtype"), (dict(rows=-1), "non-negative"), (dict(cols=1 << 31), "2^31"),
        (dict(stride=-3), "row_stride"), (dict(x=NULL), "x"), (dict(codes=NULL), "codes"), (dict(scales=NULL), "scales")]),
    ("tp_block_scores", dict(a=A, sa=A, M=2, b=A, sb=A, N=3, nb=1, bias=NULL, dt=0, out=A, work=A, bytes=1 << 40, stream=NULL), [
        (dict(dt=3), "out_dtype"), (dict(nb=0), "blocks"), (dict(M=-1), "non-negative"), (dict(N=1 << 27), "2^26"), (dict(nb=1 << 25), "blocks"),
        (dict(a=NULL), "codes_a"), (dict(sb=NULL), "scales_b"), (dict(out=NULL), "scores")]),
    ("tp_log_probs", dict(dt=0, x=A, T=2, V=3, stride=3, given=NULL, G=0, mask=NULL, ms=0, top=1, temp=1.0, go=A, h=A, l=A,
                          to=A, ti=A, st=A, work=A, bytes=1 << 40, stream=NULL), [
        (dict(dt=1), "dtype"), (dict(V=0), "at least one"), (dict(top=65), "top"), (dict(top=-1), "top"),
        (dict(temp=0.0), "temperature"), (dict(temp=-1.0), "temperature"), (dict(temp=math.nan), "temperature"),
        (dict(temp=math.inf), "temperature"), (dict(temp=1e-300), "temperature"), (dict(G=1), "given"),
        (dict(stride=-1), "strides"), (dict(T=1 << 31), "2^31"), (dict(x=NULL), "scores"), (dict(ti=NULL), "top_index")]),
    ("tp_score_images", dict(dt=0, x=A, M=2, cols=200, stride=200, b=A, sb=A, N=3, bias=NULL, odt=4, out=A, work=A,
                             bytes=1 << 40, stream=NULL), [
        (dict(dt=1), "dtype"), (dict(odt=3), "out_dtype"), (dict(cols=0), "cols"), (dict(cols=1 << 24), "blocks"),
        (dict(M=-1), "non-negative"), (dict(stride=-1), "row_stride"), (dict(x=NULL), "x"), (dict(work=NULL), "work"),
        (dict(bytes=10), "work is smaller"), (dict(sb=NULL), "scales_b"), (dict(out=NULL), "scores")]),
    ("tp_log_probs_back", dict(dt=0, x=A, T=2, V=3, stride=3, given=NULL, G=0, mask=NULL, ms=0, top=1, temp=1.0, ti=A, st=A,
                               dg=NULL, dh=NULL, dl=NULL, dt_=A, out=A, stream=NULL), [
        (dict(dt=2), "dtype"), (dict(ti=NULL), "top_index"), (dict(st=NULL), "stats"), (dict(out=NULL), "d_scores"),
        (dict(temp=0.0), "temperature")]),
    ("tp_sort_by_class", dict(b=8, ids=A, n=4, E=3, order=A, slot=A, off=A, work=A, bytes=1 << 40, stream=NULL), [
        (dict(b=2), "4 or 8"), (dict(n=-1), "slots"), (dict(n=(1 << 30) + 1), "slots"), (dict(E=0), "classes"),
        (dict(E=4097), "classes"), (dict(ids=NULL), "class_ids"), (dict(off=NULL), "offsets")]),
    ("tp_spread_rows", dict(dt=0, x=A, T=2, D=3, k=1, slot=A, kept=A, w=NULL, out=A, other=NULL, dw=NULL, stream=NULL), [
        (dict(dt=1), "dtype"), (dict(T=-1), "non-negative"), (dict(T=1 << 20, k=1 << 11), "2^31"), (dict(slot=NULL), "slot"),
        (dict(kept=NULL), "kept"), (dict(other=A), "together"), (dict(dw=A), "together"), (dict(x=NULL), "x"),
        (dict(out=NULL), "sorted")]),
    ("tp_gather_rows", dict(dt=0, y=A, T=2, D=3, k=1, slot=A, kept=A, w=NULL, out=A, other=NULL, dw=NULL, stream=NULL), [
        (dict(dt=1), "dtype"), (dict(D=-1), "non-negative"), (dict(other=A), "together"), (dict(y=NULL), "sorted"),
        (dict(out=NULL), "out")]),
])
def test_c_abi_refuses_before_anything_is_enqueued(name, good, bad):
    assert len(good) == len(capi.SIGNATURES[name])
    for change, msg in bad:
        _refused(name, list({**good, **change}.values()), msg)


ODD = _P(264)


@pytest.mark.parametrize("name,args,places", [
    ("tp_quantize_blocks", [0, A, 2, 3, 3, A, A, NULL], {5: "codes", 6: "scales"}),
    ("tp_block_scores", [A, A, 2, A, A, 3, 1, NULL, 0, A, A, 1 << 40, NULL],
     {0: "codes_a", 1: "scales_a", 3: "codes_b", 4: "scales_b", 10: "work"}),
    ("tp_score_images", [0, A, 2, 200, 200, A, A, 3, NULL, 4, A, A, 1 << 40, NULL],
     {5: "codes_b", 6: "scales_b", 11: "work"}),
    ("tp_log_probs", [0, A, 2, 3, 3, NULL, 0, NULL, 0, 1, 1.0, A, A, A, A, A, A, A, 1 << 40, NULL],
     {16: "stats", 17: "work"}),
    ("tp_log_probs_back", [0, A, 2, 3, 3, NULL, 0, NULL, 0, 1, 1.0, A, A, NULL, NULL, NULL, A, A, NULL], {12: "stats"}),
    ("tp_sort_by_class", [8, A, 4, 3, A, A, A, A, 1 << 40, NULL], {7: "work"}),
])
def test_c_abi_refuses_what_is_not_aligned(name, args, places):
    for i, what in places.items():
        _refused(name, [*args[:i], ODD, *args[i + 1:]], f"{what} must be 16-byte aligned")


def test_c_abi_refuses_small_workspaces():
    M, N, nb = 1, 16, 130
    need = capi.lib().tp_block_scores_work(M, N, nb)
    if need:
        _refused("tp_block_scores", [A, A, M, A, A, N, nb, NULL, 0, A, A, need - 1, NULL], "work is smaller")
        _refused("tp_block_scores", [A, A, M, A, A, N, nb, NULL, 0, A, NULL, need, NULL], "work")
    need = capi.lib().tp_log_probs_work(1, 1 << 20, 8)
    if need:
        _refused("tp_log_probs", [0, A, 1, 1 << 20, 0, NULL, 0, NULL, 0, 8, 1.0, A, A, A, A, A, A, A, need - 1, NULL],
                 "work is smaller")
    need = capi.lib().tp_sort_by_class_work(1 << 20, 64)
    if need:
        _refused("tp_sort_by_class", [8, A, 1 << 20, 64, A, A, A, A, need - 1, NULL], "work is smaller")


def test_c_abi_takes_empty_calls():
    lib = capi.lib()
    assert lib.tp_quantize_blocks(0, NULL, 0, 5, 5, NULL, NULL, NULL) == capi.TP_OK
    assert lib.tp_block_scores(NULL, NULL, 0, A, A, 3, 1, NULL, 0, NULL, NULL, 0, NULL) == capi.TP_OK
    assert lib.tp_spread_rows(0, NULL, 0, 5, 2, NULL, NULL, NULL, NULL, NULL, NULL, NULL) == capi.TP_OK
    assert lib.tp_gather_rows(0, NULL, 4, 0, 2, A, A, NULL, NULL, NULL, NULL, NULL) == capi.TP_OK
    assert lib.tp_scale_rows(0) == 0 and lib.tp_scale_rows(1) == 16 and lib.tp_scale_rows(17) == 32


# ----------------------------------------------------------------------------- the definitions
def test_reference_codes_are_torchs():
    x = torch.randn(4, 300, generator=torch.Generator().manual_seed(0))
    q, e = R.quantize(x)
    b = torch.nn.functional.pad(x, (0, 84)).view(4, 3, 128)
    torchs = torch.ldexp(b, -e[:, :, None].int()).to(torch.float8_e4m3fn).float().double().view(4, 384)
    assert torch.equal(q, torchs)
    most = b.abs().amax(2).double()
    unit = torch.exp2(e.double())
    assert (most <= 448 * unit).all() and (most > 224 * unit).all()


def test_reference_log_probs_are_torchs():
    g = torch.Generator().manual_seed(1)
    x = torch.randn(5, 40, generator=g, dtype=torch.float64).requires_grad_()
    mask = torch.rand(5, 40, generator=g) < 0.7
    mask[:, 3] = True
    given = torch.full((5, 1), 3)
    ups = [torch.randn(s, generator=g, dtype=torch.float64) for s in ((5, 1), (5,), (5,), (5, 4))]
    got = R.log_probs(x.detach(), given, 4, 1.7, mask, ups)
    z = (x / 1.7).masked_fill(~mask, -math.inf)
    lp = torch.log_softmax(z, 1)
    p = lp.exp()
    H = -(p * lp.masked_fill(~mask, 0)).sum(1)
    best, index = lp.topk(4, 1)
    outs = (lp.gather(1, given), H, torch.logsumexp(z, 1), best)
    for name, o in zip(("given", "entropy", "log_sum", "top"), outs):
        assert torch.allclose(got[name], o, atol=1e-12), name
    assert torch.equal(got["top_index"], index)
    (d,) = torch.autograd.grad(outs, x, ups)
    assert torch.allclose(got["d_scores"], d, atol=1e-12)


def test_reference_order():
    order, slot, offsets = R.sort_by_class(torch.tensor([[2, 0], [9, 2], [0, -1]]), 3)
    assert order.tolist() == [1, 4, 0, 3, 2, 5] and offsets.tolist() == [0, 2, 2, 4]
    assert slot.tolist() == [[2, 0], [4, 3], [1, 5]]
