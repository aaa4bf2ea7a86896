"""Pair log probabilities and 8-bit integer rows without a GPU: registrations, refusals of the Python functions and the C
ABI, and the 64-bit definitions that the GPU tests compare with, against torch's own functions."""
import ctypes
import math

import pytest
import torch

from tests import pairs_reference as R
from torch_projectors import capi, matching

_P = ctypes.c_void_p
A, NULL, ODD = _P(256), _P(None), _P(264)


@pytest.mark.parametrize("name", ["quantize_rows", "row_scores", "pair_log_probs", "pair_log_probs_back"])
def test_gpu_kernel_registered_and_no_cpu_kernel(name):
    op = f"torch_projectors::{name}"
    assert torch._C._dispatch_has_kernel_for_dispatch_key(op, "CUDA")
    assert not torch._C._dispatch_has_kernel_for_dispatch_key(op, "CPU")


@pytest.mark.parametrize("call", [
    lambda: matching.quantize_rows(torch.zeros(2, 3)),
    lambda: matching.row_scores(torch.zeros(2, 3), torch.zeros(2, 3)),
    lambda: matching.pair_log_probs(torch.zeros(2, 3), torch.zeros(4, 3)),
    lambda: matching.pair_log_probs(torch.zeros(2, 3, requires_grad=True), torch.zeros(4, 3)),
])
def test_cpu_tensors_fail_loudly(call):
    with pytest.raises(NotImplementedError):
        call()


@pytest.mark.parametrize("call,msg", [
    (lambda: matching.quantize_rows(torch.zeros(())), "at least 1 dimension"),
    (lambda: matching.row_scores(torch.zeros(2, 100), torch.zeros(3, 120)), "do not fit"),
    (lambda: matching.row_scores(torch.zeros(2, 5, 20), torch.zeros(3, 10, 12)), "do not fit"),
    (lambda: matching.pair_log_probs(torch.zeros(()), torch.zeros(2, 3)), "at least 1 dimension"),
    (lambda: matching.pair_log_probs(torch.zeros(2, 4), torch.zeros(2, 3)), "do not fit"),
    (lambda: matching.pair_log_probs(torch.zeros(2, 2, dtype=torch.complex64), torch.zeros(2, 3)), "Images of 4 values do not fit"),
    (lambda: matching.pair_log_probs(torch.zeros(2, 3), torch.zeros(4, 3), torch.zeros(3, dtype=torch.int64)), "Given"),
    (lambda: matching.pair_log_probs(torch.zeros(2, 3), torch.zeros(4, 3), torch.zeros(2, 1, dtype=torch.int64)), "Given"),
    (lambda: matching.pair_log_probs(torch.zeros(2, 3), torch.zeros(4, 3), bias=torch.zeros(2)), "Bias"),
    (lambda: matching.pair_log_probs(torch.zeros(2, 3), torch.zeros(4, 3), mask=torch.ones(2, 4, dtype=torch.bool)), "Mask"),
])
def test_python_argument_checks(call, msg):
    with pytest.raises(ValueError, match=msg):
        call()


QUANTIZE = dict(dt=0, x=A, rows=2, cols=3, stride=3, codes=A, scales=A, stream=NULL)
SCORES = dict(a=A, sa=A, M=2, b=A, sb=A, N=3, cols=200, bias=NULL, odt=0, out=A, work=A, bytes=1 << 40, stream=NULL)
IMAGES = dict(dt=0, x=A, M=2, cols=200, stride=200, b=A, sb=A, N=3, bias=NULL, odt=0, out=A, work=A, bytes=1 << 40, stream=NULL)
PAIRS = dict(dt=0, x=A, M=20, K=30, sx=30, r=A, N=40, sr=30, given=NULL, bias=NULL, mask=NULL, temp=1.0, go=NULL, l=A, st=A, work=A,
             bytes=1 << 40, stream=NULL)
BACK = dict(dt=0, x=A, M=20, K=30, sx=30, r=A, N=40, sr=30, given=NULL, bias=NULL, mask=NULL, temp=1.0, st=A, dg=NULL, dl=A, dx=A, dr=A,
            db=A, work=A, bytes=1 << 40, stream=NULL)
ROWS = [(dict(dt=1), "dtype"), (dict(M=-1), "non-negative"), (dict(N=-1), "non-negative"), (dict(M=1 << 27), "2^26"), (dict(N=(1 << 26) + 1), "2^26"),
        (dict(M=1 << 18, N=(1 << 17) + 1), "2^35"), (dict(K=0), "cols"), (dict(K=(1 << 21) + 1), "cols"), (dict(sx=-1), "strides"),
        (dict(sr=(1 << 21) + 1), "strides"), (dict(temp=0.0), "temperature"), (dict(temp=math.nan), "temperature"), (dict(temp=1e-40), "temperature"),
        (dict(x=NULL), "images"), (dict(r=NULL), "references"), (dict(work=NULL), "work must not be NULL"), (dict(bytes=15), "work is smaller"),
        (dict(work=ODD), "work must be 16-byte aligned"), (dict(st=ODD), "state must be 16-byte aligned")]


@pytest.mark.parametrize("name,good,bad", [
    ("tp_quantize_rows", QUANTIZE, [
        (dict(dt=1), "dtype"), (dict(rows=-1), "rows"), (dict(cols=0), "cols"), (dict(cols=(1 << 17) + 1), "2^17"), (dict(stride=-1), "row_stride"),
        (dict(x=NULL), "x"), (dict(codes=NULL), "codes"), (dict(scales=NULL), "scales"), (dict(codes=ODD), "codes must be 16-byte aligned")]),
    ("tp_row_scores", SCORES, [
        (dict(odt=3), "out_dtype"), (dict(M=-1), "non-negative"), (dict(N=1 << 27), "2^26"), (dict(M=1 << 20, N=(1 << 17) + 1), "2^37"), (dict(cols=0), "cols"),
        (dict(cols=(1 << 17) + 1), "2^17"), (dict(a=NULL), "codes_a"), (dict(sa=NULL), "scales_a"), (dict(b=NULL), "codes_b"), (dict(sb=NULL), "scales_b"),
        (dict(out=NULL), "scores"), (dict(a=ODD), "codes_a must be 16-byte"), (dict(b=ODD), "codes_b must be 16-byte"), (dict(work=ODD), "work must be 16-byte")]),
    ("tp_row_score_images", IMAGES, [
        (dict(dt=2), "dtype"), (dict(odt=3), "out_dtype"), (dict(M=-1), "non-negative"), (dict(stride=-1), "row_stride"), (dict(cols=0), "cols"),
        (dict(x=NULL), "x"), (dict(work=NULL), "work"), (dict(bytes=10), "work is smaller"), (dict(sb=NULL), "scales_b"), (dict(out=NULL), "scores")]),
    ("tp_pair_log_probs", PAIRS, ROWS + [(dict(l=NULL), "log_sum"), (dict(given=A), "given_log_probs")]),
    ("tp_pair_log_probs_back", BACK, ROWS + [(dict(st=NULL), "state")]),
])
def test_c_abi_refuses_before_anything_is_enqueued(name, good, bad):
    assert len(good) == len(capi.SIGNATURES[name])
    for change, msg in bad:
        assert getattr(capi.lib(), name)(*{**good, **change}.values()) == capi.TP_ERR_INVALID, change
        assert msg in capi.lib().tp_last_error().decode(), change


@pytest.mark.parametrize("M,N,K", [(1, 4096, 16640), (8, 300, 5000), (9, 1, 1), (333, 1999, 8280), (500, 4099, 2070), (4096, 36864, 4224)])
@pytest.mark.parametrize("dt", [0, 3, 4])
def test_small_workspaces_of_pairs_are_refused(M, N, K, dt):
    lib = capi.lib()
    need = lib.tp_pair_log_probs_work(dt, M, N, K)
    assert need > 0
    change = dict(dt=dt, M=M, N=N, K=K, sx=K, sr=K, bytes=need - 1)
    assert lib.tp_pair_log_probs(*{**PAIRS, **change}.values()) == capi.TP_ERR_INVALID
    assert "work is smaller" in lib.tp_last_error().decode()
    need = lib.tp_pair_log_probs_back_work(dt, M, N, K, 1, 1)
    assert need > 0 and need >= lib.tp_pair_log_probs_back_work(dt, M, N, K, 0, 1)
    change["bytes"] = need - 1
    assert lib.tp_pair_log_probs_back(*{**BACK, **change}.values()) == capi.TP_ERR_INVALID
    assert "work is smaller" in lib.tp_last_error().decode()


def test_scores_are_not_kept():
    """Of 4096 x 36864 pairs the scores would be 604 MB; the forward pass keeps tiles' parts, the gradient a piece of 128 MB and
    the gradients that its pieces add up."""
    lib = capi.lib()
    assert lib.tp_pair_log_probs_work(4, 4096, 36864, 4224) < 64 << 20
    assert lib.tp_pair_log_probs_back_work(4, 4096, 36864, 4224, 1, 1) < (128 + 70 + 64) << 20
    assert lib.tp_pair_state(4096, 36864) == 4 * 4096
    assert lib.tp_pair_state(8, 1000) == 8 * 1004 and lib.tp_pair_state(0, 10) == 0


@pytest.mark.parametrize("M,N,K", [(16, 100, 16640), (700, 900, 3000), (333, 1999, 8280)])
def test_small_workspaces_of_row_scores_are_refused(M, N, K):
    lib = capi.lib()
    need = lib.tp_row_scores_work(M, N, K)
    assert need > 0
    for change, msg in ((dict(bytes=need - 1), "work is smaller"), (dict(work=NULL), "work must not be NULL")):
        assert lib.tp_row_scores(*{**SCORES, "M": M, "N": N, "cols": K, **change}.values()) == capi.TP_ERR_INVALID
        assert msg in lib.tp_last_error().decode()


def test_c_abi_takes_empty_calls():
    lib = capi.lib()
    assert lib.tp_quantize_rows(0, NULL, 0, 5, 5, NULL, NULL, NULL) == capi.TP_OK
    assert lib.tp_row_scores(NULL, NULL, 0, A, A, 3, 100, NULL, 0, NULL, NULL, 0, NULL) == capi.TP_OK
    assert lib.tp_pair_log_probs(*{**PAIRS, "M": 0, "x": NULL, "l": NULL, "st": NULL, "work": NULL, "bytes": 0}.values()) == capi.TP_OK
    assert lib.tp_pair_log_probs_back(*{**BACK, "dx": NULL, "dr": NULL, "db": NULL}.values()) == capi.TP_OK


# ----------------------------------------------------------------------------- the definitions
def test_reference_log_probs_and_gradients_are_torchs():
    g = torch.Generator().manual_seed(0)
    x, r = torch.randn(6, 20, generator=g).requires_grad_(), torch.randn(15, 20, generator=g).requires_grad_()
    b = torch.randn(15, generator=g).requires_grad_()
    mask = torch.rand(15, generator=g) < 0.7
    mask[:4] = True
    given = torch.tensor([0, 1, -1, 2, 3, 0])
    dg, dl = torch.randn(6, generator=g), torch.randn(6, generator=g)
    w = R.pair_log_probs(x.detach(), r.detach(), given, b.detach(), 1.7, mask, dg, dl)
    z = ((x.double() @ r.double().t() + b.double()) / 1.7).masked_fill(~mask, -math.inf)
    lp = torch.log_softmax(z, 1)
    log_sum = torch.logsumexp(z, 1)
    got = lp.gather(1, given.clamp_min(0)[:, None])[:, 0] * (given >= 0)
    assert torch.allclose(w["log_sum"], log_sum, atol=1e-12) and torch.allclose(w["given"], got, atol=1e-12)
    d = torch.autograd.grad((got, log_sum), (x, r, b), (dg.double(), dl.double()))
    for name, v in zip(("d_images", "d_references", "d_bias"), d):
        assert torch.allclose(w[name], v.double(), atol=1e-6), name


def test_reference_bounds_hold_for_sums_in_32_bits():
    """torch's own sums in 32 bits stay within the bounds."""
    g = torch.Generator().manual_seed(1)
    x, r, b = torch.randn(9, 300, generator=g), torch.randn(40, 300, generator=g) * 0.2, torch.randn(40, generator=g)
    w = R.pair_log_probs(x, r, torch.arange(9), b, 1.3)
    z = (x @ r.t() + b) / 1.3
    assert ((torch.logsumexp(z, 1) - w["log_sum"]).abs() <= w["tol_log_sum"]).all()
    assert ((torch.log_softmax(z, 1).diagonal()[:9] - w["given"]).abs() <= w["tol_given"] + 2e-6).all()


def test_reference_integers():
    x = torch.tensor([[127.0, 0.5, 1.5, -2.5, -126.6, 0.0], [0.0] * 6, [1e-45, 0, 0, 0, 0, 0], [math.inf, 1, 0, 0, 0, 0]])
    codes, scale = R.quantize_rows(x)
    assert codes[0].tolist() == [127, 0, 2, -2, -127, 0] and scale[0] == 1
    assert (codes[1:] == 0).all() and scale[1] == 2.0 ** -126 and scale[2] == 2.0 ** -126 and scale[3].isnan()
    s = R.row_scores(codes[:1], scale[:1], codes[:2], scale[:2], torch.tensor([0.25, 3.0]))
    assert s.tolist() == [[127.0 ** 2 * 2 + 8 + 0.25, 3.0]]
