"""The matching operators on the GPU against their definitions in 64 bits (tests/matching_reference.py).

Tolerances, from the roundings (u the unit roundoff of a type, 2^-24 in fp32):
* codes and scales are exact;
* scores: a product is exact and each of the nb + 8 additions along a sum loses at most 2 u of the
  magnitudes' sum;
* log probabilities: (x - m) / temperature - ln s, each step within a few u of its own size, ln s within
  2e-6 (V terms of relative error about 1e-7, summed in a tree): 2e-6 (1 + |value|), the entropy twice that;
* score gradients: 1e-5 of the sum of the row's upstream magnitudes / temperature, times p (1 + |ln p| + H)
  plus the listed place's own, plus u of the storage type;
* row sums: k + 1 roundings of the magnitudes' sum, plus u of the storage type; weight gradients D / 64 + 16
  roundings.
"""
import math

import pytest
import torch

from tests import matching_reference as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def m(gpu):
    from torch_projectors import matching
    return matching


def gen(seed):
    return torch.Generator().manual_seed(seed)


def near(got, want, tol, what):
    got = got.detach().double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.equal(got.isnan(), want.isnan()), what
    inf = want.isinf()
    assert torch.equal(got[inf], want[inf]), what
    fine = torch.isfinite(want)
    off = (got - want)[fine].abs() - (tol[fine] if torch.is_tensor(tol) else tol)
    assert off.numel() == 0 or float(off.max()) <= 0, (what, float(off.max()))


# ----------------------------------------------------------------------------- blocks
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("shape", [(1, 1), (3, 127), (2, 128), (5, 129), (17, 300), (16, 256)])
def test_quantize(m, shape, dtype):
    x = (torch.randn(shape, generator=gen(1)) * torch.exp(torch.linspace(3, -9, shape[1]))).to(dtype)
    q = m.quantize_blocks(x.to(DEV))
    want, e = R.quantize(x)
    assert torch.equal(q.codes.float().double().cpu(), want)
    assert q.scales.shape == (e.shape[1], -(-shape[0] // 16) * 16)
    assert torch.equal(q.scales.cpu()[:, :shape[0]].long() - 127, e.t())
    assert (q.scales.cpu()[:, shape[0]:] == 127).all()


def test_quantize_extremes(m):
    x = torch.zeros(9, 128)
    x[1, 5] = 448.0
    x[2, 5] = 448.00003  # the next value above
    x[3, :] = 1e-42  # subnormal
    x[4, 3] = torch.finfo(F32).max
    x[5, 3] = -torch.finfo(F32).max
    x[5, 4] = 1e-30
    x[6, 0], x[6, 1], x[6, 2] = math.inf, math.nan, 7.0
    x[7, :] = -math.inf
    x[8, :] = torch.arange(128) / 16.0  # halves between codes
    q = m.quantize_blocks(x.to(DEV))
    want, e = R.quantize(x)
    got = q.codes.float().double().cpu()
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.nan_to_num(0), want.nan_to_num(0))
    assert torch.equal(q.scales.cpu()[:, :9].long() - 127, e.t())


def test_quantize_layouts(m):
    base = torch.randn(11, 700, generator=gen(2))
    for x in (base[:, 3:500], base[::2], base.t()[:300].t(), base.t(), base[4:5].expand(6, 700), base[:0]):
        q = m.quantize_blocks(_as(x))
        assert q.codes.shape[0] == x.shape[0]
        if len(x):
            assert torch.equal(q.codes.float().double().cpu(), R.quantize(x.contiguous())[0])
    c = torch.randn(3, 8, 5, dtype=torch.complex64, generator=gen(3))
    want, _ = R.quantize(torch.view_as_real(c).reshape(3, 80))
    assert torch.equal(m.quantize_blocks(c.to(DEV)).codes.float().double().cpu(), want)


def _as(x):
    """x on the GPU with its own strides and offset."""
    whole = torch.empty(0, dtype=x.dtype).set_(x.untyped_storage()).to(DEV)
    return whole.as_strided(x.shape, x.stride(), x.storage_offset())


def _scores_check(m, M, N, K, out_dtype, bias, seed=0, fall=-7.0):
    g = gen(seed)
    amp = torch.exp(torch.linspace(0, fall, K))
    a, b = torch.randn(M, K, generator=g) * amp, torch.randn(N, K, generator=g) * amp
    f = torch.randn(N, generator=g) if bias else None
    qa, qb = m.quantize_blocks(a.to(DEV)), m.quantize_blocks(b.to(DEV))
    va, vb = R.blocks_value(*qa), R.blocks_value(*qb)
    want, mag = va @ vb.t(), va.abs() @ vb.abs().t()
    if bias:
        want, mag = want + f.double(), mag + f.double().abs()
    nb = qa.codes.shape[1] // 128
    tol = (nb + 8) * 2.0 ** -23 * mag + (R.U[out_dtype] * want.abs() * 1.01 if out_dtype != F32 else 0)
    kw = dict(bias=None if f is None else f.to(DEV), out_dtype=out_dtype)
    got = m.block_scores(qa, qb, **kw)
    assert got.dtype == out_dtype
    near(got, want, tol, "scores of blocks")
    assert torch.equal(m.block_scores(a.to(DEV), qb, **kw), got)  # quantised by the call
    assert torch.equal(m.block_scores(qa, qb, **kw), got)  # the same again


@pytest.mark.parametrize("M,N,K", [
    (1, 1, 1), (1, 256, 4224), (1, 17, 300), (2, 130, 128), (7, 65, 129), (16, 64, 512), (17, 64, 640), (33, 100, 900),
    (64, 64, 256), (65, 127, 1100), (100, 1999, 384), (128, 128, 1280), (129, 257, 2000), (200, 300, 16640),
    (255, 255, 260), (256, 256, 128), (300, 513, 777), (513, 300, 1500), (1000, 70, 2112), (1025, 1030, 385),
    (3, 4099, 640), (40, 5000, 129), (2050, 9, 333)])
@pytest.mark.parametrize("out_dtype,bias", [(F32, True), (BF16, False)])
def test_scores(m, M, N, K, out_dtype, bias):
    _scores_check(m, M, N, K, out_dtype, bias)


def test_scores_values_of_all_sizes(m):
    # blocks whose scales differ by far more than fp32's precision, signs that cancel
    _scores_check(m, 40, 70, 2000, F32, False, seed=5, fall=-60.0)
    _scores_check(m, 300, 300, 2000, F32, True, seed=6, fall=30.0)


def test_scores_exact_integers(m):
    """Small integers are exact in every step: each product lands at its own place."""
    g = gen(8)
    for M, N, K in ((70, 90, 300), (300, 270, 256), (1, 40, 640), (20, 600, 130)):
        a, b = torch.randint(-4, 5, (M, K), generator=g).float(), torch.randint(-4, 5, (N, K), generator=g).float()
        assert torch.equal(m.block_scores(a.to(DEV), m.quantize_blocks(b.to(DEV))).cpu(), a @ b.t())


def test_scores_empty_and_not_finite(m):
    a, b = torch.randn(5, 300, generator=gen(1)), torch.randn(7, 300, generator=gen(2))
    assert m.block_scores(a[:0].to(DEV), b.to(DEV)).shape == (0, 7)
    assert m.block_scores(a.to(DEV), b[:0].to(DEV)).shape == (5, 0)
    a[2, 17], b[3, 200] = math.inf, math.nan
    s = m.block_scores(a.to(DEV), b.to(DEV)).cpu()
    bad = torch.zeros(5, 7, dtype=torch.bool)
    bad[2], bad[:, 3] = True, True
    assert torch.equal(s.isnan(), bad)


def test_scores_past_32_bit_offsets(m):
    N, nb = 300001, 130  # 5.0e9 bytes of codes
    codes = torch.zeros(N, nb * 128, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)
    scales = torch.full((nb, -(-N // 16) * 16), 127, dtype=torch.uint8, device=DEV)
    rows = torch.tensor([0, 1, 258111, 258112, N - 1], device=DEV)
    codes[rows] = torch.ones(5, nb * 128, device=DEV).to(torch.float8_e4m3fn)
    scales[:, rows] = torch.tensor([126, 127, 128, 129, 130], dtype=torch.uint8, device=DEV)
    for M in (1, 40, 300):
        got = m.block_scores(torch.ones(M, nb * 128, device=DEV), m.BlockScaled(codes, scales))
        want = torch.zeros(M, N, device=DEV)
        want[:, rows] = nb * 128 * torch.tensor([0.5, 1, 2, 4, 8], device=DEV)
        assert torch.equal(got, want)


# ----------------------------------------------------------------------------- log probabilities
def _probs_check(m, x, given=None, top=0, temperature=1.0, mask=None, seed=0, with_grad=True, view=None):
    """x [T, V] on the CPU; `view` its GPU tensor where that has a layout of its own."""
    T, V = x.shape
    g = gen(seed)
    G = 0 if given is None else given.shape[1]
    ups = (torch.randn(T, G, generator=g), torch.randn(T, generator=g), torch.randn(T, generator=g),
           torch.randn(T, top, generator=g))
    s = (x.to(DEV) if view is None else view).detach().requires_grad_(with_grad)
    dev = lambda v: None if v is None else v.to(DEV)  # noqa: E731
    out = m.log_probs(s, dev(given), top=top, temperature=temperature, mask=dev(mask))
    want = R.log_probs(x, given, top, temperature, mask, tuple(u if u.numel() else None for u in ups))
    two = lambda v: 2e-6 * (1 + v.abs().nan_to_num(0, 0, 0))  # noqa: E731
    if given is not None:
        near(out.given, want["given"], two(want["given"]), "given")
    near(out.log_sum, want["log_sum"], two(want["log_sum"]), "log_sum")
    near(out.entropy, want["entropy"], 2 * two(want["entropy"]), "entropy")
    if top:
        near(out.top, want["top"], two(want["top"]), "top")
        rows = ~want["log_sum"].isnan()
        assert torch.equal(out.top_index.cpu()[rows], want["top_index"][rows])
    if not with_grad:
        return out
    outs = [(o, u) for o, u in zip((out.given, out.entropy, out.log_sum, out.top), ups) if o is not None and o.numel()]
    (d,) = torch.autograd.grad([o for o, _ in outs], [s], [u.to(DEV) for _, u in outs])
    assert d.dtype == x.dtype and d.shape == x.shape
    z = x.double() / temperature
    if mask is not None:
        z = z.masked_fill(~mask.expand(T, V), -math.inf)
    lp = (z - z.amax(1, keepdim=True))
    lp = lp - torch.log(lp.exp().sum(1, keepdim=True))
    p = lp.exp().nan_to_num(0)
    total = sum(u.double().abs().reshape(T, -1).sum(1) for u in ups)[:, None]
    size = p * (1 + lp.nan_to_num(0, 0, 0).abs() + want["entropy"][:, None].nan_to_num(0))
    at = torch.zeros(T, V, dtype=torch.float64)
    for idx in (given, want["top_index"]):
        if idx is not None and idx.numel():
            for t in range(T):
                at[t, [int(v) for v in idx[t] if 0 <= int(v) < V]] = 1
    tol = 1e-5 * total / temperature * (size + 2.0 ** -4 * at) + 1e-37
    tol = tol + (R.U[x.dtype] * want["d_scores"].abs().nan_to_num(0) * 1.01 + (2.0 ** -25 if x.dtype == F16 else 0))
    rows = ~want["log_sum"].isnan()
    near(d[rows.to(DEV)], want["d_scores"][rows], tol[rows], "d_scores")
    return out


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("T,V,top", [(1, 1, 1), (3, 2, 2), (2, 63, 5), (5, 64, 64), (4, 65, 8), (3, 255, 1), (2, 257, 0),
                                     (7, 1000, 16), (2, 4096, 8), (3, 4099, 33), (1, 20011, 4)])
def test_probs(m, T, V, top, dtype):
    g = gen(V)
    x = (torch.randn(T, V, generator=g) * 3).to(dtype)
    given = torch.randint(0, V, (T, 1), generator=g)
    _probs_check(m, x, given, min(top, V), 1.5)


@pytest.mark.parametrize("T,V,top,dtype", [(1, 294912, 16, BF16), (2, 70001, 8, F32), (600, 301, 3, F32)])
def test_probs_long_and_many(m, T, V, top, dtype):
    g = gen(3)
    x = (torch.randn(T, V, generator=g) * 2).to(dtype)
    _probs_check(m, x, torch.randint(0, V, (T, 2), generator=g), top, 0.7)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shared", [True, False])
def test_probs_masks(m, shared, dtype):
    g = gen(11)
    T, V = 6, 333
    x = torch.randn(T, V, generator=g).to(dtype)
    mask = torch.rand(1 if shared else T, V, generator=g) < 0.5
    mask[0, 9] = True
    if not shared:
        mask[1] = False  # allows nothing
        mask[2] = False
        mask[2, 332] = True  # allows one
        mask[3, :] = False
        mask[3, [4, 77]] = True
    # what masked places hold is not used
    x = torch.where(mask.expand(T, V), x, torch.tensor([math.nan, math.inf, -math.inf])[torch.arange(V) % 3].to(dtype))
    given = torch.tensor([[9, -1], [5, 9], [332, 0], [4, 77], [9, 9], [-1, -1]])
    _probs_check(m, x, given, 5, 1.0, mask[0] if shared else mask)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_probs_values_at_the_ends(m, dtype):
    big = torch.finfo(dtype).max
    V = 130
    x = torch.zeros(8, V, dtype=dtype)
    x[0] = -big  # the lowest value everywhere: a uniform row
    x[1] = -math.inf  # allows nothing
    x[2, :] = -big
    x[2, 7] = 3.0  # one candidate, the others at the lowest value
    x[3, :] = -math.inf
    x[3, 100] = -big
    x[4, 5] = big
    x[5, 64:] = -math.inf
    x[6, 11] = math.nan
    x[7, :] = big
    given = torch.tensor([[3], [3], [7], [100], [5], [70], [0], [129]])
    _probs_check(m, x, given, 4, 0.5 if dtype == F16 else 1.0)
    y = m.log_probs(torch.full((2, 9), -big, dtype=dtype, device=DEV), temperature=0.25)  # scaled past the range
    assert torch.allclose(y.entropy.cpu(), torch.full((2,), math.log(9.0)), atol=4e-6)
    z = torch.zeros(1, 9, dtype=dtype, device=DEV)
    z[0, 4] = math.inf
    y = m.log_probs(z, torch.tensor([4], device=DEV))
    assert y.log_sum.item() == math.inf and y.given.isnan().all() and y.entropy.isnan().all()


def test_probs_ties_and_orders(m):
    V = 5000
    for x in (torch.zeros(1, V), -torch.zeros(1, V), torch.arange(V).float()[None] / 100, -torch.arange(V).float()[None] / 100,
              (torch.arange(V) % 7).float()[None], torch.where(torch.arange(V) % 2 == 0, 0.0, -0.0)[None]):
        for dtype in (F32, BF16):
            _probs_check(m, x.to(dtype), torch.tensor([[17]]), 20, 1.0, with_grad=False)


def test_probs_layouts_and_shapes(m):
    base = torch.randn(9, 517, generator=gen(4))
    given = torch.randint(0, 100, (9, 1), generator=gen(5))
    for x in (base[:, 1:400], base[:, 3:], base.t().contiguous().t(), base[2:3].expand(9, 517)):
        _probs_check(m, x, given, 3, view=_as(x))
    x = base[:, :510].reshape(3, 3, 510).to(DEV)
    out = m.log_probs(x, given.view(3, 3).to(DEV), top=4, mask=torch.ones(510, dtype=torch.bool, device=DEV))
    assert out.given.shape == (3, 3) and out.top.shape == (3, 3, 4) and out.log_sum.shape == (3, 3)
    flat = m.log_probs(x.view(9, 510), given.to(DEV), top=4)
    assert flat.given.shape == (9, 1)
    assert torch.equal(out.given.view(9, 1), flat.given) and torch.equal(out.top_index.view(9, 4), flat.top_index)
    one = m.log_probs(x[0, 0], given.view(-1)[0].to(DEV), top=4)
    assert one.given.shape == () and one.top.shape == (4,) and torch.equal(one.top, out.top[0, 0])
    none = m.log_probs(x[:0], given.view(3, 3)[:0].to(DEV), top=2)
    assert none.given.shape == (0, 3) and none.top.shape == (0, 3, 2)
    assert m.log_probs(x).given is None


def test_probs_given_out_of_range(m):
    out = m.log_probs(torch.zeros(4, 5, device=DEV), torch.tensor([0, -1, 5, -2], device=DEV))
    got = out.given.cpu()
    assert got[0].item() == pytest.approx(-math.log(5.0)) and got[1].item() == 0 and got[2:].isnan().all()


def test_probs_past_32_bit_offsets(m):
    stride, V = 2_300_000_001, 700
    whole = torch.zeros(2 * stride + V, dtype=BF16, device=DEV)
    s = whole.as_strided((3, V), (stride, 1))
    x = torch.randn(3, V, generator=gen(6)).to(BF16)
    s.copy_(x.to(DEV))
    _probs_check(m, x, torch.tensor([[1], [2], [3]]), 5, view=s)


@pytest.mark.parametrize("which", range(4))
def test_probs_gradient_against_differences(m, which):
    """Central differences along a direction; the step's third-order term is about h^2 = 1e-4 of the value,
    fp32 rounding of the outputs 2e-6 / h."""
    g = gen(which)
    T, V, h = 4, 300, 0.02
    x, direction = torch.randn(T, V, generator=g), torch.randn(T, V, generator=g)
    x[:, :3] += torch.tensor([6.0, 10.0, 14.0])  # the best three stay in their order within the step
    given = torch.randint(0, V, (T,), generator=g).to(DEV)
    up = torch.randn((T, 3) if which == 3 else (T,), generator=g)

    def outputs(v):
        return m.log_probs(v, given, top=3, temperature=1.3)

    def value(v):
        return (outputs(v)[which].double().cpu() * up.double()).sum()

    s = x.to(DEV).requires_grad_()
    outputs(s)[which].backward(up.to(DEV))
    slope = (s.grad.double().cpu() * direction.double()).sum()
    differences = (value((x + h * direction).to(DEV)) - value((x - h * direction).to(DEV))) / (2 * h)
    assert abs(float(slope - differences)) <= 2e-3 * float(up.abs().sum()) + 1e-3 * abs(float(slope))


# ----------------------------------------------------------------------------- rows by class
@pytest.mark.parametrize("T,k,E", [(1, 1, 1), (1, 5, 3), (16, 2, 8), (63, 1, 2), (64, 1, 64), (65, 3, 7), (1000, 2, 257),
                                   (333, 4, 4096), (5000, 3, 16), (40000, 2, 100), (100003, 1, 1000)])
@pytest.mark.parametrize("dtype", [torch.int64, torch.int32])
def test_sort(m, T, k, E, dtype):
    g = gen(T)
    classes = (torch.rand(T, k, generator=g) ** 3 * E).to(dtype)
    classes[torch.rand(T, k, generator=g) < 0.05] = -1
    classes[torch.rand(T, k, generator=g) < 0.05] = E
    if T > 1:
        classes[T // 2, 0] = torch.iinfo(dtype).max
    got = m.sort_by_class(classes.to(DEV), E)
    flat = classes.reshape(-1).long()
    key = torch.where((flat >= 0) & (flat < E), flat, E)
    order = torch.sort(key, stable=True)[1]
    slot = torch.empty_like(order)
    slot[order] = torch.arange(T * k)
    offsets = torch.searchsorted(key[order].contiguous(), torch.arange(E + 1))
    assert torch.equal(got.order.cpu().long(), order)
    assert torch.equal(got.slot.cpu().long(), slot.view(T, k))
    assert torch.equal(got.offsets.cpu().long(), offsets)


def test_sort_edges(m):
    got = m.sort_by_class(torch.empty(0, 2, dtype=torch.int64, device=DEV), 3)
    assert got.order.shape == (0,) and got.slot.shape == (0, 2) and got.offsets.tolist() == [0, 0, 0, 0]
    got = m.sort_by_class(torch.full((70000,), 2, device=DEV), 3)  # one class takes all
    assert torch.equal(got.order.cpu(), torch.arange(70000, dtype=torch.int32)) and got.offsets.tolist() == [0, 0, 0, 70000]
    got = m.sort_by_class(torch.full((100,), -5, device=DEV), 3)  # every slot is dropped
    assert got.offsets.tolist() == [0, 0, 0, 0] and got.slot.shape == (100, 1)
    a, b = (m.sort_by_class(torch.tensor([[2, 0], [1, 2]], device=DEV).t(), 3) for _ in range(2))
    assert a.order.tolist() == [2, 1, 0, 3] and torch.equal(a.order, b.order)


def _route(m, T, k, E, seed):
    g = gen(seed)
    classes = torch.randint(0, E, (T, k), generator=g)
    classes[torch.rand(T, k, generator=g) < 0.15] = -1  # dropped
    order = m.sort_by_class(classes.to(DEV), E)
    return order, order.slot.cpu(), int(order.offsets[-1])


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("T,k,E,D", [(1, 1, 1, 1), (1, 2, 4, 7), (5, 1, 3, 8), (16, 2, 8, 128), (33, 3, 5, 129), (20, 8, 16, 1235),
                                     (100, 2, 9, 64), (7, 4, 3, 4224), (3, 2, 2, 16640), (2, 1, 2, 66048), (300, 2, 6, 33)])
@pytest.mark.parametrize("weighted", [True, False])
def test_rows(m, T, k, E, D, dtype, weighted):
    g = gen(D)
    order, slot, kept = _route(m, T, k, E, D)
    u = R.U[dtype]
    tiny = 2.0 ** -25 if dtype == F16 else 0.0
    x, y = torch.randn(T, D, generator=g).to(dtype), torch.randn(T * k, D, generator=g).to(dtype)
    w = torch.rand(T, k, generator=g) if weighted else None
    d_sorted, d_sum = torch.randn(T * k, D, generator=g).to(dtype), torch.randn(T, D, generator=g).to(dtype)
    leaf = lambda v: None if v is None else v.to(DEV).requires_grad_()  # noqa: E731

    gx, gw = leaf(x), leaf(w)
    sorted_ = m.dispatch(gx, order, gw)
    assert sorted_.dtype == dtype
    want = R.spread(x, slot, kept, w)
    near(sorted_, want, (u + 2.0 ** -24) * want.abs() + tiny, "sorted")
    grads = torch.autograd.grad(sorted_, [v for v in (gx, gw) if v is not None], d_sorted.to(DEV))
    want, mag = R.gather(d_sorted, slot, kept, w)
    near(grads[0], want, u * want.abs() + (k + 1) * 2.0 ** -24 * mag * (1 + u) + tiny, "d_x")
    dot_tol = (D / 64 + 16) * 2.0 ** -24
    if weighted:
        want, mag = R.dots(x, d_sorted, slot, kept)
        near(grads[1], want, dot_tol * mag, "d_weights of dispatch")

    gy, gw = leaf(y), leaf(w)
    total = m.combine(gy, order, gw)
    want, mag = R.gather(y, slot, kept, w)
    near(total, want, u * want.abs() + (k + 1) * 2.0 ** -24 * mag * (1 + u) + tiny, "sum")
    grads = torch.autograd.grad(total, [v for v in (gy, gw) if v is not None], d_sum.to(DEV))
    want = R.spread(d_sum, slot, kept, w)
    near(grads[0], want, (u + 2.0 ** -24) * want.abs() + tiny, "d_y")
    if weighted:
        want, mag = R.dots(d_sum, y, slot, kept)
        near(grads[1], want, dot_tol * mag, "d_weights of combine")


def test_rows_complex_and_layouts(m):
    order, slot, kept = _route(m, 10, 2, 3, 0)
    g = gen(1)
    x = torch.randn(10, 6, 4, dtype=torch.complex64, generator=g)
    w = torch.rand(10, 2, generator=g)
    for view in (x, x.transpose(1, 2).contiguous().transpose(1, 2), x.conj().resolve_conj().conj()):
        s = m.dispatch(view.to(DEV), order)
        assert s.shape == (20, 6, 4) and s.dtype == torch.complex64
        real = torch.view_as_real(x).reshape(10, 48)
        assert torch.equal(torch.view_as_real(s).reshape(20, 48).double().cpu(), R.spread(real, slot, kept))
    gy, gw = s.detach().requires_grad_(), w.to(DEV).requires_grad_()
    up = torch.randn(10, 6, 4, dtype=torch.complex64, generator=g)
    back = m.combine(gy, order, gw)
    dy, dw = torch.autograd.grad(back, (gy, gw), up.to(DEV))
    pairs = lambda v: torch.view_as_real(v.cpu()).reshape(v.shape[0], -1)  # noqa: E731
    near(pairs(dy.detach()), R.spread(pairs(up), slot, kept, w), 1e-6, "complex d_y")
    near(dw, R.dots(pairs(up), pairs(s), slot, kept)[0], 1e-4, "complex d_weights")
    for view in (torch.randn(10, 40, generator=g)[:, 1:38], torch.randn(37, 10, generator=g).t()):
        assert torch.equal(m.dispatch(_as(view), order).double().cpu(), R.spread(view, slot, kept))


def test_rows_edges(m):
    order = m.sort_by_class(torch.full((4, 2), 9, device=DEV), 3)  # every slot is dropped
    x = torch.full((4, 10), math.nan, device=DEV)
    assert (m.dispatch(x, order) == 0).all()
    w = torch.ones(4, 2, device=DEV, requires_grad=True)
    y = torch.full((8, 10), math.nan, device=DEV, requires_grad=True)
    total = m.combine(y, order, w)
    assert (total == 0).all()
    dy, dw = torch.autograd.grad(total, (y, w), torch.full((4, 10), math.inf, device=DEV))
    assert (dy == 0).all() and (dw == 0).all()
    empty = m.sort_by_class(torch.empty(0, 2, dtype=torch.int64, device=DEV), 3)
    assert m.dispatch(torch.empty(0, 5, device=DEV), empty).shape == (0, 5)
    order = m.sort_by_class(torch.tensor([0, 1], device=DEV), 2)
    assert m.combine(torch.empty(2, 0, device=DEV), order).shape == (2, 0)
    z = m.dispatch(torch.empty(2, 0, device=DEV), order, torch.ones(2, device=DEV))
    assert z.shape == (2, 0)


def test_rows_past_32_bit_offsets(m):
    T, D = 66001, 33000  # 2.18e9 values, 4.4 GB
    order = m.sort_by_class((T - 1 - torch.arange(T, device=DEV)) % 4096, 4096)
    x = torch.arange(T, device=DEV, dtype=torch.int32).remainder(251).to(BF16)[:, None].expand(T, D).contiguous()
    s = m.dispatch(x, order)
    at = order.slot[:, 0].long()
    for c in (0, 1, D // 2, D - 1):
        assert torch.equal(s[:, c][at], x[:, c])
    back = m.combine(s, order)
    del s
    assert torch.equal(back, x)


@pytest.mark.parametrize("which", ("dispatch", "combine"))
def test_rows_gradient_against_differences(m, which):
    order, slot, kept = _route(m, 9, 3, 4, 2)
    g = gen(3)
    n, D, h = (9 if which == "dispatch" else 27), 50, 0.25
    f = getattr(m, which)
    x, w = torch.randn(n, D, generator=g), torch.rand(9, 3, generator=g)
    dx, dw = torch.randn(n, D, generator=g), torch.randn(9, 3, generator=g)
    up = torch.randn(27 if which == "dispatch" else 9, D, generator=g)
    gx, gw = x.to(DEV).requires_grad_(), w.to(DEV).requires_grad_()
    f(gx, order, gw).backward(up.to(DEV))
    value = lambda a, b: float((f(a.to(DEV), order, b.to(DEV)).double().cpu() * up.double()).sum())  # noqa: E731
    # linear in each: central differences are exact but for rounding
    for grad, d, plus, minus in ((gx.grad, dx, (x + h * dx, w), (x - h * dx, w)), (gw.grad, dw, (x, w + h * dw), (x, w - h * dw))):
        slope = float((grad.double().cpu() * d.double()).sum())
        size = float(up.abs().sum()) * 4
        assert abs(slope - (value(*plus) - value(*minus)) / (2 * h)) <= 1e-6 * size / h


def test_gradients_once(m):
    """A graph of the gradients is refused where it is used, not before; what needs no gradient gets none."""
    x = torch.randn(3, 20, device=DEV, requires_grad=True)
    (d,) = torch.autograd.grad(m.log_probs(x).log_sum.sum(), x, create_graph=True)
    assert torch.isfinite(d).all()
    with pytest.raises(RuntimeError, match="once"):
        d.square().sum().backward()
    order = m.sort_by_class(torch.tensor([[0, 1], [1, 1], [0, 0]], device=DEV), 2)
    w = torch.rand(3, 2, device=DEV, requires_grad=True)
    (d,) = torch.autograd.grad(m.dispatch(x, order, w).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once"):
        d.sum().backward()
    (dw,) = torch.autograd.grad(m.combine(torch.ones(6, 5, device=DEV), order, w).sum(), w)
    assert torch.equal(dw, torch.full((3, 2), 5.0, device=DEV))
    with torch.no_grad():
        assert not m.log_probs(x, top=2).top.requires_grad and not m.dispatch(x, order, w).requires_grad
    out = m.log_probs(x, top=2)
    assert out.top.requires_grad and not out.top_index.requires_grad and out.given is None


# ----------------------------------------------------------------------------- streams and graphs
def _all(m, s):
    scores = m.block_scores(s["x"], m.BlockScaled(s["codes"], s["scales"]), bias=s["bias"])
    p = m.log_probs(scores, s["given"], top=2, temperature=2.0)
    order = m.sort_by_class(p.top_index, 40)
    rows = m.dispatch(s["x"], order, p.top.exp())
    return [scores, *p, *order, rows, m.combine(rows, order, p.top.exp())]


def _state(m, seed):
    g = gen(seed)
    q = m.quantize_blocks(torch.randn(40, 700, generator=g).to(DEV))
    return dict(x=torch.randn(30, 700, generator=g).to(DEV), codes=q.codes, scales=q.scales,
                bias=torch.randn(40, generator=g).to(DEV), given=torch.randint(0, 40, (30,), generator=g).to(DEV))


def test_another_stream_and_a_graph(m):
    states = [_state(m, seed) for seed in range(4)]
    want = [[t.clone() for t in _all(m, s)] for s in states]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = _all(m, states[0])
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want[0]))
    static = {k: v.clone() for k, v in states[0].items()}
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _all(m, static)
    for n in (1, 2, 3, 0, 1):
        for k in static:
            static[k].view(torch.uint8).copy_(states[n][k].view(torch.uint8))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want[n])), n
        assert all(torch.equal(a, b) for a, b in zip(_all(m, states[n]), want[n])), n  # eager work in between


def test_probs_many_givens(m):
    """More given and listed candidates than a wavefront has lanes, with repeats."""
    g = gen(21)
    x = torch.randn(3, 900, generator=g) * 2
    given = torch.randint(0, 60, (3, 100), generator=g)
    given[torch.rand(3, 100, generator=g) < 0.1] = -1
    _probs_check(m, x, given, 40, 1.2)


def test_rows_foreign_slots_stay_in_bounds(m):
    """Places outside the sorted rows (an order from elsewhere) are not read, nor is anything written there."""
    order = m.sort_by_class(torch.tensor([0, 1, 0, 1], device=DEV), 2)
    bad = order._replace(slot=torch.tensor([[0], [-5], [1 << 30], [2]], dtype=torch.int32, device=DEV))
    x = torch.ones(4, 33, device=DEV)
    s = m.dispatch(x, bad)
    assert (s[0] == 1).all() and (s[2] == 1).all()
    w = torch.full((4, 1), 2.0, device=DEV, requires_grad=True)
    back = m.combine(x, bad, w)
    assert torch.equal(back[:, 0].detach().cpu(), torch.tensor([2.0, 0, 0, 2.0]))
    (dw,) = torch.autograd.grad(back.sum(), w)
    assert torch.equal(dw.cpu(), torch.tensor([[33.0], [0], [0], [33.0]]))


def test_one_image_of_every_type(m):
    """A single image takes its own kernel: the same scores as from its blocks."""
    g = gen(31)
    refs = m.quantize_blocks(torch.randn(37, 515, generator=g).to(DEV))
    for dtype in (F32, F16, BF16):
        x = torch.randn(3, 515, generator=g).to(dtype)[1:2]
        x[0, 100] = 0.0
        for out in (F32, BF16):
            got = m.block_scores(x.to(DEV), refs, out_dtype=out)
            assert torch.equal(got, m.block_scores(m.quantize_blocks(x.to(DEV)), refs, out_dtype=out))
        x[0, 300] = math.nan
        assert m.block_scores(x.to(DEV), refs).isnan().all()


def test_views_that_hold_other_values(m):
    """Negative and conjugate views count as what they show, in values, weights and upstream gradients."""
    g = gen(41)
    c = torch.randn(6, 40, dtype=torch.complex64, generator=g).to(DEV)
    view = c.conj().imag
    plain = view.resolve_neg().contiguous()
    assert view.is_neg() and not plain.is_neg()
    for a, b in zip(m.log_probs(view, top=3), m.log_probs(plain, top=3)):
        assert a is b is None or torch.equal(a, b)
    x, y = (v.detach().requires_grad_() for v in (view, plain))
    up = torch.randn(6, dtype=torch.complex64, generator=g).to(DEV).conj().imag
    dx, = torch.autograd.grad(m.log_probs(x).entropy, x, up)
    dy, = torch.autograd.grad(m.log_probs(y).entropy, y, up.resolve_neg())
    assert torch.equal(dx, dy)
    q, r = m.quantize_blocks(view), m.quantize_blocks(plain)
    assert torch.equal(q.codes.view(torch.uint8), r.codes.view(torch.uint8)) and torch.equal(q.scales, r.scales)
    bias = torch.randn(6, dtype=torch.complex64, generator=g).to(DEV).conj().imag
    assert torch.equal(m.block_scores(view, r, bias=bias), m.block_scores(plain, r, bias=bias.resolve_neg()))
    order = m.sort_by_class(torch.randint(0, 3, (6, 2), generator=g).to(DEV), 3)
    w = torch.randn(6, 2, dtype=torch.complex64, generator=g).to(DEV).conj().imag
    s = m.dispatch(plain, order, w.resolve_neg())
    assert torch.equal(m.dispatch(view, order, w), s)
    assert torch.equal(m.combine(-(-s), order, w), m.combine(s, order, w.resolve_neg()))
    assert torch.equal(m.dispatch(c.conj(), order, w), m.dispatch(c.conj().resolve_conj(), order, w.resolve_neg()))


def test_blocks_from_any_address(m):
    g = gen(42)
    x = torch.randn(40, 300, generator=g).to(DEV)
    q = m.quantize_blocks(torch.randn(70, 300, generator=g).to(DEV))
    moved = []
    for t in q:
        room = torch.empty(t.numel() + 3, dtype=torch.uint8, device=DEV)[3:]
        room.copy_(t.view(torch.uint8).flatten())
        moved.append(room.view(t.dtype).view(t.shape))
    assert moved[0].data_ptr() % 16
    assert torch.equal(m.block_scores(x, m.BlockScaled(*moved)), m.block_scores(x, q))


@pytest.mark.parametrize("M,N,K,out_dtype,bias", [(16, 300, 16640, F32, True), (16, 4100, 1000, BF16, False),
                                                  (24, 2000, 8320, F32, False), (20, 4099, 640, F32, True),
                                                  (32, 150, 4224, BF16, True)])
def test_scores_of_few_images(m, M, N, K, out_dtype, bias):
    _scores_check(m, M, N, K, out_dtype, bias, seed=5)


@pytest.mark.parametrize("n,E", [(2048, 4096), (2049, 4096), (4096, 16), (4097, 16), (5000, 1000), (8193, 64), (32768, 64),
                                 (32769, 64), (140000, 4096), (530001, 64)])
def test_sort_where_its_split_changes(m, n, E):
    classes = (torch.rand(n, generator=gen(n)) ** 2 * (E + 1)).long()
    got = m.sort_by_class(classes.to(DEV), E)
    order = torch.sort(classes, stable=True)[1]
    assert torch.equal(got.order.cpu().long(), order)
    assert torch.equal(got.slot.cpu().long()[order, 0], torch.arange(n))
    assert torch.equal(got.offsets.cpu().long(), torch.searchsorted(classes[order].contiguous(), torch.arange(E + 1)))


@pytest.mark.parametrize("top", [1, 4, 12, 31, 33, 64])
@pytest.mark.parametrize("kind", ["rising", "falling", "narrow", "few values", "one lane"])
def test_probs_candidates_of_every_number(m, kind, top):
    """Rows that bring many, few or clustered candidates to a wavefront's tile."""
    V, g = 9001, gen(top)
    x = torch.randn(3, V, generator=g)
    if kind in ("rising", "falling"):
        x = x.sort(1, descending=kind == "falling")[0]
    elif kind == "narrow":
        x = -20000 + x  # differ in the last bits only
    elif kind == "few values":
        x = x.sign() + (x > 2).float()
    else:
        x[:, 512:516] += 20  # neighbours, which one lane reads
        x[:, 4096:4100] += 21
    _probs_check(m, x, torch.randint(0, V, (3, 1), generator=g), top, 2.0)


def test_probs_streamed(m):
    """Scores larger than the caches: rows at both ends against the oracle."""
    T, V = 1501, 36867  # 221 MB
    for dtype in (F32, BF16):
        n = T if dtype == F32 else 2 * T
        x = (torch.randn(n, V, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV) * 2).to(dtype).requires_grad_()
        given = torch.arange(n, device=DEV)
        out = m.log_probs(x, given, top=9, temperature=1.5)
        up = [torch.linspace(-1, 1, n, device=DEV), torch.linspace(0, 0.1, n, device=DEV), torch.linspace(0.5, 0, n, device=DEV),
              torch.ones(n, 9, device=DEV) * 0.1]
        (d,) = torch.autograd.grad([out.given, out.entropy, out.log_sum, out.top], [x], up)
        rows = torch.tensor([0, 1, n // 2, n - 1])
        at = rows.to(DEV)
        want = R.log_probs(x.detach()[at].cpu(), given[at].cpu()[:, None], 9, 1.5, None,
                           (up[0][at].cpu()[:, None], up[1][at].cpu(), up[2][at].cpu(), up[3][at].cpu()))
        near(out.given[at][:, None], want["given"], 2e-5, "given")
        near(out.log_sum[at], want["log_sum"], 2e-5, "log_sum")
        near(out.entropy[at], want["entropy"], 4e-5, "entropy")
        assert torch.equal(out.top_index[at].cpu(), want["top_index"])
        near(d[at], want["d_scores"], 1e-5 + R.U[dtype] * want["d_scores"].abs() * 1.01, "d_scores")
