"""Each kernel, tile and way of splitting that the matching operators' rules choose, against their definitions in 64 bits,
computed for whole tensors on the GPU.  Sizes are chosen so that every choice runs with values that tell all places
apart; tolerances from the roundings (u a type's unit roundoff, 2^-24 in fp32):
* scores: nb + 8 additions of 2 u each of the magnitudes' sum, plus u of the result in 16 bits;
* log probabilities 2e-6 (1 + |value|), the entropy twice that; score gradients 1e-5 of the row's upstream
  magnitudes / temperature, times p (1 + |ln p| + H), plus 2^-4 of it at given and listed places, plus u of the result;
* row sums: k + 1 roundings of the magnitudes' sum, plus u of the result; weight gradients D / 64 + 16 roundings of the
  magnitudes' sum."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
U = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}


@pytest.fixture(scope="module")
def m(gpu):
    from torch_projectors import matching
    return matching


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def least(dtype):
    return 2.0 ** -25 if dtype == F16 else 1e-37  # half of the type's least step


def near(got, want, tol, what):
    got = got.detach().double()
    assert got.shape == want.shape, what
    inf = want.isinf()
    assert torch.equal(got[inf], want[inf]), what
    off = torch.where(inf, 0.0, (got - want).abs() - tol)
    assert not off.isnan().any() and float(off.max()) <= 0, (what, float(off.max()))


# ----------------------------------------------------------------------------- scores
def _value(blocks):
    rows = blocks.codes.shape[0]
    unit = torch.exp2(blocks.scales[:, :rows].t().double() - 127)
    return (blocks.codes.float().double().view(rows, -1, 128) * unit[:, :, None]).view(rows, -1)


# the first two choose tiles of 128 x 128 in one range of the blocks and in seven, the next two 256 x 256 likewise
@pytest.mark.parametrize("M,N,K,ranges", [
    (1500, 2050, 128, 1), (2050, 200, 16640, 7), (3000, 4099, 128, 1), (500, 4099, 16640, 7),
    (2500, 2500, 801, 1), (1000, 1100, 16600, 7), (4097, 4500, 100, 1), (4095, 8190, 640, 1), (333, 1999, 8280, 4),
    (257, 8000, 16640, 2)])
@pytest.mark.parametrize("out_dtype,bias", [(F32, True), (BF16, False), (F32, False), (BF16, True)])
def test_scores_by_every_tile(m, M, N, K, ranges, out_dtype, bias):
    from torch_projectors import capi
    nb = -(-K // 128)
    assert capi.lib().tp_block_scores_work(M, N, nb) == (ranges * M * N * 4 if ranges > 1 else 0)
    g = gen(M)
    fall = torch.exp(torch.linspace(0, -7, K, device=DEV))
    a, b = torch.randn(M, K, generator=g, device=DEV) * fall, torch.randn(N, K, generator=g, device=DEV) * fall
    f = torch.randn(N, generator=g, device=DEV) if bias else None
    qa, qb = m.quantize_blocks(a), m.quantize_blocks(b)
    va, vb = _value(qa), _value(qb)
    want, mag = va @ vb.t(), va.abs() @ vb.abs().t()
    if bias:
        want, mag = want + f.double(), mag + f.double().abs()
    tol = (nb + 8) * 2.0 ** -23 * mag + (U[BF16] * want.abs() * 1.01 if out_dtype == BF16 else 0.0)
    got = m.block_scores(qa, qb, bias=f, out_dtype=out_dtype)
    assert got.dtype == out_dtype
    near(got, want, tol, "scores")
    assert torch.equal(m.block_scores(a, qb, bias=f, out_dtype=out_dtype), got)
    assert torch.equal(m.block_scores(qa, qb, bias=f, out_dtype=out_dtype), got)


# ----------------------------------------------------------------------------- log probabilities
def _probs_check(m, T, V, top, dtype, mask=None, seed=0, temperature=1.5, ties=False):
    g = gen(seed)
    x = torch.randn(T, V, generator=g, device=DEV) * 3
    if ties:
        x = x.round()
    x = x.to(dtype)
    if mask is not None:  # what masked places hold is not used
        hidden = torch.tensor([math.nan, math.inf, 1e4], device=DEV, dtype=dtype)[torch.arange(V, device=DEV) % 3]
        x = torch.where(mask, x, hidden)
    given = torch.randint(0, V, (T, 2), generator=g, device=DEV)
    ups = [torch.randn(s, generator=g, device=DEV) for s in ((T, 2), (T,), (T,), (T, top))]
    s = x.requires_grad_()
    out = m.log_probs(s, given, top=top, temperature=temperature, mask=mask)
    results = [out.given, out.entropy, out.log_sum] + ([out.top] if top else [])
    (d,) = torch.autograd.grad(results, s, ups[:len(results)])

    z = x.detach().double() / temperature
    if mask is not None:
        z = torch.where(mask, z, -math.inf)
    none = (z == -math.inf).all(1, keepdim=True)
    most = torch.where(none, 0.0, z.amax(1, keepdim=True))
    z = z - most
    ls = torch.log(z.exp().sum(1, keepdim=True))
    lp = torch.where(none, -math.inf, z - ls)
    p = lp.exp()
    lp0 = torch.where(p > 0, lp, 0.0)
    H = -(p * lp0).sum(1)
    value = lambda v: 2e-6 * (1 + v.abs().nan_to_num(0, 0, 0))  # noqa: E731
    log_sum = torch.where(none, -math.inf, most + ls)[:, 0]
    near(out.log_sum, log_sum, value(log_sum), "log_sum")
    near(out.entropy, H, 2 * value(H), "entropy")
    want = lp.gather(1, given)
    near(out.given, want, value(want), "given")
    listed = torch.empty(T, 0, dtype=torch.int64, device=DEV)
    if top:
        # of the scores themselves: ties go to the lowest index
        keys = x.detach().float() if mask is None else torch.where(mask, x.detach().float(), -math.inf)
        best, listed = (v[:, :top] for v in torch.sort(keys, dim=1, descending=True, stable=True))
        listed = torch.where(best == -math.inf, -1, listed)
        assert torch.equal(out.top_index, listed)
        want = torch.where(listed < 0, -math.inf, lp.gather(1, listed.clamp_min(0)))
        near(out.top, want, value(want), "top")
    at, here, total, size = torch.zeros_like(p), torch.zeros_like(p), 0.0, 0.0
    for index, up in ((given, ups[0].double()), (listed, ups[3].double())):
        if index.numel():
            up = torch.where(index < 0, 0.0, up)
            at.scatter_add_(1, index.clamp_min(0), up)
            here.scatter_add_(1, index.clamp_min(0), (index >= 0).double())
            total, size = total + up.sum(1, keepdim=True), size + up.abs().sum(1, keepdim=True)
    dH, dL = ups[1].double()[:, None], ups[2].double()[:, None]
    want = (p * (dL - total) - dH * p * (lp0 + H[:, None]) + at) / temperature
    allowed = ~none if mask is None else mask & ~none
    want = torch.where(allowed, want, 0.0)
    size = size + dH.abs() + dL.abs()
    tol = 1e-5 * size / temperature * (p * (1 + lp0.abs() + H[:, None]) + 2.0 ** -4 * (here > 0))
    near(d, want, tol + 1.01 * U[dtype] * want.abs() + least(dtype), "d_scores")


def _masks(T, V, shared, seed):
    """Selective everywhere, with whole tiles, whole wavefronts' and whole workgroups' parts and whole rows masked out."""
    g = gen(seed)
    mask = torch.rand(1 if shared else T, V, generator=g, device=DEV) < 0.4
    mask[0, 1024:3 * 1024] = False
    if V > 20000:
        mask[-1, 8 * 1024:V - 5000] = False
    if not shared:
        mask[T // 2] = False  # allows nothing
        mask[T // 2 + 1] = False
        mask[T // 2 + 1, V - 1] = True  # allows the last
        mask[T // 2 + 2, :-1024] = False
        mask[0, :2048] = False
    return mask[0] if shared else mask


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("shared", [True, False])
@pytest.mark.parametrize("T,V,top", [(6, 4099, 5), (700, 4099, 4), (2100, 3080, 8), (4300, 2500, 3), (5, 70001, 16),
                                     (5, 294911, 8), (300, 9000, 33)])
def test_masks_over_many_tiles(m, T, V, top, shared, dtype):
    _probs_check(m, T, V, top, dtype, _masks(T, V, shared, V), seed=T)


# one wavefront a row over many tiles, two, four, eight, and several workgroups
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("T,V,top", [(4099, 6001, 8), (4100, 2049, 40), (2049, 5003, 8), (1100, 5003, 12), (513, 9001, 8),
                                     (257, 8193, 64), (31, 40000, 9)])
@pytest.mark.parametrize("ties", [False, True])
def test_every_split_of_a_row(m, T, V, top, ties, dtype):
    _probs_check(m, T, V, top, dtype, seed=V, ties=ties)


@pytest.mark.parametrize("T,V,dtype,shared", [(1501, 36867, F32, None), (4100, 26000, BF16, None), (4099, 13001, F32, True),
                                              (4098, 26001, F16, True)])
def test_streamed_scores(m, T, V, dtype, shared):
    """Scores larger than the caches (200 MB and more), one to four wavefronts a row."""
    _probs_check(m, T, V, 9, dtype, None if shared is None else _masks(T, V, shared, 3), seed=1)


# ----------------------------------------------------------------------------- rows by class
def _rows_check(m, T, k, E, D, dtype, weighted, seed=0):
    g = gen(seed)
    classes = torch.randint(0, E, (T, k), generator=g, device=DEV)
    classes[torch.rand(T, k, generator=g, device=DEV) < 0.15] = -1  # dropped
    order = m.sort_by_class(classes, E)
    kept = order.slot < order.offsets[-1]
    at = order.slot.long()
    w = torch.rand(T, k, generator=g, device=DEV) if weighted else None
    factor = torch.where(kept, 1.0 if w is None else w.double(), 0.0)
    x, d_sum = (torch.randn(T, D, generator=g, device=DEV).to(dtype) for _ in range(2))
    y, d_sorted = (torch.randn(T * k, D, generator=g, device=DEV).to(dtype) for _ in range(2))
    u, one = U[dtype], 2.0 ** -24

    def spread(v):
        out = torch.zeros(T * k, D, dtype=torch.float64, device=DEV)
        for j in range(k):
            out[at[:, j]] = factor[:, j, None] * v.double()
        return out, (u + one) * out.abs() + least(dtype)

    def gather(v):
        out = torch.zeros(T, D, dtype=torch.float64, device=DEV)
        mag = torch.zeros_like(out)
        for j in range(k):
            part = factor[:, j, None] * v[at[:, j]].double()
            out += part
            mag += part.abs()
        return out, u * out.abs() + (k + 1) * one * mag * (1 + u) + least(dtype)

    def dots(a, b):
        out, mag = (torch.zeros(T, k, dtype=torch.float64, device=DEV) for _ in range(2))
        for j in range(k):
            part = a.double() * b[at[:, j]].double()
            out[:, j], mag[:, j] = part.sum(1), part.abs().sum(1)
        return out * kept, (D / 64 + 16) * one * mag * kept

    def leaf(v):
        return None if v is None else v.clone().requires_grad_()

    gx, gw = leaf(x), leaf(w)
    s = m.dispatch(gx, order, gw)
    near(s, *spread(x), "sorted")
    grads = torch.autograd.grad(s, [v for v in (gx, gw) if v is not None], d_sorted)
    del s
    near(grads[0], *gather(d_sorted), "d_x")
    if weighted:
        near(grads[1], *dots(x, d_sorted), "d_weights of dispatch")
    gy, gw = leaf(y), leaf(w)
    total = m.combine(gy, order, gw)
    near(total, *gather(y), "sum")
    grads = torch.autograd.grad(total, [v for v in (gy, gw) if v is not None], d_sum)
    near(grads[0], *spread(d_sum), "d_y")
    if weighted:
        near(grads[1], *dots(d_sum, y), "d_weights of combine")


# four wavefronts a row with and without the weights' gradient, one and two stretches at once
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("weighted", [True, False])
@pytest.mark.parametrize("k", [1, 2, 3, 5, 8])
@pytest.mark.parametrize("T,D", [(700, 1361), (520, 4099), (2100, 641), (2050, 1281)])
def test_rows_of_four_wavefronts(m, T, D, k, weighted, dtype):
    _rows_check(m, T, k, 9, D, dtype, weighted, seed=D + k)


# 32 MB of sorted rows and more, which are streamed, by one, four and sixteen wavefronts a row
@pytest.mark.parametrize("weighted", [True, False])
@pytest.mark.parametrize("T,k,D,dtype", [
    (2048, 2, 4225, F32), (4001, 3, 2051, BF16), (1003, 5, 4099, F16), (600, 8, 8193, F32), (9000, 2, 601, F32),
    (30001, 4, 301, BF16), (7000, 8, 400, F16), (20000, 1, 513, F32), (300, 2, 33001, F32), (90, 6, 66001, BF16),
    (65000, 2, 300, F32)])
def test_streamed_rows(m, T, k, D, dtype, weighted):
    assert T * k * D * (4 if dtype == F32 else 2) >= 1 << 25
    _rows_check(m, T, k, 12, D, dtype, weighted, seed=T)
