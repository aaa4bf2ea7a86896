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


@pytest.mark.parametrize("G", [1, 3, 90])
@pytest.mark.parametrize("index", [300, 10 ** 12, -2, -(2 ** 63)])
def test_gradient_of_given_candidates_out_of_range(m, index, G):
    """Their log probability is NaN, and so is the gradient of their row, but for masked places; of a result that has no
    share in the loss (an upstream gradient of 0) there is none."""
    V = 300
    x = torch.randn(4, V, generator=gen(2))
    mask = torch.rand(V, generator=gen(3)) < 0.8
    given = torch.randint(0, V, (4, G), generator=gen(4))
    mask[given.flatten()] = True
    mask[5] = False
    given[given == 5] = -1
    fine = given.clone()
    given[1:, G // 2] = index
    fine[1:, G // 2] = -1
    up = torch.randn(4, G, generator=gen(5))
    up[2, G // 2] = 0.0

    def gradient(which):
        s = x.to(DEV).requires_grad_()
        out = m.log_probs(s, which.to(DEV), mask=mask.to(DEV))
        return out.given.detach().cpu(), torch.autograd.grad(out.given, s, up.to(DEV))[0].cpu()

    got, d = gradient(given)
    want, d_fine = gradient(fine)
    assert got[1:, G // 2].isnan().all() and int(got.isnan().sum()) == 3
    assert torch.equal(d[[0, 2]], d_fine[[0, 2]]) and torch.isfinite(d[[0, 2]]).all()
    assert d[[1, 3]][:, mask].isnan().all() and (d[:, ~mask] == 0).all()


def _gradient_in_64_bits(x, given, mask, top_index, temperature, d_given, d_top):
    """(d_scores, tolerance) from the formula, on the GPU.  An fp32 sum of n values is at most n 2^-24 of their
    magnitudes off; p is 1e-5 off, as are its logarithm and the entropy (which carry no gradient here)."""
    z = x.double() / temperature
    if mask is not None:
        z = z.masked_fill(~mask, -math.inf)
    p = torch.softmax(z, 1)
    at, mag, count = (torch.zeros_like(p) for _ in range(3))
    for index, up in ((given, d_given.double()), (top_index, d_top.double())):
        ok = index >= 0
        safe = index.clamp_min(0)
        up = torch.where(ok, up, 0.0)
        at.scatter_add_(1, safe, up)
        mag.scatter_add_(1, safe, up.abs())
        count.scatter_add_(1, safe, ok.double())
    n = given.shape[1] + top_index.shape[1]
    total, size = at.sum(1, keepdim=True), mag.sum(1, keepdim=True)
    if mask is not None:
        at, mag = at.masked_fill(~mask, 0.0), mag.masked_fill(~mask, 0.0)
    want = (at - p * total) / temperature
    u = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}[x.dtype]
    tol = ((count + 4) * 2.0 ** -24 * mag + p * (1e-5 + (n / 64 + 8) * 2.0 ** -24) * size) / temperature
    return want, tol + 1.01 * u * want.abs() + (2.0 ** -25 if x.dtype == F16 else 1e-37)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("T,V,G,places", [(3, 700, 5000, 700), (2, 5003, 3000, 5003), (2, 9000, 3001, 7), (5, 2049, 61, 2049),
                                          (2, 40001, 40001, 40001), (3, 1, 200, 1), (300, 3100, 130, 3100)])
@pytest.mark.parametrize("masked", [False, True])
def test_gradient_of_thousands_of_given_candidates(m, T, V, G, places, masked, dtype):
    """More given and listed candidates than lanes, with repeats within and between groups of lanes, -1 among them."""
    g = gen(V + G)
    x = (torch.randn(T, V, generator=g) * 2).to(dtype).to(DEV)
    given = (torch.randint(0, places, (T, G), generator=g) * 131 % V).to(DEV)
    given[torch.rand(T, G, generator=g).to(DEV) < 0.1] = -1
    mask = (torch.rand(T, V, generator=g) < 0.7).to(DEV) if masked and V > 1 else None
    if mask is not None:
        mask[:, 0] = True
    top = min(V, 7)
    d_given, d_top = torch.randn(T, G, generator=g).to(DEV), torch.randn(T, top, generator=g).to(DEV)
    s = x.clone().requires_grad_()
    out = m.log_probs(s, given, top=top, temperature=1.7, mask=mask)
    (d,) = torch.autograd.grad([out.given, out.top], [s], [d_given, d_top], retain_graph=True)
    want, tol = _gradient_in_64_bits(x, given, mask, out.top_index, 1.7, d_given, d_top)
    off = (d.double() - want).abs() - tol
    assert float(off.max()) <= 0, float(off.max())
    (again,) = torch.autograd.grad([out.given, out.top], [s], [d_given, d_top])
    assert torch.equal(d, again)


def test_gradient_of_given_candidates_is_not_quadratic_in_their_number(m):
    """Every candidate given: 16384 of 16384 in four rows are 1 MB of inputs, a fraction of a millisecond's work; each
    walked for each other would be 1e9 loads, over a tenth of a second."""
    T, V = 4, 16384
    x = torch.randn(T, V, generator=gen(6)).to(DEV).requires_grad_()
    out = m.log_probs(x, torch.randint(0, V, (T, V), generator=gen(7)).to(DEV))
    up = torch.ones_like(out.given)
    ms = []
    for _ in range(4):
        start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        start.record()
        torch.autograd.grad(out.given, x, up, retain_graph=True)
        end.record()
        torch.cuda.synchronize()
        ms.append(start.elapsed_time(end))
    assert min(ms) < 10, ms


@pytest.mark.parametrize("T,D", [(4, 33), (600, 2049)])
def test_places_from_elsewhere_leave_the_last_row_alone(m, T, D):
    """Slots outside the sorted rows write nothing: not to the last place either, which is another row's."""
    order = m.sort_by_class(torch.zeros(T, dtype=torch.int64, device=DEV), 1)
    slot = torch.arange(T, dtype=torch.int32).flip(0).view(T, 1)
    bad = torch.arange(1, T, 2)
    slot[bad, 0] = torch.tensor([-5, T, 1 << 30, -(2 ** 31)], dtype=torch.int32)[torch.arange(len(bad)) % 4]
    foreign = order._replace(slot=slot.to(DEV))
    x = torch.randn(T, D, generator=gen(8))
    w = torch.rand(T, 1, generator=gen(9))
    gx, gw = x.to(DEV).requires_grad_(), w.to(DEV).requires_grad_()
    s = m.dispatch(gx, foreign, gw)
    good = torch.arange(0, T, 2)
    at = slot[good, 0].long()
    assert at.max() == T - 1
    assert torch.equal(s.detach().cpu()[at], w[good] * x[good])
    up = torch.randn(T, D, generator=gen(10))
    dx, dw = torch.autograd.grad(s, (gx, gw), up.to(DEV))
    assert torch.equal(dx.cpu()[good], w[good] * up[at]) and (dx[bad] == 0).all() and (dw[bad] == 0).all()
    y = m.combine(s.detach(), foreign, gw).detach().cpu()
    assert torch.equal(y[good], w[good] * (w[good] * x[good])) and (y[bad] == 0).all()


def _random_blocks(m, rows, K, lo, hi, g):
    """BlockScaled with every finite code and scale bytes lo .. hi."""
    codes = torch.randint(0, 256, (rows, K), generator=g, dtype=torch.int64).to(torch.uint8)
    codes[(codes & 127) == 127] = 0
    scales = torch.full((K // 128, -(-rows // 16) * 16), 127, dtype=torch.uint8)
    scales[:, :rows] = torch.randint(lo, hi + 1, (K // 128, rows), generator=g).to(torch.uint8)
    value = codes.view(torch.float8_e4m3fn).float().double().view(rows, K // 128, 128)
    value = (value * torch.exp2(scales[:, :rows].t().double() - 127)[:, :, None]).view(rows, K)
    return m.BlockScaled(codes.to(DEV).view(torch.float8_e4m3fn), scales.to(DEV)), value


@pytest.mark.parametrize("M,N,K", [(1, 40, 1280), (9, 130, 512), (20, 33, 256), (70, 100, 768)])
@pytest.mark.parametrize("a,b", [((3, 6), (243, 246)), ((243, 246), (3, 6)), ((3, 60), (200, 230))])
def test_scores_of_blocks_at_the_ends_of_the_exact_range(m, M, N, K, a, b):
    """Scale bytes 3 .. 246: every code times its scale is a bfloat16, and the scores are exact but for the sum's
    roundings (nb + 8 of 2^-23 of the magnitudes' sum)."""
    g = gen(M)
    qa, va = _random_blocks(m, M, K, *a, g)
    qb, vb = _random_blocks(m, N, K, *b, g)
    want, mag = va @ vb.t(), va.abs() @ vb.abs().t()
    assert float(mag.max()) < 3e38
    got = m.block_scores(qa, qb).double().cpu()
    assert ((got - want).abs() <= (K // 128 + 8) * 2.0 ** -23 * mag).all()


@pytest.mark.parametrize("M,N,K", [(1, 40, 1280), (9, 130, 512), (70, 100, 768)])
def test_scores_of_blocks_below_the_exact_range(m, M, N, K):
    """Scale bytes 0 .. 2: each value to a multiple of 2^-133, bfloat16's least, at most one off."""
    g = gen(M)
    qa, va = _random_blocks(m, M, K, 0, 2, g)
    qb, vb = _random_blocks(m, N, K, 230, 240, g)
    want, mag = va @ vb.t(), va.abs() @ vb.abs().t()
    got = m.block_scores(qa, qb).double().cpu()
    tol = (K // 128 + 8) * 2.0 ** -23 * mag + 2.0 ** -133 * vb.abs().sum(1)[None]
    assert ((got - want).abs() <= tol).all()


@pytest.mark.parametrize("M", [1, 5, 40])
def test_scores_of_the_largest_float32(m, M):
    """Values from 248 2^120 = 3.297e38 up are nearest to the code 256 at that scale, 2^128, and count as infinite;
    those below as 240 2^120, finite."""
    x, b = torch.zeros(M, 200), torch.full((20, 200), 2.0 ** -30)
    limit = 248 * 2.0 ** 120
    x[:, 3], b[7, 3] = torch.nextafter(torch.tensor(limit), torch.tensor(0.0)), 0.0
    got = m.block_scores(x.to(DEV), b.to(DEV)).cpu()
    want = torch.full((M, 20), 240 * 2.0 ** 90)
    want[:, 7] = 0.0
    assert torch.equal(got, want)
    x[:, 3] = limit
    got = m.block_scores(x.to(DEV), b.to(DEV)).cpu()
    assert (got[:, [i for i in range(20) if i != 7]] == math.inf).all() and got[:, 7].isnan().all()
    x[:, 3] = -torch.finfo(F32).max
    assert (m.block_scores(x.to(DEV), b.to(DEV)).cpu()[:, 0] == -math.inf).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T,k,D", [(5, 2, 40), (700, 3, 1301), (40, 5, 4099), (300, 8, 129)])
def test_rows_with_some_places_from_elsewhere(m, T, k, D, dtype):
    """Choices without a place beside ones that have theirs, dropped ones among them, both ways and with the weights'
    gradient: the others' rows are as they are without them."""
    g = gen(T)
    classes = torch.randint(-1, 4, (T, k), generator=g)
    order = m.sort_by_class(classes.to(DEV), 4)
    slot = order.slot.cpu()
    away = torch.rand(T, k, generator=g) < 0.3
    away[0], away[1, 0] = True, False
    away |= slot == T * k - 1
    away[T // 2, k - 1] = False
    far = torch.tensor([-1, T * k, 1 << 30, -(2 ** 31)], dtype=torch.int32)
    foreign = torch.where(away, far[torch.arange(T * k).view(T, k) % 4], slot)
    order = order._replace(slot=foreign.to(DEV))
    held = ~away
    kept = held & (slot < int(order.offsets[-1]))
    x, up = torch.randn(T, D, generator=g).to(dtype), torch.randn(T, D, generator=g).to(dtype)
    w = torch.rand(T, k, generator=g)
    s = m.dispatch(x.to(DEV), order, w.to(DEV)).cpu()
    row = torch.arange(T)[:, None].expand(T, k)
    want = torch.where(kept[:, :, None], w[:, :, None] * x.float()[:, None], 0.0).to(dtype)
    assert torch.equal(s[slot[held].long()], want[held])
    y = torch.randn(T * k, D, generator=g).to(dtype)
    gy, gw = y.to(DEV).requires_grad_(), w.to(DEV).requires_grad_()
    dy, dw = torch.autograd.grad(m.combine(gy, order, gw), (gy, gw), up.to(DEV))
    want = torch.where(kept[:, :, None], w[:, :, None] * up.float()[:, None], 0.0).to(dtype)
    assert torch.equal(dy.cpu()[slot[held].long()], want[held])
    part = up.double()[row] * y.double()[slot.long()]
    want, mag = torch.where(kept, part.sum(2), 0.0), part.abs().sum(2)
    assert ((dw.double().cpu() - want).abs() <= (D / 64 + 16) * 2.0 ** -24 * mag).all() and (dw.cpu()[~kept] == 0).all()


def test_forward_mode_is_refused(m):
    """A forward-mode tangent of what is differentiable is refused, with and without grad mode, not dropped."""
    import torch.autograd.forward_ad as fw
    x = torch.randn(4, 20, device=DEV)
    order = m.sort_by_class(torch.tensor([0, 1, 0, 1], device=DEV), 2)
    w = torch.rand(4, 1, device=DEV)
    calls = [lambda d: m.log_probs(d), lambda d: m.dispatch(d, order), lambda d: m.combine(d, order, w),
             lambda d: m.dispatch(x, order, d[:, :1]), lambda d: m.combine(x, order, d[:, :1])]
    for call in calls:
        for grad in (True, False):
            with torch.set_grad_enabled(grad), fw.dual_level():
                with pytest.raises(NotImplementedError):
                    call(fw.make_dual(x, torch.ones_like(x)))
    assert torch.isfinite(m.log_probs(x).log_sum).all()


def test_log_probs_of_arguments_of_any_layout(m):
    """Masks, given candidates and upstream gradients that are views: strided, transposed, expanded."""
    g = gen(12)
    T, V = 9, 1500
    x = torch.randn(T, V, generator=g).to(DEV)
    ups = torch.randn(T, 3, generator=g).to(DEV), torch.randn(T, generator=g).to(DEV)

    def results(mask, given, up_given, up_sum):
        s = x.clone().requires_grad_()
        out = m.log_probs(s, given, top=6, mask=mask)
        (d,) = torch.autograd.grad([out.given, out.log_sum], [s], [up_given, up_sum])
        return [*out, d]

    wide = (torch.rand(T, V + 77, generator=g) < 0.6).to(DEV)
    tall = (torch.rand(V, T, generator=g) < 0.6).to(DEV)
    one = (torch.rand(V, generator=g) < 0.6).to(DEV)
    given = torch.randint(0, V, (3, T), generator=g).to(DEV)
    up_wide = torch.zeros(T, 9, device=DEV)
    up_wide[:, ::3] = ups[0]
    up_sum = torch.zeros(2 * T, device=DEV)
    up_sum[::2] = ups[1]
    for mask in (wide[:, 50:50 + V], tall.t(), one.expand(T, V), one.repeat_interleave(2)[::2]):
        want = results(mask.contiguous(), given.t().contiguous(), *ups)
        got = results(mask, given.t(), up_wide[:, ::3], up_sum[::2])
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    scalar = results(one, given.t(), torch.ones((), device=DEV).expand(T, 3), torch.ones((), device=DEV).expand(T))
    plain = results(one, given.t(), torch.ones(T, 3, device=DEV), torch.ones(T, device=DEV))
    assert all(torch.equal(a, b) for a, b in zip(scalar, plain))


def test_log_probs_of_more_dimensions_with_masks(m):
    g = gen(13)
    x = torch.randn(4, 5, 70, generator=g).to(DEV).requires_grad_()
    mask = (torch.rand(4, 5, 70, generator=g) < 0.5).to(DEV)
    given = torch.randint(0, 70, (4, 5, 2), generator=g).to(DEV)
    out = m.log_probs(x, given, top=3, mask=mask)
    flat = m.log_probs(x.view(20, 70), given.view(20, 2), top=3, mask=mask.view(20, 70))
    assert out.given.shape == (4, 5, 2) and out.top.shape == (4, 5, 3) and out.entropy.shape == (4, 5)
    for a, b in zip(out, flat):
        assert torch.equal(a.reshape(b.shape), b)
    a, b = (torch.autograd.grad(o.given.exp().sum() + o.top.sum() + o.entropy.sum(), x)[0] for o in (out, flat))
    assert torch.equal(a, b) and (a[~mask] == 0).all()
    line = x.detach()[0, 0]
    one = m.log_probs(line, given[0, 0], top=3, mask=mask[0, 0])
    assert torch.equal(one.given, out.given[0, 0]) and torch.equal(one.top_index, out.top_index[0, 0])


def test_nothing_to_do(m):
    """No rows, no choices, no candidates wanted: empty or zero results and gradients of the right shapes."""
    x = torch.empty(0, 70, device=DEV, requires_grad=True)
    out = m.log_probs(x, torch.empty(0, 2, dtype=torch.int64, device=DEV), top=3)
    (d,) = torch.autograd.grad([out.given, out.log_sum, out.top], [x], [out.given, out.log_sum, out.top])
    assert d.shape == (0, 70)
    x = torch.randn(3, 70, device=DEV, requires_grad=True)
    out = m.log_probs(x, torch.empty(3, 0, dtype=torch.int64, device=DEV))
    assert out.given.shape == (3, 0) and out.top.shape == (3, 0)
    (d,) = torch.autograd.grad(out.given.sum() + out.top.sum(), x)
    assert (d == 0).all()
    order = m.sort_by_class(torch.empty(4, 0, dtype=torch.int64, device=DEV), 3)
    assert order.slot.shape == (4, 0) and order.offsets.tolist() == [0, 0, 0, 0]
    x = torch.randn(4, 30, device=DEV, requires_grad=True)
    y = torch.empty(0, 30, device=DEV, requires_grad=True)
    w = torch.empty(4, 0, device=DEV, requires_grad=True)
    s, total = m.dispatch(x, order, w), m.combine(y, order, w)
    assert s.shape == (0, 30) and total.shape == (4, 30) and (total == 0).all()
    dx, dw = torch.autograd.grad(s, (x, w), torch.empty(0, 30, device=DEV))
    assert (dx == 0).all() and dw.shape == (4, 0)
    dy, dw = torch.autograd.grad(total, (y, w), torch.ones(4, 30, device=DEV))
    assert dy.shape == (0, 30) and dw.shape == (4, 0)


def test_rows_of_arguments_of_any_layout(m):
    """Weights and upstream gradients that are views, complex rows whose gradient comes in conjugate."""
    g = gen(14)
    classes = torch.randint(-1, 5, (3, 40), generator=g).to(DEV)
    order = m.sort_by_class(classes.t(), 5)
    same = m.sort_by_class(classes.t().contiguous(), 5)
    assert all(torch.equal(a, b) for a, b in zip(order, same))
    x = torch.randn(40, 12, 7, dtype=torch.complex64, generator=g).to(DEV)
    w = torch.rand(3, 40, generator=g).to(DEV).t()
    up = torch.randn(120, 7, 12, dtype=torch.complex64, generator=g).to(DEV).transpose(1, 2).conj()

    def results(x, w, up):
        gx, gw = x.detach().requires_grad_(), w.detach().requires_grad_()
        s = m.dispatch(gx, order, gw)
        return [s, *torch.autograd.grad(s, (gx, gw), up)]

    got = results(x.transpose(1, 2), w, up.transpose(1, 2))
    want = results(x.transpose(1, 2).contiguous(), w.contiguous(), up.transpose(1, 2).resolve_conj().contiguous())
    assert all(torch.equal(a, b) for a, b in zip(got, want))
