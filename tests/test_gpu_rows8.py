"""Scores in 8-bit integers on the GPU (matching.quantize_rows, row_scores): codes, scales and scores are those of the
definition (tests/pairs_reference.py) bit by bit, as the sums are exact and every rounding has its place."""
import math

import pytest
import torch

from tests import own_streams
from tests import pairs_reference as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def m(gpu):
    from torch_projectors import matching
    return matching


def gen(seed):
    return torch.Generator().manual_seed(seed)


def rows(n, K, dtype=F32, seed=0, fall=2.0):
    return (torch.randn(n, K, generator=gen(seed)) * torch.exp(-fall * torch.rand(1, K, generator=gen(seed + 1)))).to(dtype)


def same(q, x):
    codes, scale = R.quantize_rows(x)
    K = x.shape[1]
    assert q.codes.dtype == torch.int8 and q.codes.shape == (x.shape[0], -(-K // 128) * 128)
    assert q.scales.dtype == F32 and q.scales.shape == (x.shape[0],)
    got = q.codes.cpu().long()
    assert torch.equal(got[:, :K], codes) and (got[:, K:] == 0).all()
    assert torch.equal(q.scales.cpu().view(torch.int32), scale.view(torch.int32)) or \
        torch.equal(q.scales.cpu().isnan(), scale.isnan()) and torch.equal(q.scales.cpu().nan_to_num(0), scale.nan_to_num(0))


# one, two, four, eight and sixteen wavefronts a row, and rows that are read twice
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("n,K", [(1, 1), (3, 7), (9, 128), (5, 129), (4, 2048), (3, 2049), (6, 4097), (5, 8200), (2, 16640), (3, 33001), (2, 131072)])
def test_quantize(m, n, K, dtype):
    x = rows(n, K, dtype, seed=K)
    same(m.quantize_rows(x.to(DEV)), x)


def test_quantize_many_rows(m):
    x = rows(70001, 33, seed=1)
    same(m.quantize_rows(x.to(DEV)), x)


@pytest.mark.parametrize("K", [128, 300, 5000, 40000])
def test_quantize_ends(m, K):
    x = torch.zeros(11, K)
    x[1] = torch.arange(K) % 255 / 2.0 - 63.5  # halves between codes, where the largest is 127
    x[1, 0] = 127.0
    x[2] = 1e-42 * (torch.arange(K) % 7)  # subnormal: the scale stops at 2^-126
    x[3, K // 2] = torch.finfo(F32).max
    x[3, 0] = torch.finfo(F32).min
    x[3, 1] = 1.3e36
    x[4, K - 1] = math.inf
    x[5, K - 1] = math.nan
    x[6, 0] = -math.inf
    x[7] = -5.0
    x[8, :2] = torch.tensor([127 * 2.0 ** -126, 1.5 * 2.0 ** -126])
    x[9] = torch.linspace(-1, 1, K)
    x[10] = (torch.arange(K) % 127 + 0.5) * (1 / 3.0)  # close to borders between codes
    same(m.quantize_rows(x.to(DEV)), x)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_quotients_close_to_borders(m, dtype):
    """Values whose quotients lie at and around halves, where a reciprocal would choose the other code now and then."""
    g = gen(5)
    most = 0.3 + torch.rand(400, 1, generator=g) * 100
    x = (torch.randint(-127, 127, (400, 260), generator=g) + 0.5) * (most / 127)
    x = x * (1 + torch.randint(-3, 4, (400, 260), generator=g) * 2.0 ** -23)
    x[:, :1] = most
    x = x.to(dtype)
    same(m.quantize_rows(x.to(DEV)), x)


def test_quantize_layouts(m):
    base = rows(11, 700, seed=3).to(DEV)
    for v in (base[:, 3:300], base[::2], base.t()[:40], base[:, ::2], base[:0], base.view(11, 7, 100), base[2:3].expand(5, 700)):
        x = v.flatten(1).cpu()
        q = m.quantize_rows(v)
        if v.shape[0]:
            same(q, x)
        else:
            assert q.codes.shape == (0, 768) and q.scales.shape == (0,)
    z = torch.randn(3, 4, 5, dtype=torch.complex64, generator=gen(4))
    same(m.quantize_rows(z.to(DEV)), torch.view_as_real(z).reshape(3, -1))
    same(m.quantize_rows(z.to(DEV).conj()), torch.view_as_real(z.conj().resolve_conj()).reshape(3, -1))
    same(m.quantize_rows(z.to(DEV).conj().imag), -z.imag.reshape(3, -1))


def scores(m, M, N, K, dtype=F32, out=F32, bias=True, seed=0):
    x, r = rows(M, K, dtype, seed), rows(N, K, dtype, seed + 10)
    b = torch.randn(N, generator=gen(seed + 20)) if bias else None
    a, sa = R.quantize_rows(x)
    c, sc = R.quantize_rows(r)
    want = R.row_scores(a.to(DEV), sa.to(DEV), c.to(DEV), sc.to(DEV), None if b is None else b.to(DEV)).to(out)
    refs = m.quantize_rows(r.to(DEV))
    kw = dict(bias=None if b is None else b.to(DEV), out_dtype=out)
    for left in (x.to(DEV), m.quantize_rows(x.to(DEV))):
        got = m.row_scores(left, refs, **kw)
        assert got.dtype == out and torch.equal(got, want)
    assert torch.equal(m.row_scores(x.to(DEV), r.to(DEV), **kw), want)


# one image rounded on the way or not, few of them in ranges, tiles of each size, leftovers split
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 40, 300), (1, 300, 33000), (2, 17, 129), (16, 100, 16640), (17, 33, 5000), (30, 5000, 700),
                                   (33, 64, 128), (65, 130, 257), (333, 1999, 1000), (700, 900, 3000), (1500, 700, 260), (2500, 2500, 200)])
@pytest.mark.parametrize("out,bias", [(F32, True), (BF16, True), (F32, False)])
def test_scores(m, M, N, K, out, bias):
    scores(m, M, N, K, out=out, bias=bias, seed=M)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("M", [1, 5, 100])
def test_scores_of_half_rows(m, M, dtype):
    scores(m, M, 120, 515, dtype=dtype, out=BF16)


@pytest.mark.parametrize("M,N,K", [(4096, 4096, 600), (4097, 2100, 1300)])
def test_large_tiles(m, M, N, K):
    scores(m, M, N, K)


def test_largest_sums(m):
    """The largest codes over the longest rows: just below 2^31."""
    K = 131072
    for M in (1, 3, 40):
        x = torch.ones(M, K, device=DEV)
        x[0] = -1
        r = torch.ones(50, K, device=DEV)
        got = m.row_scores(m.quantize_rows(x), m.quantize_rows(r))
        s = torch.tensor(1.0) / 127
        want = float(torch.tensor(127.0 * 127 * K) * s * s)
        assert (got[0] == -want).all() and (got[1:] == want).all()


@pytest.mark.parametrize("M", [1, 4, 40])
def test_rows_that_are_not_finite(m, M):
    """Their scores are NaN, the others' are as without them."""
    x, r = rows(M, 300).to(DEV), rows(60, 300, seed=2).to(DEV)
    clean = m.row_scores(x, r)
    r[7, 299] = math.inf
    got = m.row_scores(x, r)
    keep = torch.arange(60, device=DEV) != 7
    assert got[:, 7].isnan().all() and torch.equal(got[:, keep], clean[:, keep])
    x[0, 3] = math.nan
    got = m.row_scores(x, r)
    assert got[0].isnan().all() and torch.equal(got[1:][:, keep], clean[1:][:, keep])


def test_codes_from_any_address(m):
    x, r = rows(20, 256).to(DEV), rows(30, 256, seed=3).to(DEV)
    a, b = m.quantize_rows(x), m.quantize_rows(r)
    want = m.row_scores(a, b)

    def moved(q):
        room = torch.empty(q.codes.numel() + 1, dtype=torch.int8, device=DEV)[1:].view(q.codes.shape)
        scales = torch.empty(2 * q.scales.numel(), device=DEV)[::2]
        return m.RowScaled(room.copy_(q.codes), scales.copy_(q.scales))

    assert torch.equal(m.row_scores(moved(a), moved(b)), want)
    wide = torch.zeros(20, 512, dtype=torch.int8, device=DEV)
    wide[:, 128:384] = a.codes
    assert torch.equal(m.row_scores(m.RowScaled(wide[:, 128:384], a.scales), b), want)


def test_offsets_past_32_bits(m):
    K, N = 131072, 33000
    codes = torch.zeros(N, K, dtype=torch.int8, device=DEV)
    codes[-1], codes[0] = 3, 1
    refs = m.RowScaled(codes, torch.ones(N, device=DEV))
    for M in (1, 2, 40):
        got = m.row_scores(m.RowScaled(torch.ones(M, K, dtype=torch.int8, device=DEV), torch.ones(M, device=DEV)), refs)
        assert (got[:, 0] == K).all() and (got[:, -1] == 3 * K).all() and (got[:, 1:-1] == 0).all()


def test_nothing_to_do(m):
    x, r = rows(3, 20).to(DEV), rows(5, 20).to(DEV)
    assert m.row_scores(x[:0], r).shape == (0, 5) and m.row_scores(x, r[:0]).shape == (3, 0)


@pytest.mark.parametrize("M", [1, 6, 300])
def test_another_stream_and_a_graph(m, M):
    states = [(rows(M, 700, seed=s).to(DEV), rows(500, 700, seed=s + 50).to(DEV), torch.randn(500, generator=gen(s)).to(DEV)) for s in range(3)]

    def step(s):
        refs = m.quantize_rows(s[1])
        return [refs.codes, refs.scales, m.row_scores(s[0], refs, bias=s[2])]

    wanted = [[t.clone() for t in step(s)] for s in states]
    torch.cuda.synchronize()
    side = own_streams.stream()
    with torch.cuda.stream(side):
        got = step(states[0])
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, wanted[0]))
    static = [t.clone() for t in states[0]]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(static)
    for n in (1, 2, 0, 1):
        for t, v in zip(static, states[n]):
            t.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, wanted[n])), n
        assert all(torch.equal(a, b) for a, b in zip(step(states[n]), wanted[n])), n


def test_search_and_posterior(m):
    """Images of known references are found among others, and the posterior of the scores is the pairs' own where the rounding
    leaves it: 1/254 of a row's largest value for each of its values."""
    g = gen(9)
    r = torch.randn(900, 400, generator=g).to(DEV) * 0.4
    of = torch.randint(0, 900, (50,), generator=g).to(DEV)
    x = r[of] + torch.randn(50, 400, generator=g).to(DEV)
    bias = -0.5 * r.square().sum(1)
    s = m.row_scores(x, r, bias=bias)
    post = m.log_probs(s, of, top=1)
    exact = m.pair_log_probs(x, r, of, bias=bias)
    assert (post.top_index[:, 0] == of).float().mean() > 0.9
    step = (x.abs().amax(1, keepdim=True) * r.norm(dim=1) + x.norm(dim=1, keepdim=True) * r.abs().amax(1)) / 254
    # rounding errors of random sign: at most a few standard deviations, step / sqrt(3) each
    assert ((s - (x @ r.t() + bias)).abs() <= 5 * step).all()
    assert ((post.log_sum - exact.log_sum).abs() <= 5 * step.amax(1)).all()


def test_refusals(m):
    q = m.quantize_rows(torch.zeros(3, 8, device=DEV))
    for call, msg in [
            (lambda: m.quantize_rows(torch.zeros(2, 3, dtype=torch.float64, device=DEV)), "float32, float16 or bfloat16"),
            (lambda: m.quantize_rows(torch.zeros(2, 0, device=DEV)), "at least one value"),
            (lambda: m.quantize_rows(torch.zeros(1, 131073, device=DEV)), "2\\^17"),
            (lambda: m.row_scores(torch.zeros(2, 200, device=DEV), q), "256 codes a row, references 128"),
            (lambda: m.row_scores(m.RowScaled(q.codes.float(), q.scales), q), "int8"),
            (lambda: m.row_scores(m.RowScaled(q.codes[:, :100], q.scales), q), "multiple of 128"),
            (lambda: m.row_scores(m.RowScaled(q.codes, q.scales[:2]), q), "scales"),
            (lambda: m.row_scores(q, q, bias=torch.zeros(2, device=DEV)), "bias"),
            (lambda: m.row_scores(q, q, out_dtype=F16), "out_dtype"),
            (lambda: m.row_scores(q, m.RowScaled(q.codes, q.scales.cpu())), "same GPU")]:
        with pytest.raises(RuntimeError, match=msg):
            call()
