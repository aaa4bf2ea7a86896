"""Pair log probabilities on the GPU (matching.pair_log_probs) against their definition in 64 bits and its bounds
(tests/pairs_reference.py), at the sizes where kernels, tiles, ranges and pieces change."""
import math

import pytest
import torch

from tests import own_streams
from tests import pairs_reference as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
INF, NAN = math.inf, math.nan


@pytest.fixture(scope="module")
def m(gpu):
    from torch_projectors import matching
    return matching


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def near(got, want, tol, what):
    assert got.shape == want.shape, (what, got.shape, want.shape)
    got = got.detach().double()
    bad = got.isnan() != want.isnan()
    assert not bad.any(), (what, "NaN", bad.nonzero()[:4].tolist())
    inf = want.isinf()
    assert torch.equal(got[inf], want[inf]), (what, "infinities")
    fine = torch.isfinite(want)
    off = ((got - want).abs() - tol)[fine]
    assert off.numel() == 0 or float(off.max()) <= 0, (what, float(off.max()), float((got - want)[fine].abs().max()))


def problem(M, N, K, dtype, seed=0, bias=True, mask=True, given=True, temperature=1.3, power=None):
    """Images that are a reference each and noise: some probabilities next to one, some spread out."""
    g = gen(seed)
    power = power or 2 * math.log(N + 1) + 3
    r = torch.randn(N, K, generator=g, device=DEV) * (power / K) ** 0.5
    of = torch.randint(0, N, (M,), generator=g, device=DEV)
    x = r[of] * (1 + torch.rand(M, 1, generator=g, device=DEV)) + torch.randn(M, K, generator=g, device=DEV)
    p = dict(images=x.to(dtype), references=r.to(dtype), temperature=temperature)
    if bias:
        p["bias"] = -0.5 * r.square().sum(1)
    if mask:
        p["mask"] = torch.rand(N, generator=g, device=DEV) < 0.75
    if given:
        p["given"] = torch.where(torch.rand(M, generator=g, device=DEV) < 0.8, of, torch.randint(-1, N, (M,), generator=g, device=DEV))
    p["d_given"] = -torch.rand(M, generator=g, device=DEV) if given else None
    p["d_log_sum"] = 0.5 * torch.randn(M, generator=g, device=DEV)
    return p


def run(m, p, wants=("images", "references", "bias"), views=None):
    """Results and gradients as a dict; `views` makes what is passed of each leaf."""
    leaf = {k: p[k].clone().requires_grad_() for k in wants if p.get(k) is not None}
    args = {k: (views or {}).get(k, lambda t: t)(leaf.get(k, p.get(k))) for k in ("images", "references", "given", "bias", "mask")}
    out = m.pair_log_probs(args["images"], args["references"], args["given"], bias=args["bias"],
                           temperature=p["temperature"], mask=args["mask"])
    got = dict(log_sum=out.log_sum)
    outs, ups = [out.log_sum], [p["d_log_sum"]]
    if out.given is not None:
        got["given"] = out.given
        outs.append(out.given)
        ups.append(p["d_given"])
    if leaf:
        for k, d in zip(leaf, torch.autograd.grad(outs, list(leaf.values()), ups)):
            got["d_" + k] = d
    return {k: v.detach() for k, v in got.items()}


def want(p):
    return R.pair_log_probs(p["images"], p["references"], p.get("given"), p.get("bias"), p["temperature"], p.get("mask"),
                            p["d_given"], p["d_log_sum"])


def check(m, p, **kw):
    got, w = run(m, p, **kw), want(p)
    assert len(got) >= 1
    for k, v in got.items():
        if k.startswith("d_"):
            assert v.dtype == (F32 if k == "d_bias" else p["images"].dtype)
        near(v, w[k], w["tol_" + k], k)
    return got


SMALL = [(1, 1, 1), (1, 2, 3), (1, 17, 64), (2, 33, 130), (3, 300, 129), (5, 16, 1025), (8, 300, 70), (9, 1, 1), (9, 65, 130),
         (16, 3, 8), (33, 129, 257), (64, 64, 64), (65, 63, 72), (130, 70, 333), (300, 257, 96)]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("M,N,K", SMALL)
def test_small(m, M, N, K, dtype):
    check(m, problem(M, N, K, dtype, seed=M + N))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("M", [1, 4, 9, 40])
@pytest.mark.parametrize("bias,mask,given", [(False, False, False), (True, False, False), (False, True, True), (False, False, True)])
def test_without_options(m, M, bias, mask, given, dtype):
    check(m, problem(M, 150, 80, dtype, seed=7, bias=bias, mask=mask, given=given))


# every tile, with and without split leftovers, whole rows and odd ones (16-bit rows of an odd size are staged)
TILES = [(100, 5000, 64), (20, 200, 4096), (333, 1999, 520), (500, 1030, 203), (700, 900, 1100), (1500, 700, 300), (2500, 2500, 72)]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("M,N,K", TILES)
def test_tiles(m, M, N, K, dtype):
    check(m, problem(M, N, K, dtype, seed=M))


@pytest.mark.parametrize("dtype,M,N,K", [(BF16, 4096, 4096, 520), (F16, 4000, 4200, 264), (F32, 4096, 2100, 264), (F32, 2049, 4100, 70),
                                         (BF16, 4097, 4000, 131)])
def test_large_tiles(m, M, N, K, dtype):
    check(m, problem(M, N, K, dtype, seed=M))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_references_in_pieces(m, dtype):
    """More references than a piece of the scores' gradient holds (128 MB: 16384 of 16-bit rows of 4096 images)."""
    p = problem(4096, 17000 if dtype == BF16 else 8300, 16, dtype, seed=3)
    check(m, p)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("M,N", [(1, 8192), (1, 8193), (3, 12288), (8, 20001)])
def test_few_images_of_many_references(m, M, N, dtype):
    """More than 8192 references of few images are joined in steps of 4096: given references in the last one, and steps
    that allow nothing."""
    p = problem(M, N, 24, dtype, seed=N)
    p["given"][0] = N - 1
    check(m, p)
    p["mask"][:4096] = False
    p["mask"][8000:] = False
    check(m, p)
    p["mask"][:] = False
    check(m, p)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("M", [3, 20])
def test_long_rows(m, M, dtype):
    """Sums of many values in one go lose what their differences need: within a few roundings of the score's own size."""
    p = problem(M, 40, 16640, dtype, seed=5, mask=False)
    got, w = run(m, p, wants=()), want(p)
    # (a sum of K terms of random sign loses sqrt(K) roundings or so, not K)
    near(got["log_sum"], w["log_sum"], 2e-5 * (1 + w["log_sum"].abs()), "log_sum")
    check(m, p)


@pytest.mark.parametrize("M", [2, 30])
def test_probability_next_to_one(m, M):
    """The logarithm of a probability next to one keeps what the others hold."""
    p = problem(M, 50, 64, F32, seed=6, mask=False, temperature=1.0, power=40.0)
    x = p["references"][:M] * 1.2
    p["images"], p["given"] = x, torch.arange(M, device=DEV)
    got, w = run(m, p), want(p)
    assert (w["given"] > -1e-3).all() and (w["given"] < 0).all()
    assert ((got["given"].double() - w["given"]).abs() <= 1e-4 * w["given"].abs()).all()
    # so does the gradient at the given reference: p - 1 is what the others hold
    p["d_log_sum"], p["d_given"] = torch.zeros(M, device=DEV), torch.ones(M, device=DEV)
    got, w = run(m, p), want(p)
    assert ((got["d_bias"].double() - w["d_bias"]).abs() <= 1e-4 * w["d_bias"].abs() + 1e-12).all()


# ----------------------------------------------------------------------------- masks and ends
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("M", [1, 8, 12, 200])
def test_nothing_allowed(m, M, dtype):
    p = problem(M, 130, 72, dtype, seed=1)
    p["mask"] = torch.zeros(130, dtype=torch.bool, device=DEV)
    p["references"][::3] = NAN
    got = run(m, p)
    assert (got["log_sum"] == -INF).all()
    none = p["given"] == -1
    assert (got["given"][~none] == -INF).all() and (got["given"][none] == 0).all()
    for k in ("d_images", "d_references", "d_bias"):
        assert (got[k] == 0).all(), k


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("held", [NAN, INF, -INF, "lowest"])
@pytest.mark.parametrize("M,N,K", [(3, 140, 72), (20, 140, 72), (300, 700, 136), (300, 700, 131)])
def test_what_masked_references_hold(m, M, N, K, held, dtype):
    p = problem(M, N, K, dtype, seed=2)
    clean = run(m, p)
    p["references"][~p["mask"]] = torch.finfo(dtype).min if held == "lowest" else held
    p["bias"][~p["mask"]] = NAN
    got = run(m, p)
    for k in got:
        assert torch.equal(got[k], clean[k]), k
        assert not got[k].isnan().any(), k  # (a given reference that is ruled out has -inf)


@pytest.mark.parametrize("M", [3, 20])
def test_bias_rules_out(m, M):
    p = problem(M, 90, 64, F32, seed=3, mask=False)
    p["bias"][::2] = -INF
    got = check(m, p)
    assert (got["d_bias"][::2] == 0).all() and (got["d_references"][::2] == 0).all()
    p["bias"][:] = torch.finfo(F32).min  # the type's lowest value is no mask: scores that lie there, all alike
    got = run(m, p)
    assert torch.isfinite(got["given"][p["given"] >= 0]).all() and torch.isfinite(got["log_sum"]).all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("M", [4, 50])
def test_images_that_are_not_finite(m, M, dtype):
    """Their own results are NaN, the others' are as without them."""
    p = problem(M, 77, 72, dtype, seed=4)
    p["given"] = p["given"].clamp_min(0)
    clean = run(m, p)
    p["images"][1, 5] = NAN
    got = run(m, p)
    assert got["log_sum"][1].isnan() and got["given"][1].isnan()
    others = torch.arange(M, device=DEV) != 1
    for k in ("log_sum", "given", "d_images"):
        assert torch.equal(got[k][others], clean[k][others]), k
    assert got["d_images"][1].isnan().all()
    for k in ("d_references", "d_bias"):
        assert got[k][p["mask"]].isnan().all() and (got[k][~p["mask"]] == 0).all(), k


@pytest.mark.parametrize("M", [4, 50])
def test_given_out_of_range(m, M):
    p = problem(M, 60, 64, F32, seed=5)
    p["given"][0], p["given"][1], p["given"][2] = 60, -2, 1 << 40
    p["d_given"][2] = 0.0  # its result is not used
    check(m, p)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_no_references_and_no_images(m, dtype):
    p = problem(5, 7, 16, dtype, mask=False)
    none = {**p, "references": p["references"][:0], "bias": p["bias"][:0]}
    out = run(m, {**none, "given": torch.tensor([-1, 0, -1, 3, -1], device=DEV), "d_given": torch.zeros(5, device=DEV)})
    assert (out["log_sum"] == -INF).all()
    assert out["given"].isnan().tolist() == [False, True, False, True, False] and out["given"][0] == 0
    assert (out["d_images"] == 0).all() and out["d_references"].shape == (0, 16) and out["d_bias"].shape == (0,)
    out = run(m, {**p, "images": p["images"][:0], "given": p["given"][:0], "d_given": p["d_given"][:0], "d_log_sum": p["d_log_sum"][:0]})
    assert out["log_sum"].shape == (0,) and (out["d_references"] == 0).all() and (out["d_bias"] == 0).all()
    assert out["d_images"].shape == (0, 16)


# ----------------------------------------------------------------------------- layouts
def _wide(t):  # rows of a wider matrix, from an odd address on
    w = torch.empty(t.shape[0], t.shape[1] + 13, dtype=t.dtype, device=t.device)
    w[:, 5:5 + t.shape[1]] = t.detach()
    return w[:, 5:5 + t.shape[1]]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("M,N,K", [(3, 140, 72), (20, 140, 72), (140, 300, 64)])
def test_layouts(m, M, N, K, dtype):
    p = problem(M, N, K, dtype, seed=8)
    plain = check(m, p)
    w = want(p)
    for views in (dict(images=_wide, references=_wide), dict(images=lambda t: t.t().contiguous().t()),
                  dict(references=lambda t: t[:, None].reshape(N, K // 8, 8)),
                  dict(bias=lambda t: torch.stack([t, t], 1)[:, 1], mask=lambda t: torch.stack([t, t], 1)[:, 0],
                       given=lambda t: torch.stack([t, t], 1)[:, 1])):
        out = m.pair_log_probs(*(views.get(k, lambda t: t)(p[k]) for k in ("images", "references", "given")),
                               bias=views.get("bias", lambda t: t)(p["bias"]), temperature=p["temperature"],
                               mask=views.get("mask", lambda t: t)(p["mask"]))
        near(out.log_sum, w["log_sum"], w["tol_log_sum"], "log_sum")
        near(out.given, w["given"], w["tol_given"], "given")
    # gradients through views: columns of a wider leaf, transposed leaves
    leaf_x = torch.zeros(M, K + 9, dtype=dtype, device=DEV)
    leaf_x[:, 3:3 + K] = p["images"]
    leaf_x.requires_grad_()
    leaf_r = p["references"].t().contiguous().requires_grad_()
    out = m.pair_log_probs(leaf_x[:, 3:3 + K], leaf_r.t(), p["given"], bias=p["bias"], temperature=p["temperature"], mask=p["mask"])
    dx, dr = torch.autograd.grad((out.log_sum, out.given), (leaf_x, leaf_r), (p["d_log_sum"], p["d_given"]))
    near(dx[:, 3:3 + K], w["d_images"], w["tol_d_images"], "d_images")
    assert (dx[:, :3] == 0).all() and (dx[:, 3 + K:] == 0).all()
    near(dr.t(), w["d_references"], w["tol_d_references"], "d_references")
    assert torch.equal(plain["log_sum"], run(m, p, wants=())["log_sum"])


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("K", [64, 70])
def test_one_row_for_all(m, K, dtype):
    """Expanded rows lie zero elements apart; their gradients are those of the one row."""
    p = problem(40, 50, K, dtype, seed=9, mask=False, given=False)
    for which in ("images", "references"):
        row = p[which][:1].clone().requires_grad_()
        n = p[which].shape[0]
        args = {k: p[k] for k in ("images", "references")}
        args[which] = row.expand(n, K)
        out = m.pair_log_probs(args["images"], args["references"], bias=p["bias"], temperature=p["temperature"])
        w = want({**p, which: row.detach().expand(n, K).contiguous()})
        near(out.log_sum, w["log_sum"], w["tol_log_sum"], which)
        (d,) = torch.autograd.grad(out.log_sum, row, p["d_log_sum"])
        # the expansion's own backward sums n rounded rows in the type
        tol = w["tol_d_" + which].sum(0) + (n + 2) * R.roundoff(dtype) * w["d_" + which].abs().sum(0)
        near(d[0], w["d_" + which].sum(0), tol, which)


def test_rows_further_apart_than_the_kernels_take(m):
    wide = torch.zeros(3, (1 << 21) + 8, device=DEV)
    p = problem(3, 30, 48, F32, seed=10)
    wide[:, 4:52] = p["images"]
    out = m.pair_log_probs(wide[:, 4:52], p["references"], p["given"], bias=p["bias"], temperature=p["temperature"], mask=p["mask"])
    w = want(p)
    near(out.log_sum, w["log_sum"], w["tol_log_sum"], "log_sum")


def test_offsets_past_32_bits(m):
    """References whose last rows lie past 2^32 bytes, few images and many."""
    N, K = 70000, 16400
    r = torch.zeros(N, K, dtype=BF16, device=DEV)
    at = torch.tensor([0, N // 2, N - 1], device=DEV)
    r[at] = torch.randn(3, K, generator=gen(11), device=DEV).to(BF16)
    for M in (3, 12):
        x = r[at[torch.arange(M, device=DEV) % 3]]
        out = m.pair_log_probs(x, r, at[torch.arange(M, device=DEV) % 3], temperature=500.0)
        z = x.double() @ r[at].double().t() / 500.0
        log_sum = torch.logsumexp(torch.cat([z, torch.full((M, 1), math.log(N - 3), device=DEV, dtype=torch.float64)], 1), 1)
        tol = (K + 16) * R.U * (x.double().square().sum(1) / 500.0) + 200 * R.U * (1 + log_sum.abs())
        near(out.log_sum, log_sum, tol, "log_sum")
        near(out.given, z.gather(1, (torch.arange(M, device=DEV) % 3)[:, None])[:, 0] - log_sum, 2 * tol, "given")


def test_complex_rows(m):
    g = gen(12)
    x = torch.randn(6, 4, 5, dtype=torch.complex64, generator=g, device=DEV).requires_grad_()
    r = torch.randn(30, 4, 5, dtype=torch.complex64, generator=g, device=DEV).requires_grad_()
    out = m.pair_log_probs(x, r)
    z = (x.detach().flatten(1)[:, None] * r.detach().flatten(1).conj()[None]).sum(2).real.double()
    near(out.log_sum, torch.logsumexp(z, 1), torch.full((6,), 1e-4, device=DEV, dtype=torch.float64), "log_sum")
    dx, dr = torch.autograd.grad(out.log_sum.sum(), (x, r))
    p = torch.softmax(z, 1)
    near(torch.view_as_real(dx).flatten(), torch.view_as_real((p.to(torch.complex128) @ r.detach().flatten(1).to(torch.complex128))).flatten(),
         1e-4, "d_images")
    near(torch.view_as_real(dr).flatten(), torch.view_as_real((p.t().to(torch.complex128) @ x.detach().flatten(1).to(torch.complex128))).flatten(),
         1e-4, "d_references")


# ----------------------------------------------------------------------------- gradients
@pytest.mark.parametrize("M", [5, 21])
@pytest.mark.parametrize("wants", [("images",), ("references",), ("bias",), ("images", "bias"), ("references", "images")])
@pytest.mark.parametrize("given", [True, False])
def test_some_gradients(m, M, wants, given):
    """What is not wanted is not formed, and does not change the rest."""
    p = problem(M, 60, 40, F32, seed=13, given=given)
    every = run(m, p)
    some = run(m, p, wants=wants)
    for k in wants:
        assert torch.equal(some["d_" + k], every["d_" + k]), k


@pytest.mark.parametrize("M", [3, 12])
def test_one_upstream_gradient(m, M):
    p = problem(M, 60, 40, F32, seed=14)
    x = p["images"].clone().requires_grad_()
    out = m.pair_log_probs(x, p["references"], p["given"], bias=p["bias"], temperature=p["temperature"], mask=p["mask"])
    (a,) = torch.autograd.grad(out.log_sum, x, p["d_log_sum"], retain_graph=True)
    (b,) = torch.autograd.grad(out.given, x, p["d_given"])
    for d, ups in ((a, dict(d_given=None)), (b, dict(d_log_sum=None))):
        w = want({**p, **ups})
        near(d, w["d_images"], w["tol_d_images"], "d_images")


@pytest.mark.parametrize("M", [3, 12])
@pytest.mark.parametrize("which", ["images", "references", "bias"])
def test_gradient_against_differences(m, M, which):
    p = problem(M, 25, 24, F32, seed=15, mask=True)
    x = p[which].clone().requires_grad_()

    def value(t):
        q = {**p, which: t}
        w = R.pair_log_probs(q["images"], q["references"], q["given"], q["bias"], q["temperature"], q["mask"])
        # (of a given reference that is ruled out the gradient is that of the log sum alone, as by log_probs)
        given = torch.where(w["given"] == -INF, -w["log_sum"], w["given"])
        return (w["log_sum"] * p["d_log_sum"].double()).sum() + (given * p["d_given"].double()).sum()

    out = m.pair_log_probs(*(x if k == which else p[k] for k in ("images", "references", "given")),
                           bias=x if which == "bias" else p["bias"], temperature=p["temperature"], mask=p["mask"])
    (d,) = torch.autograd.grad((out.log_sum, out.given), x, (p["d_log_sum"], p["d_given"]))
    for seed in range(4):
        v = torch.randn(x.shape, generator=gen(seed), device=DEV, dtype=torch.float64)
        h = 1e-4
        slope = (value(p[which].double() + h * v) - value(p[which].double() - h * v)) / (2 * h)
        off, bound = abs(float((d.double() * v).sum() - slope)), 2e-4 * float((d.double().abs() * v.abs()).sum() + 1e-3)
        assert off <= bound, (off, bound)


def test_differentiable_once(m):
    x = torch.randn(3, 8, device=DEV, requires_grad=True)
    r = torch.randn(5, 8, device=DEV)
    (d,) = torch.autograd.grad(m.pair_log_probs(x, r).log_sum.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        d.sum().backward()
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            m.pair_log_probs(torch.autograd.forward_ad.make_dual(x.detach(), torch.ones_like(x)), r)
    assert not m.pair_log_probs(x.detach(), r).log_sum.requires_grad


# ----------------------------------------------------------------------------- repeats, streams and graphs
CASES = [(4, 300, 264, F32), (12, 90, 2100, F16), (200, 700, 264, BF16), (300, 500, 131, F32)]


@pytest.mark.parametrize("M,N,K,dtype", CASES)
def test_the_same_again(m, M, N, K, dtype):
    p = problem(M, N, K, dtype, seed=16)
    first = run(m, p)
    for _ in range(3):
        for k, v in run(m, p).items():
            assert torch.equal(v, first[k]), k


@pytest.mark.parametrize("M,N,K,dtype", CASES)
def test_another_stream_and_a_graph(m, M, N, K, dtype):
    """Forward and gradient captured, replayed with other inputs and eager calls in between."""
    keys = ("images", "references", "bias", "mask", "given", "d_given", "d_log_sum")
    states = [problem(M, N, K, dtype, seed=s) for s in range(3)]

    def step(p):  # (leaves of its own: no graph of an earlier step lives when the backward pass is captured)
        x, r, b = (p[k].detach().requires_grad_() for k in ("images", "references", "bias"))
        out = m.pair_log_probs(x, r, p["given"], bias=b, temperature=p["temperature"], mask=p["mask"])
        grads = torch.autograd.grad((out.given, out.log_sum), (x, r, b), (p["d_given"], p["d_log_sum"]))
        return (out.given.detach(), out.log_sum.detach(), *grads)

    wanted = [[t.clone() for t in step(p)] for p in states]
    torch.cuda.synchronize()
    side = own_streams.stream()
    with torch.cuda.stream(side):
        got = step(states[0])
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, wanted[0]))
    static = {**states[0], **{k: states[0][k].clone() for k in keys}}
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(static)
    for n in (1, 2, 0, 1):
        for k in keys:
            static[k].copy_(states[n][k])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, wanted[n])), n
        assert all(torch.equal(a, b) for a, b in zip(step(states[n]), wanted[n])), n


def test_two_streams_at_once(m):
    ps = [problem(300, 2000, 520, BF16, seed=s) for s in range(2)]
    wanted = [run(m, p) for p in ps]
    torch.cuda.synchronize()
    streams = [own_streams.stream(i) for i in range(len(ps))]
    got = [None, None]
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = run(m, ps[i])
        torch.cuda.synchronize()
        for a, b in zip(got, wanted):
            assert all(torch.equal(a[k], b[k]) for k in b)


@pytest.mark.parametrize("M", [5, 60])
def test_two_graphs_in_turn(m, M):
    """Forward and gradient captured twice, with other inputs, and replayed alternately: what each keeps between its kernels is its own."""
    ps = [problem(M, 700, 264, F32, seed=s) for s in (21, 22)]

    def step(p):
        x, r, b = (p[k].detach().requires_grad_() for k in ("images", "references", "bias"))
        out = m.pair_log_probs(x, r, p["given"], bias=b, temperature=p["temperature"], mask=p["mask"])
        return (out.log_sum.detach(), *torch.autograd.grad((out.given, out.log_sum), (x, r, b), (p["d_given"], p["d_log_sum"])))

    wanted = [[t.clone() for t in step(p)] for p in ps]
    torch.cuda.synchronize()
    graphs, outs = [torch.cuda.CUDAGraph() for _ in ps], []
    for graph, p in zip(graphs, ps):
        with torch.cuda.graph(graph):
            outs.append(step(p))
    for n in (0, 1, 1, 0, 1):
        for t in outs[n]:
            t.zero_()
        graphs[n].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs[n], wanted[n])), n


@pytest.mark.parametrize("M", [6, 90])
def test_images_that_are_the_references(m, M):
    """One tensor on both sides has the gradients of both."""
    p = problem(M, M, 70, F32, seed=23, bias=False, mask=False, given=False)
    p["images"] = p["references"]
    w = want(p)
    both = p["references"].clone().requires_grad_()
    (got,) = torch.autograd.grad(m.pair_log_probs(both, both, temperature=p["temperature"]).log_sum, both, p["d_log_sum"])
    # (their sum is rounded once more)
    total = w["d_images"] + w["d_references"]
    near(got, total, w["tol_d_images"] + w["tol_d_references"] + R.U * total.abs(), "both")


@pytest.mark.parametrize("M", [2, 20])
def test_conjugate_rows(m, M):
    """Conjugates that are only marked as such are what they stand for."""
    g = gen(24)
    x = torch.randn(M, 40, dtype=torch.complex64, generator=g, device=DEV)
    r = torch.randn(70, 40, dtype=torch.complex64, generator=g, device=DEV) * 0.2
    assert x.conj().is_conj()
    a = m.pair_log_probs(x.conj(), r.conj())
    b = m.pair_log_probs(x.conj().resolve_conj(), r.conj().resolve_conj())
    assert torch.equal(a.log_sum, b.log_sum)
    assert torch.equal(m.row_scores(x.conj(), m.quantize_rows(r.conj())), m.row_scores(x.conj().resolve_conj(), m.quantize_rows(r.conj().resolve_conj())))


# ----------------------------------------------------------------------------- with the other operators
@pytest.mark.parametrize("M", [6, 40])
def test_same_as_log_probs_of_the_scores(m, M):
    """The likelihood of images and its gradient, with the scores in memory and without."""
    p = problem(M, 500, 96, F32, seed=17, temperature=0.8)
    r = p["references"].clone().requires_grad_()
    scores = p["images"] @ r.t() + p["bias"]
    a = m.log_probs(scores, p["given"], temperature=0.8, mask=p["mask"])
    (da,) = torch.autograd.grad((a.log_sum, a.given), r, (p["d_log_sum"], p["d_given"]))
    b = m.pair_log_probs(p["images"], r, p["given"], bias=p["bias"], temperature=0.8, mask=p["mask"])
    (db,) = torch.autograd.grad((b.log_sum, b.given), r, (p["d_log_sum"], p["d_given"]))
    w = want(p)
    near(a.log_sum, b.log_sum.detach().double(), 2 * w["tol_log_sum"], "log_sum")
    near(a.given, b.given.detach().double(), 2 * w["tol_given"] + 1e-5, "given")
    near(da, db.double(), 3 * w["tol_d_references"] + 1e-5, "d_references")


def test_refusals(m):
    x, r = torch.zeros(3, 8, device=DEV), torch.zeros(5, 8, device=DEV)
    for call, msg in [
            (lambda: m.pair_log_probs(x, r.half()), "same dtype"),
            (lambda: m.pair_log_probs(x.double(), r.double()), "float32, float16 or bfloat16"),
            (lambda: m.pair_log_probs(x, r, torch.zeros(3, dtype=torch.int32, device=DEV)), "int64"),
            (lambda: m.pair_log_probs(x, r, bias=torch.zeros(5, dtype=F16, device=DEV)), "float32"),
            (lambda: m.pair_log_probs(x, r, mask=torch.zeros(5, dtype=torch.uint8, device=DEV)), "bool"),
            (lambda: m.pair_log_probs(x, r, temperature=0.0), "temperature"),
            (lambda: m.pair_log_probs(x, r, temperature=NAN), "temperature"),
            (lambda: m.pair_log_probs(x[:, :0], r[:, :0]), "at least one value"),
            (lambda: m.pair_log_probs(x, r.cpu()), "same GPU|Expected all tensors"),
            (lambda: torch.ops.torch_projectors.pair_log_probs_back(x, r, None, None, None, 1.0, torch.zeros(4, device=DEV), None,
                                                                    torch.zeros(3, device=DEV), True, True, True), "state")]:
        with pytest.raises(RuntimeError, match=msg):
            call()
