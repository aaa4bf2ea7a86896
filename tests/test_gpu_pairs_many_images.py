"""Gradients of pair log probabilities of more images than one piece of the scores' gradient holds (32768): pieces of the images
and of the references, and counts at which a row of all images would pass what the products' offsets reach."""
import pytest
import torch

from tests import pairs_plans as P
from tests import pairs_reference as R
from tests.test_gpu_pairs import BF16, DEV, F16, F32, NAN, check, gen, m, near, problem, run, want  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("M,N,K", [(33000, 4200, 16), (40001, 4199, 9), (70000, 40, 24)])
def test_pieces_of_images(m, M, N, K, dtype):  # noqa: F811
    b = P.back_layout(P.CODES[str(dtype)], dtype != F32 and K % 8 == 0, M, N, K)
    assert b.images < M
    assert b.references < N or N < 1000
    p = problem(M, N, K, dtype, seed=M)
    got = check(m, p)
    # what is ruled out stays out of every piece, whatever it holds
    p["references"][~p["mask"]] = NAN
    p["bias"][~p["mask"]] = NAN
    for k, v in run(m, p).items():
        assert torch.equal(v, got[k]), k


@pytest.mark.parametrize("dtype,M", [(BF16, 20000000), (F16, 9000000), (F32, 5000000)])
def test_millions_of_images(m, dtype, M):  # noqa: F811
    """255 rows of 5 million float32 values pass 2^32 bytes, of 9 million 16-bit ones 2^31.

    The terms of a reference's gradient are all positive here, so that what 32 bits lose is relative to the result: scores of
    at most 20 lose 2 (6 K + 16) 2^-24 20 = 1.6e-4 of a probability, sums of 2^16 products and of 611 pieces 3e-4 at most, the
    scores' gradient and the result a rounding each."""
    N, K = 300, 8
    print(dtype, M, flush=True)
    g = gen(31)
    r = (0.3 * torch.randn(N, K, generator=g, device=DEV)).to(dtype).requires_grad_()
    bias = torch.randn(N, generator=g, device=DEV).requires_grad_()
    x = (0.5 + torch.rand(M, K, generator=g, device=DEV)).to(dtype).requires_grad_()
    up = 1e-3 * (0.5 + torch.rand(M, generator=g, device=DEV))
    out = m.pair_log_probs(x, r, bias=bias)
    dx, dr, db = torch.autograd.grad(out.log_sum, (x, r, bias), up)
    x, r, bias = x.detach(), r.detach(), bias.detach()
    want_r, want_b = torch.zeros(N, K, dtype=torch.float64, device=DEV), torch.zeros(N, dtype=torch.float64, device=DEV)
    for i in range(0, M, 1 << 20):
        part = x[i: i + (1 << 20)].double()
        G = torch.softmax(part @ r.double().t() + bias.double(), 1) * up[i: i + (1 << 20), None].double()
        want_r += G.t() @ part
        want_b += G.sum(0)
    rounding = R.roundoff(dtype) if dtype != F32 else 0.0
    near(dr, want_r, (5e-4 + 2 * rounding) * want_r, "d_references")
    near(db, want_b, 5e-4 * want_b, "d_bias")
    for rows in (slice(0, 500), slice(M // 2 - 250, M // 2 + 250), slice(M - 500, M)):
        w = R.pair_log_probs(x[rows], r, None, bias, d_log_sum=up[rows])
        near(out.log_sum[rows], w["log_sum"], w["tol_log_sum"], "log_sum")
        near(dx[rows], w["d_images"], w["tol_d_images"], "d_images")


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("M,N,K", [(3, 10000000, 4), (12, 5000000, 8), (12, 3000001, 3)])
def test_millions_of_references(m, M, N, K, dtype):  # noqa: F811
    """Thousands of parts of an image's scores, and pieces of the references.

    The native exponential has no subnormal results: probabilities below 2^-126 of the largest count as 0, which takes at most 2^-126 of the
    upstream gradients times what a gradient's other factors add up to."""
    print(dtype, M, N, flush=True)
    p = problem(M, N, K, dtype, seed=32)
    p["given"][0] = N - 1
    got, w = run(m, p), want(p)
    least = 2.0 ** -126 * float((p["d_given"].abs() + p["d_log_sum"].abs()).max()) / p["temperature"]
    lost = dict(d_images=least * p["references"].double().abs().sum(0), d_references=least * p["images"].double().abs().sum(0), d_bias=least * M)
    for k, v in got.items():
        near(v, w[k], w["tol_" + k] + lost.get(k, 0.0), k)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_some_gradients_of_pieces(m, dtype):  # noqa: F811
    """What is not wanted is not formed, and does not change the rest."""
    p = problem(33000, 4200, 16, dtype, seed=33)
    every = run(m, p)
    for wants in (("images",), ("references",), ("bias",), ("references", "bias")):
        some = run(m, p, wants=wants)
        for k in wants:
            assert torch.equal(some["d_" + k], every["d_" + k]), k


@pytest.mark.parametrize("dtype", [F32, F16])
def test_pieces_in_two_graphs(m, dtype):  # noqa: F811
    """Captured twice with other inputs and replayed in turn, with eager calls in between: what pieces add up begins anew each time."""
    ps = [problem(33000, 4200, 16, dtype, seed=s) for s in (34, 35)]

    def step(p):  # (leaves of its own)
        x, r, b = (p[k].detach().requires_grad_() for k in ("images", "references", "bias"))
        out = m.pair_log_probs(x, r, p["given"], bias=b, temperature=p["temperature"], mask=p["mask"])
        return (out.log_sum.detach(), *torch.autograd.grad((out.given, out.log_sum), (x, r, b), (p["d_given"], p["d_log_sum"])))

    wanted = [[t.clone() for t in step(p)] for p in ps]
    torch.cuda.synchronize()
    graphs, outs = [torch.cuda.CUDAGraph() for _ in ps], []
    for graph, p in zip(graphs, ps):
        with torch.cuda.graph(graph):
            outs.append(step(p))
    for n in (0, 1, 1, 0):
        for t in outs[n]:
            t.fill_(NAN)
        graphs[n].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs[n], wanted[n])), n
        assert all(torch.equal(a, b) for a, b in zip(step(ps[n]), wanted[n])), n
