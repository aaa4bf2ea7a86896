"""Timing cases of two operators of torch_projectors.matching on images and a table of references: log
probabilities of the pairs without their scores in memory, and scores in 8-bit integers with a scale for each row.

A case is a dict of plain values with a `kind`:
  "pairs"  M images of K values against N references (both of `dtype`): score = (<image, reference> + bias) /
           temperature, some references ruled out where `mask`; the log probability of a given reference and the
           log sum of each image; `train` adds the gradients of images, references and biases from upstream
           gradients of both
  "rows8"  M images of K values (`dtype`) rounded to 8-bit integers with a scale for each image, times N references
           kept that way (or, where `both`, rounded within the call too), plus a bias per reference (`out` of the
           scores)

`own` chooses who computes: plain torch operations in 32 bits, or the package's operators.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
PAD = 128  # integer codes are padded with zeros to a multiple of this


def _matching():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "torch-projectors_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from torch_projectors import matching
    return matching


def _coefficients(n):
    """Real values of one rfft image of box n."""
    return 2 * n * (n // 2 + 1)


def _pairs(name, M, N, K, dtype, train=False, mask=False, temperature=1.0):
    return dict(kind="pairs", M=M, N=N, K=K, dtype=dtype, train=train, mask=mask, temperature=temperature, name=name)


def _rows8(name, M, N, K, dtype, out="float32", both=False):
    return dict(kind="rows8", M=M, N=N, K=K, dtype=dtype, out=out, both=both, name=name)


def listed():
    return [
        # one image of a 64 box against every in-plane angle: a call of microseconds
        _pairs("pairs_one_64", 1, 256, _coefficients(64), "float32"),
        # one image of a 128 box against the poses of projection matching: as fast as the references are read
        _pairs("pairs_one_128", 1, 4096, _coefficients(128), "bfloat16"),
        # the marginal likelihood of a whole stack, no gradient
        _pairs("pairs_search_128", 4096, 8192, _coefficients(128), "float32"),
        # a step on a few images against the projections of a coarse grid
        _pairs("pairs_step_few", 4, 1152, _coefficients(64), "float32", train=True),
        # a minibatch of an odd box (rows of no whole number of 16 bytes), ragged counts, some references ruled out
        _pairs("pairs_step_ragged", 500, 4099, _coefficients(45), "float32", train=True, mask=True, temperature=1.5),
        # a ragged minibatch in half precision
        _pairs("pairs_step_half", 333, 1999, _coefficients(90), "float16", train=True, temperature=1.5),
        # refining volumes against a stack in single precision, as the operators' own projections come
        _pairs("pairs_step_stack", 2048, 8192, _coefficients(64), "float32", train=True),
        # a stack against a pose grid of which the scores alone would be 604 MB
        _pairs("pairs_step_grid", 4096, 36864, _coefficients(64), "bfloat16", train=True),
        # one image of a 64 box against every in-plane angle: a call of microseconds
        _rows8("rows8_one_64", 1, 256, _coefficients(64), "float32"),
        # one image of a 128 box against the poses of projection matching: as fast as the references are read
        _rows8("rows8_one_128", 1, 4096, _coefficients(128), "bfloat16"),
        # a batch of a ragged box and ragged counts against references of this step, scores kept in 16 bits
        _rows8("rows8_batch_90", 333, 1999, _coefficients(90), "float16", out="bfloat16", both=True),
        # a search of a particle stack over all references: the matrix units' rate
        _rows8("rows8_search_128", 4096, 8192, _coefficients(128), "float32"),
    ]


def _size(dtype):
    return 4 if dtype == "float32" else 2


def work(c):
    M, N, K, s = c["M"], c["N"], c["K"], _size(c["dtype"])
    if c["kind"] == "pairs":
        bytes_ = (M + N) * K * s + 4 * N + (N if c["mask"] else 0) + 16 * M
        flops = 2 * M * N * K
        if c["train"]:
            # upstream gradients in, the three gradients out; two more products (that a kernel which keeps no
            # scores has to form them again is its own affair)
            bytes_ += 8 * M + (M + N) * K * s + 4 * N
            flops += 4 * M * N * K
        return {"bytes": bytes_, "flops": flops}
    references = N * K * s if c["both"] else N * (-(-K // PAD) * PAD + 4)
    return {"bytes": M * K * s + references + 4 * N + M * N * _size(c["out"]), "flops": 2 * M * N * K}


def _cost(c):
    """Rough time, to keep drawn cases below the largest listed one of their kind."""
    w = work(c)
    rate = 2.5e15 if c["kind"] == "rows8" else 2e14 if c["dtype"] == "float32" else 1.2e15
    return w["bytes"] / 4e12 + w["flops"] / rate


def draw(rng):
    def logint(a, b):
        return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))

    while True:
        # whole images of an even box, or a plain number of values
        K = _coefficients(2 * logint(4, 64)) if rng.random() < 0.6 else logint(16, 16640)
        M = 1 if rng.random() < 0.15 else logint(1, 4096)
        if rng.random() < 0.6:
            c = dict(kind="pairs", M=M, N=logint(2, 36864), K=K, dtype=rng.choice(["float32", "bfloat16", "float16"]),
                     train=rng.random() < 0.6, mask=rng.random() < 0.4, temperature=rng.choice([0.7, 1.0, 1.0, 1.5]))
        else:
            c = dict(kind="rows8", M=M, N=logint(2, 36864), K=K, dtype=rng.choice(["float32", "bfloat16", "float16"]),
                     out=rng.choice(["float32", "float32", "bfloat16"]), both=rng.random() < 0.3)
        if _cost(c) <= max(_cost(d) for d in listed() if d["kind"] == c["kind"]):
            return c


# ----------------------------------------------------------------------------- inputs
def _references(rows, K, power, g):
    """Fourier coefficients of projections: amplitudes fall by two orders of magnitude from the first to the last,
    `power` is the sum of their squares."""
    x = torch.randn(rows, K, generator=g, device=g.device) * torch.exp(torch.linspace(0.0, -4.6, K, device=g.device))
    return x * (power / x.square().sum(1, keepdim=True)).sqrt()


def _to_rows8(x):
    """codes [R, K padded] (int8) and scales [R] of x [R, K]: scale = largest magnitude / 127 and code = x / scale to
    nearest even, both quotients rounded to 32 bits."""
    x = x.float()
    most = x.abs().amax(1, keepdim=True)
    # (a quotient by a number of Python's would be a product with its reciprocal)
    scales = (most / torch.full_like(most, 127.0)).clamp_min(2.0 ** -126)
    codes = torch.nn.functional.pad(torch.round(x / scales), (0, -x.shape[1] % PAD))
    return codes.to(torch.int8), scales[:, 0]


def prepare(c, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    M, N, K, dt = c["M"], c["N"], c["K"], DTYPES[c["dtype"]]
    s = dict(c)
    # images are a reference each and unit noise; with this power the right reference stands as high as the log sum
    # of all others, a little more for images that had luck with their noise
    refs = _references(N, K, 2 * math.log(N) + 4, g)
    is_of = torch.randint(0, N, (M,), generator=g, device="cuda")
    s["images"] = (refs[is_of] + torch.randn(M, K, generator=g, device="cuda")).to(dt)
    s["bias"] = -0.5 * refs.square().sum(1) + 0.1 * torch.randn(N, generator=g, device="cuda")
    if c["kind"] == "rows8":
        if c["both"]:
            s["references"] = refs.to(dt)
        else:
            s["codes"], s["scales"] = _to_rows8(refs)
        return s
    s["references"] = refs.to(dt)
    s["given"] = is_of
    s["mask"] = None
    if c["mask"]:
        s["mask"] = torch.rand(N, generator=g, device="cuda") < 0.8
        s["mask"][is_of] = True
    if c["train"]:
        for name in ("images", "references", "bias"):
            s[name].requires_grad_()
        # a mean over the images, scaled up where half precision's least numbers would swallow the gradients
        up = (1024.0 if c["dtype"] == "float16" else 1.0) / M
        s["d_given"] = -up * torch.rand(M, generator=g, device="cuda")
        s["d_log_sum"] = 0.3 * up * torch.randn(M, generator=g, device="cuda")
    return s


# ----------------------------------------------------------------------------- one pass
def run(s):
    if own:
        return (_own_pairs if s["kind"] == "pairs" else _own_rows8)(s)
    with torch.no_grad():
        return (_plain_pairs if s["kind"] == "pairs" else _plain_rows8)(s)


def _own_pairs(s):
    r = _matching().pair_log_probs(s["images"], s["references"], s["given"], bias=s["bias"],
                                   temperature=s["temperature"], mask=s["mask"])
    out = dict(given=r.given, log_sum=r.log_sum)
    if s["train"]:
        out["d_images"], out["d_references"], out["d_bias"] = torch.autograd.grad(
            (r.given, r.log_sum), (s["images"], s["references"], s["bias"]), (s["d_given"], s["d_log_sum"]))
    return out


def _own_rows8(s):
    m = _matching()
    references = s["references"] if s["both"] else m.RowScaled(s["codes"], s["scales"])
    return m.row_scores(s["images"], references, bias=s["bias"], out_dtype=DTYPES[s["out"]])


def _plain_pairs(s):
    x, r = s["images"].float(), s["references"].float()
    # (a sum over all values in one go is 1e-4 off where the scores' differences count)
    z = s["bias"].expand(x.shape[0], -1)
    for k in range(0, x.shape[1], 2048):
        z = torch.addmm(z, x[:, k: k + 2048], r[:, k: k + 2048].t())
    z = z / s["temperature"]
    if s["mask"] is not None:
        z = z.masked_fill(~s["mask"], float("-inf"))
    most = z.amax(1, keepdim=True)
    z -= most
    given = s["given"][:, None]
    z_given = z.gather(1, given)
    e = z.exp()
    e_given = e.gather(1, given)
    # what the others hold by itself: next to a probability of one a sum of all would lose it
    others = e.scatter_(1, given, 0.0).sum(1, keepdim=True)
    total = others + e_given
    log_prob = torch.where(e_given > others, -torch.log1p(others / e_given), z_given - total.log())
    out = dict(given=log_prob[:, 0], log_sum=(most + total.log())[:, 0])
    if s["train"]:
        d_given, d_log_sum = s["d_given"][:, None], s["d_log_sum"][:, None]
        d = (e / total).mul_(d_log_sum - d_given)
        d.scatter_(1, given, (d_log_sum * e_given + d_given * others) / total)
        d /= s["temperature"]
        out["d_images"] = (d @ r).to(s["images"].dtype)
        out["d_references"] = (d.t() @ x).to(s["references"].dtype)
        out["d_bias"] = d.sum(0)
    return out


def _plain_rows8(s):
    a, sa = _to_rows8(s["images"])
    b, sb = _to_rows8(s["references"]) if s["both"] else (s["codes"], s["scales"])
    return ((a.float() @ b.float().t()) * sa[:, None] * sb + s["bias"]).to(DTYPES[s["out"]])


# ----------------------------------------------------------------------------- in 64 bits
def _integers(x):
    """The integers and the scales that rows stand for: by definition the quotients are those of 32 bits."""
    x = x.float().cpu().numpy()
    scales = np.maximum(np.abs(x).max(1) / np.float32(127), np.float32(2.0 ** -126))
    codes = np.rint(x / scales[:, None])
    return torch.from_numpy(codes).to("cuda", torch.float64), torch.from_numpy(scales).to("cuda", torch.float64)


def exact(c, seed):
    s = prepare(c, seed)
    with torch.no_grad():
        if c["kind"] == "rows8":
            a, sa = _integers(s["images"])
            b, sb = _integers(s["references"]) if c["both"] else (s["codes"][:, : c["K"]].double(), s["scales"].double())
            return torch.addmm(s["bias"].double(), a * sa[:, None], (b * sb[:, None]).t())
        x, r = s["images"].double(), s["references"].double()
        T = c["temperature"]
        z = torch.addmm(s["bias"].double() / T, x, r.t(), alpha=1 / T)
        if s["mask"] is not None:
            z[:, ~s["mask"]] = -math.inf
        log_sum = torch.logsumexp(z, 1)
        rows = torch.arange(c["M"], device=z.device)
        z -= log_sum[:, None]
        out = dict(given=z[rows, s["given"]], log_sum=log_sum)
        if c["train"]:
            up = z.exp_()
            up *= (s["d_log_sum"].double() - s["d_given"].double())[:, None]
            up[rows, s["given"]] += s["d_given"].double()
            up /= T
            out.update(d_images=up @ r, d_references=up.t() @ x, d_bias=up.sum(0))
        return out
