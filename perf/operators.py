"""Timing cases of the matching operators (torch_projectors.matching): images scored against references in
8-bit blocks, log probabilities of the scored hypotheses, and rows sorted by class and back.

A case is a dict of plain values with a `kind`:
  "scores"  M images of K values against N references: the images quantised to blocks of 128 with a
            power-of-two scale each, the product with the references' blocks, plus a bias per reference
            (`dtype` of the images, `out` of the scores)
  "probs"   T rows of V scores (`dtype`): the log probability of a given candidate, the entropy, the log sum
            and the `top` best alternatives, some candidates masked where `mask`; `train` adds the gradient
            of the scores from upstream gradients of all four
  "route"   T rows of D values (`dtype`), k classes of E each: the sort, the rows in class order and the
            weighted sum back in row order; `train` adds the gradients of the rows, the classes' results
            and the weights

`own` chooses who computes: plain torch operations in 32 bits, or the package's operators.
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
BLOCK = 128  # values that share a scale
PAD = 16  # rows of the scales are padded to this


def _matching():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "torch-projectors_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from torch_projectors import matching
    return matching


def _coefficients(n):
    """Real values of one rfft image of box n."""
    return 2 * n * (n // 2 + 1)


def listed():
    return [
        # one image of a 64 box against every in-plane angle: a call of microseconds
        dict(kind="scores", M=1, N=256, K=_coefficients(64), dtype="float32", out="float32", name="scores_one_64"),
        # one image of a 128 box against the poses of projection matching: as fast as the references are read
        dict(kind="scores", M=1, N=4096, K=_coefficients(128), dtype="float32", out="float32", name="scores_one_128"),
        # a batch of a ragged box (not a whole number of blocks), ragged counts, scores kept in 16 bits
        dict(kind="scores", M=333, N=1999, K=_coefficients(90), dtype="bfloat16", out="bfloat16",
             name="scores_batch_90"),
        # a search of a particle stack over all references: the matrix units' rate
        dict(kind="scores", M=4096, N=8192, K=_coefficients(128), dtype="float32", out="float32",
             name="scores_search_128"),
        # one image's in-plane and view hypotheses
        dict(kind="probs", T=1, V=4096, top=8, dtype="float32", mask=False, train=False, name="probs_one"),
        # a few images over a fine pose grid with in-plane angles, scores in 16 bits
        dict(kind="probs", T=8, V=294912, top=16, dtype="bfloat16", mask=False, train=False, name="probs_fine_grid"),
        # a training minibatch, ragged, some hypotheses excluded
        dict(kind="probs", T=500, V=4099, top=4, dtype="float32", mask=True, train=True, name="probs_step_ragged"),
        # a particle stack over a pose grid, with the gradient
        dict(kind="probs", T=4096, V=36864, top=8, dtype="float32", mask=False, train=True, name="probs_step_stack"),
        # a handful of rows to a few classes: launches count
        dict(kind="route", T=16, k=2, E=8, D=128, dtype="bfloat16", train=False, name="route_few"),
        # images of a 64 box to their two best classes
        dict(kind="route", T=2048, k=2, E=16, D=_coefficients(64), dtype="float32", train=False, name="route_images_64"),
        # a training minibatch of a ragged width, three classes each
        dict(kind="route", T=1001, k=3, E=7, D=1235, dtype="float32", train=True, name="route_step_ragged"),
        # a large batch of feature rows in 16 bits
        dict(kind="route", T=16384, k=4, E=64, D=4096, dtype="bfloat16", train=True, name="route_step_large"),
    ]


def _size(dtype):
    return 4 if dtype == "float32" else 2


def work(c):
    if c["kind"] == "scores":
        M, N, K = c["M"], c["N"], c["K"]
        nb = -(-K // BLOCK)
        return {"bytes": M * K * _size(c["dtype"]) + N * nb * (BLOCK + 1) + 4 * N + M * N * _size(c["out"]),
                "flops": 2 * M * N * K}
    if c["kind"] == "probs":
        T, V, s = c["T"], c["V"], _size(c["dtype"])
        bytes_ = T * V * s + (V if c["mask"] else 0) + T * (8 + 12 + 12 * c["top"])
        flops = 8 * T * V
        if c["train"]:
            # the scores again, their gradient out, the upstream gradients in
            bytes_ += 2 * T * V * s + (V if c["mask"] else 0) + T * (12 + 4 * c["top"])
            flops += 6 * T * V
        return {"bytes": bytes_, "flops": flops}
    T, k, D, s = c["T"], c["k"], c["D"], _size(c["dtype"])
    S = T * k
    # class ids, both permutations, weights; rows in, sorted rows out; the classes' results in, their sum out
    bytes_ = 8 * S + 8 * S + 4 * (c["E"] + 1) + 4 * S + (T * D + S * D) * s + (S * D + T * D) * s
    flops = 2 * S * D
    if c["train"]:
        # upstream of the sorted rows in, the rows' gradient out; upstream of the sum and the results in, theirs out
        bytes_ += (S * D + T * D) * s + (T * D + S * D + S * D) * s + 8 * S
        flops += S * D + 3 * S * D
    return {"bytes": bytes_, "flops": flops}


def _cost(c):
    """Rough time, to keep drawn cases below the largest listed one of their kind."""
    w = work(c)
    return w["bytes"] / 4e12 + w["flops"] / 1.5e15


def draw(rng):
    def logint(a, b):
        return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))

    while True:
        kind = rng.choice(["scores", "probs", "route"])
        if kind == "scores":
            # whole images of an even box, or a plain number of values
            K = _coefficients(2 * logint(8, 64)) if rng.random() < 0.6 else logint(100, 16640)
            c = dict(kind=kind, M=1 if rng.random() < 0.15 else logint(1, 4096), N=logint(16, 8192), K=K,
                     dtype=rng.choice(["float32", "bfloat16"]), out=rng.choice(["float32", "float32", "bfloat16"]))
        elif kind == "probs":
            c = dict(kind=kind, T=logint(1, 4096), V=logint(2, 294912), top=rng.choice([0, 1, 2, 4, 7, 8, 16, 32]),
                     dtype=rng.choice(["float32", "bfloat16", "float16"]), mask=rng.random() < 0.4,
                     train=rng.random() < 0.5)
            c["top"] = min(c["top"], c["V"] // 2)
        else:
            c = dict(kind=kind, T=logint(1, 16384), k=rng.choice([1, 2, 2, 3, 4, 6, 8]), E=logint(2, 256),
                     D=logint(8, 16640), dtype=rng.choice(["float32", "bfloat16", "float16"]),
                     train=rng.random() < 0.5)
        largest = max(_cost(d) for d in listed() if d["kind"] == kind)
        if _cost(c) <= largest and 3072 not in c.values():
            return c


# ----------------------------------------------------------------------------- inputs
def _images(rows, K, g):
    """Fourier coefficients: amplitudes fall by three orders of magnitude from the first to the last."""
    fall = torch.exp(torch.linspace(0.0, -7.0, K, device=g.device))
    return torch.randn(rows, K, generator=g, device=g.device) * fall


def _to_blocks(x):
    """codes [R, 128 nb] (float8_e4m3fn) and scales [nb, R padded to 16] (bytes, 127 + the exponent) of x [R, K]:
    the exponent is the least that keeps the block's largest value within 448."""
    R, K = x.shape
    nb = -(-K // BLOCK)
    b = torch.nn.functional.pad(x.float(), (0, nb * BLOCK - K)).view(R, nb, BLOCK)
    mant, e = torch.frexp(b.abs().amax(2))  # largest = mant * 2^e, mant in [0.5, 1)
    e = torch.where(mant > 0.875, e - 8, e - 9)  # 448 = 0.875 * 2^9
    e = torch.where(mant == 0, torch.zeros_like(e), e.clamp_min(-127))
    codes = torch.ldexp(b, -e.unsqueeze(2)).to(torch.float8_e4m3fn).view(R, nb * BLOCK)
    scales = torch.full((nb, -(-R // PAD) * PAD), 127, dtype=torch.uint8, device=x.device)
    scales[:, :R] = (e + 127).t().to(torch.uint8)
    return codes, scales


def _from_blocks(codes, scales):
    R, Kp = codes.shape
    e = scales[:, :R].t().to(torch.int32) - 127
    return torch.ldexp(codes.float().view(R, Kp // BLOCK, BLOCK), e.unsqueeze(2)).view(R, Kp)


def prepare(c, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt = DTYPES[c["dtype"]]
    s = dict(c)
    if c["kind"] == "scores":
        refs = _images(c["N"], c["K"], g)
        s["images"] = (refs[torch.arange(c["M"], device="cuda") % c["N"]] * 0.5 + _images(c["M"], c["K"], g)).to(dt)
        s["bias"] = -0.5 * refs.square().sum(1)
        s["codes"], s["scales"] = _to_blocks(refs)
    elif c["kind"] == "probs":
        T, V = c["T"], c["V"]
        x = torch.randn(T, V, generator=g, device="cuda") * 2
        s["given"] = torch.randint(0, V, (T,), generator=g, device="cuda")
        # the present hypothesis stands out, in some rows more than in others
        x.scatter_add_(1, s["given"][:, None], 12 * torch.rand(T, 1, generator=g, device="cuda"))
        s["scores"] = x.to(dt).requires_grad_(c["train"])
        s["mask"] = None
        if c["mask"]:
            s["mask"] = torch.rand(V, generator=g, device="cuda") < 0.8
            s["mask"][s["given"]] = True
            s["mask"][: c["top"]] = True
        if c["train"]:
            s["d_given"] = -torch.rand(T, generator=g, device="cuda")
            s["d_entropy"] = torch.randn(T, generator=g, device="cuda") * 0.1
            s["d_log_sum"] = torch.randn(T, generator=g, device="cuda") * 0.1
            s["d_top"] = torch.randn(T, c["top"], generator=g, device="cuda") * 0.1
    else:
        T, k, E, D = c["T"], c["k"], c["E"], c["D"]
        # some classes are far more popular than others
        liking = torch.randn(E, generator=g, device="cuda") + torch.rand(T, k, E, generator=g, device="cuda") * 4
        s["classes"] = liking.argmax(2)
        s["weights"] = torch.softmax(torch.randn(T, k, generator=g, device="cuda"), 1).requires_grad_(c["train"])
        s["x"] = torch.randn(T, D, generator=g, device="cuda").to(dt).requires_grad_(c["train"])
        s["y"] = torch.randn(T * k, D, generator=g, device="cuda").to(dt).requires_grad_(c["train"])
        if c["train"]:
            s["d_sorted"] = torch.randn(T * k, D, generator=g, device="cuda").to(dt)
            s["d_sum"] = torch.randn(T, D, generator=g, device="cuda").to(dt)
    return s


# ----------------------------------------------------------------------------- one pass
def run(s):
    if own:
        return {"scores": _own_scores, "probs": _own_probs, "route": _own_route}[s["kind"]](s)
    with torch.no_grad():
        return {"scores": _plain_scores, "probs": _plain_probs, "route": _plain_route}[s["kind"]](s)


def _own_scores(s):
    m = _matching()
    return m.block_scores(s["images"], m.BlockScaled(s["codes"], s["scales"]), bias=s["bias"],
                          out_dtype=DTYPES[s["out"]])


def _own_probs(s):
    r = _matching().log_probs(s["scores"], s["given"], top=s["top"], temperature=1.5, mask=s["mask"])
    out = dict(given=r.given, entropy=r.entropy, log_sum=r.log_sum, top=r.top, top_index=r.top_index)
    if s["train"]:
        (out["d_scores"],) = torch.autograd.grad(
            (r.given, r.entropy, r.log_sum, r.top), (s["scores"],),
            (s["d_given"], s["d_entropy"], s["d_log_sum"], s["d_top"]))
    return out


def _own_route(s):
    m = _matching()
    r = m.sort_by_class(s["classes"], s["E"])
    xs = m.dispatch(s["x"], r)
    y = m.combine(s["y"], r, s["weights"])
    out = dict(order=r.order, slot=r.slot, offsets=r.offsets, sorted=xs, sum=y)
    if s["train"]:
        out["d_x"], out["d_y"], out["d_weights"] = torch.autograd.grad(
            (xs, y), (s["x"], s["y"], s["weights"]), (s["d_sorted"], s["d_sum"]))
    return out


def _plain_scores(s):
    images = _from_blocks(*_to_blocks(s["images"]))
    return (images @ _from_blocks(s["codes"], s["scales"]).t() + s["bias"]).to(DTYPES[s["out"]])


def _plain_probs(s):
    x = s["scores"].float()
    if s["mask"] is not None:
        x = x.masked_fill(~s["mask"], float("-inf"))
    z = (x - x.amax(1, keepdim=True)) / 1.5
    e = z.exp()
    total = e.sum(1, keepdim=True)
    lp = z - total.log()
    p = e / total
    plp = torch.where(p > 0, p * lp, torch.zeros_like(p))
    entropy = -plp.sum(1)
    best, index = torch.sort(x, dim=1, descending=True, stable=True)
    index = index[:, : s["top"]]
    del best
    out = dict(given=lp.gather(1, s["given"][:, None])[:, 0], entropy=entropy,
               log_sum=x.amax(1) / 1.5 + total.log()[:, 0], top=lp.gather(1, index), top_index=index)
    if s["train"]:
        at_all = s["d_log_sum"] - s["d_given"] - s["d_top"].sum(1)
        d = p * at_all[:, None] - s["d_entropy"][:, None] * (plp + p * entropy[:, None])
        d.scatter_add_(1, s["given"][:, None], s["d_given"][:, None])
        d.scatter_add_(1, index, s["d_top"])
        out["d_scores"] = (d / 1.5).to(s["scores"].dtype)
    return out


def _plain_route(s):
    T, k, E, D = s["T"], s["k"], s["E"], s["D"]
    classes = s["classes"].reshape(-1)
    order = torch.sort(classes, stable=True)[1]
    slot = torch.empty_like(order)
    slot[order] = torch.arange(T * k, device=order.device)
    offsets = torch.zeros(E + 1, dtype=torch.int32, device=order.device)
    offsets[1:] = (classes[:, None] == torch.arange(E, device=order.device)).sum(0).cumsum(0)
    w = s["weights"]
    y = s["y"].float()[slot].view(T, k, D)
    out = dict(order=order.to(torch.int32), slot=slot.to(torch.int32).view(T, k), offsets=offsets,
               sorted=s["x"][order // k], sum=(w[:, :, None] * y).sum(1).to(s["y"].dtype))
    if s["train"]:
        out["d_x"] = s["d_sorted"].float()[slot].view(T, k, D).sum(1).to(s["x"].dtype)
        d_sum = s["d_sum"].float()
        out["d_y"] = (w.reshape(-1)[order][:, None] * d_sum[order // k]).to(s["y"].dtype)
        out["d_weights"] = (d_sum[:, None, :] * y).sum(2)
    return out


# ----------------------------------------------------------------------------- in 64 bits
def _eight_bits(v):
    """v rounded to a 3-bit mantissa, exponents from -6 up, half to even (no value here is past 448)."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 3)
    return torch.round(v / step) * step


def exact(c, seed):
    s = prepare(c, seed)
    with torch.no_grad():
        if c["kind"] == "scores":
            x = s["images"].double()
            a = torch.zeros(c["M"], s["codes"].shape[1], dtype=torch.float64, device=x.device)
            b = s["codes"].double()
            for k in range(a.shape[1] // BLOCK):
                at = slice(k * BLOCK, (k + 1) * BLOCK)
                part = x[:, at]
                most = part.abs().amax(1, keepdim=True)
                unit = torch.exp2(torch.ceil(torch.log2(most.clamp_min(1e-300) / 448)).clamp_min(-127))
                a[:, k * BLOCK: k * BLOCK + part.shape[1]] = _eight_bits(part / unit) * unit
                b[:, at] *= torch.exp2(s["scales"][k, : c["N"]].double() - 127)[:, None]
            return a @ b.t() + s["bias"].double()
        if c["kind"] == "probs":
            z = s["scores"].double() / 1.5
            if s["mask"] is not None:
                z = torch.where(s["mask"], z, torch.full((), -math.inf, dtype=z.dtype, device=z.device))
            log_sum = torch.logsumexp(z, 1)
            z -= log_sum[:, None]
            p = z.exp()
            zp = torch.nan_to_num(z, neginf=0.0) * p
            entropy = -zp.sum(1)
            index = torch.sort(z, dim=1, descending=True, stable=True)[1][:, : c["top"]]
            rows = torch.arange(c["T"], device=z.device)
            out = dict(given=z[rows, s["given"]], entropy=entropy, log_sum=log_sum, top=z[rows[:, None], index],
                       top_index=None)
            if c["train"]:
                up = torch.zeros_like(z)
                up[rows, s["given"]] += s["d_given"].double()
                up.scatter_add_(1, index, s["d_top"].double())
                up -= p * up.sum(1, keepdim=True)
                up += p * s["d_log_sum"].double()[:, None]
                up -= (zp + p * entropy[:, None]) * s["d_entropy"].double()[:, None]
                out["d_scores"] = up / 1.5
            return out
        T, k = c["T"], c["k"]
        flat = s["classes"].flatten()
        # a slot's place: the slots of lower classes, then the earlier ones of its own
        place = torch.argsort(torch.argsort(flat * (T * k) + torch.arange(T * k, device=flat.device)))
        place = place.view(T, k)
        w, y = s["weights"].double(), s["y"].double()
        out = dict(order=None, slot=None, offsets=None, sorted=torch.empty(T * k, c["D"], dtype=torch.float64, device=y.device),
                   sum=torch.zeros(T, c["D"], dtype=torch.float64, device=y.device))
        if c["train"]:
            up, d_sum = s["d_sorted"].double(), s["d_sum"].double()
            out["d_x"] = torch.zeros_like(out["sum"])
            out["d_y"] = torch.empty_like(y)
            out["d_weights"] = torch.empty_like(w)
        for j in range(k):
            at = place[:, j]
            out["sorted"][at] = s["x"].double()
            out["sum"] += w[:, j, None] * y[at]
            if c["train"]:
                out["d_x"] += up[at]
                out["d_y"][at] = w[:, j, None] * d_sum
                out["d_weights"][:, j] = (d_sum * y[at]).sum(1)
        return out
