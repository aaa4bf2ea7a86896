"""The matching operators' definitions in 64 bits on the CPU, for the tests to compare with."""
import math

import torch

BLOCK = 128
# unit roundoffs
U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def quantize(x):
    """(code values [R, 128 nb], exponents [R, nb]) in float64: each code is the e4m3 value nearest to x 2^-e."""
    x = x.double().cpu()
    R, K = x.shape
    nb = -(-K // BLOCK)
    b = torch.nn.functional.pad(x, (0, nb * BLOCK - K)).view(R, nb, BLOCK)
    finite = torch.isfinite(b)
    most = torch.where(finite, b.abs(), torch.zeros_like(b)).amax(2)
    e = torch.zeros(R, nb, dtype=torch.int64)
    for r in range(R):
        for k in range(nb):
            m = float(most[r, k])
            if m > 0:
                f, ex = math.frexp(m / 448.0)
                e[r, k] = max(ex - 1 if f == 0.5 else ex, -127)
    v = b * torch.exp2(-e.double())[:, :, None]
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 3)
    q = torch.where(finite, torch.round(v / step) * step, torch.full_like(v, math.nan))
    return q.view(R, nb * BLOCK), e


def blocks_value(codes, scales):
    """What BlockScaled tensors stand for, in float64."""
    codes, scales = codes.cpu(), scales.cpu()
    R, Kp = codes.shape
    e = scales[:, :R].t().double() - 127
    return (codes.float().double().view(R, Kp // BLOCK, BLOCK) * torch.exp2(e)[:, :, None]).view(R, Kp)


def log_probs(scores, given=None, top=0, temperature=1.0, mask=None, ups=None):
    """Results of [T, V] scores as a dict; with ups = (d_given, d_entropy, d_log_sum, d_top) the gradient too."""
    x = scores.double().cpu()
    T, V = x.shape
    allowed = torch.ones(T, V, dtype=torch.bool) if mask is None else mask.cpu().expand(T, V)
    out = dict(entropy=torch.zeros(T), log_sum=torch.zeros(T), top=torch.full((T, top), -math.inf),
               top_index=torch.full((T, top), -1, dtype=torch.int64))
    out = {k: v.double() if v.is_floating_point() else v for k, v in out.items()}
    G = 0 if given is None else given.shape[1]
    out["given"] = torch.zeros(T, G, dtype=torch.float64)
    d = torch.zeros(T, V, dtype=torch.float64)
    for t in range(T):
        ok = allowed[t]
        z = torch.full((V,), -math.inf, dtype=torch.float64)
        z[ok] = x[t][ok] / temperature
        nan, none = bool(z.isnan().any()), bool((z == -math.inf).all())
        # relative to the largest: scores of the type's lowest value leave no room for ln V in 64 bits either
        m = z.max()
        ls = torch.log(torch.exp(z - m).sum())
        L = torch.tensor(math.nan if nan else -math.inf if none else float(m + ls), dtype=torch.float64)
        lp = torch.full_like(z, -math.inf) if none else torch.full_like(z, math.nan) if nan else (z - m) - ls
        p = lp.exp()
        H = -torch.where(p > 0, p * lp, torch.zeros_like(p)).sum() if not nan else L
        out["entropy"][t], out["log_sum"][t] = 0.0 if none else H, L
        for g in range(G):
            v = int(given[t, g])
            out["given"][t, g] = 0.0 if v == -1 else lp[v] if 0 <= v < V else math.nan
        best = [v for v in sorted(range(V), key=lambda v: (-float(z[v]), v)) if float(z[v]) > -math.inf][:top] if top else []
        for j, v in enumerate(best):
            out["top"][t, j], out["top_index"][t, j] = lp[v], v
        if top and nan:
            out["top"][t] = math.nan
        if ups is None or none:
            continue
        d_given, d_entropy, d_log_sum, d_top = ups
        at = torch.zeros(V, dtype=torch.float64)
        total = 0.0
        if d_given is not None:
            for g in range(G):
                v = int(given[t, g])
                if v >= 0:
                    total += float(d_given[t, g])
                    if ok[v]:
                        at[v] += float(d_given[t, g])
        if d_top is not None:
            for j, v in enumerate(best):
                total += float(d_top[t, j])
                at[v] += float(d_top[t, j])
        dH = 0.0 if d_entropy is None else float(d_entropy[t])
        dL = 0.0 if d_log_sum is None else float(d_log_sum[t])
        plp = torch.where(p > 0, p * lp, torch.zeros_like(p))
        row = (p * (dL - total) - dH * (plp + p * H) + at) / temperature
        d[t] = torch.where(ok, row, torch.zeros_like(row))
    out["d_scores"] = d
    return out


def sort_by_class(classes, E):
    flat = [int(c) for c in classes.reshape(-1)]
    key = [c if 0 <= c < E else E for c in flat]
    order = sorted(range(len(flat)), key=lambda i: (key[i], i))
    slot = [0] * len(flat)
    for r, i in enumerate(order):
        slot[i] = r
    offsets = [sum(k < c for k in key) for c in range(E + 1)]
    return torch.tensor(order, dtype=torch.int32), torch.tensor(slot, dtype=torch.int32).view(classes.shape), \
        torch.tensor(offsets, dtype=torch.int32)


def spread(x, slot, kept, weights=None):
    """[T, D] -> [T k, D] in float64."""
    T, k = slot.shape
    out = torch.zeros(T * k, x.shape[1], dtype=torch.float64)
    for t in range(T):
        for j in range(k):
            r = int(slot[t, j])
            if r < kept:
                out[r] = x[t].double() * (1.0 if weights is None else float(weights[t, j]))
    return out


def gather(y, slot, kept, weights=None):
    """[T k, D] -> ([T, D], sum of magnitudes) in float64."""
    T, k = slot.shape
    out = torch.zeros(T, y.shape[1], dtype=torch.float64)
    mag = torch.zeros_like(out)
    for t in range(T):
        for j in range(k):
            r = int(slot[t, j])
            if r < kept:
                v = y[r].double() * (1.0 if weights is None else float(weights[t, j]))
                out[t] += v
                mag[t] += v.abs()
    return out, mag


def dots(x, y, slot, kept):
    """<x[t], y[slot[t, j]]> and the sum of magnitudes, in float64."""
    T, k = slot.shape
    out = torch.zeros(T, k, dtype=torch.float64)
    mag = torch.zeros_like(out)
    for t in range(T):
        for j in range(k):
            r = int(slot[t, j])
            if r < kept:
                v = x[t].double() * y[r].double()
                out[t, j], mag[t, j] = v.sum(), v.abs().sum()
    return out, mag
