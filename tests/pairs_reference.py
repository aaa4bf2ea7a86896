"""64-bit definitions of the pair log probabilities and of the rows in 8-bit integers, written from their formulas.

pair_log_probs also bounds what sums in 32 bits may lose (u the unit roundoff, 2^-24 in fp32):
* a score's K products are summed in some order, in float32 rows as six products of 8-bit pieces each: at most
  6 K + 16 additions lose u of the magnitudes' sum each, what is left out 2^-21 of each product; times the temperature and plus
  the bias, each another rounding: `e_score` of the magnitudes' sum;
* probabilities: e^z by a native base-2 exponential (2 u relative), z off by twice the largest score's error (its own and the
  reference point's) and by u of its size in powers of two; sums of N in a tree of lanes: (64 + 24) u;
* gradients: G off by p's error, rounded to the rows' type where there are more than 8 images (half precision also
  loses 2^-25 of 2^-13 of the largest upstream gradient); sums of products as above, their result rounded once.
"""
import math

import torch

U = 2.0 ** -24


def roundoff(dtype):
    return torch.finfo(dtype).eps / 2


def pair_log_probs(images, references, given=None, bias=None, temperature=1.0, mask=None, d_given=None, d_log_sum=None):
    """dict of the results and gradients in float64, and of the bounds on what 32 bits may lose: tol_*.  Scores that are not
    finite are kept as they come; references that the mask rules out are not looked at."""
    dtype, dev = images.dtype, images.device
    x, r = images.double(), references.double()
    M, N, K = x.shape[0], r.shape[0], x.shape[1]
    allowed = torch.ones(N, dtype=torch.bool, device=dev) if mask is None else mask.clone()
    b = torch.zeros(N, dtype=torch.float64, device=dev) if bias is None else bias.double()
    allowed &= b != -math.inf
    r = torch.where(allowed[:, None], r, torch.zeros_like(r))
    b = torch.where(allowed, b, torch.zeros_like(b))
    z = (x @ r.t() + b) / temperature
    z[:, ~allowed] = -math.inf
    mag = (x.abs() @ r.abs().t() + b.abs()) / temperature
    e_score = (((6 if dtype == torch.float32 else 1) * K + 16) * U + 2.0 ** -21)
    off = e_score * mag
    top = z.max(1, keepdim=True).values if N else torch.full((M, 1), -math.inf, dtype=torch.float64, device=dev)
    base = torch.where(top == -math.inf, torch.zeros_like(top), top)
    e = torch.exp(z - base)
    total = e.sum(1, keepdim=True)
    none = (total == 0)[:, 0]
    out = dict(log_sum=torch.where(none, torch.full_like(base[:, 0], -math.inf), (base + total.log())[:, 0]))
    worst = torch.where(allowed, off, torch.zeros_like(off)).amax(1) if N else torch.zeros(M, dtype=torch.float64, device=dev)
    e_prob = 2 * worst + 4 * U * torch.nan_to_num(base[:, 0].abs(), posinf=0.0) + 128 * U
    out["tol_log_sum"] = worst + e_prob + 4 * U * torch.nan_to_num(out["log_sum"].abs(), posinf=0.0)
    p = torch.where(none[:, None], torch.zeros_like(e), e / torch.where(none[:, None], torch.ones_like(total), total))
    g = torch.full((M,), -1, device=dev) if given is None else given
    valid = (g >= 0) & (g < N)
    rows = torch.arange(M, device=dev)
    at = torch.where(valid, g, torch.zeros_like(g))
    if given is not None:
        own = z[rows, at] if N else torch.full((M,), math.nan, dtype=torch.float64, device=dev)
        e_own = torch.exp(own - base[:, 0])
        # the others by themselves
        others = e.clone()
        if N:
            others[rows[valid], at[valid]] = 0.0
        others = others.sum(1)
        lp = torch.where(e_own > others, -torch.log1p(others / e_own), own - out["log_sum"])
        lp = torch.where(none, torch.full_like(lp, -math.inf), lp)
        lp = torch.where(out["log_sum"].isnan(), torch.full_like(lp, math.nan), lp)
        out["given"] = torch.where(valid, lp, torch.where(g == -1, torch.zeros_like(lp), torch.full_like(lp, math.nan)))
        # what the scores lose moves it by 1 - p of that, at most
        out["tol_given"] = torch.where(
            valid, 2 * worst + 8 * U * torch.nan_to_num(out["given"].abs(), posinf=0.0, neginf=0.0) + e_prob *
            torch.nan_to_num(-torch.expm1(out["given"]), nan=1.0), torch.zeros_like(worst))
    if d_given is None and d_log_sum is None:
        return out
    dg = torch.zeros(M, dtype=torch.float64, device=dev) if d_given is None or given is None else d_given.double().clone()
    dl = torch.zeros(M, dtype=torch.float64, device=dev) if d_log_sum is None else d_log_sum.double()
    dg[g == -1] = 0.0
    dg[~valid & (g != -1) & (dg != 0)] = math.nan
    G = p * (dl - dg)[:, None]
    if given is not None and N:
        own_p = p[rows, at]
        here = torch.where(e_own > others, dl * own_p + dg * others / total[:, 0], dl * own_p + dg * (1 - own_p))
        keep = valid & allowed[at]
        G[rows[keep], at[keep]] = here[keep]
    G = torch.where(none[:, None] | ~allowed[None, :], torch.zeros_like(G), G) / temperature
    size = torch.nan_to_num((dl.abs() + dg.abs()) / temperature)
    tolG = p * size[:, None] * e_prob[:, None] * 2 + 4 * U * G.abs()
    if given is not None and N:
        tolG[rows[valid], at[valid]] += (size * e_prob)[valid] * 2 * (own_p * (1 - own_p) + U)[valid]
    out["d_bias"], out["tol_d_bias"] = G.sum(0), tolG.sum(0) + (M + 16) * U * G.abs().sum(0)
    few = M <= 8
    rounding = U if few or dtype == torch.float32 else roundoff(dtype)
    tolG = tolG + rounding * G.abs()
    if dtype == torch.float16 and not few:
        tolG = tolG + 2.0 ** -25 * 2.0 ** -13 * size.max() * 2
    pieces = (6 if dtype == torch.float32 and not few else 1)
    for name, left, right, n in (("d_images", G, r, N), ("d_references", G.t(), x, M)):
        loss = (pieces * n + 16) * U + (2.0 ** -21 if dtype == torch.float32 else 0.0)
        left_tol = tolG if name == "d_images" else tolG.t()
        value = left @ right
        out[name] = value
        out["tol_" + name] = (left_tol @ right.abs() + loss * (left.abs() @ right.abs()) + roundoff(dtype) * value.abs() * (1 + 2.0 ** -6) +
                              (2.0 ** -25 if dtype == torch.float16 else 2.0 ** -134))
    return out


def quantize_rows(x):
    """Integers [R, K] and scales [R] (float32, by definition) of rows."""
    x = x.float()
    most = x.abs().amax(1)
    scale = torch.maximum(most / torch.tensor(127.0), torch.tensor(2.0 ** -126))
    scale = torch.where(torch.isfinite(most), scale, torch.full_like(scale, math.nan))
    codes = torch.round(x / scale[:, None])
    return torch.where(codes.isnan(), torch.zeros_like(codes), codes).to(torch.int64), scale


def row_scores(a, sa, b, sb, bias=None):
    """In the order of the definition: the exact sum to float32, each product rounded, the bias added."""
    total = (a.double() @ b.double().t()).to(torch.int64)  # (below 2^53: exact)
    out = total.float() * sa[:, None] * sb[None, :]
    return out if bias is None else out + bias[None, :]
