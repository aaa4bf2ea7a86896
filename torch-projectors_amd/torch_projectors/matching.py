"""Matching images to references: what stands between projecting references and backprojecting images.

    quantize_blocks(x)                    rows in 8-bit floating point, a scale for each 128 values
    block_scores(images, references)      <image, reference> of every pair, from such rows
    log_probs(scores, given, top, ...)    log probabilities of given candidates, entropy, log sum and the
                                          best alternatives of each row; differentiable
    sort_by_class(classes, num_classes)   rows sorted by the classes that they go to
    dispatch(x, order) / combine(y, order)  rows into that order, and back with weights; differentiable

The reference leaves these steps to its users (it has no counterpart).  A search scores the images of a
stack against the projections of every class and pose (`block_scores`), turns the scores into a posterior
(`log_probs`: `top_index` and `top` are the best hypotheses and their weights), and hands each image to the
classes it goes to (`sort_by_class` of the hypotheses' classes, `dispatch`); each class's stretch
`offsets[c] : offsets[c + 1]` is then one call of a projection operator, and `combine` sums a row's results
with its weights.  In training, `log_probs` of `images @ projections.T` carries the gradient of the marginal
likelihood (`log_sum`) back to volumes and poses.

All run on the GPU only (a CPU tensor raises NotImplementedError), on the current stream, without a
synchronisation; they can be captured in a graph.  What is differentiable is so once, backwards (forward-mode
tangents raise NotImplementedError).
"""
from typing import NamedTuple, Optional

import torch

from . import ops  # noqa: F401  (the package's operators are loaded)

_OPS = torch.ops.torch_projectors


# ----------------------------------------------------------------------------- scores in 8-bit blocks
class BlockScaled(NamedTuple):
    """Rows [R, K] in 8-bit blocks of 128 values: value = code * 2^(scale - 127).

    codes   [R, 128 nb] float8_e4m3fn, nb = ceil(K / 128), zero past K
    scales  [nb, R padded to a multiple of 16] uint8
    """
    codes: torch.Tensor
    scales: torch.Tensor


def _real_rows(x, what):
    """[R, ...] -> [R, K]; complex values as (real, imaginary) pairs."""
    if x.dim() < 1:
        raise ValueError(f"{what} must have at least 1 dimension")
    if x.is_complex():
        x = torch.view_as_real(x.resolve_conj().resolve_neg())
    return x if x.dim() == 2 else x.reshape(x.shape[0], _numel(x.shape[1:]))


def _numel(shape):
    n = 1
    for s in shape:
        n *= s
    return n


def quantize_blocks(x: torch.Tensor) -> BlockScaled:
    """Rows [R, ...] (float32, float16, bfloat16 or complex64) in 8-bit blocks of 128 values.

    A block's scale is the least power of two that keeps its largest finite magnitude within 448 times
    it; the codes are rounded to nearest even.  Values that are not finite become NaN.  Not
    differentiable.

    Products take a value exactly where its block's scale byte is 3 to 246.  In blocks whose largest value is
    below 1.05e-35 (bytes 0 to 2) values count as multiples of 2^-133; values from 3.297e38 up count as infinite, as
    does what is past 2^128 in blocks from elsewhere."""
    return BlockScaled(*_OPS.quantize_blocks.default(_real_rows(x, "x")))


def block_scores(images, references, bias: Optional[torch.Tensor] = None,
                 out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """scores[m, n] = <image m, reference n> + bias[n], from 8-bit blocks, summed in float32.

    images [M, ...] and references [N, ...] are BlockScaled, or rows that are quantised here, of as many
    values on both sides (BlockScaled rows hold zeros past theirs: of them the numbers of blocks are
    compared); of complex rows the real part of the inner product is taken (their real pairs' product).  With rfft images,
    which hold one half of a symmetric plane, scale either side's columns other than x = 0 and n / 2 by two for the
    whole plane's product; with bias = -|reference|^2 / 2 the scores are the log likelihoods of unit noise
    up to a constant per image, where every image has the same transfer function (in the references).  With functions
    of their own, score images times theirs without a bias and subtract the half product of the squared functions
    and the references' squared magnitudes, which depends on the pair, too.

    bias float32 [N]; out_dtype float32 or bfloat16.  Not differentiable."""
    rows = None if isinstance(images, BlockScaled) else _real_rows(images, "images")
    if not isinstance(references, BlockScaled):
        references = _real_rows(references, "references")
        if rows is not None and rows.shape[1] != references.shape[1]:
            raise ValueError(f"Images of {rows.shape[1]} values do not fit references of {references.shape[1]}")
        references = quantize_blocks(references)
    images, image_scales = images if rows is None else (rows, None)
    return _OPS.block_scores.default(images, image_scales, references.codes, references.scales, bias, out_dtype)


# ----------------------------------------------------------------------------- log probabilities
class LogProbs(NamedTuple):
    """Results of log_probs, float32 but for the indices.

    given      log probabilities of the given candidates, of given's shape (None without)
    entropy    of each row's distribution
    log_sum    ln sum exp(score / temperature) over each row's allowed candidates
    top        [..., top] log probabilities of the best candidates, best first
    top_index  [..., top] int64, ties in the order of their indices
    """
    given: Optional[torch.Tensor]
    entropy: torch.Tensor
    log_sum: torch.Tensor
    top: torch.Tensor
    top_index: torch.Tensor


def log_probs(scores: torch.Tensor, given: Optional[torch.Tensor] = None, top: int = 0, temperature: float = 1.0,
              mask: Optional[torch.Tensor] = None) -> LogProbs:
    """Log probabilities of the softmax of scores [..., V] / temperature (float32, float16 or bfloat16).

    given   int64 [...] or [..., G]: the candidates whose log probability is wanted; -1 for none (its
            result is 0 and has no gradient); any other index out of range gives NaN, and a row of NaN
            gradients unless its own upstream gradient is 0
    top     how many of the best candidates to list, at most 64
    mask    bool [V] or of the scores' shape, True where allowed; what masked scores hold is not used

    A score of -inf is not allowed either.  A row that allows nothing has log probabilities and log_sum
    -inf, entropy 0 and no gradient; past the allowed candidates top_index is -1 and top -inf.  A NaN
    among the allowed scores makes its row's results NaN.  The gradient reaches scores from all four
    float results, in the scores' dtype."""
    if scores.dim() < 1:
        raise ValueError("Scores must have at least 1 dimension (..., candidates)")
    lead, V = scores.shape[:-1], scores.shape[-1]
    if given is not None and (given.shape[:len(lead)] != lead or given.dim() > len(lead) + 1):
        raise ValueError(f"Given candidates {tuple(given.shape)} must have the scores' leading dimensions "
                         f"{tuple(lead)} and at most one more")
    if mask is not None and mask.shape != scores.shape and mask.shape != (V,):
        raise ValueError(f"Mask {tuple(mask.shape)} must have the scores' shape {tuple(scores.shape)} or be ({V},)")
    if len(lead) == 1:
        return LogProbs(*_OPS.log_probs.default(scores, given, mask, top, temperature)[:5])
    T = _numel(lead)
    flat = given if given is None else given.reshape(T) if given.dim() == len(lead) else given.reshape(T, given.shape[-1])
    if mask is not None and mask.shape == scores.shape:
        mask = mask.reshape(T, V)
    g, entropy, log_sum, best, index, _ = _OPS.log_probs.default(scores.reshape(T, V), flat, mask, top, temperature)
    return LogProbs(None if g is None else g.view(given.shape), entropy.view(lead), log_sum.view(lead),
                    best.view(*lead, top), index.view(*lead, top))


# ----------------------------------------------------------------------------- rows by class
class ClassOrder(NamedTuple):
    """T rows with k classes each, as T k slots sorted by class (all int32).

    order    [T k] the slot (row * k + choice) at each place
    slot     [T, k] the place of each slot
    offsets  [num_classes + 1] class c has places offsets[c] : offsets[c + 1]; those from offsets[-1] on
             belong to dropped slots
    """
    order: torch.Tensor
    slot: torch.Tensor
    offsets: torch.Tensor


def sort_by_class(classes: torch.Tensor, num_classes: int) -> ClassOrder:
    """Sort the choices [T] or [T, k] (int64 or int32) of T rows by class, keeping the order of each
    class's slots.  Choices outside [0, num_classes), num_classes at most 4096, are dropped."""
    if classes.dim() not in (1, 2):
        raise ValueError("Classes must be (rows) or (rows, choices)")
    return ClassOrder(*_OPS.sort_by_class.default(classes, num_classes))


def _move(op, x, n, order, weights, what):
    slot, offsets = order.slot, order.offsets
    if x.dim() < 1 or x.shape[0] != n:
        raise ValueError(f"{what} must have {n} rows, got shape {tuple(x.shape)}")
    if weights is not None and weights.shape != slot.shape:
        if weights.dim() != 1 or (weights.shape[0], 1) != slot.shape:
            raise ValueError(f"Weights {tuple(weights.shape)} must have the classes' shape {tuple(slot.shape)}")
        weights = weights.unsqueeze(1)
    rows = _real_rows(x, what)
    out = op(rows, slot, offsets, weights, None)[0]
    if rows is x:
        return out
    if x.is_complex():
        return torch.view_as_complex(out.view(out.shape[0], *x.shape[1:], 2))
    return out.view(out.shape[0], *x.shape[1:])


def dispatch(x: torch.Tensor, order: ClassOrder, weights: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rows x [T, ...] (float32, float16, bfloat16 or complex64) in class order: [T k, ...], row t at
    each of its places slot[t, j], times weights[t, j] (float32 [T, k]) where given; zero rows where
    dropped.  Differentiable in x and weights."""
    return _move(_OPS.spread_rows.default, x, order.slot.shape[0], order, weights, "x")


def combine(y: torch.Tensor, order: ClassOrder, weights: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rows y [T k, ...] in class order back to [T, ...]: sum_j weights[t, j] y[slot[t, j]] in float32,
    rounded once, without the dropped ones.  Differentiable in y and weights."""
    return _move(_OPS.gather_rows.default, y, order.order.shape[0], order, weights, "y")
