"""The softmax cross entropy of a language model's head, without its logits.

`linear_cross_entropy(x, weight, targets)` is the mean of logsumexp(x weight^T) - (x weight^T)[target], what
limn's training example computes as log_softmax of the head's output (reference
`examples/train_stories.py:61-64`). There the logits are a (rows, vocab) tensor, and their log_softmax and its
gradient two more; here the CUSTOM kernels "xent_fwd" and "xent_bwd" (`limn_hip_xent_fwd` and
`limn_hip_xent_bwd` of include/limn_hip.h) walk the vocabulary in pieces and keep two numbers a row. Where the active
device does not register both, for float64, and where the gradient must itself be differentiable, it is
composed from limn's primitives.
"""

from __future__ import annotations

import math

from limn_amd.attend import contiguous, records, through
from limn_amd.seam import FLOATS, Tensor, accumulate_in, active_device, custom, float32, float64, int32, promote

XENT_FWD, XENT_BWD = "xent_fwd", "xent_bwd"


def linear_cross_entropy(x: Tensor, weight: Tensor, targets: Tensor, reduction: str = "mean") -> Tensor:
    """Cross entropy of x (..., width) under the head `weight` (vocab, width) at int32 targets (...).

    A target outside [0, vocab) leaves its row out. `reduction`: "mean" over the other rows (0 where there is
    none), "sum", or "none" for the rows' own losses, shaped as targets; float32 for every width but float64.
    The kernels take up to some 2^30 elements and 690000 rows of x; more raise NotImplementedError when the loss is
    realized, and go in parts whose sums are added.
    """
    if x.ndim < 1 or weight.ndim != 2:
        raise ValueError(f"linear_cross_entropy needs rows (..., width) and a (vocab, width) weight, got {x.shape} and {weight.shape}")
    if x.shape[-1] != weight.shape[1]:
        raise ValueError(f"linear_cross_entropy: widths differ, {x.shape} and {weight.shape}")
    if x.dtype not in FLOATS or weight.dtype not in FLOATS:
        raise ValueError(f"linear_cross_entropy needs float dtypes, got {x.dtype} and {weight.dtype}")
    if targets.dtype != int32 or targets.shape != x.shape[:-1]:
        raise ValueError(f"linear_cross_entropy: targets must be {x.shape[:-1]} int32, got {targets.shape} {targets.dtype}")
    if reduction not in ("mean", "sum", "none"):
        raise ValueError(f"linear_cross_entropy: reduction is mean, sum or none, not {reduction!r}")
    common, vocab = promote(x.dtype, weight.dtype), weight.shape[0]
    loss = _rows(x.cast(common), weight.cast(common), targets)
    if reduction == "none":
        return loss
    total = loss.sum()
    if reduction == "sum":
        return total
    live = ((targets >= 0) * (targets < vocab)).cast(loss.dtype).sum()
    return total * live.maximum(1.0).reciprocal()


def _rows(x: Tensor, w: Tensor, targets: Tensor) -> Tensor:
    """The rows' losses, shaped as targets. The kernels take the leading dims as one (row-major bytes)."""
    dev = active_device()
    if x.dtype == float64 or not (dev.has_custom(XENT_FWD) and dev.has_custom(XENT_BWD)):
        return _composed(x, w, targets)
    x, w, targets = contiguous(x), contiguous(w), contiguous(targets)
    rows = targets.shape
    loss, lse = custom(XENT_FWD, (x.node, w.node, targets.node), (), ((float32, rows), (float32, rows)))

    def backward(g: Tensor):
        if records(x, w):
            return through(lambda x, w: _composed(x, w, targets), (x, w), g)
        srcs = (x.node, w.node, targets.node, lse, contiguous(g).node)
        return tuple(Tensor.from_node(n) for n in custom(XENT_BWD, srcs, (), ((x.dtype, x.shape), (w.dtype, w.shape))))

    return Tensor.from_node(loss, (x, w), backward)


def _composed(x: Tensor, w: Tensor, targets: Tensor) -> Tensor:
    wide, vocab, rows = accumulate_in(x.dtype), w.shape[0], math.prod(targets.shape)
    # a row left out goes as zeros, and its logits too: what it or the weight holds is multiplied by no gradient of 0
    live = ((targets >= 0) * (targets < vocab)).reshape(rows, 1)
    kept = live.where(x.cast(wide).reshape(rows, x.shape[-1]), 0.0)
    logp = live.where(kept @ w.cast(wide).transpose(), 0.0).log_softmax(-1)
    picked = Tensor.arange(vocab).reshape(1, vocab).eq(targets.reshape(rows, 1))
    return -(picked.where(logp, 0.0)).sum(axis=-1).reshape(*targets.shape)
