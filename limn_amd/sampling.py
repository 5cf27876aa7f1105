"""A token for each row of logits, from given uniform numbers.

`sample(logits, uniforms, temperature=, top_k=, top_p=, min_p=)` is the last step of answering with a language model: what the
reference's training example does to a softmax on the host (`examples/train_stories.py`) stays on the device here, with
the filters that servers offer. It is the CUSTOM kernel "sample" (`limn_hip_sample` of include/limn_hip.h) where the active
device registers it, and composed from limn's primitives in float64 elsewhere (the filters' order from every pair of
tokens: for small vocabularies).

With w_j = exp((x_j - max x) / temperature) and the order of x descending, equal ones by index, each filter keeps a beginning
of the order: the first top_k; of those the ones before which less than top_p of their mass lies; of those the ones with w_j >=
min_p; the first always. The token is the first one whose mass with all before it passes u times the kept mass.
"""

from __future__ import annotations

import math
import sys

from limn_amd.attend import contiguous
from limn_amd.seam import FLOATS, Tensor, active_device, custom, float32, float64, int32

SAMPLE = "sample"
MOST_TOKENS = 1 << 24


def sample(logits: Tensor, uniforms: Tensor, *, temperature: float | Tensor = 1.0, top_k: int | Tensor = 0, top_p: float | Tensor = 1.0,
           min_p: float | Tensor = 0.0) -> tuple[Tensor, Tensor]:
    """Tokens (...) int32 drawn from logits (..., vocab), vocab up to 2^24, by uniforms (...) float32 in [0, 1), and the logarithms (...) float32
    of their shares of the kept mass.

    The settings are numbers, or tensors (...) with one for each row (float32, top_k int32):
    - `temperature`: 0 or below takes the largest logit (the first of equal ones), with the logarithm 0;
    - `top_k`: 0 or below, or the vocabulary or more, for no limit;
    - `top_p`: 1 or more for no limit; - `min_p`: 0 or below for none.

    A NaN among the logits counts as minus infinity; a row without anything above that gives token -1 and minus infinity. An
    infinite logit has all of the mass. A uniform number outside [0, 1) takes the nearest end, NaN the last token kept. Of tensors, a
    temperature of NaN counts as 0, and a top_p or min_p of NaN is no limit. No gradient flows.
    """
    if logits.ndim < 1 or logits.dtype not in FLOATS:
        raise ValueError(f"sample needs float logits (..., vocab), got {logits.shape} {logits.dtype}")
    if logits.shape[-1] > MOST_TOKENS:
        raise ValueError(f"sample: a vocabulary of at most {MOST_TOKENS}, not {logits.shape[-1]}")
    rows = logits.shape[:-1]
    if uniforms.shape != rows or uniforms.dtype != float32:
        raise ValueError(f"sample: uniforms must be {rows} float32, got {uniforms.shape} {uniforms.dtype}")
    rules: list[Tensor | None] = []
    for name, rule, off, dtype in (("temperature", temperature, 1.0, float32), ("top_k", top_k, 0, int32), ("top_p", top_p, 1.0, float32), ("min_p", min_p, 0.0, float32)):
        if not isinstance(rule, Tensor):
            number = int(rule) if dtype == int32 and math.isfinite(rule) else float(rule)
            if number != rule or abs(number) > 2**31 - 1:
                raise ValueError(f"sample: {name} must be a finite {'whole ' if dtype == int32 else ''}number, got {rule}")
            rules.append(None if number == off else Tensor.full(rows, number, dtype=dtype))
        elif rule.shape != rows or rule.dtype != dtype:
            raise ValueError(f"sample: {name} must be {rows} {dtype}, got {rule.shape} {rule.dtype}")
        else:
            rules.append(rule)
    logits, uniforms = logits.detach(), uniforms.detach()
    if logits.dtype == float64 or not active_device().has_custom(SAMPLE):
        return _composed(logits, uniforms, *rules)
    given = tuple(contiguous(t).node for t in rules if t is not None)
    srcs = (contiguous(logits).node, contiguous(uniforms).node, *given)
    outs = custom(SAMPLE, srcs, tuple(t is not None for t in rules), ((int32, rows), (float32, rows)))
    return tuple(Tensor.from_node(n) for n in outs)


def _composed(logits: Tensor, uniforms: Tensor, temperature, top_k, top_p, min_p) -> tuple[Tensor, Tensor]:
    """The same from limn's primitives, the order from a comparison of every pair."""
    rows, vocab = logits.shape[:-1], logits.shape[-1]
    ones = (1,) * len(rows)
    column = lambda t: t.reshape(*rows, 1)  # noqa: E731
    x = logits.cast(float64)
    infinite = (x > sys.float_info.max).cast(float64)
    there = infinite.max(-1, keepdim=True).where(infinite, x > -math.inf)  # not minus infinity, NaN (which is above nothing), or beside an infinity
    x = there.where((infinite > 0).where(0.0, x), -math.inf)
    top = x.max(-1, keepdim=True)
    some = (top > -math.inf).reshape(*rows)
    warm = Tensor.full(rows, 1.0) if temperature is None else temperature
    heat = column((warm > 0).where(warm, 1.0).cast(float64))
    w = there.where(((x - top) / heat).exp(), 0.0)
    mine, other = x.reshape(*rows, vocab, 1), x.reshape(*rows, 1, vocab)
    index = Tensor.arange(vocab)
    sooner = (index.reshape(*ones, 1, vocab) < index.reshape(*ones, vocab, 1)).cast(float64)
    ahead = (other > mine) + other.eq(mine) * sooner  # (..., token, the tokens before it)
    rank = ahead.sum(-1)
    before = (ahead * w.reshape(*rows, 1, vocab)).sum(-1)
    kept = rank < vocab
    if top_k is not None:
        kept = rank < column(((top_k > 0) * (top_k < vocab)).where(top_k, vocab).cast(float64))
    if top_p is not None:
        p = column(top_p.cast(float64))
        kept = kept * (p < 1.0).where(before < p * (kept * w).sum(-1, keepdim=True), 1.0)
    if min_p is not None:
        kept = kept * (1.0 - (w < column(min_p.cast(float64))))
    kept = (kept + rank.eq(0.0)) > 0
    mass = (kept * w).sum(-1, keepdim=True)
    # past the end, NaN too: the last one kept whose mass is one, as the kernels' whole numbers have it
    u = uniforms.cast(float64)
    short = (u < 1.0).where((kept * ((before + w) <= column(u) * mass)).sum(-1), vocab)
    heavy = w > 2.0 ** -(1 + min(52, 62 - (vocab - 1).bit_length()))
    place = (warm > 0).cast(float64) * short.minimum((kept * heavy).sum(-1) - 1.0)
    hit = rank.eq(column(place))
    token = (hit * index.cast(float64).reshape(*ones, vocab)).sum(-1).cast(int32)
    share = (warm > 0).cast(float64).where((hit * w).sum(-1) / mass.reshape(*rows), 1.0)
    return some.cast(int32).where(token, -1), some.where(share.log(), -math.inf).cast(float32)
