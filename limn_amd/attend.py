"""Attention whose scores follow rules: capped by a tanh, biased by distance, masked by document or prefix,
with query heads that share key heads and the live length of a cache.

`attend` is to these what `Tensor.attention` (reference `limn/tensor.py:509-575`) is to causal and key
masks: it emits the CUSTOM kernels "attend_fwd" and "attend_bwd" where the active device registers both
(the hip device does, `limn_hip_attend_fwd` and `limn_hip_attend_bwd` of include/limn_hip.h), and the form composed
from limn's primitives elsewhere, for float64, and where the gradient must itself be differentiable.

Query i of a sequence with L live keys sits at position p(i) = L - t_q + i (the queries are the last of its
positions), query head h reads key head h // (heads / kv_heads), and

    s[i, j] = cap(scale q_i . k_j) - slopes[h] |p(i) - j|,    cap(x) = softcap tanh(x / softcap)
    out_i   = sum_j softmax_j(s[i, j]) v_j                     over the keys j that query i sees.
"""

from __future__ import annotations

import math
from collections.abc import Callable

from limn_amd.seam import CUT_OPS, FLOATS, Node, Op, Tensor, accumulate_in, active_device, custom, float32, float64, grad, int32, promote

ATTEND_FWD, ATTEND_BWD = "attend_fwd", "attend_bwd"
MOST = 2.0**120  # of a scale or a cap: its float32 form, with the constants of the exponential, stays a normal number


def attend(q: Tensor, k: Tensor, v: Tensor, *, causal: bool = False, softcap: float = 0.0, slopes: Tensor | None = None,
           documents: Tensor | None = None, prefix: Tensor | None = None, lengths: Tensor | None = None, scale: float | None = None) -> Tensor:
    """Attention of q (..., heads, t_q, hd) over k (..., kv_heads, t_k, hd) and v (..., kv_heads, t_k, hd_v).

    - `causal`: query i sees the keys at or before its position p(i), and with `prefix` (..., int32) also the
      first prefix keys;
    - `documents` (..., t_k) int32: a query sees only keys of its own position's document; a negative document
      is padding, whose queries see nothing and whose keys are seen by none;
    - `lengths` (..., int32): only the first lengths keys are live, and the queries are the last of them (a
      cache with room for more);
    - `slopes` (heads,) float32: each head takes slopes[h] |p(i) - j| off its scores; it gets no gradient;
    - `softcap`: scores capped at +-softcap by a tanh, before the distance is taken off; 0 for none, else from 2^-120 to
      2^120;
    - `scale`: of the scores, 1 / sqrt(hd) if not given; up to 2^120 either way.

    A query that sees no key gives zeros and passes no gradient. What hidden keys hold changes nothing where the device's
    kernels run (head dims up to 256, not float64); composed of primitives, an infinity or a NaN there
    spoils the rows that do not see it too. The leading dims of q, k and v are equal, as
    are those of documents, prefix and lengths.
    """
    if min(q.ndim, k.ndim, v.ndim) < 3:
        raise ValueError(f"attend needs (..., heads, t, dim) tensors, got {q.shape}, {k.shape}, {v.shape}")
    if not all(t.dtype in FLOATS for t in (q, k, v)):
        raise ValueError(f"attend needs float dtypes, got {q.dtype}, {k.dtype}, {v.dtype}")
    lead, (heads, t_q, hd) = q.shape[:-3], q.shape[-3:]
    kv_heads, t_k = k.shape[-3:-1]
    if k.shape[:-3] != lead or v.shape[:-3] != lead or v.shape[-3] != kv_heads or v.shape[-2] != t_k or k.shape[-1] != hd:
        raise ValueError(f"attend shape mismatch: {q.shape}, {k.shape}, {v.shape}")
    if heads % kv_heads:
        raise ValueError(f"attend: {heads} query heads do not share {kv_heads} key heads evenly")
    if t_q > t_k and (causal or documents is not None or lengths is not None):
        raise ValueError(f"attend: the queries are the last of the keys' positions, got {t_q} queries and {t_k} keys")
    if prefix is not None and not causal:
        raise ValueError("attend: a prefix opens keys that causality hides; the call is not causal")
    softcap = float(softcap)
    if softcap != 0 and not 1 / MOST <= softcap <= MOST:
        raise ValueError(f"attend: softcap must be positive, between 2^-120 and 2^120, or 0 for none, got {softcap}")
    scale = hd**-0.5 if scale is None else float(scale)
    if not abs(scale) <= MOST:
        raise ValueError(f"attend: scale must be finite, between -2^120 and 2^120, got {scale}")
    if slopes is not None and (slopes.shape != (heads,) or slopes.dtype != float32):
        raise ValueError(f"attend: slopes must be ({heads},) float32, got {slopes.shape} {slopes.dtype}")
    for name, t, shape in (("documents", documents, lead + (t_k,)), ("prefix", prefix, lead), ("lengths", lengths, lead)):
        if t is not None and (t.shape != shape or t.dtype != int32):
            raise ValueError(f"attend: {name} must be {shape} int32, got {t.shape} {t.dtype}")
    width = promote(promote(q.dtype, k.dtype), v.dtype)
    q, k, v = (t.cast(width) for t in (q, k, v))
    rules = (slopes, documents, prefix, lengths)
    dev = active_device()
    if width == float64 or max(hd, v.shape[-1]) > 256 or not (dev.has_custom(ATTEND_FWD) and dev.has_custom(ATTEND_BWD)):
        return _composed(q, k, v, *rules, causal, scale, softcap)
    q, k, v = contiguous(q), contiguous(k), contiguous(v)
    given = tuple(contiguous(t) for t in rules if t is not None)
    # which rules are given travels in the params: srcs hold only those
    params = (bool(causal), scale, softcap, tuple(t is not None for t in rules))
    outs = ((width, lead + (heads, t_q, v.shape[-1])), (float32, lead + (heads, t_q, 1)))
    out, lse = custom(ATTEND_FWD, tuple(t.node for t in (q, k, v, *given)), params, outs)

    def backward(g: Tensor):
        if records(q, k, v):
            return through(lambda *qkv: _composed(*qkv, *rules, causal, scale, softcap), (q, k, v), g)
        do = contiguous(g)
        srcs = tuple(t.node for t in (q, k, v, *given)) + (out, lse, do.node)
        return tuple(Tensor.from_node(n) for n in custom(ATTEND_BWD, srcs, params, tuple((t.dtype, t.shape) for t in (q, k, v))))

    return Tensor.from_node(out, (q, k, v), backward)


def contiguous(t: Tensor) -> Tensor:
    """t as row-major bytes: itself when it already is a buffer or a cut, else a copy."""
    if t.node.op is Op.BUFFER or t.node.op in CUT_OPS:
        return t
    return Tensor.from_node(Node(Op.CONTIGUOUS, (t.node,), t.dtype, t.shape), (t,), lambda g: (g,))


def records(*tensors: Tensor) -> bool:
    """Whether an op on these tensors would record a derivation now: inside a backward pass, whether the
    gradient must itself be differentiable."""
    return Tensor.from_node(tensors[0].node, tensors, lambda g: (g,) * len(tensors)).requires_grad


def through(build: Callable[..., Tensor], inputs: tuple[Tensor, ...], g: Tensor) -> tuple[Tensor | None, ...]:
    """The cotangents that g on build(*inputs) gives each input, by limn's own rules for its graph. It is built of a tensor of
    its own for each input: g comes from the inputs too, one input may be another's, or made from it, and none of those paths
    is the input's share here."""
    own = [Tensor.from_node(t.node, (t,), lambda c: (c,)) for t in inputs]
    found = iter(grad((build(*own) * g).sum(), [t for t in own if t.requires_grad], create_graph=True))
    return tuple(next(found) if t.requires_grad else None for t in own)


def _tanh_terms(count: int) -> list[float]:
    """The first coefficients of tanh(z) / z in powers of z^2, from tanh' = 1 - tanh^2."""
    terms = [1.0]
    while len(terms) < count:
        n = len(terms)
        terms.append(-sum(terms[i] * terms[n - 1 - i] for i in range(n)) / (2 * n + 1))
    return terms


def _capped(s: Tensor, softcap: float, wide) -> Tensor:
    """softcap tanh(s / softcap), to a few half steps of itself: 1 - 2 / (1 + e^2z) is off by half steps of 1, however
    small z is, so up to |z| = 1/2 the series takes its place (its first term left out is past the last bit)."""
    inverse = 1.0 / softcap
    z = s * inverse
    near = s.minimum(0.625 * softcap).maximum(-0.625 * softcap)  # no more than the series is good for, where it is not taken
    square = (near * inverse) * (near * inverse)
    terms = _tanh_terms(16 if wide == float64 else 7)
    ratio = square * terms[-1] + terms[-2]
    for c in reversed(terms[:-2]):
        ratio = ratio * square + c
    # past +-40 tanh is +-1 in any float width, and the exponential finite
    far = (1.0 - 2.0 * ((z * 2.0).minimum(80.0).maximum(-80.0).exp() + 1.0).reciprocal()) * softcap
    return ((z * z) <= 0.25).where(near * ratio, far)


def _composed(q: Tensor, k: Tensor, v: Tensor, slopes, documents, prefix, lengths, causal: bool, scale: float, softcap: float) -> Tensor:
    """The same from limn's primitives, the scores and weights at the accumulation width. (A weight of 0
    times a hidden key's infinity or NaN is NaN here; the kernels leave hidden keys out altogether.)"""
    lead, (heads, t_q, hd) = q.shape[:-3], q.shape[-3:]
    kv_heads, t_k = k.shape[-3:-1]
    group, wide, ones = heads // kv_heads, accumulate_in(q.dtype), (1,) * len(lead)
    rows = q.cast(wide).reshape(*lead, kv_heads, group, t_q, hd)
    keys = k.cast(wide).reshape(*lead, kv_heads, 1, t_k, hd)
    values = v.cast(wide).reshape(*lead, kv_heads, 1, t_k, v.shape[-1])
    s = (rows @ keys.transpose(-2, -1)) * scale
    if softcap:
        s = _capped(s, softcap, wide)
    key = Tensor.arange(t_k).reshape(*ones, 1, 1, 1, t_k)
    at = Tensor.arange(t_q).reshape(*ones, 1, 1, t_q, 1)
    length = None if lengths is None else lengths.minimum(t_k).maximum(0).reshape(*lead, 1, 1, 1, 1)
    at = at + (t_k - t_q if length is None else length - t_q)
    if slopes is not None:
        far = (at - key).maximum(key - at).cast(wide)
        s = s - slopes.detach().cast(wide).reshape(*ones, kv_heads, group, 1, 1) * far
    seen = (key < t_k) * (at <= at)  # ones of the pairs' shape: the rules below take pairs away
    if length is not None:
        seen = seen * (key < length)
    if causal:
        reach = key <= at
        if prefix is not None:
            near = key < prefix.reshape(*lead, 1, 1, 1, 1)
            reach = reach + near - reach * near
        seen = seen * reach
    if documents is not None:
        doc = documents.reshape(*lead, 1, 1, 1, t_k)
        # a row's document: the one at its position, picked by a sum over keys (-1 before the first key)
        row_doc = (key.eq(at) * (doc + 1)).sum(axis=-1, keepdim=True) - 1
        seen = seen * row_doc.eq(doc) * (doc >= 0)
    seen = seen.cast(wide)
    low = -1e30 if wide != float64 else -1e300
    s = seen.where(s, low)
    e = seen.where((s - s.max(-1, keepdim=True).detach()).exp(), 0.0)
    total = e.sum(axis=-1, keepdim=True)
    weights = e * (total + total.eq(0.0)).reciprocal()
    return (weights @ values).reshape(*lead, heads, t_q, v.shape[-1]).cast(q.dtype)
