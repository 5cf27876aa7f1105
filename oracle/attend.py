"""Attention with score rules and the head's cross entropy from their definitions, in float64 (TEST INFRASTRUCTURE
ONLY; see oracle/__init__.py), each with a bound on what rounding may change of every result.

`attend` returns the forward and the gradients of limn_hip_attend_fwd / limn_hip_attend_bwd, one head at a time,
hidden pairs left out of every sum (a hidden row's infinities and NaN are never multiplied).

The bounds are first-order bounds on the kernels' roundings, with u the half
step of the storage type (torch.finfo(t).eps / 2) and f that of float32, 2^-24:
  - a score is a float32 sum of hd products: off by at most e = (hd + 8) f scale sum|q||k|, plus f times the
    distance term, plus 4 f |s|, and where it is capped 16 f |cap tanh(x / cap)| more: near 0 a polynomial of relative
    error 2^-25.9 and two products (with their constants, 7 f); past |x / cap| = 1/2, where tanh is .46, 1 - 2 w with
    w = 1 / (1 + e) off by 3.5 f absolutely (an exponential and a reciprocal of 2 f each, w <= .27), the exponent's two
    constants and products by 4 f relatively (times 2z / sinh 2z <= .85), the product with the cap by 3 f. Half
    widths under caps up to 64 take the latter alone, w up to 1: 8 f of the cap;
  - a probability is then off by a factor of at most 1 + 2 max_j e + 8 f (its own and the sum's scores, one
    exponential, the sum), and by u more where it is rounded to be an operand (half widths);
  - a sum of n terms in float32 adds (n + 8) f times the sum of its terms' magnitudes;
  - delta = rowsum(dout * out) takes out as stored: off by u rowsum|dout||out|, and out's own error;
  - a probability below the least normal float32 number, 2^-126, may be 0 (the exponential gives no subnormal
    numbers): it is off by up to that number, which no relative bound covers;
  - a float16 operand below 2^-14, the least normal one, is off by up to 2^-25 absolutely: the kernels multiply
    the forward's weights by 2^7 and the dV product's by 2^14 first, so 2^-32 and 2^-39 of a weight; the
    score gradients, scale apart, by 2^8, so 2^-33;
  - a float32 operand goes as three bfloat16 numbers, each rounded from what the ones before leave: 24 bits, or as
    many as there are above bfloat16's least step, 2^-133, so it is off by up to 2^-134 and a product by that
    times the other operand (a weight by less than 2^-126, which it already is);
  - every stored result rounds once more: u times its value, and up to the least number of its type where the
    value is below it (float32 and bfloat16 sums and stores may take subnormal numbers as 0).
"""

from __future__ import annotations

import numpy as np

HALF_STEP = {"float32": 2.0**-24, "float16": 2.0**-11, "bfloat16": 2.0**-8}
LEAST = {"float32": 2.0**-126, "float16": 2.0**-24, "bfloat16": 2.0**-126}
F, TINY = 2.0**-24, 2.0**-126


def seen_pairs(t_q, t_k, length, causal, prefix, documents):
    """(t_q, t_k) truth values, and the queries' positions."""
    at = np.arange(length - t_q, length)[:, None]
    key = np.arange(t_k)[None, :]
    seen = np.broadcast_to(key < length, (t_q, t_k)).copy()
    if causal:
        seen &= (key <= at) | (key < (0 if prefix is None else prefix))
    if documents is not None:
        rows = np.where(at >= 0, documents[np.clip(at, 0, t_k - 1)], -1)
        seen &= (rows == documents[None, :]) & (rows >= 0)
    return seen, at


def _product(a, b):
    """a @ b over the pairs where a is not zero: a zero times an infinity or a NaN is left out."""
    with np.errstate(invalid="ignore", over="ignore"):
        if np.isfinite(b).all():
            return a @ b
        return np.stack([(np.where(row[:, None] != 0, row[:, None] * b, 0.0)).sum(0) for row in a])


def attend(q, k, v, *, causal=False, softcap=0.0, slopes=None, documents=None, prefix=None, lengths=None, scale=None, dout=None, dtype="float32"):
    """out, lse (and with dout dq, dk, dv) of (batch, heads, t, dim) arrays, and each one's bound: a dict of
    (value, bound) pairs."""
    batch, heads, t_q, hd = q.shape
    kv_heads, t_k = k.shape[1:3]
    group, hd_v = heads // kv_heads, v.shape[-1]
    scale = hd**-0.5 if scale is None else scale
    u, least = HALF_STEP[dtype], LEAST[dtype]
    operand = 0.0 if dtype == "float32" else u
    small = 1.0 if dtype == "float16" else 0.0
    lost = 2.0**-134 if dtype == "float32" else 0.0
    q, k, v = (np.asarray(x, dtype=np.float64) for x in (q, k, v))
    shapes = dict(out=q.shape[:-1] + (hd_v,), lse=q.shape[:-1], dq=q.shape, dk=k.shape, dv=v.shape)
    got = {n: np.zeros(s) for n, s in shapes.items()}
    off = {n: np.zeros(s) for n, s in shapes.items()}
    fine = lambda x: np.where(np.isfinite(x), np.abs(x), 0.0)  # noqa: E731
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        for b in range(batch):
            length = t_k if lengths is None else int(np.clip(lengths[b], 0, t_k))
            seen, at = seen_pairs(t_q, t_k, length, causal, None if prefix is None else int(prefix[b]), None if documents is None else documents[b])
            far = np.abs(at - np.arange(t_k)[None, :]).astype(np.float64)
            for h in range(heads):
                Q, K, V = q[b, h], k[b, h // group], v[b, h // group]
                x = np.where(seen, Q @ K.T, 0.0) * scale
                e = (hd + 8) * F * abs(scale) * (fine(Q) @ fine(K).T) + 4 * F * np.abs(x) + lost * abs(scale) * (fine(Q).sum(1)[:, None] + fine(K).sum(1)[None, :])
                bent = 1.0
                s = x
                if softcap:
                    t = np.tanh(x / softcap)
                    s, bent = softcap * t, 1 - t * t
                    e = e + (8 * F * softcap if dtype != "float32" and softcap <= 64 else 16 * F * np.abs(s))
                if slopes is not None:
                    s = s - slopes[h] * far
                    e = e + 4 * F * slopes[h] * far + 4 * F * np.abs(s)
                s = np.where(seen, s, -np.inf)
                top = np.max(s, axis=1, keepdims=True, initial=-np.inf)
                base = np.where(np.isneginf(top), 0.0, top)
                w = np.where(seen, np.exp(s - base), 0.0)
                total = w.sum(1, keepdims=True)
                p = np.where(total == 0, 0.0, w / np.where(total == 0, 1.0, total))
                n = seen.sum(1, keepdims=True)
                rel = 2 * np.max(np.where(seen, e, 0.0), axis=1, keepdims=True) + (n + 16) * F
                got["out"][b, h] = _product(p, V)
                off["out"][b, h] = (rel + operand) * (p @ fine(V)) + (TINY + small * 2.0**-32) * (seen @ fine(V)) + u * fine(got["out"][b, h]) + least
                got["lse"][b, h] = np.where(total == 0, -np.inf, base + np.log(total))[:, 0]
                off["lse"][b, h] = rel[:, 0] + 4 * F * fine(got["lse"][b, h])
                if dout is None:
                    continue
                G = np.asarray(dout[b, h], dtype=np.float64)
                O = got["out"][b, h]
                dp = np.where(seen, G @ V.T, 0.0)
                delta = (np.where(n > 0, G, 0.0) * O).sum(1, keepdims=True)
                ddelta = (fine(G) * (off["out"][b, h] + hd_v * F * fine(O))).sum(1, keepdims=True)
                ddp = (hd_v + 8) * F * (fine(G) @ fine(V).T) + lost * (fine(G).sum(1)[:, None] + fine(V).sum(1)[None, :])
                ds = np.where(seen, p * (dp - delta) * scale * bent, 0.0)
                size = np.where(seen, p * abs(scale) * bent, 0.0)
                dds = np.abs(ds) * (rel + 8 * F + operand) + size * (ddelta + ddp) + np.where(seen, TINY * (1 + fine(dp - delta) * abs(scale)) + small * 2.0**-33 * abs(scale), 0.0)
                if softcap:  # 1 - tanh^2, off by twice the tanh's own 4 f and by the score's
                    dds = dds + np.where(seen, np.abs(p * (dp - delta)) * abs(scale), 0.0) * (16 * F + 2 * e / softcap)
                kv = h // group
                got["dq"][b, h] = _product(ds, K)
                off["dq"][b, h] = dds @ fine(K) + lost * np.abs(ds).sum(1, keepdims=True) + (n + 8) * F * (np.abs(ds) @ fine(K)) + u * fine(got["dq"][b, h]) + least
                m = seen.sum(0)[:, None] * group
                got["dk"][b, kv] += _product(ds.T, Q)
                off["dk"][b, kv] += dds.T @ fine(Q) + lost * np.abs(ds).sum(0)[:, None] + (m + 8) * F * (np.abs(ds).T @ fine(Q))
                got["dv"][b, kv] += _product(p.T, G)
                off["dv"][b, kv] += (p * (rel + operand) + (TINY + small * 2.0**-39) * seen).T @ fine(G) + (m + 8) * F * (p.T @ fine(G))
    for name in ("dk", "dv"):
        off[name] += u * fine(got[name]) + least
    names = ("out", "lse") if dout is None else ("out", "lse", "dq", "dk", "dv")
    return {n: (got[n], off[n]) for n in names}


def xent(x, w, targets, g=None, dtype="float32"):
    """loss, lse of rows x under the head w (and with cotangents g of the losses dx and dw), and each one's
    bound: a dict of (value, bound) pairs."""
    x, w = np.asarray(x, dtype=np.float64), np.asarray(w, dtype=np.float64)
    rows, width = x.shape
    vocab = w.shape[0]
    u, least = HALF_STEP[dtype], LEAST[dtype]
    operand = 0.0 if dtype == "float32" else u
    live = (targets >= 0) & (targets < vocab)
    at = np.where(live, targets, 0)
    xs = np.where(live[:, None], x, 0.0)
    with np.errstate(invalid="ignore", over="ignore"):
        z = x @ w.T
        top = z.max(1, keepdims=True)
        lse = (top + np.log(np.exp(z - top).sum(1, keepdims=True)))[:, 0]
        # a float32 operand is the sum of three bfloat16 numbers, each rounded from what the ones before leave: 24 bits,
        # or as many as there are above bfloat16's least step, 2^-133, so the operand is off by up to half of that and a
        # product by 2^-134 times the other operand
        lost = 2.0**-134 if dtype == "float32" else 0.0
        lost_z = lost * (np.abs(x).sum(1) + np.abs(w).sum(1).max())
        e = ((width + 8) * F * (np.abs(x) @ np.abs(w).T)).max(1) + 4 * F * np.abs(z).max(1) + lost_z
        rel = 2 * e + (vocab**0.5 + 32) * F  # the sum of positive terms runs in many short chains
        loss = np.where(live, lse - z[np.arange(rows), at], 0.0)
    out = dict(loss=(loss, np.where(live, rel + e + 8 * F * np.abs(lse), 0.0)), lse=(lse, rel + 8 * F * np.abs(lse)))
    if g is None:
        return out
    g = np.where(live, np.asarray(g, dtype=np.float64), 0.0)[:, None]
    zs = np.where(live[:, None], z, 0.0)
    p = np.where(live[:, None], np.exp(zs - np.where(live, lse, 0.0)[:, None]), 0.0)
    hit = np.zeros_like(p)
    hit[np.arange(rows), at] = live
    dz = g * (p - hit)
    # p's own error, the difference's rounding, and dz rounded to be an operand
    ddz = np.abs(g) * (p * np.where(live, rel + e + 8 * F * np.abs(lse) + 8 * F, 0.0)[:, None] + TINY) + np.abs(dz) * (operand + 4 * F)
    dx, dw = dz @ w, dz.T @ xs
    dxo = ddz @ np.abs(w) + (vocab + 8) * F * (np.abs(dz) @ np.abs(w)) + u * np.abs(dx) + least
    dwo = ddz.T @ np.abs(xs) + (rows + 8) * F * (np.abs(dz).T @ np.abs(xs)) + u * np.abs(dw) + least
    # a dz, or a float32 one's last part, below its type's least normal number is off by a part of that number; float16's
    # are multiplied by a power of two that brings the largest |g| to 2^14 or more, so 2^-25 2^-14 of that is left
    tiny = 2.0**-39 * np.abs(g).max(initial=0.0) + TINY if dtype == "float16" else TINY
    dxo = dxo + tiny * np.abs(w).sum(0) + lost * np.abs(dz).sum(1, keepdims=True)
    dwo = dwo + tiny * np.abs(xs).sum(0) + lost * np.abs(dz).sum(0)[:, None]
    out.update(dx=(dx, dxo), dw=(dw, dwo))
    return out


def within(got, value, bound, what=""):
    """got equals value up to bound, and its infinities and NaN are value's."""
    got, value = np.asarray(got, dtype=np.float64), np.asarray(value, dtype=np.float64)
    assert got.shape == value.shape, (what, got.shape, value.shape)
    fine = np.isfinite(value)
    same = np.where(fine, np.isfinite(got), (got == value) | (np.isnan(got) & np.isnan(value)))
    assert same.all(), f"{what}: {np.count_nonzero(~same)} of {same.size} are finite on one side only, first at {np.argwhere(~same)[0]}"
    far = np.where(fine, np.abs(np.where(fine, got, 0.0) - np.where(fine, value, 0.0)) - np.broadcast_to(bound, value.shape), 0.0)
    worst = np.unravel_index(np.argmax(far), far.shape) if far.size else ()
    assert not far.size or far[worst] <= 0, f"{what}: off by {abs(got[worst] - value[worst]):.3g} at {worst} (value {value[worst]:.3g}), bound {np.broadcast_to(bound, value.shape)[worst]:.3g}"
