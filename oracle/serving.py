"""Attention over a paged cache, sampling and 8-bit linear layers from their definitions, in float64 (TEST INFRASTRUCTURE ONLY; see
oracle/__init__.py), with a bound on what rounding may change of every computed number.

The bounds are first-order bounds on the kernels' roundings, as oracle/attend.py derives them, with u the half step of the
storage type and F that of float32:
  - paged: those of oracle/attend.py's forward: a score is a float32 sum of hd products, a cap adds 16 F of its result (or 8 F of
    the cap, for half widths under caps up to 64), a weight that is an operand is rounded to the half width, and so on;
  - sample: weights are 64-bit numbers, masses whole multiples of 2^-bits of the largest weight, each rounded by half of that: a
    mass of n tokens is off by n 2^-bits / 2, where the kept mass is at least 1, and the logarithm of a share by that and float32's
    half step of itself. Tokens are compared as they are: two borders as close as that to u times the mass, or to top_p's,
    would be a row in some millions;
  - int8: the sums are exact; (float) of one, its product with each scale and the sum with the bias round once each: 3 F of the
    product, F of the sum, then u of the result. x / s rounds once before it is rounded to a whole number, here as in the kernels
    (float32), so the whole numbers are the same.
"""

from __future__ import annotations

import numpy as np

from oracle.attend import F, HALF_STEP, LEAST, TINY, _product


def same_kind(got, want):
    """got with NaN where want says NaN and got has an infinity: what an infinite value gives under a weight that may be 0."""
    return np.where(np.isnan(want) & np.isinf(got), np.nan, got)


PAST = {"float32": 2.0**128, "bfloat16": 2.0**128 * (1 - 2.0**-9), "float16": 65520.0}  # from here on a number rounds to infinity


def paged(q, k, v, key_pages, value_pages, starts, lengths, table, *, softcap=0.0, slopes=None, scale=None, dtype="float32"):
    """out (tokens, heads, hd) with its bound, and the pages as the call leaves them: (out, bound), key_pages, value_pages. An infinity
    in out is given as NaN where one of the infinite values that make it has a weight which may come to 0 as an operand or beside a
    larger score of another part, below 2^-31 for float16 (2^-25, half its least number, and 2^7 that weights are multiplied by, and
    one bit for the weight's error), 2^-124 else (float32's least normal number and two bits): 0 times an infinity is NaN, so a kernel may
    give either there (see `same_kind`)."""
    tokens, heads, hd = q.shape
    pages, kv_heads, page, _ = key_pages.shape
    scale = hd**-0.5 if scale is None else scale
    group, u, least = heads // kv_heads, HALF_STEP[dtype], LEAST[dtype]
    operand, small, lost = (0.0 if dtype == "float32" else u), (1.0 if dtype == "float16" else 0.0), (2.0**-134 if dtype == "float32" else 0.0)
    keys, values = key_pages.copy(), value_pages.copy()
    live = [(max(0, min(int(starts[s]), tokens)), max(0, min(int(starts[s + 1]), tokens)), int(np.clip(lengths[s], 0, table.shape[1] * page))) for s in range(len(lengths))]
    place = lambda s, j: (table[s, j // page], j % page) if 0 <= table[s, j // page] < pages else None  # noqa: E731
    if k is not None:
        for s, (b, e, length) in enumerate(live):
            for r in range(b, e):
                p = length - e + r
                at = place(s, p) if p >= 0 else None
                if at is not None:
                    keys[at[0], :, at[1]], values[at[0], :, at[1]] = k[r], v[r]
    out, off = np.zeros(q.shape), np.zeros(q.shape)
    fine = lambda x: np.where(np.isfinite(x), np.abs(x), 0.0)  # noqa: E731
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        for s, (b, e, length) in enumerate(live):
            if e <= b:
                continue
            at = np.arange(length - e + b, length)[:, None]
            where = [place(s, j) for j in range(length)]
            there = np.array([w is not None for w in where], bool)
            K, V = (np.zeros((length, kv_heads, hd)) for _ in range(2))
            for j, w in enumerate(where):
                if w is not None:
                    K[j], V[j] = keys[w[0], :, w[1]], values[w[0], :, w[1]]
            seen = (np.arange(length)[None, :] <= at) & there[None, :]
            far = np.maximum(at - np.arange(length)[None, :], 0).astype(np.float64)
            n = seen.sum(1, keepdims=True)
            for h in range(heads):
                Q, Kh, Vh = np.asarray(q[b:e, h], np.float64), K[:, h // group], V[:, h // group]
                x = np.where(seen, Q @ Kh.T, 0.0) * scale
                err = (hd + 8) * F * abs(scale) * (fine(Q) @ fine(Kh).T) + 4 * F * np.abs(x) + lost * abs(scale) * (fine(Q).sum(1)[:, None] + fine(Kh).sum(1)[None, :])
                if softcap:
                    x = softcap * np.tanh(x / softcap)
                    err = err + 16 * F * np.abs(x) + (8 * F * softcap if dtype != "float32" and softcap <= 64 else 0.0)
                if slopes is not None:
                    x = x - slopes[h] * far
                    err = err + 4 * F * abs(slopes[h]) * far + 4 * F * np.abs(x)
                x = np.where(seen, x, -np.inf)
                top = np.max(x, axis=1, keepdims=True, initial=-np.inf)
                w = np.where(seen, np.exp(x - np.where(np.isneginf(top), 0.0, top)), 0.0)
                total = w.sum(1, keepdims=True)
                p = np.where(total == 0, 0.0, w / np.where(total == 0, 1.0, total))
                rel = 2 * np.max(np.where(seen, err, 0.0), axis=1, keepdims=True, initial=0.0) + (n + 16) * F
                out[b:e, h] = _product(p, Vh)
                faint = seen & (w < (2.0**-31 if dtype == "float16" else 2.0**-124) * np.maximum(total, 1.0))
                out[b:e, h] = np.where(np.isinf(out[b:e, h]) & (faint.astype(float) @ (~np.isfinite(Vh)) > 0), np.nan, out[b:e, h])
                off[b:e, h] = (rel + operand) * (p @ fine(Vh)) + (TINY + small * 2.0**-32) * (seen @ fine(Vh)) + u * fine(out[b:e, h]) + least
    return (out, off), keys, values


def sample(logits, uniforms, temperature=None, top_k=None, top_p=None, min_p=None):
    """tokens, and logprobs with their bound: (rows,) arrays."""
    rows, vocab = logits.shape
    tokens, logs = np.full(rows, -1, np.int32), np.full(rows, -np.inf)
    bits = min(52, 62 - int(np.ceil(np.log2(vocab))))
    for r in range(rows):
        x = np.asarray(logits[r], np.float64)
        x = np.where(np.isnan(x), -np.inf, x) + 0.0
        if not (x > -np.inf).any():
            continue
        order = np.argsort(-x, kind="stable")
        t = 1.0 if temperature is None else float(temperature[r])
        if not t > 0:
            tokens[r], logs[r] = order[0], 0.0
            continue
        with np.errstate(invalid="ignore", over="ignore"):
            w = np.where(x[order] == x[order[0]], 1.0, np.exp((x[order] - x[order[0]]) / t))
        end = vocab
        if top_k is not None and 0 < top_k[r] < vocab:
            end = int(top_k[r])
        if top_p is not None and top_p[r] < 1:
            before = np.concatenate([[0.0], np.cumsum(w[:end])[:-1]])
            end = max(1, int((before < float(top_p[r]) * w[:end].sum()).sum()))
        if min_p is not None and min_p[r] > 0:
            end = min(end, max(1, int((w >= float(min_p[r])).sum())))
        mass = np.cumsum(w[:end])
        u = float(uniforms[r])
        u = min(max(u, 0.0), 1.0) if u == u else 1.0
        at = min(int(np.searchsorted(mass, u * mass[-1], side="right")), int((w[:end] > 2.0 ** -(bits + 1)).sum()) - 1)
        tokens[r], logs[r] = order[at], np.log(w[at]) - np.log(mass[-1])
    return tokens, (logs, np.where(np.isfinite(logs), F * np.abs(logs) + vocab * 2.0**-bits + 2.0**-46, 0.0))


def quantized(x):
    """x (rows, width) as whole numbers and scales, in float32 arithmetic as the operator is defined."""
    x = np.asarray(x, np.float32)
    odd = ~np.isfinite(x).all(1)
    with np.errstate(invalid="ignore"):
        scales = np.maximum(np.abs(np.where(odd[:, None], 0, x)).max(1) / np.float32(127), np.float32(2.0**-126))
        values = np.where(odd[:, None], 0, np.rint(x / scales[:, None]))
    return values.astype(np.int8), np.where(odd, np.float32(np.nan), scales).astype(np.float32)


def int8_linear(x, weight, scales, bias=None, dtype="float32"):
    """The layer's output and its bound."""
    values, s = quantized(x)
    whole = values.astype(np.int64) @ weight.astype(np.int64).T
    y = whole * scales.astype(np.float64) * s.astype(np.float64)[:, None]
    off = 3 * F * np.abs(y) + TINY
    if bias is not None:
        y = y + np.asarray(bias, np.float64)
        off = off + F * np.abs(y)
    off = off + HALF_STEP[dtype] * np.abs(y) + LEAST[dtype]
    return np.where(np.abs(y) >= PAST[dtype], np.copysign(np.inf, y), y), off
