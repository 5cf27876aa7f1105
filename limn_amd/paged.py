"""Attention of new tokens over a paged cache: what a server of a language model runs in every layer of every step.

The cache is a pool of pages that sequences of any length take their places from: key_pages and value_pages (pages,
kv_heads, page, hd), and a table of each sequence's pages. The new tokens of all sequences are packed, one behind another,
whatever each has: a part of a prompt, or the one token that was drawn last. `attend_paged` puts their keys and values in
their places and lets their queries attend, in one CUSTOM kernel "attend_paged" (`limn_hip_attend_paged` of
include/limn_hip.h) where the active device registers it, and composed from limn's primitives elsewhere and for float64.

Row i of the n new tokens of sequence s, which has L = lengths[s] positions with them, sits at position p(i) = L - n + i,
key j of the sequence in place j % page of page table[s, j // page], query head h reads key head h // (heads / kv_heads), and

    s[i, j] = cap(scale q_i . k_j) - slopes[h] (p(i) - j),    cap(x) = softcap tanh(x / softcap)
    out_i   = sum_j softmax_j(s[i, j]) v_j                    over the keys j <= p(i).
"""

from __future__ import annotations

import numpy as np

from limn_amd.attend import MOST, _capped, contiguous, records
from limn_amd.seam import FLOATS, Op, Tensor, accumulate_in, active_device, custom, float32, float64, int32, promote

ATTEND_PAGED = "attend_paged"


def attend_paged(q: Tensor, k: Tensor | None, v: Tensor | None, key_pages: Tensor, value_pages: Tensor, starts: Tensor, lengths: Tensor, table: Tensor,
                 *, softcap: float = 0.0, slopes: Tensor | None = None, scale: float | None = None, heads: int = 0) -> Tensor:
    """Attention of packed new tokens q (tokens, heads, hd) over a paged cache, which takes up their k and v (tokens, kv_heads, hd).

    - `key_pages`, `value_pages` (pages, kv_heads, page, hd): the cache, realized buffers; written in place when the result
      is realized. k and v None: the cache holds the new tokens already.
    - `starts` (sequences + 1,) int32, ascending: sequence s has the rows starts[s] to starts[s + 1]; rows of no sequence give
      zeros and write nothing.
    - `lengths` (sequences,) int32: each one's positions, its new tokens the last of them. A length below the number of
      new tokens leaves the first of them without a position: they see nothing and give zeros.
    - `table` (sequences, table_pages) int32: the pages of each one's positions. Behind the last position it may hold
      anything. Keys of a page number that is not in the cache are not there: nothing is written, and no query sees them.
      Sequences may share pages that none of them writes to in this call; a page that is written stands in the table once.
    - `slopes` (heads,) float32, `softcap`, `scale`: as in `attend`.
    - `heads`: q holds all that is new, each token's queries, keys and values one behind another, (tokens, (heads + 2 kv_heads) hd), as
      a layer's one product gives them; k and v are None then, and nothing is copied apart.

    The result is (tokens, heads, hd). What a key that a query does not see holds, infinities and NaN among them, changes nothing in its row.

    There is no gradient: the call is for answering (under `no_grad`, or on tensors that need none). Nothing else of the batch that
    realizes the result may read the pages, or write what it reads: the order between them is not set.
    """
    together = heads > 0
    if heads < 0 or q.ndim != (2 if together else 3) or key_pages.ndim != 4:
        raise ValueError(f"attend_paged needs (tokens, heads, hd) queries, or all in one with `heads`, and (pages, kv_heads, page, hd) pages, got {q.shape} and {key_pages.shape}")
    (pages, kv_heads, page, hd), tokens = key_pages.shape, q.shape[0]
    heads = heads or q.shape[1]
    if q.shape[1:] != (((heads + 2 * kv_heads) * hd,) if together else (heads, hd)) or value_pages.shape != key_pages.shape:
        raise ValueError(f"attend_paged shape mismatch: {q.shape}, {key_pages.shape}, {value_pages.shape}")
    if heads % kv_heads:
        raise ValueError(f"attend_paged: {heads} query heads do not share {kv_heads} key heads evenly")
    width = key_pages.dtype
    if width not in FLOATS or value_pages.dtype != width:
        raise ValueError(f"attend_paged needs pages of one float dtype, got {key_pages.dtype} and {value_pages.dtype}")
    if any(t.node.op is not Op.BUFFER for t in (key_pages, value_pages)) or key_pages.node.arg is value_pages.node.arg:
        raise ValueError("attend_paged writes its pages in place: they must be two realized buffers")
    if (k is None) != (v is None) or (together and k is not None):
        raise ValueError("attend_paged: new keys and new values go together, and not beside queries that hold them")
    fresh = () if k is None else (k, v)
    if any(t.shape != (tokens, kv_heads, hd) for t in fresh):
        raise ValueError(f"attend_paged: new keys and values must be {(tokens, kv_heads, hd)}, got {k.shape} and {v.shape}")
    if not all(t.dtype in FLOATS and promote(t.dtype, width) == width for t in (q, *fresh)):
        raise ValueError(f"attend_paged: the pages are {width}, got {[t.dtype for t in (q, *fresh)]}")
    if table.ndim != 2:
        raise ValueError(f"attend_paged: the table must be (sequences, table_pages), got {table.shape}")
    sequences = table.shape[0]
    for name, t, shape in (("starts", starts, (sequences + 1,)), ("lengths", lengths, (sequences,)), ("table", table, table.shape)):
        if t.shape != shape or t.dtype != int32:
            raise ValueError(f"attend_paged: {name} must be {shape} int32, got {t.shape} {t.dtype}")
    if slopes is not None and (slopes.shape != (heads,) or slopes.dtype != float32):
        raise ValueError(f"attend_paged: slopes must be ({heads},) float32, got {slopes.shape} {slopes.dtype}")
    softcap = float(softcap)
    if softcap != 0 and not 1 / MOST <= softcap <= MOST:
        raise ValueError(f"attend_paged: softcap must be positive, between 2^-120 and 2^120, or 0 for none, got {softcap}")
    scale = hd**-0.5 if scale is None else float(scale)
    if not abs(scale) <= MOST:
        raise ValueError(f"attend_paged: scale must be finite, between -2^120 and 2^120, got {scale}")
    if records(q, *fresh):
        raise ValueError("attend_paged has no gradient: call it under no_grad, or on tensors that need none")
    q, *fresh = (t.cast(width) for t in (q, *fresh))
    if width == float64 or hd > 256 or not active_device().has_custom(ATTEND_PAGED):
        if together:
            at, kv = heads * hd, kv_heads * hd
            q, *fresh = (t.reshape(tokens, -1, hd) for t in (q[:, :at], q[:, at : at + kv], q[:, at + kv :]))
        return _composed(q, *(fresh or (None, None)), key_pages, value_pages, starts, lengths, table, slopes, scale, softcap)
    if any(isinstance(t.node.arg, np.ndarray) for t in (key_pages, value_pages)):
        raise ValueError("attend_paged writes its pages in place: they must lie on the device")
    given = (starts, lengths, table) + (() if slopes is None else (slopes,))
    srcs = tuple(contiguous(t).node for t in (q, *fresh, key_pages, value_pages, *given))
    (out,) = custom(ATTEND_PAGED, srcs, (scale, softcap, bool(fresh), slopes is not None, together), ((width, (tokens, heads, hd)),))
    return Tensor.from_node(out)


def _composed(q, k, v, key_pages, value_pages, starts, lengths, table, slopes, scale: float, softcap: float) -> Tensor:
    """The same from limn's primitives: the pages are assigned whole, and every token gathers its own keys."""
    (tokens, heads, hd), (pages, kv_heads, page, _) = q.shape, key_pages.shape
    sequences, table_pages = table.shape
    places, wide = table_pages * page, accumulate_in(q.dtype)
    row, seq = Tensor.arange(tokens), Tensor.arange(sequences)
    first, end = starts[:sequences].reshape(1, sequences), starts[1:].reshape(1, sequences)
    mine = (row.reshape(tokens, 1) >= first) * (row.reshape(tokens, 1) < end)  # (tokens, sequences)
    length = lengths.maximum(0).minimum(places).reshape(1, sequences)
    known = mine.sum(-1)
    at = (mine * (length - end)).sum(-1) + row  # p, where known
    # (rows are gathered by numbers that lie inside whatever the tensors hold)
    own = table.gather_rows((mine * seq.reshape(1, sequences)).sum(-1).minimum(sequences - 1))  # (tokens, table_pages)
    inside = (own >= 0) * (own < pages)
    own = inside.where(own, 0)
    pools = []
    for pool, fresh in ((key_pages, k), (value_pages, v)):
        if fresh is not None:
            n = Tensor.arange(table_pages).reshape(1, table_pages)
            of = (at.reshape(tokens, 1) >= (n + 1) * page).sum(-1).reshape(tokens, 1)
            here = n.eq(of) * inside * (known * (at >= 0)).reshape(tokens, 1)  # its page's column
            slot = (here * (own * page + (at.reshape(tokens, 1) - of * page) + 1)).sum(-1) - 1  # -1: none
            cell = Tensor.arange(pages * page).reshape(pages * page, 1)
            writes = cell.eq(slot.reshape(1, tokens))
            writer = (writes * row.reshape(1, tokens)).sum(-1).minimum(tokens - 1)
            new = fresh.reshape(tokens, kv_heads * hd).gather_rows(writer).reshape(pages, page, kv_heads, hd).permute(0, 2, 1, 3)
            hit = writes.sum(-1).reshape(pages, 1, page, 1)
            pool.assign(contiguous(hit.where(new, Tensor.from_node(pool.node))))
        flat = Tensor.from_node(contiguous(Tensor.from_node(pool.node).permute(0, 2, 1, 3)).node).reshape(pages * page, kv_heads * hd)
        where = (own.reshape(tokens, table_pages, 1) * page + Tensor.arange(page).reshape(1, 1, page)).reshape(tokens, places)
        pools.append(flat.gather_rows(where).reshape(tokens, places, kv_heads, 1, hd).permute(0, 2, 3, 1, 4).cast(wide))
    keys, values = pools  # (tokens, kv_heads, 1, places, hd)
    group = heads // kv_heads
    s = (q.cast(wide).reshape(tokens, kv_heads, group, 1, hd) @ keys.transpose(-2, -1)) * scale
    if softcap:
        s = _capped(s, softcap, wide)
    key, p = Tensor.arange(places).reshape(1, places), at.reshape(tokens, 1)
    if slopes is not None:
        far = (p - key).cast(wide).reshape(tokens, 1, 1, 1, places)
        s = s - slopes.detach().cast(wide).reshape(1, kv_heads, group, 1, 1) * far
    there = inside.reshape(tokens, table_pages, 1).expand(tokens, table_pages, page).reshape(tokens, places)
    seen = ((key <= p) * known.reshape(tokens, 1) * there).reshape(tokens, 1, 1, 1, places).cast(wide)
    s = seen.where(s, -1e30 if wide != float64 else -1e300)
    e = seen.where((s - s.max(-1, keepdim=True)).exp(), 0.0)
    total = e.sum(axis=-1, keepdim=True)
    weights = e * (total + total.eq(0.0)).reciprocal()
    values = seen.transpose(-2, -1).where(values, 0.0)  # an infinity or a NaN times a weight of 0 is NaN
    return (weights @ values).reshape(tokens, heads, hd).cast(q.dtype)
