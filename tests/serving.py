"""Inputs for the tests of what answering with a language model takes: a paged cache in any state, logits, 8-bit layers."""

from __future__ import annotations

import numpy as np

from conftest import DTYPES, storage_values

from limn_amd.gpt import mixed, normed
from limn_amd.seam import Tensor, float32, int32


def paged_inputs(seed, dtype="float32", counts=(1,), lengths=(5,), heads=2, kv_heads=None, hd=8, page=4, spare=0, table_pages=None, slopes=False, std=1.0, rows_before=0):
    """Packed tokens, pools whose pages are dealt at random, a table with -1 behind each sequence's pages."""
    rng = np.random.default_rng(seed)
    kv = kv_heads or heads
    stored = lambda *shape, by=1.0: storage_values((rng.standard_normal(shape) * by).astype(np.float32), DTYPES[dtype])  # noqa: E731
    starts = rows_before + np.concatenate([[0], np.cumsum(counts)])
    tokens = int(starts[-1]) + spare
    table_pages = table_pages or max(1, -(-max(lengths) // page))
    pages = len(counts) * table_pages + 2
    deal = rng.permutation(pages)
    table = np.full((len(counts), table_pages), -1, np.int32)
    for s, length in enumerate(lengths):
        n = min(table_pages, -(-length // page))
        table[s, :n] = deal[s * table_pages : s * table_pages + n]
    return dict(q=stored(tokens, heads, hd, by=std), k=stored(tokens, kv, hd), v=stored(tokens, kv, hd), key_pages=stored(pages, kv, page, hd),
                value_pages=stored(pages, kv, page, hd), starts=starts.astype(np.int32), lengths=np.array(lengths, np.int32), table=table,
                slopes=(2.0 ** -np.arange(1, heads + 1)).astype(np.float32) if slopes else None)


def logit_rows(seed, rows, vocab, dtype="float32", spread=2.5):
    rng = np.random.default_rng(seed)
    return storage_values((rng.standard_normal((rows, vocab)) * spread).astype(np.float32), DTYPES[dtype]), rng.random(rows).astype(np.float32), rng


PROMPTS = [[1, 2, 3, 4, 5], [7], [9, 8, 7, 6, 5, 4, 3, 2, 1, 0, 11], [30, 31]]


def whole_logits(model, tokens) -> np.ndarray:
    """The logits (tokens, vocab) of a whole sequence through the model as training runs it."""
    x = model.tok(Tensor(np.array([tokens], dtype=np.int32), dtype=int32))
    if model.slopes is None:
        x = x + model.pos(Tensor.arange(len(tokens)))
    x = x.cast(model.cfg.dtype)
    for block in model.blocks:
        x = block(x, model.slopes, None)
    return mixed(model.head, normed(model.ln, x)).cast(float32).numpy()[0]
