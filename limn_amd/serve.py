"""Answering with the GPT of `limn_amd.gpt`: prompts of any lengths in, the tokens that follow them out.

What the reference's training example does at its end (`examples/train_stories.py`, one prompt, the whole of it through the
model again for every token), as a server does it: the prompts' tokens are packed and go through the model once, in parts of
at most `part` tokens, and leave their keys and values in the pages of a cache; then each step takes one token a sequence over
the cache (`attend_paged`) and draws the next one on the device (`sample`). A step's whole state is in place, tokens,
lengths and what was drawn, so a captured step replays without the host in between. The weights are cast once (`held`), or
brought to 8 bits (`int8_linear`).
"""

from __future__ import annotations

import copy
from collections.abc import Sequence

import numpy as np

from limn_amd.attend import contiguous
from limn_amd.gpt import GPT, Held, Linear, mixed
from limn_amd.int8 import quantize_rows
from limn_amd.sampling import sample
from limn_amd.seam import DType, Tensor, capture, float32, int32, no_grad, realize

PAGE = 64  # positions in a page: a table of 4 bytes for every 64, and half a page without use for each sequence


def held(model: GPT, int8: bool = False) -> GPT:
    """The model for answering: its linear layers cast to the configuration's dtype once, where training casts them at every use;
    with `int8` those of its blocks brought to 8 bits, a scale for each output. The rest is shared with `model`."""
    dtype = model.cfg.dtype

    def kept(layer: Linear, small: bool = False) -> Held:
        bias = None if layer.bias is None else layer.bias.detach().cast(dtype)
        weight, scales = quantize_rows(layer.weight) if small else (layer.weight.detach().cast(dtype), None)
        realize(*(t for t in (weight, bias, scales) if t is not None))
        return Held(weight, bias, scales)

    out = copy.copy(model)
    out.head, out.blocks = kept(model.head), [copy.copy(block) for block in model.blocks]
    for block in out.blocks:
        for name in ("qkv", "proj", "up", "down"):
            setattr(block, name, kept(getattr(block, name), int8))
    return out


class Cache:
    """The keys and values of a model's blocks, in pages, and which sequence has which of them (on the host)."""

    def __init__(self, model: GPT, pages: int, page: int = PAGE, dtype: DType | None = None):
        cfg = model.cfg
        shape = (pages, cfg.key_heads, page, cfg.dim // cfg.heads)
        self.page = page
        self.free = list(range(pages))[::-1]
        zero = Tensor.zeros((1, 1, 1, 1), dtype=dtype or cfg.dtype).expand(*shape)
        self.layers = [(contiguous(zero), contiguous(zero)) for _ in model.blocks]  # filled on the device
        realize(*(pool for pools in self.layers for pool in pools))
        self.tables: dict[int, list[int]] = {}

    def reserve(self, sequence: int, length: int) -> None:
        """Pages for the first `length` positions of a sequence, those it has first."""
        more = -(-length // self.page) - len(self.tables.get(sequence, ()))
        if more > len(self.free):
            raise ValueError(f"Cache: {length} positions of sequence {sequence} take {more} more pages, {len(self.free)} are free")
        self.tables.setdefault(sequence, []).extend(self.free.pop() for _ in range(more))

    def drop(self, sequence: int) -> None:
        """The sequence is over: its pages are free."""
        self.free.extend(self.tables.pop(sequence)[::-1])

    def table(self, sequences: Sequence[int]) -> Tensor:
        """The sequences' pages (sequences, the most that one has) int32, -1 behind the last."""
        rows = [self.tables[s] for s in sequences]
        if not rows:
            raise ValueError("Cache: a table is of at least one sequence")
        out = np.full((len(rows), max(1, *(len(r) for r in rows))), -1, dtype=np.int32)
        for to, row in zip(out, rows):
            to[: len(row)] = row
        return Tensor(out, dtype=int32)


def in_vocabulary(name: str, model: GPT, prompts: Sequence[Sequence[int]]) -> None:
    if any(not 0 <= t < model.cfg.vocab for p in prompts for t in p):
        raise ValueError(f"{name}: tokens must lie in [0, {model.cfg.vocab})")


def prefill(model: GPT, cache: Cache, sequences: Sequence[int], prompts: Sequence[Sequence[int]], table: Tensor, part: int = 4096) -> Tensor:
    """The prompts through the model, their keys and values into the cache: the logits (sequences, vocab) behind each one's last token.
    Parts hold at most `part` tokens and end anywhere; each sequence goes on in the next one where it ended. For answering: under
    `no_grad`, with pages reserved for the prompts, at least one token each. The device compiles the model's small kernels for every number of
    tokens that a part has, and keeps them; the prompts' last part has what is left."""
    if part < 1 or len(prompts) == 0 or len(sequences) != len(prompts) or any(len(p) == 0 for p in prompts):
        raise ValueError(f"prefill needs a part of at least 1 and a prompt of at least one token for each sequence, got {part}, {len(sequences)} sequences and prompts of {[len(p) for p in prompts]}")
    longest = max(len(p) for p in prompts)
    in_vocabulary("prefill", model, prompts)
    if not model.cfg.distance and longest > model.cfg.ctx:
        raise ValueError(f"prefill: learned positions end at {model.cfg.ctx}, a prompt of {longest} tokens does not fit")
    short = [s for s, p in zip(sequences, prompts) if len(cache.tables.get(s, ())) * cache.page < len(p)]
    if short:
        raise ValueError(f"prefill: the prompts of the sequences {short} have more positions than pages are reserved for")
    if table.ndim != 2 or table.shape[0] != len(prompts) or table.shape[1] * cache.page < longest:
        raise ValueError(f"prefill: a table of {table.shape} does not hold {len(prompts)} prompts of up to {longest} tokens in pages of {cache.page}")
    todo, done = [list(p) for p in prompts], [0] * len(prompts)
    logits: Tensor | None = None
    while any(at < len(p) for at, p in zip(done, todo)):
        tokens, positions, starts, ends, room = [], [], [0], [], part
        for s, p in enumerate(todo):
            take = min(room, len(p) - done[s])
            tokens += p[done[s] : done[s] + take]
            positions += range(done[s], done[s] + take)
            done[s] += take
            room -= take
            starts.append(len(tokens))
            ends.append(len(tokens) - 1 if take and done[s] == len(p) else -1)
        numbers = lambda t: Tensor(np.array(t, dtype=np.int32), dtype=int32)  # noqa: E731
        rows = model.extend(numbers(tokens), numbers(positions), cache.layers, (numbers(starts), numbers(done), table))
        end = numbers(ends)
        here = mixed(model.head, rows.gather_rows(end.maximum(0)))
        logits = here if logits is None else (end.reshape(-1, 1) >= 0).where(here, logits)
        realize(logits)
    return logits


def generate(model: GPT, prompts: Sequence[Sequence[int]], count: int, *, temperature: float = 1.0, top_k: int = 0, top_p: float = 1.0, min_p: float = 0.0,
             seed: int = 0, int8: bool = False, page: int = PAGE, part: int = 4096, captured: bool = True) -> tuple[np.ndarray, np.ndarray]:
    """`count` tokens behind each prompt: (prompts, count) int32, and the logarithms float32 of their shares (see `sample`).

    Prompts are token numbers, at least one; with learned positions a prompt and its answer fit into the model's context.

    `int8` halves the blocks' weights in memory; it is no faster for one token a sequence: each product needs its rows rounded first. (64
    sequences, us a step held and in 8 bits: 8 layers 512 wide 864 and 988, 4 layers 1024 wide 575 and 608, 2048 716 and 735, 4096 1160 and 1164.)
    """
    cfg, n = model.cfg, len(prompts)
    if n == 0 or count < 1 or part < 1 or page < 1 or any(len(p) == 0 for p in prompts):
        raise ValueError("generate needs prompts of at least one token, and a count, part and page of at least 1")
    in_vocabulary("generate", model, prompts)
    if not cfg.distance and max(len(p) for p in prompts) + count > cfg.ctx + 1:
        raise ValueError(f"generate: learned positions end at {cfg.ctx}, a prompt of {max(len(p) for p in prompts)} tokens and {count} more do not fit")
    rules = dict(temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
    lengths = [len(p) + count - 1 for p in prompts]  # the last token drawn is not read
    with no_grad():
        model = held(model, int8)
        cache = Cache(model, sum(-(-length // page) for length in lengths), page)
        for s, length in enumerate(lengths):
            cache.reserve(s, length)
        table, starts = cache.table(range(n)), Tensor(np.arange(n + 1, dtype=np.int32), dtype=int32)
        uniforms = Tensor(np.random.default_rng(seed).random((count, n), dtype=np.float32))
        now = Tensor(np.array([len(p) for p in prompts], dtype=np.int32), dtype=int32)
        at, column = Tensor.zeros((1,), dtype=int32), Tensor(np.arange(count, dtype=np.int32).reshape(count, 1), dtype=int32)
        tokens, shares = Tensor.zeros((n,), dtype=int32), Tensor.zeros((count, n), dtype=float32)
        answers = Tensor.zeros((count, n), dtype=int32)

        def draw(logits: Tensor) -> tuple[Tensor, ...]:
            """The next tokens, written down in the row `at`."""
            drawn, share = sample(logits, uniforms.gather_rows(at).reshape(n), **rules)
            here = column.eq(at)
            state = (answers.assign(here.where(drawn.reshape(1, n), answers.detach())), shares.assign(here.where(share.reshape(1, n), shares.detach())),
                     at.assign(at.detach() + 1), tokens.assign(drawn.maximum(0)))
            realize(*state)
            return state

        def step() -> tuple[Tensor, ...]:
            length = now.detach() + 1
            rows = model.extend(tokens.detach(), now.detach(), cache.layers, (starts, length, table))
            logits = mixed(model.head, rows)
            now.assign(length)
            realize(logits, now)
            return draw(logits)

        draw(prefill(model, cache, range(n), prompts, table, part))
        run = capture(step) if captured else step
        for _ in range(count - 1):
            run()
        return answers.numpy().T.copy(), shares.numpy().T.copy()
