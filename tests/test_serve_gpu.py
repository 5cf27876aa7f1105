"""Answering with the GPT on the MI355X: paged attention, sampling and 8-bit layers together, captured and replayed, against
the numpy oracle's whole model on whole sequences."""

from __future__ import annotations

from dataclasses import replace

import numpy as np
import pytest

from limn_amd.gpt import GPT, GPTConfig, make_trainer, synthetic_batch
from limn_amd.seam import bfloat16, float16, float32, no_grad, set_seed
from limn_amd.seam import device as limn_device
from limn_amd.serve import Cache, generate, held, prefill
from oracle.numpy_device import NumpyDevice
from serving import whole_logits

pytestmark = pytest.mark.gpu

SMALL = GPTConfig(vocab=64, ctx=192, dim=128, layers=2, heads=2, batch=2, dtype=bfloat16)
EVERY = replace(SMALL, kv_heads=1, softcap=4.0, distance=True)
WIDE = replace(EVERY, dim=256, heads=2, kv_heads=2, vocab=1500)  # heads of 128, a vocabulary of more than a sorted row
PROMPTS = [list(range(5)), [7], [i * 7 % 64 for i in range(130)], [i * 5 % 64 for i in range(64)], [i * 3 % 64 for i in range(63)]]

# Off by this part of the largest logit. float32: as on the CPU, with sums of up to 512 terms in chains of 64. Halves: of the
# two layers some 10 values each are rounded one after another (bf16 by 2^-8 at most of the value) by the device and, at other
# places, by the oracle, which rounds every node: 40 * 2^-8 if all went one way, and 3e-2 as they go both ways (40 of them 6 2^-8).
# 8-bit inputs: an input at the border of two whole numbers goes the other way, by 1 of 127, in each of the 8 layers.
WORST = {bfloat16: 3e-2, float16: 6e-3, float32: 2.3e-3}
WORST_INT8 = 8 / 127


def model_of(cfg: GPTConfig) -> GPT:
    set_seed(5)
    return GPT(cfg)


def logits_of(cfg: GPTConfig, small: bool, sequences) -> list[np.ndarray]:
    """The oracle's, (tokens, vocab) for each sequence."""
    limn_device.active_device = NumpyDevice()
    with no_grad():
        kept = held(model_of(cfg), small)
        return [whole_logits(kept, s).astype(np.float64) for s in sequences]


@pytest.mark.parametrize("small", [False, True], ids=["held", "int8"])
@pytest.mark.parametrize("cfg", [SMALL, replace(EVERY, dtype=float16), WIDE, replace(SMALL, dtype=float32), replace(WIDE, dtype=float32)],
                         ids=["bf16", "every-f16", "wide-bf16", "f32", "wide-f32"])
@pytest.mark.parametrize("part, page", [(4096, 64), (50, 16)])
def test_prompts_match_the_oracles_whole_model(hipdev, cfg, small, part, page):
    limn_device.active_device = hipdev
    with no_grad():
        model = held(model_of(cfg), small)
        cache = Cache(model, 40, page)
        for s, p in enumerate(PROMPTS):
            cache.reserve(s, len(p))
        got = prefill(model, cache, range(len(PROMPTS)), PROMPTS, cache.table(range(len(PROMPTS))), part).numpy().astype(np.float64)
    want = np.stack([rows[-1] for rows in logits_of(cfg, small, PROMPTS)])
    assert np.abs(got - want).max() <= (WORST[cfg.dtype] + small * WORST_INT8) * np.abs(want).max()


@pytest.mark.parametrize("small", [False, True], ids=["held", "int8"])
@pytest.mark.parametrize("cfg", [SMALL, WIDE, replace(EVERY, dtype=float32)], ids=["bf16", "wide-bf16", "every-f32"])
def test_answers_match_the_oracles_whole_model(hipdev, cfg, small):
    """Forty steps, most of them replayed: each token's share is the one that the whole model on the whole sequence gives it."""
    limn_device.active_device = hipdev
    answers, shares = generate(model_of(cfg), PROMPTS, 40, seed=3, int8=small, temperature=0.8)
    assert ((answers >= 0) & (answers < cfg.vocab)).all()
    whole = logits_of(cfg, small, [[*p, *a] for p, a in zip(PROMPTS, answers)])
    worst = WORST[cfg.dtype] + small * WORST_INT8
    for p, answer, share, rows in zip(PROMPTS, answers, shares, whole):
        rows = rows[len(p) - 1 : -1]
        off = worst * np.abs(rows).max()
        warm = rows / 0.8
        want = np.take_along_axis(warm, answer[:, None], 1)[:, 0] - np.log(np.exp(warm).sum(1))
        assert np.abs(share - want).max() <= 2 * off / 0.8


@pytest.mark.parametrize("small", [False, True], ids=["held", "int8"])
@pytest.mark.parametrize("rules", [dict(temperature=0.0), dict(top_k=20, top_p=0.9, min_p=0.01)], ids=["largest", "filters"])
@pytest.mark.parametrize("cfg", [SMALL, WIDE], ids=["bf16", "wide-bf16"])
def test_captured_answers_are_the_uncaptured_ones(hipdev, cfg, rules, small):
    """Bit for bit, with training of the same model and another answer between two of them (replays of the first program's kind
    before and after eager work)."""
    limn_device.active_device = hipdev
    set_seed(5)
    model, _, train = make_trainer(replace(cfg, ctx=192))
    plain = generate(model, PROMPTS, 24, seed=2, int8=small, captured=False, **rules)
    for _ in range(2):
        got = generate(model, PROMPTS, 24, seed=2, int8=small, **rules)
        for a, b in zip(got, plain):
            np.testing.assert_array_equal(a, b)
        other = generate(model, PROMPTS[:2], 9, seed=9, int8=not small)
        assert other[0].shape == (2, 9)
    x, y = synthetic_batch(replace(cfg, ctx=192), np.random.default_rng(1))
    train(x, y)
    assert np.isfinite(generate(model, PROMPTS, 4, int8=small, **rules)[1]).all()
