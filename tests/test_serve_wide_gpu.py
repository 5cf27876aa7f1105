"""Answers of models that attend through the composed form on the MI355X (float64, head dims past 256), captured and not, against the numpy
oracle's whole model on whole sequences."""

from __future__ import annotations

import numpy as np
import pytest

from limn_amd.gpt import GPTConfig
from limn_amd.seam import device as limn_device
from limn_amd.seam import float32, float64
from limn_amd.serve import generate
from serving import PROMPTS
from test_serve_gpu import logits_of, model_of

pytestmark = pytest.mark.gpu

# Off by this part of the largest logit. float32: test_serve_gpu's bound for sums of up to 512 terms; a head's dim of 260 stays below. float64: the
# oracle's logits are rounded to float32 before they are compared, by 2^-24 of them
CONFIGS = {
    "f64": (GPTConfig(vocab=64, ctx=64, dim=48, layers=2, heads=4, batch=2, kv_heads=2, softcap=3.0, distance=True, dtype=float64), 2.0**-24),
    "f32-260": (GPTConfig(vocab=64, ctx=64, dim=520, layers=2, heads=2, batch=2, dtype=float32), 2.3e-3),
}


@pytest.mark.parametrize("name", CONFIGS)
def test_answers_match_the_oracles_whole_model(hipdev, name):
    cfg, worst = CONFIGS[name]
    limn_device.active_device = hipdev
    got = generate(model_of(cfg), PROMPTS, 12, seed=3, temperature=0.8, page=8, part=9)
    for a, b in zip(got, generate(model_of(cfg), PROMPTS, 12, seed=3, temperature=0.8, page=8, part=9, captured=False)):
        np.testing.assert_array_equal(a, b)
    answers, shares = got
    for p, answer, share, rows in zip(PROMPTS, answers, shares, logits_of(cfg, False, [[*p, *a] for p, a in zip(PROMPTS, answers)])):
        warm = rows[len(p) - 1 : -1] / 0.8
        want = np.take_along_axis(warm, answer[:, None], 1)[:, 0] - np.log(np.exp(warm).sum(1))
        assert np.abs(share - want).max() <= 2 * worst * np.abs(warm).max() + 2.0**-24 * np.abs(want).max()  # a share is float32
