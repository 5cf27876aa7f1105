"""Caps far above the scores they are for, and scores about half the cap, where the kernels change from one form of tanh to
another: every kernel of attend against the definition in float64. A capped score may be off by a part of itself (16 half
steps of float32, see oracle/attend.py), not of the cap."""

from __future__ import annotations

import numpy as np
import pytest

from oracle.attend import attend as definition
from oracle.attend import within
from test_attend_float_tiles_gpu import check as check_tiles
from test_attend_gpu import TYPES, check, draw, served

pytestmark = pytest.mark.gpu

CAPS = [1.0, 100.0, 1e4, 1e6, 1e30]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [33, 64, 80, 128, 160])
@pytest.mark.parametrize("softcap", CAPS)
def test_trained(hipdev, dtype, hd, softcap):
    _, (q, k, v, do) = draw(hd, dtype, 1, 4, 2, 200, 200, hd, hd, std=2.0)
    check(hipdev, q, k, v, do, dtype, {}, dict(causal=True, softcap=softcap))
    check(hipdev, q, k, v, do, dtype, dict(slopes=np.array([0.5, 0.1, 0.02, 0.0], np.float32)), dict(softcap=softcap))


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("softcap", CAPS)
def test_trained_on_float32_tiles(hipdev, hd, softcap):
    _, (q, k, v, do) = draw(hd, "float32", 1, 4, 2, 200, 200, hd, hd, std=2.0)
    check_tiles(hipdev, q, k, v, do, {}, dict(causal=True, softcap=softcap))
    check_tiles(hipdev, q, k, v, do, dict(slopes=np.array([0.5, 0.1, 0.02, 0.0], np.float32)), dict(softcap=softcap))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scale", [0.3, -0.3])
@pytest.mark.parametrize("heads,kv_heads,t_q,t_k,dim", [(8, 2, 1, 300, 64), (4, 4, 5, 2100, 128), (2, 1, 70, 1100, 80)])
@pytest.mark.parametrize("softcap", CAPS)
def test_against_a_cache(hipdev, dtype, heads, kv_heads, t_q, t_k, dim, scale, softcap):
    _, (q, k, v, _) = draw(t_k, dtype, 1, heads, kv_heads, t_q, t_k, dim, dim)
    out, lse = served(hipdev, q, k, v, dtype, {}, causal=True, softcap=softcap, scale=scale)
    want = definition(q, k, v, dtype=dtype, causal=True, softcap=softcap, scale=scale)
    within(out, *want["out"], "out")
    within(lse, *want["lse"], "lse")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [64, 128])
def test_an_infinite_score_is_the_cap(hipdev, dtype, hd):
    """A query with an infinity: its scores are infinities of the keys' signs, and the cap makes them finite."""
    _, (q, k, v, _) = draw(hd, dtype, 1, 2, 1, 130, 130, hd, hd)
    q[0, 0, 77, 3] = np.inf
    out, _ = served(hipdev, q, k, v, dtype, {}, softcap=5.0)
    p = np.exp(np.where(k[0, 0, :, 3] > 0, 5.0, -5.0).astype(np.float64) - 5.0)
    half = dict(float32=2.0**-24, float16=2.0**-11, bfloat16=2.0**-8)[dtype]
    # weights and result rounded to the type, and sums of 130 terms of one exponential each
    bound = (2 * half + 200 * 2.0**-24) * (p @ np.abs(v[0, 0])) / p.sum()
    within(out[0, 0, 77], p @ v[0, 0] / p.sum(), bound)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [33, 64, 128])
@pytest.mark.parametrize("scale", [1e-20, 1e-29, 1e-31, 1e-39, 1e-50, -1e-39])
def test_scales_of_nothing(hipdev, dtype, hd, scale):
    """Equal weights: out, the logsumexp, and the values' gradient of a mean. The tiles take the score units of a scale's inverse."""
    _, (q, k, v, do) = draw(hd, dtype, 1, 2, 1, 150, 150, hd, hd)
    check(hipdev, q, k, v, do, dtype, {}, dict(causal=True, scale=scale))
    out, lse = served(hipdev, q, k, v, dtype, {}, causal=True, scale=scale)
    want = definition(q, k, v, dtype=dtype, causal=True, scale=scale)
    within(lse, *want["lse"], "lse")
    if dtype == "float32" and hd % 4 == 0:
        check_tiles(hipdev, q, k, v, do, {}, dict(causal=True, scale=scale))
