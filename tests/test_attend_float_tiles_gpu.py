"""attend's float32 tiles on bf16 matrix cores, which calls with more than 256 tiles of 32 rows go to: every case is a
small one repeated over the batch until it has that many, each repeat against float64 and bit for bit the first."""

from __future__ import annotations

import numpy as np
import pytest

from oracle.attend import attend as definition
from oracle.attend import within
from test_attend_gpu import draw, packed, trained

pytestmark = pytest.mark.gpu


def check(dev, q, k, v, do, rules, flags):
    batch, heads, t_q, _ = q.shape
    reps = 256 // (batch * heads * ((t_q + 31) // 32)) + 1
    many = lambda x: np.tile(x, (reps, *[1] * (x.ndim - 1)))  # noqa: E731
    got = trained(dev, *(many(x) for x in (q, k, v, do)), "float32", {n: x if n == "slopes" else many(x) for n, x in rules.items()}, flags)
    want = definition(q, k, v, dout=do, dtype="float32", **flags, **rules)
    most = float(np.finfo(np.float32).max)
    for name, x in got.items():
        first, (value, bound) = x[:batch], want[name]
        value = np.where(np.abs(value) > 2.0 * most, np.copysign(np.inf, value), value)  # no float32 holds it
        within(first, value, bound, name)
        for r in range(1, reps):
            np.testing.assert_array_equal(x[r * batch : (r + 1) * batch], first)
    return {n: x[:batch] for n, x in got.items()}


@pytest.mark.parametrize("t_q,t_k", [(64, 64), (65, 65), (97, 200), (128, 128), (129, 300), (300, 300)])
@pytest.mark.parametrize("hd", [4, 36, 64, 68, 100, 128])
def test_sizes(hipdev, hd, t_q, t_k):
    _, (q, k, v, do) = draw(t_q * 1000 + t_k + hd, "float32", 1, 2, 1, t_q, t_k, hd, hd)
    check(hipdev, q, k, v, do, {}, dict(causal=True))
    check(hipdev, q, k, v, do, dict(slopes=np.array([0.25, 0.0625], np.float32)), dict(softcap=5.0))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("causal,softcap,alibi,documents,prefix,ragged", [
    (True, 3.0, False, False, False, False), (True, 0.0, True, False, False, False), (True, 0.0, False, True, False, False),
    (True, 0.0, False, False, True, False), (True, 0.0, False, False, False, True), (True, 3.0, True, True, True, True),
    (False, 3.0, True, True, False, True), (False, 0.0, False, True, False, False)])
def test_rules(hipdev, dim, causal, softcap, alibi, documents, prefix, ragged):
    t_q, t_k = (230, 290) if ragged else (290, 290)
    rng, (q, k, v, do) = draw(dim + 2 * causal, "float32", 3, 4, 2, t_q, t_k, dim, dim, std=3.0 if softcap else 1.0)
    rules = {}
    if alibi:
        rules["slopes"] = np.array([0.5, 0.1, 0.02, 0.0], np.float32)
    if documents:
        rules["documents"] = packed(rng, 3, t_k, 60)
    if prefix:
        rules["prefix"] = np.array([0, 77, 250], np.int32)
    if ragged:
        rules["lengths"] = np.array([290, 131, 3], np.int32)  # one shorter than its queries
    check(hipdev, q, k, v, do, rules, dict(causal=causal, softcap=softcap))


def test_documents_in_any_order_and_rows_that_see_nothing(hipdev):
    rng, (q, k, v, do) = draw(5, "float32", 3, 2, 2, 200, 200, 64, 64)
    docs = rng.integers(-1, 4, (3, 200)).astype(np.int32)
    docs[1] = -1
    for causal in (False, True):
        got = check(hipdev, q, k, v, do, dict(documents=docs), dict(causal=causal))
        assert not got["out"][1].any() and not got["dk"][1].any() and not got["dq"][1].any()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_infinities_and_nan_in_hidden_places(hipdev, dim, bad):
    rng, (q, k, v, do) = draw(dim, "float32", 2, 4, 2, 170, 170, dim, dim)
    docs = np.repeat(np.arange(4), 50)[None, :170].repeat(2, 0).astype(np.int32)
    docs[:, 160:] = -1
    for x in (q, k, v, do):
        x[:, :, 160:] = bad
    v[0, 0, 77, 5] = bad
    do[0, 1, 120, 7] = bad
    check(hipdev, q, k, v, do, dict(documents=docs), dict(causal=True))
    rng, (q, k, v, do) = draw(dim + 2, "float32", 1, 2, 1, 100, 100, dim, dim)
    v[0, 0, 90, 3] = bad  # rows 90 to 99 see it
    k[0, 0, 99, 3] = bad if np.isnan(bad) else 0.0
    check(hipdev, q, k, v, do, {}, dict(causal=True))
    check(hipdev, q, k, v, do, {}, dict())


def test_numbers_that_no_bf16_holds(hipdev):
    """float32's largest numbers round past bf16's; subnormal ones below its least step. A query of the largest against
    keys of the smallest is an ordinary score."""
    _, (q, k, v, do) = draw(21, "float32", 1, 2, 1, 100, 100, 64, 64)
    most = np.finfo(np.float32).max
    v[0, 0, 40, :2] = (most, -most)
    do[:, :, :, :2] = 0.0  # their product with dout would leave float32
    q[0, 1, 70] = 0.0
    q[0, 1, 70, 3] = most
    k[0, 0, :, 3] *= 1e-38
    check(hipdev, q, k, v, do, {}, dict(causal=True, scale=1.0))
    _, (q, k, v, do) = draw(22, "float32", 1, 2, 1, 100, 100, 128, 128)
    scale = np.exp2(np.random.default_rng(22).integers(-60, 61, 128)).astype(np.float32)
    check(hipdev, q * scale, k / scale, v, do, {}, dict(causal=True))


def test_far_and_near_scores(hipdev):
    _, (q, k, v, do) = draw(11, "float32", 1, 2, 1, 130, 130, 64, 64, std=60.0)
    check(hipdev, q, k, v, do, {}, dict(causal=True))
    check(hipdev, np.zeros_like(q), k, v, do, {}, dict(causal=True))
    check(hipdev, q, k, v, do, dict(slopes=np.array([100.0, 1e-6], np.float32)), dict(causal=True, softcap=50.0, scale=0.01))


@pytest.mark.parametrize("bits", [-40, 40])
def test_cotangents_of_every_size(hipdev, bits):
    _, (q, k, v, do) = draw(71 + bits, "float32", 1, 2, 1, 190, 190, 64, 64)
    check(hipdev, q, k, v, do * np.float32(2.0**bits), {}, dict(causal=True))
