"""sample on the MI355X: the C ABI and limn_amd.sampling on the hip device, against the definition in float64 (oracle/serving.py)."""

from __future__ import annotations

import numpy as np
import pytest

from conftest import DTYPES, storage_values, upload
from limn_amd.dtypes import ABI_CODE, from_storage
from limn_amd.hip import runtime
from limn_amd.sampling import sample
from limn_amd.seam import Tensor, capture, float32, int32, realize, use_device
from oracle.attend import within
from oracle.serving import sample as oracle
from serving import logit_rows

pytestmark = pytest.mark.gpu
TYPES = ["float32", "bfloat16", "float16"]
GUARD = 64
KINDS = dict(temperature=float32, top_k=int32, top_p=float32, min_p=float32)


def called(dev, logits, u, dtype, apart=0, shift=0, logprobs=True, **rules):
    t, (rows, vocab) = DTYPES[dtype], logits.shape
    wide = np.full((rows, vocab + apart), np.inf, np.float32)  # between the rows: nothing that may be read
    wide[:, :vocab] = logits
    x = upload(dev, np.concatenate([np.full(shift, np.inf, np.float32), wide.reshape(-1)]), t).arg
    given = [None if rules.get(n) is None else upload(dev, np.asarray(rules[n]), kind).arg for n, kind in KINDS.items()]
    us, outs = upload(dev, u, float32).arg, [dev._alloc(rows * 4 + GUARD) for _ in range(2)]
    for b in outs:
        dev.copyin(b, np.full(b.nbytes, 0xAB, np.uint8))
    need = dev.lib.limn_hip_sample_workspace(ABI_CODE[t], rows, vocab)
    ws = dev._alloc(need + GUARD)
    dev.copyin(ws, np.full(ws.nbytes, 0xFF, np.uint8))
    runtime.check_limn(dev.lib.limn_hip_sample(x.ptr + shift * t.itemsize, us.ptr, *(None if b is None else b.ptr for b in given), outs[0].ptr, outs[1].ptr if logprobs else None,
                                               ABI_CODE[t], rows, vocab, vocab + apart, ws.ptr, need, None))
    dev.finish()
    assert (dev.copyout(ws)[need:] == 0xFF).all()
    raws = [dev.copyout(b) for b in outs]
    assert all((raw[rows * 4 :] == 0xAB).all() for raw in raws)
    return from_storage(raws[0][: rows * 4], int32, (rows,)), from_storage(raws[1][: rows * 4], float32, (rows,))


def check(dev, logits, u, dtype, apart=0, shift=0, **rules):
    rules = {n: np.full(len(logits), r, np.int32 if n == "top_k" else np.float32) if np.isscalar(r) else r for n, r in rules.items()}
    tokens, logs = called(dev, logits, u, dtype, apart, shift, **rules)
    want, (lp, bound) = oracle(logits, u, **rules)
    np.testing.assert_array_equal(tokens, want)
    within(logs, lp, bound, "logprob")
    return tokens


SIZES = [(1, 1), (3, 2), (5, 17), (33, 256), (7, 1000), (64, 1025), (9, 4099), (4, 32000), (3, 50257), (2, 131072), (1, 300001), (300, 64)]
SETTINGS = [dict(), dict(top_k=1), dict(top_k=50), dict(top_p=0.9), dict(min_p=0.05), dict(temperature=0.7, top_k=40, top_p=0.95, min_p=0.02), dict(temperature=3.0, top_p=0.5), dict(temperature=0.0)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab", SIZES)
def test_sizes(hipdev, rows, vocab, dtype):
    logits, u, _ = logit_rows(rows + vocab, rows, vocab, dtype)
    for kw in SETTINGS:
        check(hipdev, logits, u, dtype, **kw)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("spread", [0.0, 0.01, 0.5, 8.0, 100.0])
@pytest.mark.parametrize("vocab", [100, 5000, 70000])
def test_spreads(hipdev, vocab, spread, dtype):
    """From rows of equal logits to rows with one that counts."""
    logits, u, _ = logit_rows(1, 6, vocab, dtype, spread)
    for kw in SETTINGS:
        check(hipdev, logits, u, dtype, **kw)


@pytest.mark.parametrize("dtype", TYPES)
def test_settings_of_every_row(hipdev, dtype):
    logits, u, rng = logit_rows(2, 200, 3001, dtype)
    for _ in range(4):
        check(hipdev, logits, rng.random(200).astype(np.float32), dtype, temperature=rng.choice([-1.0, 0.0, 1e-30, 0.01, 0.5, 1.0, 2.0, 1e30, np.nan, np.inf], 200).astype(np.float32),
              top_k=rng.choice([-3, 0, 1, 2, 10, 3000, 3001, 2**31 - 1], 200).astype(np.int32), top_p=rng.choice([-1.0, 0.0, 1e-9, 0.3, 0.99, 1.0, 2.0, np.nan], 200).astype(np.float32),
              min_p=rng.choice([-1.0, 0.0, 1e-9, 0.1, 1.0, 5.0, np.nan], 200).astype(np.float32))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [40, 3000, 66000])
def test_ties(hipdev, vocab, dtype):
    """Few values, so that every border falls among equal ones: they go by their index."""
    rng = np.random.default_rng(3)
    logits = rng.integers(-2, 3, (40, vocab)).astype(np.float32)
    logits[:10] *= rng.choice([-0.0, 0.0], (10, vocab)).astype(np.float32)  # both zeros are equal
    u = rng.random(40).astype(np.float32)
    u[:4] = [0.0, 0.25, 0.5, 0.75]
    for kw in SETTINGS + [dict(top_k=vocab // 2), dict(top_p=0.25), dict(top_p=0.5, top_k=8)]:
        check(hipdev, logits, u, dtype, **kw)


@pytest.mark.parametrize("dtype", TYPES)
def test_infinities_nan_and_masks(hipdev, dtype):
    rng = np.random.default_rng(4)
    low = {"float32": -3.4028234663852886e38, "bfloat16": -3.3895313892515355e38, "float16": -65504.0}[dtype]
    logits = storage_values(rng.standard_normal((12, 777)).astype(np.float32), DTYPES[dtype])
    logits[0] = -np.inf
    logits[1] = np.nan
    logits[2, 5:] = -np.inf
    logits[3, 5:] = low  # masked by the type's lowest value
    logits[4] = low
    logits[5, [3, 700]] = np.inf
    logits[6, ::2] = np.nan
    logits[7] = np.nan
    logits[7, 12] = -np.inf
    logits[8, 1:] = -np.inf
    logits[9, 6] = -low
    logits[10] = -low
    u = rng.random(12).astype(np.float32)
    for kw in SETTINGS + [dict(top_k=700)]:
        tokens = check(hipdev, logits, u, dtype, **kw)
        assert (tokens[[0, 1, 7]] == -1).all()


def test_uniforms_at_the_ends_and_outside(hipdev):
    logits, _, _ = logit_rows(5, 8, 500)
    u = np.array([0.0, np.nextafter(np.float32(1), np.float32(0)), 1.0, 2.0, -1.0, np.nan, np.inf, -np.inf], np.float32)
    for kw in (dict(), dict(top_k=7), dict(top_p=0.8), dict(min_p=0.1)):
        check(hipdev, logits, u, "float32", **kw)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("apart,shift", [(0, 1), (1, 0), (7, 3), (8, 8)])
def test_rows_apart_and_shifted(hipdev, apart, shift, dtype):
    for vocab in (999, 20000):
        logits, u, _ = logit_rows(6, 5, vocab, dtype)
        check(hipdev, logits, u, dtype, apart=apart, shift=shift, top_k=30, top_p=0.9)
        check(hipdev, logits, u, dtype, apart=apart, shift=shift)


def test_draws_follow_the_shares(hipdev):
    """4096 evenly spread numbers hit each token as often as its share says, up to one at each end of its interval."""
    logits = np.repeat(np.log(np.arange(1, 9, dtype=np.float64))[None], 4096, 0).astype(np.float32)
    tokens, _ = called(hipdev, logits, ((np.arange(4096) + 0.5) / 4096).astype(np.float32), "float32", logprobs=False)
    assert (np.abs(np.bincount(tokens, minlength=8) - 4096 * np.arange(1, 9) / 36) <= 1.001).all()


def test_through_the_tensor_api_captured(hipdev):
    use_device(hipdev)
    logits, u, rng = logit_rows(7, 24, 2000, "bfloat16")
    t = Tensor.from_node(upload(hipdev, logits.reshape(4, 6, 2000), DTYPES["bfloat16"]))

    def step(x, u):
        got = sample(x, u, temperature=0.8, top_k=30, top_p=0.9)
        realize(*got)
        return got

    run = capture(step)
    rules = dict(temperature=np.full(24, 0.8, np.float32), top_k=np.full(24, 30), top_p=np.full(24, 0.9, np.float32))
    for _ in range(6):
        u = rng.random(24).astype(np.float32)
        tokens, logs = run(t, Tensor(u.reshape(4, 6)).realize())
        want, (lp, bound) = oracle(logits, u, **rules)
        np.testing.assert_array_equal(tokens.numpy().reshape(-1), want)
        within(logs.numpy().reshape(-1), lp, bound, "logprob")
        assert (Tensor(np.ones(1000)) * 3.0).sum().item() == 3000.0
