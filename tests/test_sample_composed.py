"""sample composed of limn's primitives where rows hold NaN and infinities, numbers lie outside their ranges and settings are NaN or
infinite: what the kernel does, by the same oracle."""

from __future__ import annotations

import numpy as np
import pytest

from conftest import DTYPES
from limn_amd.sampling import sample
from limn_amd.seam import Tensor, float32, float64, int32, realize, set_device
from oracle.attend import within
from oracle.serving import sample as oracle
from serving import logit_rows

KINDS = dict(temperature=float32, top_k=int32, top_p=float32, min_p=float32)


@pytest.fixture(autouse=True)
def numpy_device():
    set_device("numpy")


def check(logits, u, dtype="float32", **rules):
    rows = {n: np.broadcast_to(np.asarray(r, np.int32 if n == "top_k" else np.float32), u.shape) for n, r in rules.items()}
    with np.errstate(all="ignore"):
        tokens, logs = realize(*(got := sample(Tensor(logits, dtype=DTYPES[dtype]), Tensor(u, dtype=float32), **{n: Tensor(r, dtype=KINDS[n]) for n, r in rows.items()}))) and got
        tokens, logs = tokens.numpy(), logs.numpy()
    want, (lp, bound) = oracle(logits, u, **rows)
    np.testing.assert_array_equal(tokens, want)
    within(logs, lp, bound, "logprob")
    return tokens, logs


SETTINGS = [dict(), dict(top_k=3), dict(top_p=0.6), dict(min_p=0.2), dict(temperature=0.4, top_k=5, top_p=0.9, min_p=0.01), dict(temperature=0.0)]


@pytest.mark.parametrize("kw", SETTINGS, ids=str)
@pytest.mark.parametrize("dtype", ["float32", "float64"])
def test_infinities_nan_and_masks(kw, dtype):
    low = float(np.finfo(np.float32 if dtype == "float32" else np.float64).min)
    logits, u, _ = logit_rows(1, 12, 23)
    logits = logits.astype(np.float64 if dtype == "float64" else np.float32)
    logits[0] = -np.inf
    logits[1] = np.nan
    logits[2, 5:] = -np.inf
    logits[3, 5:] = low
    logits[4] = low
    logits[5, [3, 20]] = np.inf
    logits[6, ::2] = np.nan
    logits[7] = np.nan
    logits[7, 12] = -np.inf
    logits[8, 1:] = -np.inf
    logits[9, 6] = -low
    logits[10, ::3], logits[10, 7] = np.nan, np.inf
    tokens, _ = check(logits, u, dtype, **kw)
    assert (tokens[[0, 1, 7]] == -1).all()


def test_uniforms_at_the_ends_and_outside():
    logits, _, _ = logit_rows(5, 9, 50)
    logits[:, 40:] = -np.inf
    u = np.array([0.0, np.nextafter(np.float32(1), np.float32(0)), 1.0, 2.0, -1.0, np.nan, np.inf, -np.inf, 0.5], np.float32)
    for kw in (dict(), dict(top_k=7), dict(top_p=0.8), dict(min_p=0.1)):
        tokens, logs = check(logits, u, **kw)
        assert np.isfinite(logs).all() and (tokens < 40).all()


def test_settings_that_are_nan_or_infinite():
    logits, u, rng = logit_rows(2, 200, 31)
    check(logits, u, temperature=rng.choice([-1.0, 0.0, 1e-30, 0.01, 0.5, 1.0, 2.0, 1e30, np.nan, np.inf], 200), top_k=rng.choice([-3, 0, 1, 2, 10, 30, 31, 2**31 - 1], 200),
          top_p=rng.choice([-1.0, 0.0, 1e-9, 0.3, 0.99, 1.0, 2.0, np.nan], 200), min_p=rng.choice([-1.0, 0.0, 1e-9, 0.1, 1.0, 5.0, np.nan], 200))


def test_an_infinite_temperature_draws_evenly_from_what_is_there():
    logits = np.array([[3.0, -np.inf, 1.0, np.nan, 2.0, 0.0]] * 4, np.float32)
    u = np.array([0.1, 0.3, 0.6, 0.9], np.float32)
    tokens, logs = sample(Tensor(logits), Tensor(u), temperature=Tensor(np.full(4, np.inf, np.float32)))
    np.testing.assert_array_equal(tokens.numpy(), [0, 4, 2, 5])
    np.testing.assert_allclose(logs.numpy(), np.log(0.25), rtol=2.0**-23)


@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
def test_numbers_that_are_no_numbers_are_refused(value):
    logits, u, _ = logit_rows(3, 2, 5)
    for name in KINDS:
        with pytest.raises(ValueError, match="finite"):
            sample(Tensor(logits), Tensor(u), **{name: value})
