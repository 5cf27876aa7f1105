"""Caps far above the scores they are for, and scores about a cap, in the form composed from limn's primitives."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

from limn_amd.attend import attend
from limn_amd.hip import runtime
from limn_amd.seam import Tensor, float32, float64, grad, set_device
from oracle.attend import attend as definition
from oracle.attend import within


@pytest.fixture(autouse=True)
def _numpy():
    set_device("numpy")


def drawn(spread, seed=0):
    rng = np.random.default_rng(seed)
    q, k, v, do = (rng.standard_normal(s).astype(np.float32) for s in ((1, 2, 9, 16), (1, 1, 9, 16), (1, 1, 9, 8), (1, 2, 9, 8)))
    return q * np.float32(spread), k, v, do


@pytest.mark.parametrize("spread", [0.01, 1.0, 4.0])
@pytest.mark.parametrize("softcap", [1.0, 50.0, 1e3, 1e5, 1e8, 1e30])
def test_a_cap_is_as_exact_as_the_scores_under_it(softcap, spread):
    """float32: a score is off by a part of itself, not of the cap, so out and the gradients are what an uncapped call's are."""
    q, k, v, do = drawn(spread)
    tq, tk, tv = (Tensor(x, dtype=float32, requires_grad=True) for x in (q, k, v))
    out = attend(tq, tk, tv, causal=True, softcap=softcap)
    got = [out, *grad((out * Tensor(do, dtype=float32)).sum(), [tq, tk, tv])]
    want = definition(q, k, v, dout=do, causal=True, softcap=softcap, dtype="float32")
    for name, t in zip(("out", "dq", "dk", "dv"), got):
        within(t.numpy(), *want[name], name)


@pytest.mark.parametrize("softcap", [0.5, 1.0, 4.0, 1e6])
def test_scores_on_both_sides_of_half_the_cap_in_float64(softcap):
    q, k, v, do = (x.astype(np.float64) for x in drawn(2.0, seed=1))
    q[0, 0, 3] = 0.0
    tq, tk, tv = (Tensor(x, dtype=float64, requires_grad=True) for x in (q, k, v))
    out = attend(tq, tk, tv, softcap=softcap)
    got = [out, *grad((out * Tensor(do, dtype=float64)).sum(), [tq, tk, tv])]
    want = definition(q, k, v, dout=do, softcap=softcap)
    for name, t in zip(("out", "dq", "dk", "dv"), got):
        within(t.numpy(), want[name][0], 1e-12, name)


def test_an_infinite_score_is_the_cap():
    q, k, v, _ = drawn(1.0, seed=2)
    q[0, 0, 0, 0] = np.inf  # every score of this row is an infinity of its key's sign
    out = attend(*(Tensor(x, dtype=float32) for x in (q, k, v)), softcap=5.0)
    p = np.exp(np.where(k[0, 0, :, 0] > 0, 5.0, -5.0) - 5.0)
    row, want = out.numpy()[0, 0, 0], p @ v[0, 0] / p.sum()
    within(row, want, 64 * 2.0**-24 * (p @ np.abs(v[0, 0])) / p.sum())  # an exponential, two sums of 9, a quotient: under 64 half steps


@pytest.mark.parametrize("kw,message", [
    (dict(softcap=1e39), "softcap"), (dict(softcap=1e-39), "softcap"), (dict(softcap=float("inf")), "softcap"), (dict(softcap=-1e-3), "softcap"),
    (dict(scale=1e39), "scale"), (dict(scale=-1e39), "scale"), (dict(scale=float("nan")), "scale")])
def test_numbers_that_float32_does_not_hold_are_refused(kw, message):
    """By the function, and by the C ABI before anything is launched (the pointers are never read)."""
    with pytest.raises(ValueError, match=message):
        attend(*(Tensor(x, dtype=float32) for x in drawn(1.0)[:3]), **kw)
    lib, fake = runtime.kernels(), ctypes.c_void_p(0x1000)
    rules = (dict(scale=0.25, softcap=0.0) | kw)
    tail = (1, 1, 2, 1, 9, 9, 16, 16, 0, rules["scale"], rules["softcap"], fake, 1 << 40, None)
    for status in (lib.limn_hip_attend_fwd(*[fake] * 3, *[None] * 4, *[fake] * 2, *tail), lib.limn_hip_attend_bwd(*[fake] * 3, *[None] * 4, *[fake] * 6, *tail)):
        assert status == 1 and message in lib.limn_hip_last_error().decode()


@pytest.mark.parametrize("scale", [0.0, 1e-39, -1e-39, 1e-30])
def test_scales_of_nothing(scale):
    q, k, v, do = drawn(1.0, seed=3)
    tq, tk, tv = (Tensor(x, dtype=float32, requires_grad=True) for x in (q, k, v))
    out = attend(tq, tk, tv, causal=True, scale=scale)
    got = [out, *grad((out * Tensor(do, dtype=float32)).sum(), [tq, tk, tv])]
    want = definition(q, k, v, dout=do, causal=True, scale=scale, dtype="float32")
    for name, t in zip(("out", "dq", "dk", "dv"), got):
        within(t.numpy(), *want[name], name)
