"""Rows without a target in linear_cross_entropy's composed form: whatever they hold, and whatever the weight holds, they give
nothing and get zeros."""

from __future__ import annotations

import numpy as np
import pytest

from limn_amd.seam import Tensor, float32, float64, grad, int32, set_device
from limn_amd.xent import linear_cross_entropy
from oracle.attend import within, xent


@pytest.fixture(autouse=True)
def _numpy():
    set_device("numpy")


def run(x, w, targets, dtype):
    tx, tw = (Tensor(a, dtype=dtype, requires_grad=True) for a in (x, w))
    loss = linear_cross_entropy(tx, tw, Tensor(targets, dtype=int32))
    return [t.numpy() for t in (loss, *grad(loss, [tx, tw]))]


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("dtype", [float32, float64])
def test_infinities_and_nan_in_rows_left_out(bad, dtype):
    rng = np.random.default_rng(0)
    x, w = rng.standard_normal((6, 5)), rng.standard_normal((7, 5))
    targets = np.array([2, -1, 6, 7, 0, 3], np.int32)
    want = run(x, w, targets, dtype)
    x[[1, 3]] = bad
    for a, b in zip(run(x, w, targets, dtype), want):
        np.testing.assert_array_equal(a, b)
    exact = xent(np.nan_to_num(x, posinf=0, neginf=0), w, targets, np.full(6, 0.25), "float32")
    within(want[1], *exact["dx"])
    assert not want[1][[1, 3]].any()


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_a_weight_that_is_not_finite(bad):
    rng = np.random.default_rng(1)
    x, w = rng.standard_normal((6, 5)), rng.standard_normal((7, 5))
    w[4, 2] = bad
    targets = np.array([2, -1, 6, 7, 0, 3], np.int32)
    assert not run(x, w, targets, float32)[1][[1, 3]].any()
    for got in run(x, w, np.full(6, -1, np.int32), float32):
        assert not got.any()
