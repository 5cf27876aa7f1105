"""Rows without a target under a weight that is not finite: limn_hip_xent_bwd gives them zeros, and nothing of them to the weight."""

from __future__ import annotations

import numpy as np
import pytest

from test_xent_gpu import TYPES, called, draw

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("rows,width,vocab", [(140, 64, 300), (70, 60, 5003), (9, 64, 20011), (700, 513, 4000)])
def test_a_weight_that_is_not_finite(hipdev, dtype, bad, rows, width, vocab):
    """One tile, a width that is no multiple of 8, slices that a second kernel folds, and many tiles."""
    rng, x, w, targets = draw(rows, dtype, rows, width, vocab, left_out=0.4)
    w[vocab // 2, 3] = bad
    w[0] = bad
    out = (targets < 0) | (targets >= vocab)
    got = called(hipdev, x, w, targets, rng.standard_normal(rows).astype(np.float32), dtype)
    assert not got["loss"][out].any() and not got["dx"][out].any()
    got = called(hipdev, x, w, np.full(rows, -1, np.int32), np.ones(rows, np.float32), dtype)
    assert not got["loss"].any() and not got["dx"].any() and not got["dw"].any()
