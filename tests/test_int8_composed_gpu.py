"""quantize_rows' and int8_linear's composed form on the hip device (float64): rows with infinities and NaN."""

from __future__ import annotations

import numpy as np
import pytest

from conftest import upload
from limn_amd.int8 import int8_linear, quantize_rows
from limn_amd.seam import Tensor, float32, float64, int8, realize, use_device
from oracle.serving import quantized

pytestmark = pytest.mark.gpu


def test_rows_with_infinities_and_nan(hipdev):
    use_device(hipdev)
    x = np.random.default_rng(6).standard_normal((6, 300))
    x[1, 3], x[2, 299], x[4, 0] = np.inf, np.nan, -np.inf
    on = lambda a, kind: Tensor.from_node(upload(hipdev, a, kind))  # noqa: E731
    values, scales = quantize_rows(on(x, float64))
    w = np.eye(5, 300, dtype=np.int8)
    y = int8_linear(on(x, float64), on(w, int8), on(np.ones(5, np.float32), float32))
    realize(values, scales, y)
    odd = np.isin(np.arange(6), [1, 2, 4])
    want, s = quantized(x)
    np.testing.assert_array_equal(np.isnan(scales.numpy()), odd)
    np.testing.assert_allclose(scales.numpy()[~odd], s[~odd], rtol=2.0**-23)
    assert (values.numpy()[odd] == 0).all() and (np.abs(values.numpy().astype(int) - want) <= 1).all()
    assert np.isnan(y.numpy()[odd]).all() and np.isfinite(y.numpy()[~odd]).all()
