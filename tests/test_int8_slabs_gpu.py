"""int8_linear on weights of aligned rows that do not begin aligned, larger than the room for their copy, on the MI355X: the bits of the
same weight where it is aligned."""

from __future__ import annotations

import numpy as np
import pytest

from test_int8_gpu import TYPES, called, check, layer

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,width,outputs", [(1, 4096, 16400), (16, 4096, 16384), (40, 16384, 9001), (300, 16384, 4100), (3, 1 << 17, 600)])
def test_slabs(hipdev, rows, width, outputs, dtype):
    x, w, s, b = layer(rows, dtype, rows, width, outputs, bias=True)
    got = called(hipdev, x, w, s, b, dtype, w_shift=5)
    np.testing.assert_array_equal(got, called(hipdev, x, w, s, b, dtype))
    if rows < 40:
        check(hipdev, x, w, s, b, dtype, w_shift=4)
