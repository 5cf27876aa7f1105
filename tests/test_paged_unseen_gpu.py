"""The composed form of attend_paged on the hip device (head dims past 256): what a query does not see changes nothing in its row."""

from __future__ import annotations

import numpy as np
import pytest

from conftest import DTYPES, download
from limn_amd.paged import attend_paged
from limn_amd.seam import realize, use_device
from oracle.attend import within
from oracle.serving import paged
from serving import paged_inputs
from test_paged_gpu import spoil, tensors

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_places_that_nobody_sees(hipdev, dtype):
    use_device(hipdev)
    x = spoil(paged_inputs(4, dtype=dtype, counts=(3, 1, 5), lengths=(7, 1, 5), heads=4, kv_heads=2, hd=260, spare=2, rows_before=1))
    t = tensors(hipdev, x, dtype)
    (got,) = realize(attend_paged(**t))
    (want, bound), keys, values = paged(**x, dtype=dtype)
    got = download(hipdev, got, DTYPES[dtype], x["q"].shape)
    within(got, want, bound, "out")
    assert np.isfinite(got).all()
    np.testing.assert_array_equal(t["key_pages"].numpy(), keys)
    np.testing.assert_array_equal(t["value_pages"].numpy(), values)
