"""attend_paged composed of limn's primitives: what a query does not see changes nothing in its row, infinities and NaN among it."""

from __future__ import annotations

import numpy as np
import pytest

from limn_amd.paged import attend_paged
from limn_amd.seam import realize, set_device
from oracle.attend import within
from oracle.serving import paged, same_kind
from serving import paged_inputs
from test_paged_gpu import spoil
from test_serving import PAGED, tensors


def check(x, dtype):
    set_device("numpy")
    t = tensors(x, dtype)
    kind = "float32" if dtype == "float64" else dtype
    with np.errstate(invalid="ignore"):
        out = attend_paged(**t, softcap=3.0)
        realize(out)
    (want, bound), keys, values = paged(**x, softcap=3.0, dtype=kind)
    got = out.numpy()
    within(same_kind(got, want), want, bound, "out")
    np.testing.assert_array_equal(t["key_pages"].numpy(), keys)
    np.testing.assert_array_equal(t["value_pages"].numpy(), values)
    return got


@pytest.mark.parametrize("dtype", ["float32", "float64", "bfloat16"])
@pytest.mark.parametrize("case", PAGED, ids=str)
def test_places_that_nobody_sees(case, dtype):
    """Pages of nobody, places behind the last position, rows of no sequence."""
    got = check(spoil(paged_inputs(1, **{**case, "dtype": "float32" if dtype == "float64" else dtype})), dtype)
    assert np.isfinite(got).all()


@pytest.mark.parametrize("dtype", ["float32", "float64", "bfloat16"])
def test_pages_that_are_not_there(dtype):
    """The page read in the place of one outside the cache holds NaN."""
    x = paged_inputs(2, dtype="float32" if dtype == "float64" else dtype, counts=(2, 1), lengths=(9, 6), page=2)
    x["table"][0, 1] = 99
    unused = sorted(set(range(len(x["key_pages"]))) - set(x["table"].ravel().tolist()))
    for n in ("key_pages", "value_pages"):
        x[n][unused] = np.nan
    if 0 not in unused:
        x["table"][x["table"] == 0] = unused[0]
        for n in ("key_pages", "value_pages"):
            x[n][unused[0]], x[n][0] = 0.5, np.nan
    assert np.isfinite(check(x, dtype)).all()


@pytest.mark.parametrize("dtype", ["float32", "float64"])
def test_later_tokens(dtype):
    x = paged_inputs(3, counts=(5,), lengths=(8,), page=4, heads=2)
    x["v"][3, :, ::3], x["v"][4], x["k"][4] = np.inf, np.nan, np.nan
    got = check(x, dtype)
    assert np.isfinite(got[:3]).all() and not np.isfinite(got[3:]).all()


def test_no_row_is_gathered_from_outside():
    """A page that two sequences write to, and starts that do not ascend: nobody's promise, and no read past a tensor."""
    set_device("numpy")
    x = paged_inputs(5, counts=(3, 2, 4, 3, 1), lengths=(5, 6, 4, 9, 3))
    t = tensors({**x, "table": np.repeat(x["table"][3:4], 5, 0)}, "float32")
    assert attend_paged(**t).numpy().shape == x["q"].shape
    t = tensors({**x, "starts": np.array([0, 13, 0, 13, 0, 13], np.int32)}, "float32")
    assert attend_paged(**t).numpy().shape == x["q"].shape
    t = tensors({**x, "starts": np.array([-9, 13, -2, 99, 5, 2**31 - 1], np.int32), "lengths": np.array([-5, 2**31 - 1, 0, 7, -(2**31)], np.int32)}, "float32")
    assert attend_paged(**t).numpy().shape == x["q"].shape
