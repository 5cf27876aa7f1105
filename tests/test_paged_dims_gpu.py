"""attend_paged at float32 head dims that end among a lane's eight (68, 76, ... 124), on the MI355X: keys in the pages and new ones, in
parts, queries, keys and values in one, values at the very end of their buffers."""

from __future__ import annotations

import numpy as np
import pytest

from conftest import DTYPES, download, upload
from limn_amd.paged import attend_paged
from limn_amd.seam import Tensor, int32, realize, use_device
from oracle.attend import within
from oracle.serving import paged
from serving import paged_inputs
from test_paged_gpu import check, spoil

pytestmark = pytest.mark.gpu

CASES = [
    dict(counts=(1,), lengths=(1,), heads=1, page=1),
    dict(counts=(1, 1, 1), lengths=(70, 1, 33), heads=4, kv_heads=2, page=16),
    dict(counts=(3, 1, 0, 2), lengths=(60, 17, 9, 2), heads=6, kv_heads=2, page=8, spare=3, rows_before=2, slopes=True),
    dict(counts=(1, 2), lengths=(3100, 90), heads=4, kv_heads=1, page=32),  # in parts
    dict(counts=(40, 1), lengths=(50, 2500), heads=2, page=24),  # row tiles of 32
]


@pytest.mark.parametrize("hd", [68, 76, 84, 92, 100, 108, 116, 124])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_dims_that_end_among_eight(hipdev, case, hd):
    x = paged_inputs(hd + len(case), hd=hd, **case)
    check(hipdev, x, "float32")
    check(hipdev, spoil(x), "float32", softcap=5.0)


@pytest.mark.parametrize("hd", [68, 124])
def test_values_at_the_end_of_their_buffers(hipdev, hd):
    """A live key in the pool's last place, the last new token's row the last of k and v."""
    x = paged_inputs(1, hd=hd, counts=(1, 3), lengths=(32, 48), heads=4, kv_heads=2, page=16)
    last = len(x["key_pages"]) - 1
    x["table"][x["table"] == last] = x["table"][0, 1]
    x["table"][0, 1] = last  # positions 16 to 31 of the first sequence, its new one the last of them
    assert len(np.unique(x["table"][x["table"] >= 0])) == 5
    check(hipdev, x, "float32")
    check(hipdev, {**x, "k": None, "v": None}, "float32")


@pytest.mark.parametrize("hd", [68, 100])
def test_later_values_stay_out_of_earlier_rows(hipdev, hd):
    """An infinity in the dims that two lanes read is given back once, to the rows that see it."""
    x = paged_inputs(2, hd=hd, counts=(9,), lengths=(40,), heads=2, page=16)
    x["v"][4, :, hd - 6 :] = np.inf
    x["v"][7, :, hd - 1] = -np.inf
    got = check(hipdev, x, "float32")["out"]
    assert np.isfinite(got[:4]).all() and np.isfinite(got[..., : hd - 6]).all()
    assert (got[4:7, :, hd - 6 :] == np.inf).all() and np.isnan(got[7:, :, hd - 1]).all() and (got[7:, :, hd - 6 : hd - 1] == np.inf).all()


@pytest.mark.parametrize("hd", [68, 100])
def test_queries_keys_and_values_in_one(hipdev, hd):
    use_device(hipdev)
    x = paged_inputs(3, hd=hd, counts=(1, 9, 1), lengths=(50, 40, 9), heads=4, kv_heads=2, page=16, spare=2)
    t = DTYPES["float32"]
    on = lambda a, kind=t: Tensor.from_node(upload(hipdev, a, kind))  # noqa: E731
    pools = [on(x[n]) for n in ("key_pages", "value_pages")]
    together = on(np.concatenate([x[n].reshape(len(x["q"]), -1) for n in ("q", "k", "v")], 1))
    (got,) = realize(attend_paged(together, None, None, *pools, *(on(x[n], int32) for n in ("starts", "lengths", "table")), heads=4))
    (want, bound), keys, values = paged(**x)
    within(download(hipdev, got, t, x["q"].shape), want, bound, "out")
    for pool, w in zip(pools, (keys, values)):
        np.testing.assert_array_equal(download(hipdev, pool.node.arg, t, w.shape), w)
