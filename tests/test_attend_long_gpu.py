"""attend against caches so long that a key head's rows, or bytes, pass 32 bits; few of their keys are live."""

from __future__ import annotations

import numpy as np
import pytest

from conftest import DTYPES
from limn_amd.dtypes import ABI_CODE, from_storage, to_storage
from limn_amd.hip import runtime
from limn_amd.seam import float32
from oracle.attend import attend as definition
from oracle.attend import within
from test_attend_gpu import draw

pytestmark = pytest.mark.gpu


def on(dev, values, dtype):
    host = to_storage(values, dtype)
    buf = dev._alloc(host.nbytes)
    dev.copyin(buf, host.view(np.uint8).reshape(-1))
    return buf


@pytest.mark.parametrize("dtype,hd", [("float16", 1), ("float32", 1), ("bfloat16", 8)])
def test_few_live_keys_of_a_long_cache(hipdev, dtype, hd):
    """2^26 + 64 places for one key head of 32 query heads, the first 40 live: forward, and a backward whose gradients
    behind the live keys are zeros. Places behind them hold 1."""
    t, heads, t_q, live, places = DTYPES[dtype], 32, 3, 40, (1 << 26) + 64
    rng, (q, k, v, do) = draw(hd, dtype, 1, heads, 1, t_q, live, hd, hd)
    slopes = (0.9 ** np.arange(1, heads + 1)).astype(np.float32)
    sizes = (1, heads, 1, t_q, places, hd, hd)
    padded = []
    for x in (k, v):
        one = to_storage(np.ones((1,), np.float32), t)
        host = np.full(places * hd, one[0], dtype=one.dtype)
        host[: live * hd] = to_storage(x, t).reshape(-1)
        buf = hipdev._alloc(host.nbytes)
        hipdev.copyin(buf, host.view(np.uint8))
        padded.append(buf)
    bq, bdo, bs, bl = on(hipdev, q, t), on(hipdev, do, t), on(hipdev, slopes, float32), hipdev._alloc(4)
    hipdev.copyin(bl, np.array([live], np.int32).view(np.uint8))
    out, lse, dq = hipdev._alloc(bq.nbytes), hipdev._alloc(heads * t_q * 4), hipdev._alloc(bq.nbytes)
    dk, dv = hipdev._alloc(padded[0].nbytes), hipdev._alloc(padded[0].nbytes)
    for b in (dk, dv):
        hipdev.copyin(b, np.full(b.nbytes, 0xAB, np.uint8))
    head = (bq.ptr, padded[0].ptr, padded[1].ptr, bs.ptr, None, None, bl.ptr)
    tail = (ABI_CODE[t], *sizes, 1, hd**-0.5, 0.0)
    for backward, buffers in ((0, (out.ptr, lse.ptr)), (1, (out.ptr, lse.ptr, bdo.ptr, dq.ptr, dk.ptr, dv.ptr))):
        need = hipdev.lib.limn_hip_attend_workspace(ABI_CODE[t], *sizes, backward)
        ws = hipdev._alloc(max(need, 1))
        entry = hipdev.lib.limn_hip_attend_bwd if backward else hipdev.lib.limn_hip_attend_fwd
        runtime.check_limn(entry(*head, *buffers, *tail, ws.ptr, need, None))
        hipdev.finish()
    want = definition(q, k, v, dout=do, dtype=dtype, causal=True, slopes=slopes)
    within(from_storage(hipdev.copyout(out), t, q.shape), *want["out"], "out")
    within(hipdev.copyout(lse).view(np.float32).reshape(1, heads, t_q), *want["lse"], "lse")
    within(from_storage(hipdev.copyout(dq), t, q.shape), *want["dq"], "dq")
    for name, b in (("dk", dk), ("dv", dv)):
        raw = hipdev.copyout(b)
        within(from_storage(raw[: live * hd * t.itemsize], t, k.shape), *want[name], name)
        assert not raw[live * hd * t.itemsize :].any(), name
    del padded, dk, dv, ws
    hipdev.trim()
