"""limn_hip_attend_fwd and limn_hip_attend_bwd on buffers of their own: workspaces that begin as NaN, so that nothing is read
before it is written, and guard bytes behind every output and workspace that must stay."""

from __future__ import annotations

import numpy as np
import pytest

from conftest import DTYPES, upload
from limn_amd.dtypes import ABI_CODE, from_storage
from limn_amd.hip import runtime
from limn_amd.seam import float32, int32
from oracle.attend import attend as definition
from oracle.attend import within
from test_attend_gpu import draw, packed

pytestmark = pytest.mark.gpu

GUARD = 512


def called(dev, q, k, v, do, dtype, rules, causal, softcap):
    t = DTYPES[dtype]
    batch, heads, t_q, hd = q.shape
    kv_heads, t_k, hd_v = v.shape[1:]
    sizes = (batch, heads, kv_heads, t_q, t_k, hd, hd_v)
    ins = [upload(dev, x, t).arg for x in (q, k, v)]
    grad_out = upload(dev, do, t).arg
    given = [upload(dev, rules[n], float32 if n == "slopes" else int32).arg if n in rules else None for n in ("slopes", "documents", "prefix", "lengths")]
    shapes = dict(out=(do.shape, t), lse=(q.shape[:3], float32), dq=(q.shape, t), dk=(k.shape, t), dv=(v.shape, t))
    sized = {n: int(np.prod(s)) * kind.itemsize for n, (s, kind) in shapes.items()}
    outs = {n: dev._alloc(nb + GUARD) for n, nb in sized.items()}
    for b in outs.values():
        dev.copyin(b, np.full(b.nbytes, 0xAB, np.uint8))
    head = [b.ptr for b in ins] + [b.ptr if b else None for b in given]
    tail = (ABI_CODE[t], *sizes, int(causal), hd**-0.5, softcap)
    for backward in (0, 1):
        need = dev.lib.limn_hip_attend_workspace(ABI_CODE[t], *sizes, backward)
        ws = dev._alloc(need + GUARD)
        fill = np.full(need + GUARD, 0xFF, np.uint8)
        fill[need:] = 0xAB
        dev.copyin(ws, fill)
        if backward:
            status = dev.lib.limn_hip_attend_bwd(*head, outs["out"].ptr, outs["lse"].ptr, grad_out.ptr, *(outs[n].ptr for n in ("dq", "dk", "dv")), *tail, ws.ptr, need, None)
        else:
            status = dev.lib.limn_hip_attend_fwd(*head, outs["out"].ptr, outs["lse"].ptr, *tail, ws.ptr, need, None)
        runtime.check_limn(status)
        dev.finish()
        assert (dev.copyout(ws)[need:] == 0xAB).all()
    got = {}
    for n, (shape, kind) in shapes.items():
        raw = dev.copyout(outs[n])
        assert (raw[sized[n] :] == 0xAB).all(), n
        got[n] = from_storage(raw[: sized[n]], kind, shape)
    return got


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("hd", [64, 88, 128])
@pytest.mark.parametrize("heads,kv_heads,t_q,t_k,causal,softcap,names", [
    (4, 4, 333, 333, True, 0.0, ""), (4, 1, 333, 333, True, 5.0, "documents"), (4, 2, 200, 777, True, 0.0, "documents prefix"),
    (2, 2, 190, 475, False, 0.0, "documents lengths"), (4, 2, 257, 300, True, 0.0, "lengths prefix slopes"), (8, 1, 640, 641, True, 4.0, "documents lengths slopes")])
def test_nothing_is_read_before_it_is_written(hipdev, dtype, hd, heads, kv_heads, t_q, t_k, causal, softcap, names):
    rng, (q, k, v, do) = draw(heads + t_q + hd, dtype, 2, heads, kv_heads, t_q, t_k, hd, hd)
    every = dict(documents=packed(rng, 2, t_k, 60), prefix=np.array([70, 0], np.int32), lengths=np.array([t_k, t_k // 2 + 5], np.int32),
                 slopes=(0.5 ** np.arange(1, heads + 1)).astype(np.float32))
    rules = {n: every[n] for n in names.split()}
    reps = 256 // (2 * heads * ((t_q + 31) // 32)) + 1 if dtype == "float32" else 1  # float32: as many tiles as the tiled kernels take
    many = lambda x: np.tile(x, (reps, *[1] * (x.ndim - 1)))  # noqa: E731
    got = called(hipdev, *(many(x) for x in (q, k, v, do)), dtype, {n: x if n == "slopes" else many(x) for n, x in rules.items()}, causal, softcap)
    want = definition(q, k, v, dout=do, dtype=dtype, causal=causal, softcap=softcap, **rules)
    for name, x in got.items():
        within(x[:2], *want[name], f"{name} {dtype}")
        for r in range(1, reps):
            np.testing.assert_array_equal(x[2 * r : 2 * r + 2], x[:2])
