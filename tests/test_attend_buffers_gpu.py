"""limn_hip_attend_fwd and limn_hip_attend_bwd on buffers aligned to their elements alone, on a stream of the caller's, and at
the number of positions from which on the tiled kernels hand over to the general ones."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

from conftest import DTYPES
from limn_amd.dtypes import ABI_CODE, from_storage, to_storage
from limn_amd.hip import runtime
from limn_amd.seam import float32, int32
from oracle.attend import attend as definition
from oracle.attend import within
from test_attend_gpu import draw, packed

pytestmark = pytest.mark.gpu

GUARD = 512
RULES = ("slopes", "documents", "prefix", "lengths")


def both(dev, q, k, v, do, dtype, rules, causal=True, softcap=0.0, shift=0, stream=None):
    """Forward and backward with every typed buffer `shift` bytes past an allocation's start, guards on both of its sides, and
    workspaces that begin as NaN."""
    t = DTYPES[dtype]
    batch, heads, t_q, hd = q.shape
    kv_heads, t_k, hd_v = v.shape[1:]
    sizes = (batch, heads, kv_heads, t_q, t_k, hd, hd_v)

    def put(values, kind, at=0):
        host = to_storage(values, kind).view(np.uint8).reshape(-1)
        buf = dev._alloc(host.nbytes + at + GUARD)
        dev.copyin(buf, np.concatenate([np.full(at, 0xAB, np.uint8), host, np.full(GUARD, 0xAB, np.uint8)]))
        return buf

    ins = [put(x, t, shift) for x in (q, k, v, do)]
    given = [put(rules[n], float32 if n == "slopes" else int32) if n in rules else None for n in RULES]
    shapes = dict(out=(do.shape, t), lse=(q.shape[:3], float32), dq=(q.shape, t), dk=(k.shape, t), dv=(v.shape, t))
    at = {n: 4 * (shift > 0) if n == "lse" else shift for n in shapes}
    outs = {n: dev._alloc(int(np.prod(s)) * kind.itemsize + at[n] + GUARD) for n, (s, kind) in shapes.items()}
    for b in outs.values():
        dev.copyin(b, np.full(b.nbytes, 0xAB, np.uint8))
    ptr = {n: b.ptr + at[n] for n, b in outs.items()}
    head = [b.ptr + shift for b in ins[:3]] + [b.ptr if b else None for b in given]
    tail = (ABI_CODE[t], *sizes, int(causal), hd**-0.5, softcap)
    spaces = []
    for backward in (0, 1):
        need = dev.lib.limn_hip_attend_workspace(ABI_CODE[t], *sizes, backward)
        ws = dev._alloc(need + GUARD)
        dev.copyin(ws, np.concatenate([np.full(need, 0xFF, np.uint8), np.full(GUARD, 0xAB, np.uint8)]))
        spaces.append((ws, need))
    dev.finish()
    (ws, need), (ws_b, need_b) = spaces
    runtime.check_limn(dev.lib.limn_hip_attend_fwd(*head, ptr["out"], ptr["lse"], *tail, ws.ptr, need, stream))
    runtime.check_limn(dev.lib.limn_hip_attend_bwd(*head, ptr["out"], ptr["lse"], ins[3].ptr + shift, *(ptr[n] for n in ("dq", "dk", "dv")), *tail, ws_b.ptr, need_b, stream))
    if stream is None:
        dev.finish()
    else:
        runtime.check(dev.api.hipStreamSynchronize(stream), "waiting for a stream")
    for w, n in spaces:
        assert (dev.copyout(w)[n:] == 0xAB).all()
    got = {}
    for n, (shape, kind) in shapes.items():
        raw, size = dev.copyout(outs[n]), int(np.prod(shape)) * kind.itemsize
        assert (raw[: at[n]] == 0xAB).all() and (raw[at[n] + size :] == 0xAB).all(), n
        got[n] = from_storage(raw[at[n] : at[n] + size].copy(), kind, shape)
    return got


def check(got, want, batch):
    for name, x in got.items():
        within(x[:batch], *want[name], name)
        for r in range(batch, len(x), batch):
            np.testing.assert_array_equal(x[r : r + batch], x[:batch])


@pytest.mark.parametrize("dtype,shift", [("bfloat16", 2), ("bfloat16", 8), ("float16", 2), ("float16", 8), ("float32", 4), ("float32", 8)])
@pytest.mark.parametrize("hd", [64, 100, 128])
@pytest.mark.parametrize("heads,kv_heads,t_q,t_k,names", [(4, 1, 1, 300, "lengths slopes"), (2, 2, 3, 2100, "lengths"), (4, 2, 190, 190, "documents"), (2, 1, 130, 1100, "prefix"), (4, 4, 300, 300, "")])
def test_buffers_aligned_to_their_elements(hipdev, dtype, shift, hd, heads, kv_heads, t_q, t_k, names):
    rng, (q, k, v, do) = draw(t_q + hd, dtype, 2, heads, kv_heads, t_q, t_k, hd, hd)
    every = dict(documents=packed(rng, 2, t_k, 60), prefix=np.array([70, 0], np.int32), lengths=np.array([t_k, t_k // 2 + 5], np.int32),
                 slopes=(0.5 ** np.arange(1, heads + 1)).astype(np.float32))
    rules = {n: every[n] for n in names.split()}
    got = both(hipdev, q, k, v, do, dtype, rules, softcap=5.0 * (hd == 64), shift=shift)
    check(got, definition(q, k, v, dout=do, dtype=dtype, causal=True, softcap=5.0 * (hd == 64), **rules), 2)


def test_float32_buffers_of_as_many_rows_as_the_tiles_take(hipdev):
    _, (q, k, v, do) = draw(3, "float32", 1, 4, 2, 200, 200, 64, 64)
    many = [np.tile(x, (10, 1, 1, 1)) for x in (q, k, v, do)]
    want = definition(q, k, v, dout=do, dtype="float32", causal=True)
    for shift in (0, 4):
        check(both(hipdev, *many, "float32", {}, shift=shift), want, 1)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("heads,kv_heads,t_q,t_k", [(4, 1, 1, 5000), (4, 2, 333, 333), (8, 1, 70, 2100)])
def test_a_stream_of_the_callers(hipdev, dtype, heads, kv_heads, t_q, t_k):
    rng, (q, k, v, do) = draw(t_k, dtype, 1, heads, kv_heads, t_q, t_k, 128, 128)
    rules = dict(documents=packed(rng, 1, t_k, 900)) if t_q == t_k else dict(lengths=np.array([t_k - 9], np.int32))
    stream = ctypes.c_void_p()
    runtime.check(hipdev.api.hipStreamCreateWithFlags(ctypes.byref(stream), 1), "creating a stream")  # hipStreamNonBlocking
    try:
        for _ in range(3):
            got = both(hipdev, q, k, v, do, dtype, rules, softcap=4.0, stream=stream)
    finally:
        runtime.check(hipdev.api.hipStreamDestroy(stream), "destroying a stream")
    check(got, definition(q, k, v, dout=do, dtype=dtype, causal=True, softcap=4.0, **rules), 1)


@pytest.mark.parametrize("dtype,hd", [("bfloat16", 64), ("float16", 128)])
@pytest.mark.parametrize("t_k", [1 << 17, (1 << 17) + 1])
def test_positions_past_the_tiles_lists(hipdev, dtype, hd, t_k):
    """131072 positions fill the lists of streamed tiles; one more goes to the general kernels. Documents of some 40000."""
    rng, (q, k, v, do) = draw(t_k % 1000, dtype, 1, 1, 1, 140, t_k, hd, hd)
    rules = dict(documents=packed(rng, 1, t_k, 40000, padded=False), prefix=np.array([1000], np.int32))
    rules["documents"][0, 500:2000] = rules["documents"][0, -1]
    got = both(hipdev, q, k, v, do, dtype, rules)
    check(got, definition(q, k, v, dout=do, dtype=dtype, causal=True, **rules), 1)
    del rules["documents"]
    got = both(hipdev, q, k, v, do, dtype, dict(lengths=np.array([t_k - 70], np.int32)), softcap=4.0)
    check(got, definition(q, k, v, dout=do, dtype=dtype, causal=True, softcap=4.0, lengths=np.array([t_k - 70], np.int32)), 1)
