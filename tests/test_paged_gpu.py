"""attend_paged on the MI355X: the C ABI and limn_amd.paged on the hip device, against the definition in float64 within the bounds on
rounding that oracle/serving.py derives. Every output has guard bytes behind it that must stay."""

from __future__ import annotations

import numpy as np
import pytest

from conftest import DTYPES, download, upload
from limn_amd.dtypes import ABI_CODE, from_storage, to_storage
from limn_amd.hip import runtime
from limn_amd.paged import attend_paged
from limn_amd.seam import Tensor, capture, float32, int32, realize, use_device
from oracle.attend import within
from oracle.serving import paged, same_kind
from serving import paged_inputs

pytestmark = pytest.mark.gpu
TYPES = ["float32", "bfloat16", "float16"]
GUARD = 256


def called(dev, x, dtype, softcap=0.0, scale=None, apart=0, shift=0):
    """limn_hip_attend_paged on buffers of its own: rows `apart` elements further apart than they are long, q `shift` elements
    behind its buffer's start."""
    t = DTYPES[dtype]
    (tokens, heads, hd), (pages, kv, page, _) = x["q"].shape, x["key_pages"].shape
    scale = hd**-0.5 if scale is None else scale

    def rows(a):
        if a is None:
            return None
        wide = np.full((tokens, a.shape[1] * hd + apart), np.nan, np.float32)
        wide[:, : a.shape[1] * hd] = a.reshape(tokens, -1)
        flat = np.concatenate([np.full(shift, np.nan, np.float32), wide.reshape(-1)])
        return upload(dev, flat, t).arg

    q, k, v = rows(x["q"]), rows(x["k"]), rows(x["v"])
    ints = [upload(dev, x[n], int32).arg for n in ("starts", "lengths", "table")]
    slopes = None if x["slopes"] is None else upload(dev, x["slopes"], float32).arg
    nb = {"out": x["q"].size * t.itemsize, "keys": x["key_pages"].size * t.itemsize, "values": x["key_pages"].size * t.itemsize}
    outs = {n: dev._alloc(b + GUARD) for n, b in nb.items()}
    for n, b in outs.items():
        raw = np.full(b.nbytes, 0xAB, np.uint8)
        if n != "out":
            raw[: nb[n]] = to_storage(x["key_pages" if n == "keys" else "value_pages"], t).view(np.uint8).reshape(-1)
        dev.copyin(b, raw)
    sizes = (tokens, len(x["lengths"]), heads, kv, hd, pages, page, x["table"].shape[1])
    need = dev.lib.limn_hip_attend_paged_workspace(ABI_CODE[t], *sizes)
    ws = dev._alloc(need + GUARD)
    dev.copyin(ws, np.full(ws.nbytes, 0xFF, np.uint8))  # NaN, should any of it be read before it is written
    at = lambda b: None if b is None else b.ptr + shift * t.itemsize  # noqa: E731
    runtime.check_limn(dev.lib.limn_hip_attend_paged(at(q), at(k), at(v), outs["keys"].ptr, outs["values"].ptr, *(b.ptr for b in ints), None if slopes is None else slopes.ptr,
                                                     outs["out"].ptr, ABI_CODE[t], *sizes, heads * hd + apart, kv * hd + apart, kv * hd + apart, scale, softcap, ws.ptr, need, None))
    dev.finish()
    assert (dev.copyout(ws)[need:] == 0xFF).all()
    got = {}
    for n, b in outs.items():
        raw = dev.copyout(b)
        assert (raw[nb[n] :] == 0xAB).all(), n
        got[n] = from_storage(raw[: nb[n]], t, x["q"].shape if n == "out" else x["key_pages"].shape)
    return got


def check(dev, x, dtype, softcap=0.0, scale=None, **kw):
    got = called(dev, x, dtype, softcap, scale, **kw)
    (want, bound), keys, values = paged(**x, softcap=softcap, scale=scale, dtype=dtype)
    within(same_kind(got["out"], want), want, bound, f"out {dtype}")
    np.testing.assert_array_equal(got["keys"], keys)
    np.testing.assert_array_equal(got["values"], values)
    return got


CASES = [
    dict(counts=(1,), lengths=(1,), hd=16, heads=1),
    dict(counts=(1,), lengths=(33,), hd=64, heads=8, page=16),
    dict(counts=(1, 1, 1), lengths=(700, 1, 64), hd=64, heads=8, kv_heads=2, page=16),
    dict(counts=(1,) * 9, lengths=(1, 2, 31, 32, 33, 63, 64, 65, 300), hd=128, heads=16, kv_heads=2, page=24),
    dict(counts=(1, 1), lengths=(2600, 90), hd=128, heads=10, kv_heads=2, page=32, slopes=True),
    dict(counts=(5, 1, 0, 2), lengths=(300, 17, 9, 2), hd=40, heads=6, kv_heads=2, page=8, spare=3, rows_before=2),
    dict(counts=(16,), lengths=(16,), hd=80, heads=4, kv_heads=4, page=5),
    dict(counts=(70, 1), lengths=(500, 400), hd=128, heads=8, kv_heads=2, page=48),
    dict(counts=(130, 1, 257), lengths=(130, 1000, 900), hd=64, heads=4, kv_heads=2, page=16, spare=5),
    dict(counts=(300,), lengths=(1500,), hd=96, heads=3, kv_heads=1, page=64, slopes=True),
    dict(counts=(129, 3), lengths=(200, 64), hd=72, heads=2, page=256),
    dict(counts=(9, 130), lengths=(4, 100), hd=64, heads=2, page=16),  # more rows than positions
    dict(counts=(2, 3), lengths=(1000, 50), hd=64, heads=2, page=16, table_pages=5),  # past the table
    dict(counts=(20, 2), lengths=(40, 90), hd=33, heads=3, page=7),  # a head dim of the general kernel
    dict(counts=(3, 1), lengths=(40, 200), hd=200, heads=2, page=16),
    dict(counts=(2,), lengths=(9,), hd=1, heads=2, page=1),
    dict(counts=(64,) * 3, lengths=(64, 300, 65), hd=32, heads=20, kv_heads=4, page=1),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", CASES, ids=str)
def test_sizes(hipdev, case, dtype):
    check(hipdev, paged_inputs(len(str(case)), dtype=dtype, **case), dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cap", [0.5, 30.0, 1000.0])
@pytest.mark.parametrize("case", [CASES[3], CASES[5], CASES[8], CASES[9], CASES[13]], ids=str)
def test_caps(hipdev, case, cap, dtype):
    check(hipdev, paged_inputs(7, dtype=dtype, std=4.0, **case), dtype, softcap=cap)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", [CASES[2], CASES[7], CASES[8]], ids=str)
@pytest.mark.parametrize("scale", [0.0, -0.3, 2.0**-110, 3.0])
def test_scales(hipdev, case, scale, dtype):
    check(hipdev, paged_inputs(8, dtype=dtype, **case), dtype, scale=scale)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("apart,shift", [(8, 8), (1, 0), (0, 3), (16, 0)])
def test_rows_apart_and_shifted(hipdev, apart, shift, dtype):
    """The rows of one projection, and starts that are aligned to an element alone."""
    for case in (CASES[2], CASES[7]):
        check(hipdev, paged_inputs(9, dtype=dtype, **case), dtype, apart=apart, shift=shift)


def spoil(x, pages=(), tail=True):
    """Infinities and NaN wherever nothing may be read: pages of nobody, places behind the last position, rows of no sequence."""
    kv_heads, page = x["key_pages"].shape[1:3]
    used = set()
    for s, length in enumerate(x["lengths"]):
        for t, p in enumerate(x["table"][s]):
            if p >= 0 and t * page < length:
                used.add(int(p))
                if length < (t + 1) * page:
                    for pool, bad in (("key_pages", np.nan), ("value_pages", np.inf)):
                        x[pool][p, :, length - t * page :] = bad
    for p in set(range(len(x["key_pages"]))) - used:
        x["key_pages"][p], x["value_pages"][p] = np.inf, np.nan
    for r in range(len(x["q"])):
        if not x["starts"][0] <= r < x["starts"][-1]:
            for n in "qkv":
                x[n][r] = np.nan
    return x


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", CASES[1:14], ids=str)
def test_what_nobody_sees_changes_nothing(hipdev, case, dtype):
    check(hipdev, spoil(paged_inputs(10, dtype=dtype, **case)), dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", [CASES[5], CASES[7], CASES[8], CASES[9], CASES[13]], ids=str)
def test_later_tokens_change_nothing_in_earlier_rows(hipdev, case, dtype):
    """Infinities and NaN in the keys and values of some new tokens: rows before them stay as they are."""
    x = paged_inputs(11, dtype=dtype, **case)
    for s in range(len(case["counts"])):
        b, e = x["starts"][s], x["starts"][s + 1]
        if e - b > 2:
            x["v"][b + (e - b) // 2, :, ::3] = np.inf
            x["v"][e - 1], x["k"][e - 1] = np.nan, np.nan
    got = check(hipdev, x, dtype)
    assert np.isfinite(got["out"]).any() and not np.isfinite(got["out"]).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", [CASES[2], CASES[3], CASES[5], CASES[8], CASES[9], CASES[13]], ids=str)
def test_bad_pages(hipdev, case, dtype):
    """Page numbers outside the cache: holes among the old keys, new tokens' pages, a whole sequence."""
    x = paged_inputs(12, dtype=dtype, **case)
    x["table"][0, 0] = 2**31 - 1
    x["table"][0, -1] = -1
    if x["table"].shape[1] > 3:
        x["table"][-1, 2] = len(x["key_pages"])
        x["table"][-1, 3] = -(2**31)
    if len(x["table"]) > 2:
        x["table"][1] = -1
    check(hipdev, x, dtype)


@pytest.mark.parametrize("dtype", TYPES)
def test_odd_lengths_and_starts(hipdev, dtype):
    """Lengths below zero and past the table, starts outside the tokens."""
    x = paged_inputs(13, dtype=dtype, counts=(2, 70, 1), lengths=(40, 90, 30), hd=64, heads=4, kv_heads=2, page=16)
    x["lengths"][0], x["lengths"][2] = -7, 2**31 - 1
    x["starts"] = np.array([-5, 2, 72, 2**31 - 1], np.int32)
    check(hipdev, x, dtype)


@pytest.mark.parametrize("dtype", TYPES)
def test_shared_pages_and_a_cache_that_holds_the_tokens(hipdev, dtype):
    x = paged_inputs(14, dtype=dtype, counts=(1, 1, 80), lengths=(200, 150, 240), hd=64, heads=4, kv_heads=2, page=16)
    x["table"][1, :8] = x["table"][2, :8] = x["table"][0, :8]  # a common beginning
    check(hipdev, x, dtype)
    x["k"] = x["v"] = None
    check(hipdev, x, dtype)


def test_two_calls_give_the_same_bits(hipdev):
    x = paged_inputs(15, dtype="bfloat16", counts=(1, 200, 3), lengths=(3000, 2000, 900), hd=128, heads=8, kv_heads=2, page=16)
    a, b = (called(hipdev, x, "bfloat16")["out"] for _ in range(2))
    np.testing.assert_array_equal(a, b)


def tensors(dev, x, dtype):
    kinds = dict(starts=int32, lengths=int32, table=int32, slopes=float32)
    return {n: None if a is None else Tensor.from_node(upload(dev, a, kinds.get(n, DTYPES[dtype]))) for n, a in x.items()}


@pytest.mark.parametrize("dtype", TYPES)
def test_through_the_tensor_api(hipdev, dtype):
    use_device(hipdev)
    x = paged_inputs(16, dtype=dtype, counts=(1, 9, 1), lengths=(50, 40, 9), hd=64, heads=4, kv_heads=2, page=16, spare=2, slopes=True)
    t = tensors(hipdev, x, dtype)
    out = attend_paged(**t, softcap=20.0)
    (got,) = realize(out)
    (want, bound), keys, values = paged(**x, softcap=20.0, dtype=dtype)
    within(download(hipdev, got, DTYPES[dtype], x["q"].shape), want, bound, "out")
    np.testing.assert_array_equal(download(hipdev, t["key_pages"].node.arg, DTYPES[dtype], x["key_pages"].shape), keys)
    np.testing.assert_array_equal(download(hipdev, t["value_pages"].node.arg, DTYPES[dtype], x["key_pages"].shape), values)


def test_captured_steps_grow_the_cache(hipdev):
    """A captured step replayed over a growing sequence, other work between the replays: every step against the definition with the
    cache as it is by then."""
    use_device(hipdev)
    x = paged_inputs(17, dtype="bfloat16", counts=(1, 1), lengths=(12, 1), hd=64, heads=4, kv_heads=2, page=8, table_pages=4)
    x["table"][:] = np.arange(8).reshape(2, 4)
    pools = {n: Tensor.from_node(upload(hipdev, x[n], DTYPES["bfloat16"])) for n in ("key_pages", "value_pages")}

    def step(q, k, v, starts, lengths, table):
        out = attend_paged(q, k, v, pools["key_pages"], pools["value_pages"], starts, lengths, table)
        scaled = out * 2.0
        realize(out, scaled)
        return out, scaled

    run = capture(step)
    rng = np.random.default_rng(18)
    for i in range(8):
        for n in "qkv":
            x[n] = from_storage(to_storage(rng.standard_normal(x[n].shape).astype(np.float32), DTYPES["bfloat16"]).view(np.uint8).reshape(-1), DTYPES["bfloat16"], x[n].shape)
        x["lengths"] += 1
        t = tensors(hipdev, {n: x[n] for n in ("q", "k", "v", "starts", "lengths", "table")}, "bfloat16")
        out, scaled = run(*t.values())
        (want, bound), x["key_pages"], x["value_pages"] = paged(**x, dtype="bfloat16")
        within(out.numpy(), want, bound, f"step {i}")
        within(scaled.numpy(), 2 * out.numpy(), 0.0, f"step {i}")
        assert (Tensor(np.ones(1000)) * 3.0).sum().item() == 3000.0


def test_a_longer_cache_than_32_bits_reach(hipdev):
    """Pools past 2^32 bytes: a sequence whose pages lie at both ends."""
    t, kv, page, hd = DTYPES["bfloat16"], 8, 256, 128
    pages = (1 << 32) // (kv * page * hd * 2) + 40
    x = paged_inputs(19, dtype="bfloat16", counts=(1, 70), lengths=(600, 700), heads=8, hd=hd, page=page)
    small = x["key_pages"].shape[0]
    where = np.concatenate([[pages - 1, pages - 20], np.arange(1, small - 2), [pages - 5]])[:small]
    pools = {}
    for n in ("key_pages", "value_pages"):
        pools[n] = hipdev._alloc(pages * kv * page * hd * 2)
        for i, p in enumerate(where):
            raw = to_storage(x[n][i], t).view(np.uint8).reshape(-1)
            runtime.check(hipdev.api.hipMemcpy(pools[n].ptr + int(p) * raw.nbytes, raw.ctypes.data, raw.nbytes, 1), "uploading a page")
    table = np.where(x["table"] >= 0, where[np.maximum(x["table"], 0)], -1).astype(np.int32)
    bufs = [upload(hipdev, x[n], t).arg for n in "qkv"]
    ints = [upload(hipdev, a, int32).arg for a in (x["starts"], x["lengths"], table)]
    out = hipdev._alloc(x["q"].size * 2)
    sizes = (71, 2, 8, 8, hd, pages, page, table.shape[1])
    need = hipdev.lib.limn_hip_attend_paged_workspace(3, *sizes)
    ws = hipdev._alloc(need)
    runtime.check_limn(hipdev.lib.limn_hip_attend_paged(*(b.ptr for b in bufs), pools["key_pages"].ptr, pools["value_pages"].ptr, *(b.ptr for b in ints), None, out.ptr, 3, *sizes,
                                                        8 * hd, kv * hd, kv * hd, hd**-0.5, 0.0, ws.ptr, need, None))
    hipdev.finish()
    (want, bound), _, _ = paged(**x, dtype="bfloat16")
    within(download(hipdev, out, t, x["q"].shape), want, bound, "out")
    del pools
    hipdev.trim()
