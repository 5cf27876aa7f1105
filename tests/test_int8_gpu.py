"""quantize_rows and int8_linear on the MI355X: the C ABI and limn_amd.int8 on the hip device, against the definition (oracle/serving.py)."""

from __future__ import annotations

import numpy as np
import pytest

from conftest import DTYPES, download, storage_values, upload
from limn_amd.dtypes import ABI_CODE, from_storage
from limn_amd.hip import runtime
from limn_amd.int8 import int8_linear, quantize_rows
from limn_amd.seam import Tensor, capture, float32, int8, realize, use_device
from oracle.attend import within
from oracle.serving import int8_linear as oracle
from oracle.serving import quantized

pytestmark = pytest.mark.gpu
TYPES = ["float32", "bfloat16", "float16"]
GUARD = 256


def layer(seed, dtype, rows, width, outputs, bias=False, std=1.0):
    rng = np.random.default_rng(seed)
    stored = lambda *shape: storage_values((rng.standard_normal(shape) * std).astype(np.float32), DTYPES[dtype])  # noqa: E731
    w = rng.integers(-127, 128, (outputs, width)).astype(np.int8)
    return stored(rows, width), w, (rng.random(outputs) * 0.01 + 0.001).astype(np.float32), stored(outputs) if bias else None


def called(dev, x, w, scales, bias, dtype, shift=0, w_shift=0):
    """limn_hip_int8_linear; x and the bias `shift` elements, the weight `w_shift` bytes behind their buffers' starts."""
    t, (rows, width), outputs = DTYPES[dtype], x.shape, len(w)
    off = lambda a: upload(dev, np.concatenate([np.full(shift, np.nan, np.float32), a.reshape(-1)]), t).arg  # noqa: E731
    xs, ss, bs = off(x), upload(dev, scales, float32).arg, None if bias is None else off(bias)
    ws8 = upload(dev, np.concatenate([np.full(w_shift, 77, np.int8), w.reshape(-1)]), int8).arg
    need = dev.lib.limn_hip_int8_linear_workspace(ABI_CODE[t], rows, width, outputs)
    ws, out = dev._alloc(need + GUARD), dev._alloc(rows * outputs * t.itemsize + GUARD)
    dev.copyin(ws, np.full(ws.nbytes, 0xFF, np.uint8))
    dev.copyin(out, np.full(out.nbytes, 0xAB, np.uint8))
    at = lambda b: None if b is None else b.ptr + shift * t.itemsize  # noqa: E731
    runtime.check_limn(dev.lib.limn_hip_int8_linear(at(xs), ws8.ptr + w_shift, ss.ptr, at(bs), out.ptr, ABI_CODE[t], rows, width, outputs, ws.ptr, need, None))
    dev.finish()
    raw = dev.copyout(out)
    assert (raw[rows * outputs * t.itemsize :] == 0xAB).all() and (dev.copyout(ws)[need:] == 0xFF).all()
    return from_storage(raw[: rows * outputs * t.itemsize], t, (rows, outputs))


def check(dev, x, w, scales, bias, dtype, **kw):
    got = called(dev, x, w, scales, bias, dtype, **kw)
    within(got, *oracle(x, w, scales, bias, dtype), f"y {dtype}")
    return got


SIZES = [(1, 1, 1), (1, 64, 64), (3, 24, 17), (1, 760, 1000), (16, 512, 1536), (17, 128, 33), (32, 1000, 300), (33, 257, 65), (64, 4096, 128), (65, 130, 513), (130, 96, 1025), (257, 777, 129),
         (300, 1536, 512), (1021, 48, 257), (5, 20000, 40), (2100, 300, 2049), (4100, 70, 4099), (1, 512, 300), (2, 4096, 64), (3, 1024, 1000), (16, 512, 33), (2, 8192, 40), (1, 8192, 17), (5, 1536, 16385), (7, 48, 2048)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,width,outputs", SIZES)
def test_sizes(hipdev, rows, width, outputs, dtype):
    check(hipdev, *layer(rows + width, dtype, rows, width, outputs, bias=rows % 2 == 1), dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shift,w_shift", [(1, 0), (0, 1), (3, 4), (8, 16)])
def test_shifted_buffers(hipdev, shift, w_shift, dtype):
    for size in ((4, 512, 100), (200, 512, 300), (40, 100, 77)):
        check(hipdev, *layer(5, dtype, *size, bias=True), dtype, shift=shift, w_shift=w_shift)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [3, 150])
def test_numbers_of_every_size(hipdev, rows, dtype):
    """Rows of zeros, of the type's least and largest numbers, of one number beside zeros."""
    x, w, s, b = layer(6, dtype, rows, 200, 90, bias=True)
    info = dict(float32=(1e-38, 1e37, 1e-45), bfloat16=(1e-38, 1e37, 1e-40), float16=(6e-8, 6e4, 6e-8))[dtype]
    x[0] = 0
    x[1] = storage_values(x[1] * np.float32(info[0]), DTYPES[dtype])
    x[2] = storage_values(np.clip(x[2], -1, 1) * np.float32(info[1]), DTYPES[dtype])
    if rows > 3:
        x[3], x[4] = 0, storage_values(np.full(200, info[2], np.float32), DTYPES[dtype])
        x[3, 77] = 2.0
    check(hipdev, x, w, s, None if dtype == "float32" else b, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [6, 200])
def test_rows_with_infinities_and_nan(hipdev, rows, dtype):
    """They are NaN, and no other row is."""
    x, w, s, _ = layer(7, dtype, rows, 300, 70)
    x[1, 3], x[2, 299], x[4, 0] = np.inf, np.nan, -np.inf
    got = check(hipdev, x, w, s, None, dtype)
    assert np.isnan(got[[1, 2, 4]]).all() and np.isfinite(np.delete(got, [1, 2, 4], 0)).all()


def test_sums_are_exact_at_the_widest(hipdev):
    """2^17 products of 127 and -128."""
    x, w = np.full((2, 1 << 17), 1.0, np.float32), np.full((33, 1 << 17), -128, np.int8)
    x[1] = -1
    w[1] = 127
    got = check(hipdev, x, w, np.full(33, 1.0, np.float32), None, "float32")
    assert np.unique(np.abs(got)).size == 2


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,width", [(1, 1), (5, 17), (300, 129), (7, 4096), (2, 70001)])
def test_quantized_rows(hipdev, rows, width, dtype):
    use_device(hipdev)
    x, _, _, _ = layer(8, dtype, rows, width, 1)
    if rows > 4:
        x[1], x[2, width // 2], x[3] = 0, np.nan, storage_values(np.full(width, 1e-30, np.float32), DTYPES[dtype])
    values, scales = quantize_rows(Tensor.from_node(upload(hipdev, x, DTYPES[dtype])))
    v, s = realize(values, scales)
    want, ws = quantized(x)
    np.testing.assert_array_equal(download(hipdev, v, int8, x.shape), want)
    np.testing.assert_array_equal(download(hipdev, s, float32, (rows,)), ws)


def test_through_the_tensor_api_captured(hipdev):
    use_device(hipdev)
    t = DTYPES["bfloat16"]
    x, w, s, b = layer(9, "bfloat16", 30, 256, 500, bias=True)
    w8, ws, bt = (Tensor.from_node(upload(hipdev, a, kind)) for a, kind in ((w, int8), (s, float32), (b, t)))

    def step(x):
        y = int8_linear(x, w8, ws, bt)
        realize(y)
        return y

    run = capture(step)
    rng = np.random.default_rng(10)
    for _ in range(6):
        x = storage_values(rng.standard_normal((5, 6, 256)).astype(np.float32), t)
        y = run(Tensor.from_node(upload(hipdev, x, t)))
        within(y.numpy().reshape(30, 500), *oracle(x.reshape(30, 256), w, s, b, "bfloat16"), "y")
        assert (Tensor(np.ones(1000)) * 3.0).sum().item() == 3000.0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,width,outputs", [(1, 512, 300), (2, 1024, 77), (3, 320, 64), (7, 1040, 33), (16, 512, 1000)])
def test_few_rows_have_the_bits_of_many(hipdev, rows, width, outputs, dtype):
    """Rows alone and among forty, rows of zeros, infinities, NaN, the least and the largest numbers among them."""
    x, w, s, b = layer(11, dtype, 40, width, outputs, bias=True)
    t = np.float16 if dtype == "float16" else np.float32
    for r, value in enumerate([None, 0.0, np.inf, np.nan, None, float(np.finfo(t).max) / 2, float(np.finfo(t).tiny), -np.inf]):
        if value is not None:
            x[r, : width if value == 0 else 3] = value
    many = called(hipdev, x, w, s, b, dtype)
    for first in (0, 1, 2, 5):
        got = called(hipdev, x[first : first + rows], w, s, b, dtype)
        np.testing.assert_array_equal(got, many[first : first + rows])
