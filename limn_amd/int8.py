"""Linear layers in 8-bit integers, for answering with a trained model: half the weight's bytes, twice the matrix rate.

`quantize_rows` brings the rows of a weight to 8 bits once, a scale each; `int8_linear` brings the rows of its input to 8 bits
as they come, a scale for each token, and multiplies in whole numbers:

    s = max(max |x| / 127, 2^-126),   x8 = round(x / s),   y = (x8 . w8) s scale + bias.

Both are CUSTOM kernels ("quantize_rows", "int8_linear": `limn_hip_quantize_rows` and `limn_hip_int8_linear` of
include/limn_hip.h) where the active device registers them, and composed from limn's primitives elsewhere and for float64 (x / s
there is a product with 1 / s, which rounds a number at the border of two the other way now and then).
"""

from __future__ import annotations

import math

from limn_amd.attend import contiguous, records
from limn_amd.seam import FLOATS, Tensor, active_device, custom, float32, float64, int8, int32, promote

QUANTIZE_ROWS, INT8_LINEAR = "quantize_rows", "int8_linear"
WIDEST = 1 << 17  # products of 127 * 128 whose sum a 32-bit integer holds


def quantize_rows(x: Tensor) -> tuple[Tensor, Tensor]:
    """x (..., width) as int8 (..., width) and a float32 scale for each row (...). A row with an infinity or a NaN has the scale NaN
    and zeros."""
    if x.ndim < 1 or x.dtype not in FLOATS:
        raise ValueError(f"quantize_rows needs a float tensor (..., width), got {x.shape} {x.dtype}")
    x = x.detach()
    if x.dtype == float64 or not active_device().has_custom(QUANTIZE_ROWS):
        values, scales = _rounded(x)
        return values.cast(int8), scales.reshape(*x.shape[:-1])
    values, scales = custom(QUANTIZE_ROWS, (contiguous(x).node,), (), ((int8, x.shape), (float32, x.shape[:-1])))
    return Tensor.from_node(values), Tensor.from_node(scales)


def int8_linear(x: Tensor, weight: Tensor, scales: Tensor, bias: Tensor | None = None) -> Tensor:
    """x (..., width) through a layer whose `weight` (outputs, width) is int8 with float32 `scales` (outputs,), and `bias`
    (outputs,) of x's dtype: (..., outputs) of x's dtype. A width of up to 2^17.

    There is no gradient: the call is for answering (under `no_grad`, or on tensors that need none).
    """
    if x.ndim < 1 or x.dtype not in FLOATS or weight.ndim != 2 or weight.dtype != int8:
        raise ValueError(f"int8_linear needs float rows (..., width) and an int8 weight (outputs, width), got {x.shape} {x.dtype} and {weight.shape} {weight.dtype}")
    outputs, width = weight.shape
    if x.shape[-1] != width:
        raise ValueError(f"int8_linear: widths differ, {x.shape} and {weight.shape}")
    if width > WIDEST:
        raise ValueError(f"int8_linear: sums of up to {WIDEST} products are exact, not of {width}")
    if scales.shape != (outputs,) or scales.dtype != float32:
        raise ValueError(f"int8_linear: scales must be ({outputs},) float32, got {scales.shape} {scales.dtype}")
    if bias is not None and (bias.shape != (outputs,) or bias.dtype not in FLOATS or promote(bias.dtype, x.dtype) != x.dtype):
        raise ValueError(f"int8_linear: the bias must be ({outputs},) of {x.dtype}, got {bias.shape} {bias.dtype}")
    if records(x, scales, *(() if bias is None else (bias,))):
        raise ValueError("int8_linear has no gradient: call it under no_grad, or on tensors that need none")
    rows = x.shape[:-1]
    bias = None if bias is None else bias.cast(x.dtype)
    if x.dtype == float64 or not active_device().has_custom(INT8_LINEAR):
        values, s = _rounded(x)
        count = math.prod(rows)
        whole = values.cast(int32).reshape(count, width) @ weight.cast(int32).transpose()
        wide = float64 if x.dtype == float64 else float32
        y = whole.cast(wide) * scales.cast(wide) * s.cast(wide).reshape(count, 1)
        y = y if bias is None else y + bias.cast(wide)
        return y.cast(x.dtype).reshape(*rows, outputs)
    srcs = (contiguous(x).node, contiguous(weight).node, contiguous(scales).node) + (() if bias is None else (contiguous(bias).node,))
    (out,) = custom(INT8_LINEAR, srcs, (bias is not None,), ((x.dtype, rows + (outputs,)),))
    return Tensor.from_node(out)


def _rounded(x: Tensor) -> tuple[Tensor, Tensor]:
    """Rows as whole float32 numbers from -127 to 127, and their scales (..., 1)."""
    x = x.cast(float32)
    scales = (x.maximum(-x).max(-1, keepdim=True) / 127.0).maximum(2.0**-126)
    fine = scales < math.inf
    magic = 1.5 * 2.0**23  # a float32 this large has no bits below 1: adding it rounds to whole numbers, ties to even
    return fine.where(((x * scales.reciprocal()) + magic) - magic, 0.0), fine.where(scales, math.nan)
