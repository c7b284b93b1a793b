"""Microscaled 4-bit floating point (e2m1 codes, 32 neighbours of a row under one
power of two): rows coded and decoded, and products on the scaled matrix units.

These wrap the ``tkv_hip_dev_*_mxfp4`` entry points and the typed linear (device
pointers, asynchronous on the context's stream).  Each is a class that converts
its arguments once and launches when called.  A resident weight is
``device.QuantizedLinear.from_float(..., fmt=device.WEIGHT_MXFP4)`` or
``from_mxfp4``.  No counterpart in the reference.

Layout: a row of k elements is blocks(k) blocks, 16 bytes of codes (element 2i in
the low half of byte i) and one scale byte, 2^(byte - 127), each; codes
[rows, blocks, 16], scales [rows, blocks].
"""
from __future__ import annotations

from typing import Optional

from .attention import BF16, F16, F32, _Call
from .device import Context, QuantizedLinear, _vp

BLOCK = 32


def blocks(k: int) -> int:
    """Blocks of a row of k elements."""
    return -(-int(k) // BLOCK)


class Quantize(_Call):
    """Codes and scales of x, rows of `type` `stride` elements apart: the scale a
    block's largest binade less 2, codes to the nearest value, ties to even."""

    def __init__(self, ctx: Context, type: int, x, stride: int, rows: int, cols: int, codes, scales):
        self._also = (x, codes, scales)
        super().__init__("tkv_hip_dev_quantize_mxfp4", ctx, int(type), _vp(x), int(stride), int(rows),
                         int(cols), _vp(codes), _vp(scales))


class Dequantize(_Call):
    """The values of codes and scales, into rows of `type` `stride` elements apart."""

    def __init__(self, ctx: Context, codes, scales, rows: int, cols: int, type: int, y, stride: int):
        self._also = (codes, scales, y)
        super().__init__("tkv_hip_dev_dequantize_mxfp4", ctx, _vp(codes), _vp(scales), int(rows), int(cols),
                         int(type), _vp(y), int(stride))


class Matmul(_Call):
    """y[m, n] = a[m, k] . w[n, k]^T + bias[n], both in codes and scales, y of
    type_out with rows `stride` (None: n) elements apart."""

    def __init__(self, ctx: Context, a, a_scales, w, w_scales, m: int, n: int, k: int, type_out: int, y,
                 stride: Optional[int] = None, bias=None):
        self._also = (a, a_scales, w, w_scales, y, bias)
        super().__init__("tkv_hip_dev_matmul_mxfp4", ctx, _vp(a), _vp(a_scales), _vp(w), _vp(w_scales), int(m),
                         int(n), int(k), _vp(bias), int(type_out), _vp(y), int(n if stride is None else stride))


class Linear(_Call):
    """The linear of a resident MXFP4 weight on m rows of type_in, stride_x
    elements apart: their codes, the product and the weight's bias, into rows of
    type_out stride_y apart."""

    def __init__(self, ctx: Context, weight: QuantizedLinear, type_in: int, x, stride_x: int, m: int,
                 type_out: int, y, stride_y: Optional[int] = None):
        self._also = (weight, x, y)
        super().__init__("tkv_hip_linear_forward_typed", ctx, weight.handle, int(type_in), _vp(x), int(stride_x),
                         int(m), int(type_out), _vp(y), int(weight.n if stride_y is None else stride_y))


__all__ = ["BF16", "BLOCK", "Dequantize", "F16", "F32", "Linear", "Matmul", "Quantize", "blocks"]
