"""Attention beside the quantized linears: rotary positions, a paged cache,
attention of whole prompts and of new tokens over the cache.

These wrap the ``tkv_hip_kv_*``, ``tkv_hip_dev_rope_*`` and
``tkv_hip_dev_attention_*`` entry points (device pointers, asynchronous on the
context's stream).  Each operator is a class that checks and lays out its
arguments once and launches when called, so a loop whose buffers stay the same
pays for one foreign call per step; lengths, positions, slots and page tables
are device arrays that the call reads anew.  No counterpart on the reference's
quantization path, which ends at the linears.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import NamedTuple, Optional, Sequence

import numpy as np

from . import _lib
from .device import Context, DeviceBuffer, QuantizedLinear, _vp

F32, F16, BF16, I8 = 0, 1, 2, 3
ROPE_HALF, ROPE_PAIRS = 0, 1


class Rows(NamedTuple):
    """A device tensor [tokens, heads, head_dim] inside a larger one: address
    (or DeviceBuffer) and strides in elements."""
    data: object
    stride_token: int
    stride_head: int


class _Rows(C.Structure):
    _fields_ = [("data", C.c_void_p), ("stride_token", C.c_int64), ("stride_head", C.c_int64)]


def _rows(r: Optional[Rows]):
    if r is None:
        return None
    return _Rows(_vp(r.data).value, int(r.stride_token), int(r.stride_head))


class KVCache:
    """A paged cache: K and V [num_pages, heads, page_size, head_dim], slot s of
    the pool in page s // page_size.  Memory of its own, or the caller's
    (k, v and, for I8, k_scales and v_scales)."""

    def __init__(self, ctx: Context, type: int, num_pages: int, page_size: int, heads: int,
                 head_dim: int, k=None, v=None, k_scales=None, v_scales=None):
        h = C.c_int64()
        self.handle = 0
        _lib.check(_lib.lib().tkv_hip_kv_create(
            ctx.handle, int(type), int(num_pages), int(page_size), int(heads), int(head_dim),
            _vp(k), _vp(v), _vp(k_scales), _vp(v_scales), C.byref(h)))
        self.handle = h.value
        self.ctx, self.type, self.num_pages, self.page_size = ctx, int(type), int(num_pages), int(page_size)
        self.heads, self.head_dim = int(heads), int(head_dim)
        self._kept = (k, v, k_scales, v_scales)  # buffers handed over stay alive
        p = [C.c_void_p() for _ in range(4)]
        _lib.check(_lib.lib().tkv_hip_kv_info(self.handle, *(C.byref(x) for x in p)))
        self.k, self.v, self.k_scales, self.v_scales = (x.value for x in p)

    def close(self) -> None:
        if self.handle:
            _lib.check(_lib.lib().tkv_hip_kv_free(self.handle))
            self.handle = 0

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class _Call:
    """An entry point and its arguments, converted once; calling it launches.
    The addresses are those of its construction, so a cache, weight or buffer that
    was closed since is refused."""

    def __init__(self, name, ctx, *args):
        lib = _lib.lib()
        types = getattr(lib, name).argtypes[1:]
        # a function object without argtypes takes the converted arguments as they
        # are: 0.8 us less per call than converting 19 of them
        self._fn = lib._FuncPtr((name, lib))
        self._ctx, self._kept = ctx, args
        given = [x.data if isinstance(x, Rows) else x for x in self._also]
        given += [x for cache in given if isinstance(cache, KVCache) for x in cache._kept]
        self._held = [x for x in given if isinstance(x, (KVCache, QuantizedLinear, DeviceBuffer))]
        self._args = tuple(C.cast(C.byref(a), C.c_void_p) if isinstance(a, C.Structure)
                           else C.c_void_p() if a is None else a if isinstance(a, t) else t(a)
                           for t, a in zip(types, args))

    def __call__(self) -> None:
        for held in self._held:
            if isinstance(held, DeviceBuffer):
                if not held.ptr and held.nbytes:
                    raise ValueError("a buffer of this call is closed")
            elif not held.handle:
                raise ValueError("the cache or weight of this call is closed")
        rc = self._fn(C.c_int64(self._ctx.handle), *self._args)
        if rc:
            _lib.check(rc)


# ---- rotary positions ---------------------------------------------------------

def rope_inv_freq(rot_dim: int, base: float = 10000.0, factor: float = 1.0, by_parts: bool = False,
                  original_positions: int = 0, low_turns: float = 1.0,
                  high_turns: float = 32.0) -> np.ndarray:
    """The rot_dim / 2 inverse frequencies base^(-2 i / rot_dim) in f64, for
    contexts `factor` times longer than trained for: all slowed by `factor`
    (linear interpolation), or by_parts: those that turn at least `high_turns`
    times over original_positions kept, those below `low_turns` slowed, a linear
    mix between.  A larger `base` is the remaining usual scaling."""
    if rot_dim < 2 or rot_dim % 2:
        raise ValueError("rot_dim: a positive even number")
    if factor <= 0 or base <= 0:
        raise ValueError("base and factor: positive")
    inv = float(base) ** (-np.arange(0, rot_dim, 2, dtype=np.float64) / rot_dim)
    if not by_parts:
        return inv / factor
    if original_positions <= 0 or high_turns <= low_turns:
        raise ValueError("by_parts: original_positions > 0 and high_turns > low_turns")
    turns = original_positions * inv / (2.0 * math.pi)
    keep = np.clip((turns - low_turns) / (high_turns - low_turns), 0.0, 1.0)
    return inv * (keep + (1.0 - keep) / factor)


def rope_table(ctx: Context, positions: int, inv_freq, amplitude: float = 1.0) -> DeviceBuffer:
    """amplitude * (cos, sin)(p * inv_freq[i]) of every position, f32
    [positions, rot_dim / 2, 2], computed in f64 on the device."""
    inv = np.ascontiguousarray(inv_freq, np.float64).reshape(-1)
    table = DeviceBuffer.empty(ctx, (int(positions), inv.size, 2), np.float32)
    _lib.check(_lib.lib().tkv_hip_dev_rope_table(ctx.handle, int(positions), 2 * inv.size,
                                                 inv.ctypes.data_as(C.c_void_p), float(amplitude),
                                                 _vp(table)))
    return table


class RopeAppend(_Call):
    """Rotate q and k by their positions (table given), convert q, k and v to
    type_out, and append k and v to the cache (given, with one pool slot per
    token).  q_out / k_out: where the rotated rows go, each may be left out."""

    def __init__(self, ctx: Context, type_in: int, tokens: int, heads_q: int, heads_kv: int,
                 head_dim: int, q: Optional[Rows], k: Optional[Rows] = None,
                 v: Optional[Rows] = None, positions=None, table=None, table_len: int = 0,
                 rot_dim: int = 0, layout: int = ROPE_HALF, q_out: Optional[Rows] = None,
                 k_out: Optional[Rows] = None, type_out: Optional[int] = None,
                 cache: Optional[KVCache] = None, slots=None):
        self._also = (q, k, v, positions, table, q_out, k_out, cache, slots)
        super().__init__(
            "tkv_hip_dev_rope_append", ctx, int(type_in), int(tokens), int(heads_q),
            int(heads_kv), int(head_dim), _rows(q), _rows(k), _rows(v), _vp(positions), _vp(table),
            int(table_len), int(rot_dim), int(layout), _rows(q_out), _rows(k_out),
            int(type_in if type_out is None else type_out), cache.handle if cache else 0, _vp(slots))


class HeadNorm(NamedTuple):
    """Norms per head: x / sqrt(mean(x^2) + eps) * gain, gains f32 [head_dim] on
    the device (None: ones) for the queries' heads and for the keys'."""
    eps: float
    q_gain: object = None
    k_gain: object = None


class Rope(NamedTuple):
    """A rotation: the table (rope_table), int32 device positions, `axes` rows of
    them stride_axis apart, and the axis of each pair (rope_pair_axes)."""
    table: object
    table_len: int
    rot_dim: int
    layout: int
    positions: object
    axes: int = 1
    stride_axis: int = 0
    pair_axis: Optional[Sequence[int]] = None


class _HeadNorm(C.Structure):
    _fields_ = [("eps", C.c_float), ("q_gain", C.c_void_p), ("k_gain", C.c_void_p)]


class _Rope(C.Structure):
    _fields_ = [("table", C.c_void_p), ("table_len", C.c_int64), ("rot_dim", C.c_int64), ("layout", C.c_int32),
                ("axes", C.c_int32), ("positions", C.c_void_p), ("stride_axis", C.c_int64),
                ("pair_axis", C.c_void_p)]


def rope_pair_axes(sections: Sequence[int], interleaved: bool = False) -> list:
    """The axis of each of sum(sections) pairs: the axes' sections behind each
    other, or interleaved (one pair of each axis in turn, as long as it has any)."""
    left = [int(n) for n in sections]
    if not 1 <= len(left) <= 4 or min(left) < 0 or sum(left) == 0:
        raise ValueError("sections: the pairs of 1 to 4 axes")
    if not interleaved:
        return [axis for axis, n in enumerate(left) for _ in range(n)]
    out = []
    while any(left):
        for axis, n in enumerate(left):
            if n:
                out.append(axis)
                left[axis] -= 1
    return out


class NormRopeAppend(_Call):
    """RopeAppend with norms of each head of q and k before the rotation, and
    with positions on several axes.  norm or rope None: without it."""

    def __init__(self, ctx: Context, type_in: int, tokens: int, heads_q: int, heads_kv: int,
                 head_dim: int, q: Optional[Rows], k: Optional[Rows] = None,
                 v: Optional[Rows] = None, norm: Optional[HeadNorm] = None, rope: Optional[Rope] = None,
                 q_out: Optional[Rows] = None, k_out: Optional[Rows] = None,
                 type_out: Optional[int] = None, cache: Optional[KVCache] = None, slots=None):
        self._also = (q, k, v, q_out, k_out, cache, slots) + tuple(norm or ())[1:]
        n = r = None
        if norm is not None:
            n = _HeadNorm(float(norm.eps), _vp(norm.q_gain).value, _vp(norm.k_gain).value)
        if rope is not None:
            self._also += (rope.table, rope.positions)
            self._axes = None
            if rope.pair_axis is not None:
                pairs = [int(x) for x in rope.pair_axis]
                if len(pairs) != int(rope.rot_dim) // 2 or not all(0 <= x <= 255 for x in pairs):
                    raise ValueError("pair_axis: the axis of each of rot_dim / 2 pairs")
                self._axes = (C.c_uint8 * len(pairs))(*pairs)  # kept: read at every call
            r = _Rope(_vp(rope.table).value, int(rope.table_len), int(rope.rot_dim), int(rope.layout),
                      int(rope.axes), _vp(rope.positions).value, int(rope.stride_axis),
                      C.cast(self._axes, C.c_void_p).value if self._axes is not None else None)
        super().__init__(
            "tkv_hip_dev_norm_rope_append", ctx, int(type_in), int(tokens), int(heads_q),
            int(heads_kv), int(head_dim), _rows(q), _rows(k), _rows(v), n, r, _rows(q_out), _rows(k_out),
            int(type_in if type_out is None else type_out), cache.handle if cache else 0, _vp(slots))


# ---- attention ----------------------------------------------------------------

class AttentionPrompt(_Call):
    """Attention of packed prompts: sequence s has the query rows cu_q[s] ..
    cu_q[s + 1] and the key rows cu_k[s] .. cu_k[s + 1] (cu_k None: cu_q's;
    int32 device arrays) of the tokens_k that k and v have, which goes with cu_k.
    scale None: 1 / sqrt(head_dim)."""

    def __init__(self, ctx: Context, type: int, tokens: int, heads_q: int, heads_kv: int,
                 head_dim: int, sequences: int, q: Rows, k: Rows, v: Rows, out: Rows, cu_q,
                 cu_k=None, tokens_k: Optional[int] = None, scale: Optional[float] = None,
                 causal: bool = True, window: int = 0, type_out: Optional[int] = None):
        if cu_k is not None and tokens_k is None:
            raise ValueError("cu_k without tokens_k: keys past it are cut off")
        self._also = (q, k, v, out, cu_q, cu_k)
        super().__init__(
            "tkv_hip_dev_attention_prompt", ctx, int(type), int(tokens),
            int(tokens if tokens_k is None else tokens_k), int(heads_q), int(heads_kv),
            int(head_dim), int(sequences), _rows(q), _rows(k), _rows(v), _rows(out),
            int(type if type_out is None else type_out), _vp(cu_q), _vp(cu_k),
            1.0 / math.sqrt(head_dim) if scale is None else float(scale), int(bool(causal)),
            int(window))


class AttentionPaged(_Call):
    """Attention of new tokens over a paged cache that holds them already:
    sequence s has the query rows cu_q[s] .. cu_q[s + 1] (cu_q None: the one row
    s) and the first kv_lens[s] tokens of the pages page_table[s, :] (int32
    device arrays, table_stride entries a row).  max_q and max_kv: the longest
    of both, for the launch shape alone (0: not known)."""

    def __init__(self, ctx: Context, type: int, tokens: int, heads_q: int, cache: KVCache,
                 sequences: int, q: Rows, out: Rows, page_table, table_stride: int, kv_lens,
                 cu_q=None, max_q: int = 0, max_kv: int = 0, scale: Optional[float] = None,
                 causal: bool = True, window: int = 0, type_out: Optional[int] = None):
        self._also = (q, out, cache, page_table, kv_lens, cu_q)
        super().__init__(
            "tkv_hip_dev_attention_paged", ctx, int(type), int(tokens), int(heads_q),
            cache.handle, int(sequences), _rows(q), _rows(out),
            int(type if type_out is None else type_out), _vp(page_table), int(table_stride),
            _vp(cu_q), _vp(kv_lens), int(max_q), int(max_kv),
            1.0 / math.sqrt(cache.head_dim) if scale is None else float(scale), int(bool(causal)),
            int(window))
