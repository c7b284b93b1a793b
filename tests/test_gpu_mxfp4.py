"""GPU tests of microscaled 4-bit floating point (tokenvector.inference_amd.mxfp4)
against plain numpy forms.

Codes and scales are equal to those of the definition in 64 bits, and so are the
values read back.  Products: where every partial sum is a multiple of one power
of two below 2^24 of it, f32 sums are exact in any order, and the outputs have to
be equal to the exact ones rounded once; with scales far apart, each matrix
instruction (64 or 128 terms) may be off by 2^-20 of its largest term or sum, so
an output by (K / 64 + 2) 2^-20 of the sum of magnitudes.
"""
import sys

import numpy as np
import pytest
import torch

from tokenvector.inference_amd import _lib
from tokenvector.inference_amd import attention as A
from tokenvector.inference_amd import device as D
from tokenvector.inference_amd import mxfp4 as X

pytestmark = pytest.mark.gpu

TORCH = {A.F32: torch.float32, A.F16: torch.float16, A.BF16: torch.bfloat16}
RAW = {A.F32: np.int32, A.F16: np.int16, A.BF16: np.int16}
NAME = {A.F32: "f32", A.F16: "f16", A.BF16: "bf16"}
GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], np.float64)
GRID = np.concatenate([GRID, -GRID])
TYPES = [A.F32, A.F16, A.BF16]


def say(*a):
    print(*a, flush=True)
    sys.stdout.flush()


@pytest.fixture(scope="module")
def ctx(hip):
    c = D.Context(0)
    yield c
    c.close()


def _bits(x, typ):
    t = torch.from_numpy(np.ascontiguousarray(x, np.float32)).to(TORCH[typ])
    return t.view(torch.int32 if typ == A.F32 else torch.int16).numpy()


def _values(raw, typ):
    return torch.from_numpy(np.ascontiguousarray(raw)).view(TORCH[typ]).float().numpy()


def _round(x, typ):
    return _values(_bits(x, typ), typ)


def same(got, want):
    bad = np.argwhere(~((got == want) | ((got != got) & (want != want))))
    assert len(bad) == 0, f"{len(bad)} of {got.size} differ, first at {bad[0]}: {got[tuple(bad[0])]}, not {want[tuple(bad[0])]}"


def code_of(x):
    """Codes [rows, blocks, 16] and scales [rows, blocks] of x, from the definition."""
    rows, cols = x.shape
    b = X.blocks(cols)
    p = np.zeros((rows, b * 32), np.float64)
    p[:, :cols] = x
    p = p.reshape(rows, b, 32)
    top = np.abs(p).max(-1)
    bad = ~np.isfinite(p).all(-1)
    e = np.where(bad | (top == 0), -127, np.clip(np.frexp(np.where(bad, 1.0, top))[1] - 3, -127, 127))
    y = np.where(bad[..., None], 0.0, p) / np.exp2(e.astype(np.float64))[..., None]
    a = np.abs(y)
    c = np.zeros(y.shape, np.uint8)
    for edge, at in ((0.25, False), (0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)):
        c += (a >= edge) if at else (a > edge)
    c |= np.where(np.signbit(y), 8, 0).astype(np.uint8)
    c[bad] = 0
    c = c.reshape(rows, b, 16, 2)
    return c[..., 0] | c[..., 1] << 4, np.where(bad, 255, e + 127).astype(np.uint8)


def value_of(codes, scales, cols):
    """What codes and scales stand for, in 64 bits."""
    v = GRID[np.stack([codes & 15, codes >> 4], -1)].reshape(codes.shape[0], -1, 32)
    unit = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127))
    return (v * unit[..., None]).reshape(codes.shape[0], -1)[:, :cols]


class Guarded:
    """A device buffer of `n` bytes with 256 others before and after that have to
    stay as they are."""

    def __init__(self, ctx, n, fill=None, shift=0):
        self.n, self.shift = n, 256 + shift
        host = np.full(n + 512 + shift, 0xA5, np.uint8)
        if fill is not None:
            host[self.shift:self.shift + n] = np.ascontiguousarray(fill).view(np.uint8).reshape(-1)
        self.buf, self.host = D.DeviceBuffer.from_host(ctx, host), host
        self.ptr = self.buf.ptr + self.shift

    def read(self, dtype, shape, what):
        got = self.buf.download()
        assert np.array_equal(got[:self.shift], self.host[:self.shift]), f"{what}: wrote before its buffer"
        end = self.shift + self.n
        assert np.array_equal(got[end:], self.host[end:]), f"{what}: wrote past its buffer"
        return got[self.shift:end].view(dtype).reshape(shape)


def _rows_buffer(ctx, x, typ, stride, shift=0):
    """x as rows of `typ`, `stride` elements apart, NaN between them."""
    raw = _bits(x, typ)
    host = np.full((x.shape[0], stride), -1, raw.dtype)
    host[:, :x.shape[1]] = raw
    size = host.dtype.itemsize
    flat = host.reshape(-1)[:(x.shape[0] - 1) * stride + x.shape[1]]
    return Guarded(ctx, flat.size * size, flat, shift)


def _special(rng, rows, cols):
    """Magnitudes over f32's range, midpoints of the grid, zeros, subnormals."""
    b = X.blocks(cols) * 32
    x = rng.standard_normal((rows, b)) * np.exp2(rng.integers(-150, 127, (rows, b // 32)).repeat(32, 1))
    mid = rng.choice([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 7.99], (rows, b)) * rng.choice([-1, 1], (rows, b))
    mid = mid * np.exp2(rng.integers(-130, 124, (rows, b // 32)).repeat(32, 1))
    x = np.where((np.arange(b // 32) % 3 == 1).repeat(32)[None], mid, x)
    x = np.where((rng.random((rows, b // 32)) < 0.1).repeat(32, 1), rng.choice([0.0, -0.0], (rows, b)), x)
    with np.errstate(over="ignore"):
        return np.clip(x[:, :cols], -3.4e38, 3.4e38).astype(np.float32)


@pytest.mark.parametrize("typ", TYPES, ids=NAME.get)
@pytest.mark.parametrize("rows,cols,pad,shift", [(1, 1, 0, 0), (1, 31, 0, 0), (1, 32, 0, 0), (1, 4096, 0, 0),
                                                 (3, 33, 0, 0), (5, 2000, 48, 0), (7, 96, 1, 0), (300, 4104, 8, 0),
                                                 (64, 768, 0, 4), (1000, 40, 24, 0), (2, 16384, 0, 0)])
def test_codes_and_values(ctx, typ, rows, cols, pad, shift):
    say(f"code {rows}x{cols} {NAME[typ]} pad {pad} shift {shift}")
    rng = np.random.default_rng(rows * 7 + cols)
    x = _round(_special(rng, rows, cols), typ)
    x = np.where(np.isfinite(x), x, 0.0).astype(np.float32)
    src = _rows_buffer(ctx, x, typ, cols + pad, shift)
    b = X.blocks(cols)
    codes, scales = Guarded(ctx, rows * b * 16), Guarded(ctx, rows * b)
    X.Quantize(ctx, typ, src.ptr, cols + pad, rows, cols, codes.ptr, scales.ptr)()
    want_c, want_s = code_of(x)
    got_s = scales.read(np.uint8, (rows, b), "scales")
    got_c = codes.read(np.uint8, (rows, b, 16), "codes")
    same(got_s, want_s)
    same(got_c, want_c)
    for out in TYPES:
        size = np.dtype(RAW[out]).itemsize
        y = _rows_buffer(ctx, np.zeros((rows, cols), np.float32), out, cols + pad, shift)
        X.Dequantize(ctx, codes.ptr, scales.ptr, rows, cols, out, y.ptr, cols + pad)()
        flat = y.read(RAW[out], -1, "values")
        assert flat.itemsize == size
        got = np.full(rows * (cols + pad), -1, RAW[out])
        got[:flat.size] = flat
        got = got.reshape(rows, cols + pad)
        with np.errstate(over="ignore"):
            want = value_of(want_c, want_s, cols).astype(np.float32)
        assert np.array_equal(got[:, :cols], _bits(want, out))
        assert (got[:, cols:].reshape(-1) == -1).all(), "wrote between the rows"


def test_blocks_that_are_not_finite(ctx):
    """Their scale is NaN, and no neighbour's is."""
    x = np.random.default_rng(5).standard_normal((4, 256)).astype(np.float32)
    x[0, 40], x[1, 95], x[2, 255], x[3, 0] = np.nan, np.inf, -np.inf, -np.nan
    for typ in TYPES:
        src = _rows_buffer(ctx, x, typ, 256)
        codes, scales = Guarded(ctx, 4 * 8 * 16), Guarded(ctx, 4 * 8)
        X.Quantize(ctx, typ, src.ptr, 256, 4, 256, codes.ptr, scales.ptr)()
        want_c, want_s = code_of(_round(x, typ))
        assert (want_s == 255).sum() == 4
        assert np.array_equal(scales.read(np.uint8, (4, 8), "scales"), want_s)
        assert np.array_equal(codes.read(np.uint8, (4, 8, 16), "codes"), want_c)


def test_every_code_and_scale_read_back(ctx):
    codes = np.tile(np.arange(256, dtype=np.uint8).reshape(1, 16, 16), (256, 1, 1))
    scales = np.repeat(np.arange(256, dtype=np.uint8)[:, None], 16, 1)
    dc, ds = D.DeviceBuffer.from_host(ctx, codes), D.DeviceBuffer.from_host(ctx, scales)
    with np.errstate(over="ignore"):
        want = value_of(codes, scales, 512).astype(np.float32)
    for typ in TYPES:
        y = D.DeviceBuffer.empty(ctx, (256, 512), RAW[typ])
        X.Dequantize(ctx, dc, ds, 256, 512, typ, y, 512)()
        got, w = _values(y.download(), typ), _round(want, typ)
        assert np.array_equal(np.isnan(got), np.isnan(w)) and np.isnan(w).any()
        assert np.array_equal(got[~np.isnan(w)], w[~np.isnan(w)])
        assert np.array_equal(np.signbit(got[:255]), np.signbit(w[:255]))


def _operand(rng, rows, k, spread):
    """Random codes, zeros past k, scales within `spread` of 1."""
    b = X.blocks(k)
    c = rng.integers(0, 16, (rows, b * 32)).astype(np.uint8)
    c[:, k:] = 0
    c = c.reshape(rows, b, 16, 2)
    s = rng.integers(127 - spread, 128 + spread, (rows, b)).astype(np.uint8)
    return c[..., 0] | c[..., 1] << 4, s


def _product(ctx, a, w, m, n, k, out, bias=None, pad=0):
    d = [Guarded(ctx, x.size, x) for x in (*a, *w)]
    db = D.DeviceBuffer.from_host(ctx, bias) if bias is not None else None
    y = _rows_buffer(ctx, np.zeros((m, n), np.float32), out, n + pad)
    X.Matmul(ctx, *(x.ptr for x in d), m, n, k, out, y.ptr, n + pad, bias=db)()
    return _unpad(y, m, n, out, pad)


def _unpad(y, m, n, out, pad):
    flat = y.read(RAW[out], -1, "product")
    got = np.full(m * (n + pad), -1, RAW[out])
    got[:flat.size] = flat
    got = got.reshape(m, n + pad)
    assert (got[:, n:].reshape(-1) == -1).all(), "wrote between the rows"
    return _values(np.ascontiguousarray(got[:, :n]), out)


SIZES = [(1, 1, 1), (1, 7, 31), (2, 3, 32), (1, 64, 96), (3, 17, 64), (16, 16, 128), (16, 130, 4100), (17, 33, 256),
         (32, 100, 1000), (33, 65, 257), (64, 64, 256), (65, 130, 511), (63, 1000, 512), (100, 5, 2048), (128, 300, 1024),
         (129, 127, 288), (256, 256, 544), (1000, 768, 768), (333, 1000, 2000), (2049, 2100, 640),
         (4111, 4120, 1056), (4096, 4096, 1024), (3999, 4071, 1100), (3, 16390, 64), (20, 8200, 96), (9, 8211, 2080), (60, 16390, 288), (1, 16400, 544),
         (48, 8200, 4000), (30, 16400, 320)]


@pytest.mark.parametrize("m,n,k", SIZES)
@pytest.mark.parametrize("out", TYPES, ids=NAME.get)
def test_product_exact(ctx, m, n, k, out):
    """Scales 2^-1 .. 2^1: products are multiples of 2^-4 and below 2^8, sums (of
    random signs, K of at most 4100) far below 2^20, so exact in f32."""
    say(f"product {m}x{n}x{k} {NAME[out]}")
    rng = np.random.default_rng(m * 31 + n * 7 + k)
    a, w = _operand(rng, m, k, 1), _operand(rng, n, k, 1)
    exact = value_of(*a, k) @ value_of(*w, k).T
    assert np.abs(exact).max() < 2.0 ** 19
    bias = np.round(rng.standard_normal(n) * 64).astype(np.float32) / 16 if (m + n) % 2 else None
    pad = (m * n) % 3 * 8
    got = _product(ctx, a, w, m, n, k, out, bias, pad)
    want = exact if bias is None else exact + bias.astype(np.float64)
    same(got, _round(want.astype(np.float32), out))


@pytest.mark.parametrize("m,n,k", [(1, 33, 2000), (20, 64, 512), (96, 200, 1056), (260, 300, 768), (5, 7, 131071)])
def test_product_of_scales_far_apart(ctx, m, n, k):
    say(f"product {m}x{n}x{k}, scales far apart")
    rng = np.random.default_rng(k)
    a, w = _operand(rng, m, k, 12), _operand(rng, n, k, 12)
    va, vw = value_of(*a, k), value_of(*w, k)
    got = _product(ctx, a, w, m, n, k, A.F32)
    bound = ((k / 64 + 2) * 2.0 ** -20) * (np.abs(va) @ np.abs(vw).T) + 2.0 ** -24 * np.abs(va @ vw.T)
    worst = np.max(np.abs(got - va @ vw.T) / np.maximum(bound, 1e-300))
    assert worst <= 1.0, worst


@pytest.mark.parametrize("m", [1, 40, 300])
def test_product_ends_of_the_scales(ctx, m):
    """2^127 on one side, 2^-127 on the other; and terms of 2^-254, which are zeros."""
    rng = np.random.default_rng(m)
    a, w = _operand(rng, m, 160, 0), _operand(rng, 70, 160, 0)
    exact = value_of(*a, 160) @ value_of(*w, 160).T
    a[1][:], w[1][:] = 254, 0
    assert np.array_equal(_product(ctx, a, w, m, 70, 160, A.F32), exact.astype(np.float32))
    a[1][:, :4], a[1][:, 4] = 0, 254
    only = value_of(a[0], a[1] * 0 + 127, 160)[:, 128:] @ value_of(w[0], w[1] + 127, 160)[:, 128:].T
    assert np.array_equal(_product(ctx, a, w, m, 70, 160, A.F32), only.astype(np.float32))


@pytest.mark.parametrize("m", [1, 9, 100, 600])
def test_nan_blocks_stay_in_their_row_and_column(ctx, m):
    rng = np.random.default_rng(m)
    n, k = 300, 500
    a, w = _operand(rng, m, k, 1), _operand(rng, n, k, 1)
    exact = value_of(*a, k) @ value_of(*w, k).T
    a[1][m // 2, 15] = 255  # the last block, not whole
    w[1][[0, 77, 299], [0, 7, 15]] = 255
    got = _product(ctx, a, w, m, n, k, A.F32)
    exact[m // 2] = np.nan
    exact[:, [0, 77, 299]] = np.nan
    assert np.array_equal(np.isnan(got), np.isnan(exact))
    assert np.array_equal(got[~np.isnan(got)], exact[~np.isnan(exact)].astype(np.float32))


@pytest.mark.parametrize("typ", TYPES, ids=NAME.get)
@pytest.mark.parametrize("m,n,k,pad,shift", [(1, 130, 800, 0, 0), (4, 64, 4096, 8, 0), (13, 768, 768, 5, 0),
                                             (32, 2304, 768, 0, 0), (33, 96, 1000, 0, 4), (200, 768, 768, 0, 0),
                                             (1500, 1024, 320, 8, 0), (2, 16400, 800, 0, 0), (16, 8210, 2100, 4, 0),
                                             (7, 40, 4000, 0, 0), (16, 33, 8200, 0, 0),
                                             (2, 50, 16000, 0, 0), (5, 8200, 2000, 8, 0), (3, 16400, 4096, 0, 0),
                                             (1, 8200, 8192, 0, 0), (1, 16384, 16352, 0, 0), (30, 16400, 96, 0, 0)])
def test_linear(ctx, typ, m, n, k, pad, shift):
    """The activation's codes are the definition's, so the outputs are those of
    the codes' values: exact sums where the scales are near each other."""
    say(f"linear {m}x{n}x{k} {NAME[typ]} pad {pad} shift {shift}")
    rng = np.random.default_rng(m + n + k)
    x = _round(rng.uniform(0.6, 1.9, (m, k)).astype(np.float32) * rng.choice([-1.0, 1.0], (m, k)), typ)
    w, bias = _operand(rng, n, k, 1), rng.integers(-64, 64, n).astype(np.float32) / 8
    exact = value_of(*code_of(x), k) @ value_of(*w, k).T + bias
    dw, ds, db = (D.DeviceBuffer.from_host(ctx, v) for v in (*w, bias))
    lin = D.QuantizedLinear.from_mxfp4(ctx, dw, ds, n, k, db)
    for b in (dw, ds, db):
        b.close()  # the weight is a copy
    assert (lin.n, lin.k, lin.format) == (n, 32 * X.blocks(k), D.WEIGHT_MXFP4)
    src = _rows_buffer(ctx, x, typ, k + pad, shift)
    for out in TYPES:
        y = _rows_buffer(ctx, np.zeros((m, n), np.float32), out, n + pad)
        X.Linear(ctx, lin, typ, src.ptr, k + pad, m, out, y.ptr, n + pad)()
        same(_unpad(y, m, n, out, pad), _round(exact.astype(np.float32), out))
    if typ == A.F32 and not pad and not shift:
        y = Guarded(ctx, m * n * 4)
        for mode in (D.ACT_PER_TENSOR, D.ACT_PER_TOKEN):
            lin.forward(src.ptr, m, y.ptr, mode)
            assert np.array_equal(y.read(np.float32, (m, n), "forward"), exact.astype(np.float32))
    lin.close()


@pytest.mark.parametrize("typ", TYPES, ids=NAME.get)
@pytest.mark.parametrize("cols", [2, 5, 7, 8, 9, 12, 15, 39, 63, 71, 1001, 4095])
def test_rows_that_start_anywhere(ctx, typ, cols):
    """Rows of every remainder of 8, at every place of a 16-byte line, NaN before,
    between and behind them: coded, read back and multiplied."""
    say(f"rows of {cols} {NAME[typ]}")
    rng = np.random.default_rng(cols)
    size, b = np.dtype(RAW[typ]).itemsize, X.blocks(cols)
    for rows, pad in ((11, 1), (3, 0), (1, 0), (70, 3)):
        x = _round(_special(rng, rows, cols), typ)
        x = np.where(np.isfinite(x), x, 0.0).astype(np.float32)
        src = _rows_buffer(ctx, x, typ, cols + pad, size)
        codes, scales = Guarded(ctx, rows * b * 16), Guarded(ctx, rows * b)
        X.Quantize(ctx, typ, src.ptr, cols + pad, rows, cols, codes.ptr, scales.ptr)()
        want_c, want_s = code_of(x)
        same(scales.read(np.uint8, (rows, b), "scales"), want_s)
        same(codes.read(np.uint8, (rows, b, 16), "codes"), want_c)
        y = _rows_buffer(ctx, np.zeros((rows, cols), np.float32), typ, cols + pad, size)
        X.Dequantize(ctx, codes.ptr, scales.ptr, rows, cols, typ, y.ptr, cols + pad)()
        with np.errstate(over="ignore"):
            want = value_of(want_c, want_s, cols).astype(np.float32)
        assert np.array_equal(_unpad(y, rows, cols, typ, pad), _round(want, typ))
        # the weight's rows as many, so that the outputs' have odd strides too
        n = cols + 60
        z = _round(rng.uniform(0.6, 1.9, (rows, cols)).astype(np.float32), typ)
        src = _rows_buffer(ctx, z, typ, cols + pad, size)
        w = _operand(rng, n, cols, 1)
        lin = D.QuantizedLinear.from_mxfp4(ctx, *(D.DeviceBuffer.from_host(ctx, v) for v in w), n, cols)
        y = _rows_buffer(ctx, np.zeros((rows, n), np.float32), typ, n + pad, size)
        X.Linear(ctx, lin, typ, src.ptr, cols + pad, rows, typ, y.ptr, n + pad)()
        exact = value_of(*code_of(z), cols) @ value_of(*w, cols).T
        same(_unpad(y, rows, n, typ, pad), _round(exact.astype(np.float32), typ))
        lin.close()


@pytest.mark.parametrize("typ", TYPES, ids=NAME.get)
@pytest.mark.parametrize("m", [1, 5, 16, 17, 70])
def test_values_that_the_linear_multiplies(ctx, typ, m):
    """A weight with a one in each row gives the activation's values back: those of
    the definition, over the type's range (f32 sums have no subnormal terms)."""
    k = 200
    rng = np.random.default_rng(m)
    x = _round(_special(rng, m, k), typ)
    x = np.where(np.isfinite(x), x, 0.0).astype(np.float32)
    w = np.eye(k, dtype=np.float32)
    lin = D.QuantizedLinear.from_float(ctx, D.DeviceBuffer.from_host(ctx, w), k, k, None, D.WEIGHT_MXFP4)
    src = _rows_buffer(ctx, x, typ, k)
    y = D.DeviceBuffer.empty(ctx, (m, k), np.float32)
    X.Linear(ctx, lin, typ, src.ptr, k, m, A.F32, y)()
    with np.errstate(over="ignore"):
        want = value_of(*code_of(x), k).astype(np.float32)
    got = y.download()
    seen = (np.abs(want) >= 2.0 ** -126) & np.isfinite(want)
    same(got[seen], want[seen])
    assert np.all(np.abs(got[np.abs(want) < 2.0 ** -126]) < 2.0 ** -126)
    lin.close()


@pytest.mark.parametrize("typ", TYPES, ids=NAME.get)
@pytest.mark.parametrize("m", [3, 20])
def test_activations_that_are_not_finite(ctx, typ, m):
    rng = np.random.default_rng(m)
    n, k = 40, 300
    x = _round(rng.uniform(0.6, 1.9, (m, k)).astype(np.float32), typ)
    x[0, 299], x[m - 1, 5] = np.inf, np.nan
    w = _operand(rng, n, k, 1)
    lin = D.QuantizedLinear.from_mxfp4(ctx, *(D.DeviceBuffer.from_host(ctx, v) for v in w), n, k)
    src = _rows_buffer(ctx, x, typ, k)
    y = D.DeviceBuffer.empty(ctx, (m, n), np.float32)
    X.Linear(ctx, lin, typ, src.ptr, k, m, A.F32, y)()
    got = y.download()
    assert np.isnan(got[[0, m - 1]]).all()
    exact = value_of(*code_of(x[1:m - 1]), k) @ value_of(*w, k).T
    same(got[1:m - 1], exact.astype(np.float32))
    lin.close()


def test_weight_from_floats(ctx):
    rng = np.random.default_rng(3)
    n, k = 100, 500
    w = (rng.standard_normal((n, k)) * 0.02).astype(np.float32)
    codes, scales = code_of(w)
    lin = D.QuantizedLinear.from_float(ctx, D.DeviceBuffer.from_host(ctx, w), n, k, None, D.WEIGHT_MXFP4)
    assert (lin.n, lin.k, lin.format) == (n, 512, D.WEIGHT_MXFP4)
    back = D.DeviceBuffer.empty(ctx, (n, k), np.float32)
    X.Dequantize(ctx, lin.codes, lin.scales, n, k, A.F32, back, k)()
    assert np.array_equal(back.download(), value_of(codes, scales, k).astype(np.float32))
    x = _round(rng.standard_normal((6, k)).astype(np.float32), A.F32)
    dx, y = D.DeviceBuffer.from_host(ctx, x), D.DeviceBuffer.empty(ctx, (6, n), np.float32)
    lin.forward(dx, 6, y)
    va, vw = value_of(*code_of(x), k), value_of(codes, scales, k)
    bound = (k / 64 + 2) * 2.0 ** -20 * (np.abs(va) @ np.abs(vw).T) + 2.0 ** -24 * np.abs(va @ vw.T)
    assert np.all(np.abs(y.download() - va @ vw.T) <= bound)
    lin.close()


def test_nothing_to_do(ctx):
    y = Guarded(ctx, 64)
    X.Quantize(ctx, A.F32, None, 32, 0, 32, None, None)()
    X.Dequantize(ctx, None, None, 0, 32, A.F32, None, 32)()
    X.Matmul(ctx, None, None, None, None, 0, 4, 32, A.F32, None)()
    X.Matmul(ctx, None, None, None, None, 4, 0, 32, A.F32, None)()
    y.read(np.uint8, 64, "nothing")


@pytest.mark.parametrize("m", [1, 70, 700])
def test_captured_and_replayed(ctx, m):
    """The linear into a graph, replayed with new activations, eager calls of other
    sizes on the same workspaces between."""
    rng = np.random.default_rng(m)
    n, k = 520, 1000
    w = _operand(rng, n, k, 1)
    own = D.Context(0)
    dw, ds = (D.DeviceBuffer.from_host(own, v) for v in w)
    lin = D.QuantizedLinear.from_mxfp4(own, dw, ds, n, k)
    x = D.DeviceBuffer.empty(own, (m, k), np.float32)
    y = D.DeviceBuffer.empty(own, (m, n), np.float32)
    call = X.Linear(own, lin, A.F32, x, k, m, A.F32, y)
    call()
    with D.Graph(own) as g:
        call()
    big_x = D.DeviceBuffer.from_host(own, rng.standard_normal((m + 900, k)).astype(np.float32))
    big_y = D.DeviceBuffer.empty(own, (m + 900, n), np.float32)
    for turn in range(3):
        xs = (rng.uniform(0.6, 1.9, (m, k)) * rng.choice([-1.0, 1.0], (m, k))).astype(np.float32)
        x.upload(xs)
        D.memset(own, y, 0, y.nbytes)
        g.launch()
        exact = value_of(*code_of(xs), k) @ value_of(*w, k).T
        assert np.array_equal(y.download(), exact.astype(np.float32)), turn
        X.Linear(own, lin, A.F32, big_x, k, m + 900, A.F32, big_y)()
        own.synchronize()
    g.close()
    lin.close()
    for b in (dw, ds, x, y, big_x, big_y):
        b.close()
    own.close()


LONG = [(1, 16, 16384), (1, 384, 15808), (6, 721, 15969), (7, 384, 12736), (12, 960, 9600), (16, 40, 8193),
        (17, 130, 16352), (33, 200, 9000), (64, 640, 16000), (64, 16, 131040),
        (70, 64, 16384), (65, 33, 20001), (100, 640, 16000), (129, 300, 12001), (200, 1000, 9000), (256, 1030, 8192)]


@pytest.mark.parametrize("m,n,k", LONG)
def test_long_rows_of_few_outputs(ctx, m, n, k):
    """Sums over parts of K, joined: exact, the same in every call, beside attention
    that counts its own arrivals, and in graphs that take turns."""
    say(f"long rows {m}x{n}x{k}")
    rng = np.random.default_rng(m + n + k)
    a, w = _operand(rng, m, k, 1), _operand(rng, n, k, 1)
    exact = (value_of(*a, k) @ value_of(*w, k).T).astype(np.float32)
    for out in (A.F32, A.BF16):
        same(_product(ctx, a, w, m, n, k, out, pad=3), _round(exact, out))
    own = D.Context(0)
    dw, ds = (D.DeviceBuffer.from_host(own, v) for v in w)
    lin = D.QuantizedLinear.from_mxfp4(own, dw, ds, n, k)
    rows = [m, max(1, m // 2)]
    x = D.DeviceBuffer.empty(own, (m, k), np.float32)
    ys = [D.DeviceBuffer.empty(own, (r, n), np.float32) for r in rows]
    calls = [X.Linear(own, lin, A.F32, x, k, r, A.F32, y) for r, y in zip(rows, ys)]
    # one query of four heads over 3000 keys, whose splits are joined the same way
    q, kv, o = (D.DeviceBuffer.from_host(own, rng.standard_normal(s).astype(np.float32))
                for s in ((1, 4, 64), (3000, 2, 64), (1, 4, 64)))
    ends = [D.DeviceBuffer.from_host(own, np.array([0, t], np.int32)) for t in (1, 3000)]
    heads = [A.Rows(t, t.shape[1] * 64, 64) for t in (q, kv, kv, o)]
    attend = A.AttentionPrompt(own, A.F32, 1, 4, 2, 64, 1, *heads, ends[0], ends[1], 3000)
    for call in (*calls, attend):
        call()
    first = o.download()
    graphs = []
    for call in calls:
        with D.Graph(own) as g:
            call()
        graphs.append(g)
    for turn in range(3):
        xs = (rng.uniform(0.6, 1.9, (m, k)) * rng.choice([-1.0, 1.0], (m, k))).astype(np.float32)
        x.upload(xs)
        exact = (value_of(*code_of(xs), k) @ value_of(*w, k).T).astype(np.float32)
        for y, call, g in zip(ys, calls, graphs):
            for go in (g.launch, call, g.launch):
                D.memset(own, y, 0, y.nbytes)
                go()
                attend()
                assert np.array_equal(y.download(), exact[:y.shape[0]]), turn
        assert np.array_equal(o.download(), first)
    for g in graphs:
        g.close()
    lin.close()
    for b in (dw, ds, x, *ys, q, kv, o, *ends):
        b.close()
    own.close()


def test_two_contexts_at_once(ctx):
    """Each has its own stream and workspaces; one weight."""
    rng = np.random.default_rng(11)
    n, k, ms = 768, 768, (5, 900)
    w = _operand(rng, n, k, 1)
    dw, ds = (D.DeviceBuffer.from_host(ctx, v) for v in w)
    lin = D.QuantizedLinear.from_mxfp4(ctx, dw, ds, n, k)
    both = [D.Context(0) for _ in ms]
    xs = [(rng.uniform(0.6, 1.9, (m, k)) * rng.choice([-1.0, 1.0], (m, k))).astype(np.float32) for m in ms]
    dx = [D.DeviceBuffer.from_host(c, x) for c, x in zip(both, xs)]
    dy = [D.DeviceBuffer.empty(c, (m, n), np.float32) for c, m in zip(both, ms)]
    calls = [X.Linear(c, lin, A.F32, x, k, m, A.F32, y) for c, x, m, y in zip(both, dx, ms, dy)]
    for _ in range(20):
        for call in calls:
            call()
    for x, y in zip(xs, dy):
        exact = value_of(*code_of(x), k) @ value_of(*w, k).T
        assert np.array_equal(y.download(), exact.astype(np.float32))
    for b in (*dx, *dy):
        b.close()
    lin.close()
    for c in both:
        c.close()


def test_other_weights_refuse_the_typed_linear(ctx):
    w = D.DeviceBuffer.from_host(ctx, np.ones((32, 128), np.float32))
    lin = D.QuantizedLinear.from_float(ctx, w, 32, 128)
    x, y = D.DeviceBuffer.empty(ctx, (2, 128), np.float32), D.DeviceBuffer.empty(ctx, (2, 32), np.float32)
    with pytest.raises(_lib.TkvHipError) as e:
        X.Linear(ctx, lin, A.F32, x, 128, 2, A.F32, y, 32)()
    assert e.value.rc == _lib.UNSUPPORTED
    lin.close()
