"""GPU tests of the 4-bit entry points where offsets pass 32 bits and grids one
dimension: operands of zeros but for a few rows at their ends."""
import sys

import numpy as np
import pytest

from tokenvector.inference_amd import _lib
from tokenvector.inference_amd import attention as A
from tokenvector.inference_amd import device as D
from tokenvector.inference_amd import mxfp4 as X
from test_gpu_mxfp4 import code_of, value_of

pytestmark = pytest.mark.gpu


def say(*a):
    print(*a, flush=True)
    sys.stdout.flush()


@pytest.fixture(scope="module")
def ctx(hip):
    c = D.Context(0)
    yield c
    c.close()


class _At:
    """A part of a device buffer, for copies."""

    def __init__(self, buf, offset, shape, dtype):
        self.ctx, self.ptr, self.shape, self.dtype = buf.ctx, buf.ptr + offset, shape, np.dtype(dtype)
        self.nbytes = int(np.prod(shape)) * self.dtype.itemsize
        assert offset + self.nbytes <= buf.nbytes

    upload, download = D.DeviceBuffer.upload, D.DeviceBuffer.download


def _coded(ctx, rows, k, tail, scale=127):
    """Codes of zeros, scales 1, and `tail`'s codes and scales in the last rows."""
    b = X.blocks(k)
    codes, scales = D.DeviceBuffer(ctx, rows * b * 16), D.DeviceBuffer(ctx, rows * b)
    D.memset(ctx, codes, 0, codes.nbytes)
    D.memset(ctx, scales, scale, scales.nbytes)
    c, s = tail
    first = rows - c.shape[0]
    _At(codes, first * b * 16, c.shape, np.uint8).upload(c)
    _At(scales, first * b, s.shape, np.uint8).upload(s)
    return codes, scales


def _small(rng, rows, k):
    x = rng.choice([-1.0, 1.0, 2.0, -3.0, 0.5], (rows, k)).astype(np.float32)
    return code_of(x)


@pytest.mark.parametrize("m", [1, 40, 100])
def test_weight_of_more_than_4_gb(ctx, m):
    n, k = 66000, 131040
    say(f"product {m}x{n}x{k}")
    rng = np.random.default_rng(m)
    a, w = _small(rng, m, k), _small(rng, 20, k)
    wc, ws = _coded(ctx, n, k, w)
    ac, as_ = (D.DeviceBuffer.from_host(ctx, v) for v in a)
    y = D.DeviceBuffer.empty(ctx, (m, n), np.float32)
    X.Matmul(ctx, ac, as_, wc, ws, m, n, k, A.F32, y)()
    got = y.download()
    exact = value_of(*a, k) @ value_of(*w, k).T
    assert np.array_equal(got[:, -20:], exact.astype(np.float32)) and not got[:, :-20].any()
    for b in (wc, ws, ac, as_, y):
        b.close()


def test_most_weight_rows(ctx):
    """2^28 - 1 of them: more workgroups than a dimension of the grid takes."""
    n, k = (1 << 28) - 1, 32
    rng = np.random.default_rng(1)
    a, w = _small(rng, 1, k), _small(rng, 40, k)
    wc, ws = _coded(ctx, n, k, w)
    ac, as_ = (D.DeviceBuffer.from_host(ctx, v) for v in a)
    y = D.DeviceBuffer(ctx, 4 * n)
    X.Matmul(ctx, ac, as_, wc, ws, 1, n, k, A.F32, y)()
    exact = (value_of(*a, k) @ value_of(*w, k).T).astype(np.float32)[0]
    assert np.array_equal(_At(y, 4 * (n - 40), 40, np.float32).download(), exact)
    assert not _At(y, 4 * (n - 1040), 1000, np.float32).download().any()
    for b in (wc, ws, ac, as_, y):
        b.close()


def test_many_rows(ctx):
    """Tiles beyond one dimension of the grid."""
    m, k = (1 << 28) + 77, 32
    rng = np.random.default_rng(2)
    a, w = _small(rng, 100, k), _small(rng, 1, k)
    ac, as_ = _coded(ctx, m, k, a)
    wc, ws = (D.DeviceBuffer.from_host(ctx, v) for v in w)
    y = D.DeviceBuffer(ctx, 2 * m)
    X.Matmul(ctx, ac, as_, wc, ws, m, 1, k, A.BF16, y)()
    exact = (value_of(*a, k) @ value_of(*w, k).T)[:, 0].astype(np.float32)
    got = _At(y, 2 * (m - 100), 100, np.uint16).download().astype(np.uint32) << 16
    want = exact.view(np.uint32)
    assert not (want & 0xFFFF).any() and np.array_equal(got, want)
    assert not _At(y, 2 * (m - 5100), 5000, np.uint16).download().any()
    for b in (wc, ws, ac, as_, y):
        b.close()


def test_activations_of_more_than_2_31_elements(ctx):
    """Coded and read back, and through a linear."""
    m, k, n = 66000, 32768, 16
    rng = np.random.default_rng(3)
    x = rng.choice([-1.5, 1.0, 2.0, -3.0, 0.75], (30, k)).astype(np.float32)
    codes, scales = code_of(x)
    src = D.DeviceBuffer(ctx, 2 * m * k)
    D.memset(ctx, src, 0, src.nbytes)
    _At(src, 2 * (m - 30) * k, (30, k), np.uint16).upload((x.view(np.uint32) >> 16).astype(np.uint16))
    b = X.blocks(k)
    dc, ds = D.DeviceBuffer(ctx, m * b * 16), D.DeviceBuffer(ctx, m * b)
    X.Quantize(ctx, A.BF16, src, k, m, k, dc, ds)()
    assert np.array_equal(_At(dc, (m - 30) * b * 16, codes.shape, np.uint8).download(), codes)
    assert np.array_equal(_At(ds, (m - 30) * b, scales.shape, np.uint8).download(), scales)
    back = D.DeviceBuffer(ctx, 2 * m * k)
    X.Dequantize(ctx, dc, ds, m, k, A.BF16, back, k)()
    v = value_of(codes, scales, k)
    got = _At(back, 2 * (m - 30) * k, (30, k), np.uint16).download().astype(np.uint32) << 16
    assert np.array_equal(got, v.astype(np.float32).view(np.uint32))
    w = _small(rng, n, k)
    lin = D.QuantizedLinear.from_mxfp4(ctx, *(D.DeviceBuffer.from_host(ctx, t) for t in w), n, k)
    y = D.DeviceBuffer.empty(ctx, (m, n), np.float32)
    X.Linear(ctx, lin, A.BF16, src, k, m, A.F32, y)()
    out = y.download()
    assert np.array_equal(out[-30:], (v @ value_of(*w, k).T).astype(np.float32)) and not out[:-30].any()
    lin.close()
    for buf in (src, dc, ds, back, y):
        buf.close()


def test_workspace_that_cannot_be_had(ctx):
    """The refusal leaves nothing behind: the next call is as if it had not been."""
    own = D.Context(0)
    rng = np.random.default_rng(4)
    w = _small(rng, 64, 64)
    lin = D.QuantizedLinear.from_mxfp4(own, *(D.DeviceBuffer.from_host(own, t) for t in w), 64, 64)
    x = rng.choice([-1.5, 1.0, 2.0], (70, 64)).astype(np.float32)
    dx, y = D.DeviceBuffer.from_host(own, x), D.DeviceBuffer.empty(own, (70, 64), np.float32)
    with pytest.raises(_lib.TkvHipError) as e:  # 2^31 - 1 rows of two blocks: more than half a TB with the slabs' start
        X.Matmul(own, dx, dx, dx, dx, (1 << 31) - 1, 70, 131040, A.F32, y, 70)()
    assert e.value.rc == _lib.OOM
    lin.forward(dx, 70, y)
    exact = value_of(*code_of(x), 64) @ value_of(*w, 64).T
    assert np.array_equal(y.download(), exact.astype(np.float32))
    lin.close()
    for b in (dx, y):
        b.close()
    own.close()


def test_scales_of_many_rows_laid_out(ctx):
    """Rows whose scales' slabs take more workgroups than a dimension of the grid,
    161 GB in all: 2^29 and more of two K slices each, the second one block."""
    m, n, k = (1 << 29) + 77, 65, 288
    import torch
    if torch.cuda.mem_get_info(0)[0] < 180 << 30:
        pytest.skip("161 GB of operands and outputs")
    say(f"product {m}x{n}x{k}")
    rng = np.random.default_rng(6)
    a, w = _small(rng, 100, k), _small(rng, n, k)
    a[1][:, 8] = rng.integers(126, 129, 100)
    ac, as_ = _coded(ctx, m, k, a)
    wc, ws = (D.DeviceBuffer.from_host(ctx, v) for v in w)
    y = D.DeviceBuffer(ctx, 2 * m * n)
    X.Matmul(ctx, ac, as_, wc, ws, m, n, k, A.BF16, y)()
    exact = (value_of(*a, k) @ value_of(*w, k).T).astype(np.float32).view(np.uint32)
    want = (exact + 0x7FFF + ((exact >> 16) & 1)) >> 16  # to nearest even
    got = _At(y, 2 * (m - 100) * n, (100, n), np.uint16).download()
    assert np.array_equal(got, want)
    assert not _At(y, 2 * (m - 5100) * n, (5000, n), np.uint16).download().any()
    for b in (wc, ws, ac, as_, y):
        b.close()


def test_rows_of_more_than_one_launch(ctx):
    """More blocks than a launch of the coding takes, marked at the ends of both."""
    cols = 32768
    b = X.blocks(cols)
    per = (1 << 29) // b  # rows of a launch
    m = per + 5
    say(f"code {m}x{cols}")
    rng = np.random.default_rng(8)
    x = rng.choice([-1.5, 1.0, 2.0, -3.0, 0.75], (15, cols)).astype(np.float32)
    codes, scales = code_of(x)
    marked = ((0, slice(0, 5)), (per - 5, slice(5, 15)))
    src = D.DeviceBuffer(ctx, 2 * m * cols)
    dc, ds = D.DeviceBuffer(ctx, m * b * 16), D.DeviceBuffer(ctx, m * b)
    D.memset(ctx, src, 0, src.nbytes)
    for at, r in marked:
        raw = (x[r].view(np.uint32) >> 16).astype(np.uint16)
        _At(src, 2 * at * cols, raw.shape, np.uint16).upload(raw)
    X.Quantize(ctx, A.BF16, src, cols, m, cols, dc, ds)()
    for at, r in marked:
        assert np.array_equal(_At(dc, at * b * 16, codes[r].shape, np.uint8).download(), codes[r])
        assert np.array_equal(_At(ds, at * b, scales[r].shape, np.uint8).download(), scales[r])
    assert not _At(dc, 5 * b * 16, (100, b, 16), np.uint8).download().any()
    assert not _At(dc, (per - 105) * b * 16, (100, b, 16), np.uint8).download().any()
    D.memset(ctx, src, 0xFF, src.nbytes)
    X.Dequantize(ctx, dc, ds, m, cols, A.BF16, src, cols)()
    for at, r in marked:
        got = _At(src, 2 * at * cols, x[r].shape, np.uint16).download().astype(np.uint32) << 16
        assert np.array_equal(got, value_of(codes[r], scales[r], cols).astype(np.float32).view(np.uint32))
    assert not _At(src, 2 * (per - 105) * cols, (100, cols), np.uint16).download().any()
    for buf in (src, dc, ds):
        buf.close()
