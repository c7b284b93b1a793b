"""GPU tests of products and linears of 4-bit operands by the kernel that their sizes
take: one size of whole tiles or blocks and one with edges for each kernel that the
other tests' sizes leave out (test_mxfp4_plan.py holds the sizes to their kernels, and
the kernels to the sizes).  Scales 2^-1 .. 2^1: sums are exact in f32, as there."""
import numpy as np
import pytest

from tokenvector.inference_amd import attention as A
from tokenvector.inference_amd import device as D
from tokenvector.inference_amd import mxfp4 as X
from test_gpu_mxfp4 import (NAME, TYPES, _operand, _product, _round, _rows_buffer, _unpad, code_of, ctx,  # noqa: F401
                            same, say, value_of)

pytestmark = pytest.mark.gpu

# kernel: tiles, or few rows with their blocks of 16 tokens, 16-row blocks and waves
PRODUCTS = [("tile 128 slabs", 2048, 4096, 4096), ("tile 128 slabs", 2047, 4093, 4000),
            ("tile 64 slabs", 300, 8000, 4200), ("tile 64 ring slabs", 65, 3001, 4500),
            ("few rows 1 4 8", 5, 16400, 8200), ("few rows 1 4 8", 16, 16384, 8192)]
LINEARS = [("tile 256 slabs", 3999, 4071, 1100), ("tile 128 slabs", 2048, 4096, 2000),
           ("tile 64 slabs", 1000, 2304, 256), ("tile 64 slabs", 2003, 1997, 300), ("tile 64 slabs", 5000, 611, 1542),
           ("tile 128x64 slabs", 2500, 2304, 768),
           ("few coding 1 1 16", 4, 2048, 8192), ("few coding 1 1 16", 3, 2050, 8196), ("few coding 1 1 16", 3, 2043, 8195),
           ("few slabs 1 1 8 split", 16, 33, 9420), ("few slabs 2 1 8 split", 32, 640, 16000),
           ("few slabs 1 4 8", 14, 16400, 8200), ("few slabs 2 1 8", 24, 500, 3000), ("few slabs 2 1 8", 19, 515, 4001),
           ("few slabs 2 2 8", 24, 8200, 1000), ("few slabs 2 2 8", 31, 8209, 333), ("few slabs 4 1 8", 60, 500, 2000),
           ("few slabs 4 1 8", 49, 530, 2500), ("few slabs 4 2 8", 60, 8200, 500), ("few slabs 4 2 8", 64, 8230, 801)]


@pytest.mark.parametrize("kernel,m,n,k", PRODUCTS)
@pytest.mark.parametrize("out", TYPES, ids=NAME.get)
def test_product(ctx, kernel, m, n, k, out):  # noqa: F811
    say(f"{kernel}: product {m}x{n}x{k} {NAME[out]}")
    rng = np.random.default_rng(m + n + k)
    a, w = _operand(rng, m, k, 1), _operand(rng, n, k, 1)
    bias = np.round(rng.standard_normal(n) * 64).astype(np.float32) / 16
    exact = value_of(*a, k) @ value_of(*w, k).T
    assert np.abs(exact).max() < 2.0 ** 19
    pad = m % 2 * 3
    same(_product(ctx, a, w, m, n, k, out, bias, pad), _round((exact + bias).astype(np.float32), out))


@pytest.mark.parametrize("kernel,m,n,k", LINEARS)
@pytest.mark.parametrize("typ", TYPES, ids=NAME.get)
def test_linear(ctx, kernel, m, n, k, typ):  # noqa: F811
    say(f"{kernel}: linear {m}x{n}x{k} {NAME[typ]}")
    rng = np.random.default_rng(m + n + k)
    x = _round(rng.uniform(0.6, 1.9, (m, k)).astype(np.float32) * rng.choice([-1.0, 1.0], (m, k)), typ)
    w, bias = _operand(rng, n, k, 1), rng.integers(-64, 64, n).astype(np.float32) / 8
    exact = value_of(*code_of(x), k) @ value_of(*w, k).T + bias
    lin = D.QuantizedLinear.from_mxfp4(ctx, *(D.DeviceBuffer.from_host(ctx, v) for v in w), n, k,
                                       D.DeviceBuffer.from_host(ctx, bias))
    pad = n % 2 * 5
    src = _rows_buffer(ctx, x, typ, k + pad)
    for out in (A.F32, typ):
        y = _rows_buffer(ctx, np.zeros((m, n), np.float32), out, n + pad)
        X.Linear(ctx, lin, typ, src.ptr, k + pad, m, out, y.ptr, n + pad)()
        same(_unpad(y, m, n, out, pad), _round(exact.astype(np.float32), out))
    lin.close()
