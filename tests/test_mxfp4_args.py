"""Arguments that the 4-bit entry points refuse on the host, before any device,
and the Python side of their calls."""
import ctypes as C

import pytest

from tokenvector.inference_amd import _lib
from tokenvector.inference_amd import attention as A
from tokenvector.inference_amd import device as D
from tokenvector.inference_amd import mxfp4 as X

P = 1 << 20  # an address, 16-byte aligned, that nothing reads


def test_blocks():
    assert [X.blocks(k) for k in (1, 32, 33, 768)] == [1, 1, 2, 24]


@pytest.mark.parametrize("args", [
    (A.I8, P, 32, 1, 32, P, P), (7, P, 32, 1, 32, P, P), (A.F32, P, 32, -1, 32, P, P), (A.F32, P, 32, 1, 0, P, P),
    (A.F32, P, 31, 2, 32, P, P), (A.F32, P, 32, 1 << 31, 32, P, P), (A.F32, P, 1 << 31, 1, 1 << 31, P, P),
    (A.F32, None, 32, 1, 32, P, P), (A.F32, P, 32, 1, 32, None, P), (A.F32, P, 32, 1, 32, P, None),
    (A.F32, P, 32, 1, 32, P + 8, P), (A.F32, P + 2, 32, 1, 32, P, P), (A.BF16, P + 1, 32, 1, 32, P, P)])
def test_quantize_and_dequantize(args):
    L = _lib.lib()
    typ, x, stride, rows, cols, codes, scales = args
    assert L.tkv_hip_dev_quantize_mxfp4(0, typ, x, stride, rows, cols, codes, scales) == _lib.BAD_ARG
    assert L.tkv_hip_dev_dequantize_mxfp4(0, codes, scales, rows, cols, typ, x, stride) == _lib.BAD_ARG


@pytest.mark.parametrize("change,rc", [
    ({"a": None}, _lib.BAD_ARG), ({"w": P + 8}, _lib.BAD_ARG), ({"a": P + 4}, _lib.BAD_ARG), ({"y": None}, _lib.BAD_ARG),
    ({"as_": None}, _lib.BAD_ARG), ({"ws": None}, _lib.BAD_ARG), ({"m": -1}, _lib.BAD_ARG), ({"n": -1}, _lib.BAD_ARG),
    ({"k": 0}, _lib.BAD_ARG), ({"typ": A.I8}, _lib.BAD_ARG), ({"stride": 63}, _lib.BAD_ARG), ({"y": P + 2}, _lib.BAD_ARG),
    ({"k": 1 << 17}, _lib.UNSUPPORTED), ({"m": 1 << 31}, _lib.UNSUPPORTED),
    ({"n": 1 << 28, "stride": 1 << 28}, _lib.UNSUPPORTED)])
def test_matmul(change, rc):
    v = {"a": P, "as_": P, "w": P, "ws": P, "m": 4, "n": 64, "k": 64, "typ": A.F32, "y": P, "stride": 64, **change}
    assert _lib.lib().tkv_hip_dev_matmul_mxfp4(0, v["a"], v["as_"], v["w"], v["ws"], v["m"], v["n"], v["k"], None,
                                               v["typ"], v["y"], v["stride"]) == rc


def test_linear_and_weight():
    L = _lib.lib()
    h = C.c_int64()
    assert L.tkv_hip_linear_forward_typed(0, 0, A.F32, P, 64, 1, A.F32, P, 64) == _lib.BAD_ARG
    for codes, scales, n, k, out in ((None, P, 4, 32, C.byref(h)), (P, None, 4, 32, C.byref(h)),
                                     (P, P, 0, 32, C.byref(h)), (P, P, 4, 0, C.byref(h)), (P, P, 4, 32, None)):
        assert L.tkv_hip_weight_create_mxfp4(0, codes, scales, n, k, None, out) == _lib.BAD_ARG


def test_no_device_is_reported():
    L = _lib.lib()
    if L.tkv_hip_device_count() > 0:
        pytest.skip("a gfx950 device is visible: the no-device path cannot be observed")
    h = C.c_int64()
    assert L.tkv_hip_dev_quantize_mxfp4(0, A.F32, P, 32, 1, 32, P, P) == _lib.NO_DEVICE
    assert L.tkv_hip_dev_dequantize_mxfp4(0, P, P, 1, 32, A.F32, P, 32) == _lib.NO_DEVICE
    assert L.tkv_hip_dev_matmul_mxfp4(0, P, P, P, P, 1, 1, 32, None, A.F32, P, 1) == _lib.NO_DEVICE
    assert L.tkv_hip_weight_create_mxfp4(0, P, P, 1, 32, None, C.byref(h)) == _lib.NO_DEVICE


class _Ctx:
    handle = 0


class _Memory(D.DeviceBuffer):
    def __init__(self):
        self.ptr, self.nbytes, self.ctx = P, 64, None

    def close(self):
        self.ptr = 0


class _Weight(D.QuantizedLinear):
    def __init__(self):
        self.handle, self.n, self.k = P, 64, 64

    def close(self):
        self.handle = 0


@pytest.mark.parametrize("closed", ["weight", "buffer"])
def test_call_of_a_closed_weight_or_buffer(closed):
    weight, buffer, launched = _Weight(), _Memory(), []
    call = X.Linear(_Ctx, weight, A.F32, buffer, 64, 1, A.F32, buffer)
    call._fn = lambda *args: launched.append(args) and 0
    call()
    {"weight": weight, "buffer": buffer}[closed].close()
    with pytest.raises(ValueError, match="closed"):
        call()
    assert len(launched) == 1
