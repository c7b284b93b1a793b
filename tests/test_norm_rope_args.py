"""Arguments of the norm-and-rotation entry point that are refused on the host,
before any device, and the axes of the pairs."""
import ctypes as C

import pytest

from tokenvector.inference_amd import _lib
from tokenvector.inference_amd import attention as A
from tokenvector.inference_amd import device as D

P = 1 << 20


def _call(norm=None, rope=None, typ=A.F32, tokens=1, hq=1, hkv=1, d=64, rows=True):
    r = C.byref(A._Rows(P, 64, 64)) if rows else None
    n = C.byref(A._HeadNorm(*norm)) if norm else None
    ro = C.byref(A._Rope(*rope)) if rope else None
    return _lib.lib().tkv_hip_dev_norm_rope_append(0, typ, tokens, hq, hkv, d, r, r, r, n, ro, r, r, A.F32, 0, None)


AXES = (C.c_uint8 * 32)(*([0, 1, 2, 0] * 8))


def _rope(**change):
    v = {"table": P, "table_len": 10, "rot_dim": 64, "layout": 0, "axes": 3, "positions": P, "stride_axis": 4,
         "pair_axis": C.cast(AXES, C.c_void_p).value, **change}
    return tuple(v.values())


@pytest.mark.parametrize("norm", [(0.0, None, None), (-1e-6, None, None), (float("nan"), None, None),
                                  (float("inf"), None, None), (1e-6, P + 2, None), (1e-6, None, P + 1)])
def test_norm(norm):
    assert _call(norm) == _lib.BAD_ARG


@pytest.mark.parametrize("change", [
    {"table": None}, {"table": P + 4}, {"rot_dim": 63}, {"rot_dim": 0}, {"rot_dim": 128}, {"table_len": -1}, {"layout": 2},
    {"axes": 0}, {"axes": 5}, {"axes": 2}, {"positions": None}, {"pair_axis": None}])
def test_rope(change):
    """(axes 2: the pairs name a third)"""
    assert _call((1e-6, None, None), _rope(**change)) == _lib.BAD_ARG


@pytest.mark.parametrize("change", [{"typ": A.I8}, {"tokens": -1}, {"tokens": 1 << 31}, {"d": 257}, {"d": 0},
                                    {"hq": -1}, {"hkv": 65536}, {"rows": False}])
def test_sizes(change):
    assert _call((1e-6, None, None), _rope(), **change) == _lib.BAD_ARG


def test_no_device_is_reported():
    if _lib.lib().tkv_hip_device_count() > 0:
        pytest.skip("a gfx950 device is visible: the no-device path cannot be observed")
    assert _call((1e-6, P, P), _rope()) == _lib.NO_DEVICE
    assert _call() == _lib.NO_DEVICE


def test_pair_axes():
    assert A.rope_pair_axes([4]) == [0, 0, 0, 0]
    assert A.rope_pair_axes([2, 1, 1]) == [0, 0, 1, 2]
    assert A.rope_pair_axes([3, 1, 2], interleaved=True) == [0, 1, 2, 0, 2, 0]
    for bad in ([], [0], [1, -1], [1, 1, 1, 1, 1]):
        with pytest.raises(ValueError):
            A.rope_pair_axes(bad)


class _Ctx:
    handle = 0


class _Memory(D.DeviceBuffer):
    def __init__(self):
        self.ptr, self.nbytes, self.ctx = P, 64, None

    def close(self):
        self.ptr = 0


@pytest.mark.parametrize("which", range(5))
def test_call_of_a_closed_buffer(which):
    """Gains, table and positions among them."""
    b, launched = [_Memory() for _ in range(5)], []
    rows = A.Rows(b[4], 64, 64)
    call = A.NormRopeAppend(_Ctx, A.F32, 1, 1, 0, 64, rows, norm=A.HeadNorm(1e-6, b[0], b[1]),
                            rope=A.Rope(b[2], 4, 64, A.ROPE_HALF, b[3]))
    call._fn = lambda *args: launched.append(args) and 0
    call()
    b[which].close()
    with pytest.raises(ValueError, match="closed"):
        call()
    assert len(launched) == 1


def test_axes_of_the_pairs_are_complete():
    rope = A.Rope(P, 4, 64, A.ROPE_HALF, P, 2, 4, [0, 1])
    with pytest.raises(ValueError, match="pair_axis"):
        A.NormRopeAppend(_Ctx, A.F32, 1, 1, 0, 64, A.Rows(P, 64, 64), rope=rope)
