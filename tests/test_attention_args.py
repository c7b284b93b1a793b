"""The attention entry points' argument checks that need no device, and the
rotation frequencies."""
import ctypes as C

import numpy as np
import pytest

from tokenvector.inference_amd import _lib
from tokenvector.inference_amd import attention as A


def test_bad_arguments_before_any_device():
    L = _lib.lib()
    h = C.c_int64()
    assert L.tkv_hip_kv_create(0, 7, 1, 16, 1, 64, None, None, None, None, C.byref(h)) == _lib.BAD_ARG
    assert L.tkv_hip_kv_create(0, A.F32, 1, 16, 1, 300, None, None, None, None, C.byref(h)) == _lib.BAD_ARG
    assert L.tkv_hip_kv_create(0, A.F32, 1, 16, 1, 64, None, None, None, None, None) == _lib.BAD_ARG
    assert L.tkv_hip_kv_info(0, None, None, None, None) == _lib.BAD_ARG
    assert L.tkv_hip_kv_free(0) == _lib.OK
    assert L.tkv_hip_dev_rope_table(0, 4, 3, None, 1.0, None) == _lib.BAD_ARG
    rows = A._Rows(16, 64, 64)
    r = C.byref(rows)
    assert L.tkv_hip_dev_attention_prompt(0, A.F32, 1, 1, 3, 2, 64, 1, r, r, r, r, A.F32, 16, None, 1.0, 1,
                                          0) == _lib.BAD_ARG
    assert L.tkv_hip_dev_attention_paged(0, A.F32, 1, 1, 0, 1, r, r, A.F32, 16, 1, None, 16, 0, 0, 1.0, 1,
                                         0) == _lib.BAD_ARG
    assert L.tkv_hip_dev_rope_append(0, A.I8, 1, 1, 1, 64, r, r, r, None, None, 0, 0, 0, r, r, A.F32, 0,
                                     None) == _lib.BAD_ARG


def test_no_device_is_reported():
    L = _lib.lib()
    if L.tkv_hip_device_count() > 0:
        pytest.skip("a gfx950 device is visible: the no-device path cannot be observed")
    h = C.c_int64()
    rows = A._Rows(16, 64, 64)
    r = C.byref(rows)
    assert L.tkv_hip_kv_create(0, A.F32, 1, 16, 1, 64, None, None, None, None, C.byref(h)) == _lib.NO_DEVICE
    assert L.tkv_hip_dev_attention_prompt(0, A.F32, 1, 1, 2, 2, 64, 1, r, r, r, r, A.F32, 16, None, 1.0, 1,
                                          0) == _lib.NO_DEVICE
    assert L.tkv_hip_dev_rope_append(0, A.F32, 1, 1, 1, 64, r, r, r, None, None, 0, 0, 0, r, r, A.F32, 0,
                                     None) == _lib.NO_DEVICE


def test_frequencies():
    inv = A.rope_inv_freq(64)
    assert inv.dtype == np.float64 and inv.shape == (32,)
    assert inv[0] == 1.0 and np.isclose(inv[-1], 10000.0 ** (-62 / 64), rtol=1e-15)
    assert np.array_equal(A.rope_inv_freq(64, factor=4.0), inv / 4.0)
    parts = A.rope_inv_freq(64, factor=4.0, by_parts=True, original_positions=8192)
    turns = 8192 * inv / (2 * np.pi)
    assert np.array_equal(parts[turns >= 32], inv[turns >= 32])
    assert np.array_equal(parts[turns <= 1], (inv / 4.0)[turns <= 1])
    mid = (turns > 1) & (turns < 32)
    assert mid.any() and np.all((parts[mid] < inv[mid]) & (parts[mid] > inv[mid] / 4.0))
    for bad in ({"rot_dim": 3}, {"rot_dim": 0}, {"rot_dim": 8, "factor": 0.0}, {"rot_dim": 8, "by_parts": True}):
        with pytest.raises(ValueError):
            A.rope_inv_freq(**bad)
