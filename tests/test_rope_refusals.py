"""Rotations whose angles are no numbers are refused before a device is touched."""
import ctypes as C

import pytest

import edgexpu_amd as E


@pytest.mark.parametrize("factors,base,scale", [
    ([1.0, 0.0, 1.0, 1.0], 1e4, 1.0), ([1.0, 1.0, 1.0, -0.0], 1e4, 1.0), ([float("nan"), 1.0, 1.0, 1.0], 1e4, 1.0),
    ([1.0, 1.0, 1.0, 1e-40], 1e-200, 1e200), (None, 1e-300, 1e100), (None, 1e4, 1e301),
])
def test_angles_that_are_no_numbers(factors, base, scale):
    L = E.HipLib()
    L.clear_error()
    f = None if factors is None else (C.c_float * 4)(*factors)
    assert not L.rope_create(8, base, scale, f, 0)
    code, msg = L.last_error()
    L.clear_error()
    assert code == -2 and "rope_create" in msg, (code, msg)
