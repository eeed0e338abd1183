"""rp_unpack takes the type that was packed, and checks it (nothing is launched)."""

import ctypes

import pytest

from redpanda_amd import _lib

FAKE = 0x100000  # never dereferenced: validation only


@pytest.fixture(scope="module")
def lib():
    return _lib.open_library()


@pytest.mark.parametrize("held", [-1, 3, 77])
def test_an_unknown_type_is_refused(lib, held):
    a = _lib.PackArgs(rows=4, d=40, dtype=0, dtype_held=held, x=FAKE, x_sr=40, q=2 * FAKE, e=3 * FAKE)
    assert lib.rp_unpack(ctypes.byref(a), None) < 0
    assert "packed" in lib.rp_last_error().decode()
