"""Refusals of the entry point for some of band attention's gradients."""
import ctypes

import pytest

from interactron_amd import _lib
from tests.test_band_cpu import c_band


@pytest.mark.parametrize("want, dq, dk, dv, ws, code", [
    (0, 4096, 4096, 4096, 4096, -1), (4, 4096, 4096, 4096, 4096, -1), (-1, 4096, 4096, 4096, 4096, -1), (1, None, 4096, 4096, 4096, -1), (1, 4104, None, None, 4096, -1),
    (2, 4096, None, 4096, 4096, -1), (2, 4096, 4096, None, 4096, -1), (2, None, 4104, 4096, 4096, -1), (3, None, 4096, 4096, 4096, -1),
    (1, 4096, None, None, None, -3), (2, None, 4096, 4096, None, -3), (1, 4096, 4104, 4104, None, -3), (2, 4104, 4096, 4096, None, -3)])
def test_wrong_pointers(want, dq, dk, dv, ws, code):
    L = _lib.load()
    rc = L.ix_band_attn_bwd_some(ctypes.byref(c_band()), want, 4096, 4096, 4096, 4096, 1280, 256, 64, dq, dk, dv, ws, 1 << 30 if ws else 0, None)
    assert rc == code and L.ix_last_error()
