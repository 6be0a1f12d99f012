"""A scale is refused where its product with log2(e) is no float32 any more, not only where it is none itself."""
import ctypes

import pytest
import torch

from interactron_amd import _lib, hipops
from tests.test_band_cpu import c_band, qkv
from tests.test_cache_cpu import c_cache

BAD = [2.36e38, -2.36e38, 2.99e38, 3.4e38, float("inf"), float("-inf"), float("nan")]


@pytest.mark.parametrize("scale", BAD)
def test_band_attention(scale):
    with pytest.raises(ValueError, match="scale"):
        hipops.band_attention(*qkv(), scale=scale)


@pytest.mark.parametrize("scale", [2.34e38, -2.34e38, 0.0, 1e-45])
def test_scales_that_are_none_of_these(scale):
    with pytest.raises(_lib.HipLibraryError, match="GPU"):   # (these are CPU tensors)
        hipops.band_attention(*qkv(), scale=scale)


@pytest.mark.parametrize("scale", BAD)
def test_c_entries(scale):
    L, n = _lib.load(), ctypes.c_size_t(0)
    band = ctypes.byref(c_band(scale=scale))
    assert L.ix_band_attn_fwd(band, 4096, 4096, 4096, 4096, 1 << 30, None) == -1 and b"scale" in L.ix_last_error()
    assert L.ix_workspace_bytes_band_attn_bwd(band, ctypes.byref(n)) == -1 and b"scale" in L.ix_last_error()
    rc = L.ix_cache_attn(ctypes.byref(c_cache()), 4096, 256, 64, 4096, 4, scale, 0, 0, 0, 4096, 1 << 30, None)
    assert rc == -1 and b"scale" in L.ix_last_error()
