"""Memory that is read and written by one call of the paged cache is refused at the C boundary (pointers are never followed)."""
import ctypes

import pytest

from interactron_amd import _lib
from tests.test_cache_cpu import c_cache

POOL = 6 * 2 * 16 * 64 * 2   # bytes of c_cache's pools
K, V, FREE = 1 << 20, 2 << 20, 4 << 20


def append(c, k, v, T=3):
    # rows [2][T][2][64] of bf16, dense
    return _lib.load().ix_cache_append(ctypes.byref(c), k, v, T, T * 128, 128, 64, T * 128, 128, 64, None, None, None)


@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("at", [K, K + POOL - 16, K - 2 * 3 * 2 * 64 * 2 + 16, K + 1024, V, V + POOL - 16, V - 16])
def test_new_rows_inside_a_pool(which, at):
    rows = dict(dict(k=FREE, v=FREE), **{which: at})
    assert append(c_cache(k=K, v=V), **rows) == -1 and b"parts of the cache's own pools" in _lib.load().ix_last_error()


@pytest.mark.parametrize("k, v", [(K, K), (K, K + POOL - 16), (K + 16, K)])
def test_pools_that_share_memory(k, v):
    L, c = _lib.load(), c_cache(k=k, v=v)
    assert append(c, FREE, FREE) == -1 and b"share memory" in L.ix_last_error()
    assert L.ix_cache_compact(ctypes.byref(c), FREE, FREE, 8, None) == -1 and b"share memory" in L.ix_last_error()
