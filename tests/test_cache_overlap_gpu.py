"""Pools and new rows that lie next to each other in one allocation, or are the same."""
import pytest
import torch

from interactron_amd import _lib, hipops

pytestmark = pytest.mark.gpu


def test_one_allocation():
    both = torch.zeros(3, 6, 2, 16, 64, device="cuda", dtype=torch.bfloat16)
    both[2] = torch.randn(6, 2, 16, 64)
    table, lens = torch.arange(4, dtype=torch.int32, device="cuda").view(2, 2), torch.zeros(2, dtype=torch.int32, device="cuda")
    cache = hipops.PagedCache(both[0], both[1], table, lens)
    new = both[2].permute(0, 2, 1, 3)[:2]   # [2, 16, 2, 64] right behind the pools
    hipops.cache_append(cache, new, new)
    assert torch.equal(both[0, table[:, 0].long()], new.transpose(1, 2)) and torch.equal(both[0], both[1]) and lens.tolist() == [16, 16]
    for own in (both[0], both[1]):
        with pytest.raises(_lib.HipLibraryError, match="own pools"):
            hipops.cache_append(cache, own.permute(0, 2, 1, 3)[:2], new)
    assert lens.tolist() == [16, 16]
    # the last page of the values' pool and what lies behind it
    with pytest.raises(_lib.HipLibraryError, match="own pools"):
        hipops.cache_append(cache, new, both.view(18, 2, 16, 64).permute(0, 2, 1, 3)[11:13])


def test_keys_that_are_the_values():
    """reading them is no trouble, writing is refused"""
    pool = torch.randn(6, 2, 16, 64, device="cuda")
    table, lens = torch.arange(4, dtype=torch.int32, device="cuda").view(2, 2), torch.full((2,), 30, dtype=torch.int32, device="cuda")
    cache, apart = hipops.PagedCache(pool, pool, table, lens), hipops.PagedCache(pool, pool.clone(), table, lens)
    q, new = torch.randn(2, 4, 64, device="cuda"), torch.randn(2, 1, 2, 64, device="cuda")
    assert torch.equal(hipops.cache_attention(q, cache), hipops.cache_attention(q, apart))
    kept, left = torch.zeros(2, 2, 8, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    for call in (lambda: hipops.cache_append(cache, new, new), lambda: hipops.cache_compact(cache, kept, left)):
        with pytest.raises(_lib.HipLibraryError, match="share memory"):
            call()
