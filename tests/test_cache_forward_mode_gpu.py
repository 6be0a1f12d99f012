"""The paged cache refuses tensors that carry a forward-mode derivative."""
import pytest
import torch
import torch.autograd.forward_ad as fwd_ad

from interactron_amd import _lib, hipops
from tests.test_cache_gpu import FP32, make, query

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("grad_mode", [True, False])
def test_tangents_are_refused(grad_mode):
    cache = make([40, 60], dtype=FP32, pages=6)
    q, new = query(cache, 4), torch.randn(2, 1, cache.kv_heads, cache.hd, device="cuda")
    lens = cache.lens.clone()
    with fwd_ad.dual_level(), torch.set_grad_enabled(grad_mode):
        dual = lambda t: fwd_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in (lambda: hipops.cache_attention(dual(q), cache), lambda: hipops.cache_append(cache, dual(new), new),
                     lambda: hipops.cache_append(cache, new, dual(new)), lambda: hipops.PagedCache(dual(cache.k), cache.v, cache.table, cache.lens),
                     lambda: hipops.PagedCache(cache.k, cache.v, cache.table, cache.lens, dual(cache.weight))):
            with pytest.raises(_lib.HipLibraryError, match="forward-mode"):
                call()
        hipops.cache_attention(q, cache)
    assert torch.equal(cache.lens, lens)
