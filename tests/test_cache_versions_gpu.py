"""The calls that write a paged cache in place are seen by autograd, as torch's own in-place operations are."""
import pytest
import torch

from tests.test_cache_gpu import BF16, FP32, make, query

pytestmark = pytest.mark.gpu

CHANGED = "modified by an inplace operation"


def rows(cache, T=1):
    return torch.randn(cache.batch, T, cache.kv_heads, cache.hd, device="cuda").to(cache.dtype)


def write(cache, how):
    from interactron_amd import hipops
    if how == "append":
        hipops.cache_append(cache, rows(cache), rows(cache))
    elif how == "accumulate":
        hipops.cache_attention(query(cache, 4), cache, accumulate=True)
    elif how == "compact":
        kept, left = hipops.cache_select(cache.weight, cache.lens, 20)
        hipops.cache_compact(cache, kept, left)
    elif how == "evict":
        hipops.cache_evict(cache, 20)
    else:   # (reads only)
        hipops.cache_attention(query(cache, 4), cache)
        hipops.cache_select(cache.weight, cache.lens, 20)


WRITES = {"append": {"k", "v", "lens", "weight"}, "accumulate": {"weight"}, "compact": {"k", "v", "lens", "weight"},
          "evict": {"k", "v", "lens", "weight"}, "read": set()}


@pytest.mark.parametrize("how", list(WRITES))
def test_version_counters(how):
    cache = make([40, 60], dtype=FP32)
    before = {x: getattr(cache, x)._version for x in ("k", "v", "table", "lens", "weight")}
    write(cache, how)
    assert {x for x in before if getattr(cache, x)._version != before[x]} == WRITES[how]


@pytest.mark.parametrize("name", ["k", "v", "weight"])
@pytest.mark.parametrize("how", list(WRITES))
def test_a_graph_that_saved_a_tensor_of_the_cache(how, name):
    cache = make([40, 60], dtype=FP32)
    x = torch.ones((), device="cuda", requires_grad=True)
    loss = (getattr(cache, name) * x).sum()
    want = getattr(cache, name).sum()
    write(cache, how)
    if name in WRITES[how]:
        with pytest.raises(RuntimeError, match=CHANGED):
            loss.backward()
    else:
        loss.backward()
        assert torch.allclose(x.grad, want)


@pytest.mark.parametrize("how", ["append", "evict"])
@pytest.mark.parametrize("lens", ["q_lens", "kv_lens"])
def test_lengths_of_band_attention_that_a_cache_holds(how, lens):
    """the gradients read the lengths again: after the call they stand for other positions"""
    from interactron_amd import hipops
    cache = make([40, 60], dtype=BF16, pages=6)
    q, k, v = (torch.randn(2, 64, 2, 64, device="cuda").to(BF16).requires_grad_(True) for _ in range(3))
    out = hipops.band_attention(q, k, v, window=9, **{lens: cache.lens})
    write(cache, how)
    with pytest.raises(RuntimeError, match=CHANGED):
        out.sum().backward()


def test_tensors_made_in_inference_mode():
    with torch.inference_mode():
        cache = make([40, 60], dtype=BF16, pages=6)
        for how in WRITES:
            write(cache, how)
    with torch.no_grad():   # (they have no counters and no graph can save them)
        write(cache, "append")
    assert cache.lens.tolist() == [21, 21]
