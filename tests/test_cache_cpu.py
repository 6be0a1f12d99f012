"""Refusals of the paged cache: at the Python entry points and at the C boundary, before anything is launched."""
import ctypes

import pytest
import torch

from interactron_amd import _lib, hipops


def parts(total=6, kv=2, page=16, hd=64, batch=2, pages=3, dtype=torch.bfloat16, weight=True):
    return dict(k=torch.zeros(total, kv, page, hd, dtype=dtype), v=torch.zeros(total, kv, page, hd, dtype=dtype),
                table=torch.zeros(batch, pages, dtype=torch.int32), lens=torch.zeros(batch, dtype=torch.int32),
                weight=torch.zeros(batch, kv, pages * page) if weight else None)


def test_cpu_tensors_are_refused():
    with pytest.raises(_lib.HipLibraryError, match="GPU"):
        hipops.PagedCache(**parts())


@pytest.mark.parametrize("change, words", [
    (dict(k=torch.zeros(6, 2, 16, 64, dtype=torch.float64)), "cache keys"),
    (dict(k=torch.zeros(6, 2, 16, dtype=torch.bfloat16)), "cache keys"),
    (dict(k=torch.zeros(6, 2, 16, 48, dtype=torch.bfloat16)), "head dim 48"),
    (dict(k=torch.zeros(6, 2, 24, 64, dtype=torch.bfloat16)), "page of 24"),
    (dict(k=torch.zeros(6, 2, 8, 64, dtype=torch.bfloat16)), "page of 8"),
    (dict(k=torch.zeros(6, 2, 2048, 64, dtype=torch.bfloat16)), "page of 2048"),
    (dict(k=torch.zeros(0, 2, 16, 64, dtype=torch.bfloat16)), "empty"),
    (dict(v=torch.zeros(6, 2, 16, 64, dtype=torch.float16)), "cache values"),
    (dict(v=torch.zeros(5, 2, 16, 64, dtype=torch.bfloat16)), "cache values"),
    (dict(k=torch.zeros(6, 2, 64, 16, dtype=torch.bfloat16).transpose(2, 3)), "contiguous"),
    (dict(table=torch.zeros(2, 3, dtype=torch.int64)), "page table"),
    (dict(table=torch.zeros(6, dtype=torch.int32)), "page table"),
    (dict(table=torch.zeros(2, 0, dtype=torch.int32)), "empty"),
    (dict(lens=torch.zeros(3, dtype=torch.int32)), "lengths"),
    (dict(lens=torch.zeros(2, dtype=torch.int64)), "lengths"),
    (dict(weight=torch.zeros(2, 2, 47)), "weights"),
    (dict(weight=torch.zeros(2, 2, 48, dtype=torch.float16)), "weights"),
])
def test_cache_of_the_wrong_form_is_refused(change, words):
    with pytest.raises(ValueError, match=words):
        hipops.PagedCache(**dict(parts(), **change))


@pytest.mark.parametrize("name", ["k", "v", "weight"])
def test_cache_tensors_with_a_gradient_are_refused(name):
    made = dict(parts(), weight=torch.zeros(2, 2, 48))
    made[name].requires_grad_(True)
    with pytest.raises(_lib.HipLibraryError, match="gradient"):
        hipops.PagedCache(**made)


@pytest.mark.parametrize("args, words", [
    (dict(budget=0), "budget"), (dict(budget=2.5), "budget"), (dict(budget=True), "budget"), (dict(budget=49), "budget"),
    (dict(budget=8, sinks=5, recent=4), "first"), (dict(budget=8, sinks=-1), "sinks"), (dict(budget=8, recent=-2), "recent"),
    (dict(budget=8, lens=torch.zeros(2)), "lens"), (dict(budget=8, lens=torch.zeros(3, dtype=torch.int32)), "lens"),
    (dict(budget=8, weight=torch.zeros(2, 2, 48, dtype=torch.float64)), "weight"), (dict(budget=8, weight=torch.zeros(4, 48)), "weight"),
    (dict(budget=8, weight=torch.zeros(2, 48, 2).transpose(1, 2)), "weight"), (dict(budget=8, weight=torch.zeros(2, 2, 0)), "weight"),
])
def test_select_refuses(args, words):
    with pytest.raises(ValueError, match=words):
        hipops.cache_select(**dict(dict(weight=torch.zeros(2, 2, 48), lens=torch.zeros(2, dtype=torch.int32)), **args))


def test_select_refuses_cpu_tensors():
    with pytest.raises(_lib.HipLibraryError, match="GPU"):
        hipops.cache_select(torch.zeros(2, 2, 48), torch.zeros(2, dtype=torch.int32), 8)


def c_cache(**change):
    """A cache whose pointers are never followed: every call on it has to be refused by the host checks"""
    f = dict(k=4096, v=4096, table=4096, lens=4096, weight=4096, pages_total=6, dtype=1, kv_heads=2, page=16, hd=64, batch=2, pages=3)
    f.update(change)
    return hipops.cache._CacheC(*[f[n] for n, _ in hipops.cache._CacheC._fields_])


BAD_CACHES = [dict(k=None), dict(v=None), dict(table=None), dict(lens=None), dict(dtype=3), dict(dtype=-1), dict(hd=96), dict(page=24), dict(page=8),
              dict(page=2048), dict(batch=0), dict(batch=70000), dict(kv_heads=0), dict(pages=0), dict(pages_total=0), dict(pages_total=1 << 31),
              dict(pages=1 << 26), dict(k=4100)]


@pytest.mark.parametrize("change", BAD_CACHES, ids=str)
def test_c_entries_refuse_a_bad_cache(change):
    L, c = _lib.load(), c_cache(**change)
    n = ctypes.c_size_t(0)
    calls = [(L.ix_workspace_bytes_cache_attn, (ctypes.byref(c), 4, 0, 0, 0, ctypes.byref(n))),
             (L.ix_cache_attn, (ctypes.byref(c), 4096, 256, 64, 4096, 4, 0.125, 0, 0, 0, 4096, 1 << 30, None)),
             (L.ix_cache_append, (ctypes.byref(c), 4096, 4096, 1, 128, 128, 64, 128, 128, 64, None, None, None)),
             (L.ix_cache_compact, (ctypes.byref(c), 4096, 4096, 8, None))]
    for fn, args in calls:
        assert fn(*args) == -1 and L.ix_last_error()


@pytest.mark.parametrize("entry, args, code", [
    ("attn", dict(heads=3), -1), ("attn", dict(heads=0), -1), ("attn", dict(heads=8192), -1), ("attn", dict(q=None), -1), ("attn", dict(q=4104), -1),
    ("attn", dict(sq_h=60), -1), ("attn", dict(window=-1), -1), ("attn", dict(sinks=-1), -1), ("attn", dict(accumulate=1, ws=4096, nbytes=16), -3),
    ("attn", dict(accumulate=1, ws=None), -3), ("attn", dict(accumulate=1, weight=None), -1),
    ("append", dict(T=-1), -1), ("append", dict(k=None), -1), ("append", dict(v=4104), -1), ("append", dict(st=60), -1),
    ("compact", dict(kept=None), -1), ("compact", dict(left=None), -1), ("compact", dict(left=8192), -1), ("compact", dict(budget=0), -1),
    ("select", dict(weight=None), -1), ("select", dict(budget=0), -1), ("select", dict(budget=64), -1), ("select", dict(sinks=5, recent=4), -1),
    ("select", dict(sinks=-1), -1), ("select", dict(batch=0), -1), ("select", dict(lens=12288), -1), ("select", dict(lens=12292), -1),
    ("append", dict(T=(1 << 30) - 1), -1), ("compact", dict(left=8196), -1), ("append", dict(counts=8196), -1), ("append", dict(at=8188), -1),
])
def test_c_entries_refuse_bad_arguments(entry, args, code):
    L = _lib.load()
    a = dict(q=4096, sq_b=256, sq_h=64, out=4096, heads=4, window=0, sinks=0, accumulate=0, ws=None, nbytes=0, k=4096, v=4096, T=1, st=128, kept=4096,
             left=12288, budget=8, weight=4096, lens=8192, batch=2, recent=0, counts=None, at=None)
    a.update(args)
    c = c_cache(lens=8192, weight=a["weight"])
    if entry == "attn":
        rc = L.ix_cache_attn(ctypes.byref(c), a["q"], a["sq_b"], a["sq_h"], a["out"], a["heads"], 0.125, a["window"], a["sinks"], a["accumulate"], a["ws"], a["nbytes"], None)
    elif entry == "append":
        rc = L.ix_cache_append(ctypes.byref(c), a["k"], a["v"], a["T"], 128, a["st"], 64, 128, 128, 64, a["counts"], a["at"], None)
    elif entry == "compact":
        rc = L.ix_cache_compact(ctypes.byref(c), a["kept"], a["left"], a["budget"], None)
    else:
        rc = L.ix_cache_select(a["weight"], a["lens"], 4096, a["left"], a["batch"], 2, 48, a["budget"], a["sinks"], a["recent"], None)
    assert rc == code, (rc, L.ix_last_error())
