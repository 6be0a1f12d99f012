"""hipops.cache -- a paged cache of keys and values for sequences that grow token by token: writing new tokens, attention of one new token
per sequence, and cutting the cache back to the tokens that have had the most attention (csrc/cache.hip).

    cache = hipops.PagedCache(k, v, table, lens, weight)      # tensors of the caller; nothing is copied
    hipops.cache_append(cache, new_k, new_v)                  # [B, T, kv_heads, hd] each, at the end of every sequence
    out = hipops.cache_attention(q, cache, accumulate=True)   # q [B, heads, hd] -> [B, heads, hd]
    hipops.cache_evict(cache, budget, sinks=4, recent=256)    # in place; the pages behind the budget are free again

None of these has a backward.  All of them are ordered on the current stream, never wait for the GPU, take their sizes from the shapes
alone (the lengths stay on the device; a call's pieces and workspace follow the table's capacity, so a table much larger than the lengths costs
a second launch) and may be captured into a HIP graph.

For stacks of causal layers, where a token's keys and values stay what they were when it came.  The package's own fusion transformer is none:
every token attends to all frames, so a new frame changes the earlier tokens from the second layer on, and it is run over all frames again
(reference models/interactron.py:166-190); no model of the package holds a cache.  Several new tokens of a sequence at once attend through
band_attention over dense keys.
"""
import ctypes

import torch

from .. import _lib
from . import core
from .core import _L, _chk, _no_tangents, _stream

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_HEAD_DIMS = (32, 64, 128)
_PAGES = (16, 32, 64, 128, 256, 512, 1024)
_CACHE_NAMES = ("cache keys", "cache values", "the page table", "the lengths", "the weights")


class _CacheC(ctypes.Structure):   # struct ix_paged_cache of include/interactron_hip.h
    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("table", ctypes.c_void_p), ("lens", ctypes.c_void_p),
                ("weight", ctypes.c_void_p), ("pages_total", ctypes.c_int64), ("dtype", ctypes.c_int), ("kv_heads", ctypes.c_int),
                ("page", ctypes.c_int), ("hd", ctypes.c_int), ("batch", ctypes.c_int), ("pages", ctypes.c_int)]


_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
# for tensors that a kernel has written: a graph that saved one of them raises at its backward pass, as it does after torch's own in-place
# operations, instead of computing with the new values  (the accessor without the wrapper's checks is 1 us cheaper)
_written = getattr(torch._C, "_increment_version", torch.autograd.graph.increment_version)


def _here(names, *ts):
    """The current stream, after checking that every tensor lives on the device this process computes on."""
    dev = core._dev[0]
    if dev is None:
        for t, name in zip(ts, names):
            if t is not None and not t.is_cuda:
                raise _lib.HipLibraryError("%s must live on the GPU: the HIP path has no CPU fallback" % name)
        _stream()   # (binds the device)
        dev = torch.cuda.current_device() if core._dev[0] is None else core._dev[0]
    for t in ts:
        if t is not None and t.get_device() != dev:
            name = next(n for x, n in zip(ts, names) if x is t)
            if not t.is_cuda:
                raise _lib.HipLibraryError("%s must live on the GPU: the HIP path has no CPU fallback" % name)
            raise _lib.HipLibraryError("%s lives on cuda:%d but this process computes on cuda:%d (one process per GPU)" % (name, t.get_device(), dev))
    if _device() != dev:
        raise _lib.HipLibraryError("the current device is cuda:%d but this process computes on cuda:%d (one process per GPU)" % (_device(), dev))
    return _stream()


def _whole(t, name, dtype, shape):
    if t.dtype is not dtype or t.shape != shape:
        raise ValueError("%s must be %s %s, got %s %s" % (name, dtype, list(shape), t.dtype, list(t.shape)))
    if not t.is_contiguous():
        raise ValueError("%s must be contiguous: it is used in place" % name)


def _count(x, name, least=0):
    if isinstance(x, bool) or not isinstance(x, int) or x < least or x >= 1 << 30:
        raise ValueError("%s must be a whole number from %d to 2^30 - 1, got %r" % (name, least, x))
    return x


def _scale(scale, hd):
    """A softmax's factor; exponents are taken to base 2, so scale log2(e) has to be a float32 too"""
    scale = hd ** -0.5 if scale is None else float(scale)
    if not abs(scale) < 2.35e38:   # (and no NaN)
        raise ValueError("scale must be a finite number below 2.35e38, got %r" % scale)
    return scale


class PagedCache:
    """Keys and values of `batch` sequences in pages of a shared pool.

    k, v     [pages_total, kv_heads, page, hd], float32, bfloat16 or float16; hd 32, 64 or 128; page a power of two, 16 .. 1024
    table    int32 [batch, pages]: the pages of every sequence in order; token t is row t % page of page table[b, t // page].  Entries
             behind a sequence's length may hold anything; one that is outside the pool counts as masked and is never written through.
             Sequences may share pages that all of them only read; a page that is written has one place in the table.
    lens     int32 [batch]: tokens held
    weight   float32 [batch, kv_heads, pages * page] or None: the attention each token has had so far
    The tensors are written in place, so none of them may require a gradient, and they cannot be exchanged for others (make another cache:
    it costs nothing but the checks).  A call that writes some of them raises their version counters: a graph that saved one (the lengths of
    band_attention, say) refuses its backward pass afterwards.  (The replay of a captured call does not, like that of torch's own.)
    """
    __slots__ = ("_k", "_v", "_table", "_lens", "_weight", "kv_heads", "hd", "page", "batch", "pages", "capacity", "dtype", "c", "ref", "_all")

    k = property(lambda self: self._k)
    v = property(lambda self: self._v)
    table = property(lambda self: self._table)
    lens = property(lambda self: self._lens)
    weight = property(lambda self: self._weight)

    def __init__(self, k, v, table, lens, weight=None):
        shape, dtype = k.shape, k.dtype
        code = _DTYPES.get(dtype)
        if len(shape) != 4 or code is None:
            raise ValueError("cache keys must be [pages_total, kv_heads, page, hd] in float32, bfloat16 or float16, got %s %s" % (dtype, list(shape)))
        total, kv, page, hd = shape
        if hd not in _HEAD_DIMS:
            raise ValueError("a cache of head dim %d: %s are supported" % (hd, _HEAD_DIMS))
        if page not in _PAGES:
            raise ValueError("a page of %d tokens: powers of two from 16 to 1024 are supported" % page)
        if table.dim() != 2 or not table.numel() or not total or not kv:
            raise ValueError("an empty cache, or a page table that is not [batch, pages]: %s, %s" % (list(shape), list(table.shape)))
        B, pages = table.shape
        if not (v.shape == shape and v.dtype is dtype and table.dtype is torch.int32 and lens.dtype is torch.int32 and lens.shape == (B,) and
                k.is_contiguous() and v.is_contiguous() and table.is_contiguous() and lens.is_contiguous()):
            _whole(k, "cache keys", dtype, shape)   # (says which)
            _whole(v, "cache values", dtype, shape)
            _whole(table, "the page table", torch.int32, (B, pages))
            _whole(lens, "the lengths", torch.int32, (B,))
        if weight is not None:
            _whole(weight, "the weights", torch.float32, (B, kv, pages * page))
        if B > 65535 or kv > 1024 or pages * page >= 1 << 30 or total >= 1 << 31:
            raise ValueError("a cache of %d sequences, %d key heads, %d tokens a sequence is too large" % (B, kv, pages * page))
        if k.requires_grad or v.requires_grad or (weight is not None and weight.requires_grad):
            raise _lib.HipLibraryError("the tensors of a cache are written in place: none of them may require a gradient")
        _no_tangents("a paged cache", (k, v, weight))
        dev, at = core._dev[0], k.get_device()
        if at != dev or v.get_device() != at or table.get_device() != at or lens.get_device() != at or (weight is not None and weight.get_device() != at):
            _here(_CACHE_NAMES, k, v, table, lens, weight)   # (says which; or binds the device at the first call)
        pk, pv = k.data_ptr(), v.data_ptr()
        if (pk | pv) & 15:
            raise ValueError("cache keys and values must start on 16 bytes")
        self._k, self._v, self._table, self._lens, self._weight, self.dtype = k, v, table, lens, weight, dtype
        self.kv_heads, self.hd, self.page, self.batch, self.pages, self.capacity = kv, hd, page, B, pages, pages * page
        self.c = _CacheC(pk, pv, table.data_ptr(), lens.data_ptr(), None if weight is None else weight.data_ptr(), total, code, kv, page, hd, B, pages)
        self.ref = ctypes.byref(self.c)
        self._all = (k, v, lens) if weight is None else (k, v, lens, weight)   # what cache_append and cache_compact write


def _rows(t, name, cache, shape):
    """t with rows that the kernels can read, and its strides: last dimension dense, every row on 16 bytes (copied where it is not)"""
    if t.dtype is not cache.dtype or t.shape != shape:
        raise ValueError("%s must be %s %s like the cache, got %s %s" % (name, cache.dtype, list(shape), t.dtype, list(t.shape)))
    strides, per = t.stride(), 3 if cache.c.dtype == 0 else 7   # (elements of 16 bytes, less one)
    if strides[-1] != 1 or t.data_ptr() & 15 or (strides[0] | strides[1] | strides[-2]) & per:
        t = t.clone(memory_format=torch.contiguous_format)
        strides = t.stride()
    return t, strides


def _per_sequence(t, name, cache):
    if t is not None:
        _whole(t, name, torch.int32, (cache.batch,))
        return t.data_ptr()


def cache_append(cache, k, v, counts=None, at=None):
    """Writes k, v [B, T, kv_heads, hd] as tokens at[b] .. at[b] + counts[b] - 1 of every sequence and sets the lengths to at + counts.

    at: int32 [B], default: the cache's lengths (the new tokens follow the old ones; an earlier place takes tokens back, behind a later one
    lies whatever the pages held).  counts: int32 [B], default T (rows behind a sequence's count are padding and not read).  Tokens beyond
    the capacity are dropped.  New tokens have had no attention yet: their weight is 0.  k and v must not be parts of the cache's own pools, nor
    the pools of each other."""
    if k.dim() != 4:
        raise ValueError("new keys must be [batch, tokens, kv_heads, hd], got %s" % list(k.shape))
    T = k.shape[1]
    shape = (cache.batch, T, cache.kv_heads, cache.hd)
    k, (kb, kt, kh, _) = _rows(k, "new keys", cache, shape)
    v, (vb, vt, vh, _) = _rows(v, "new values", cache, shape)
    n, start = _per_sequence(counts, "counts", cache), _per_sequence(at, "at", cache)
    if (k.requires_grad or v.requires_grad) and torch.is_grad_enabled():
        raise _lib.HipLibraryError("cache_append has no backward: call it under torch.no_grad()")
    _no_tangents("cache_append", (k, v))
    s = _here(("new keys", "new values", "counts", "at"), k, v, counts, at)
    rc = _L().ix_cache_append(cache.ref, k.data_ptr(), v.data_ptr(), T, kb, kt, kh, vb, vt, vh, n, start, s)
    if rc:
        _chk(rc, "ix_cache_append")
    _written(cache._all)


_attn_ws_bytes = {}   # workspace of ix_cache_attn by sizes


def _attention_ws(cache, H, window, sinks, accumulate):
    c = cache.c
    key = (c.dtype, c.kv_heads, c.page, c.hd, c.batch, c.pages, H, window, sinks, accumulate)
    need = _attn_ws_bytes.get(key)
    if need is None:
        n = ctypes.c_size_t(0)
        _chk(_L().ix_workspace_bytes_cache_attn(cache.ref, H, window, sinks, accumulate, ctypes.byref(n)), "ix_workspace_bytes_cache_attn")
        if len(_attn_ws_bytes) >= 4096:
            _attn_ws_bytes.clear()
        need = _attn_ws_bytes[key] = n.value
    return need


def cache_attention(q, cache, scale=None, window=None, sinks=0, accumulate=False):
    """Attention of one new token per sequence: q [B, heads, hd] stands at the last token of its sequence -> [B, heads, hd].

    heads is a multiple of the cache's kv_heads; head h reads key head h // (heads // kv_heads).  scale: default 1 / sqrt(hd).  window:
    only the last `window` tokens and the first `sinks` are seen (default: all).  accumulate: the attention that every token gets here,
    summed over the heads that share its key head, is added to cache.weight.  An empty sequence gives zeros."""
    if q.dim() != 3 or q.shape[1] == 0 or q.shape[1] % cache.kv_heads:
        raise ValueError("q must be [batch, heads, hd] with a multiple of %d heads, got %s" % (cache.kv_heads, list(q.shape)))
    H = q.shape[1]
    if H > 4096:
        raise ValueError("%d query heads: at most 4096 are supported" % H)
    shape = (cache.batch, H, cache.hd)
    if q.requires_grad and torch.is_grad_enabled():
        raise _lib.HipLibraryError("cache_attention has no backward: call it under torch.no_grad()")
    _no_tangents("cache_attention", (q,))
    q, (qb, qh, _) = _rows(q, "q", cache, shape)
    w, sinks, accumulate = 0 if window is None else _count(window, "window", 1), _count(sinks, "sinks"), 1 if accumulate else 0
    if accumulate and cache.weight is None:
        raise ValueError("accumulate: the cache holds no weights")
    scale = _scale(scale, cache.hd)
    s = _here(("q",), q)
    out, ws, need = q.new_empty(shape), None, _attention_ws(cache, H, w, sinks, accumulate)
    if need:   # (a buffer per call: calls on other streams and captured graphs share none)
        ws = torch.empty(need, dtype=torch.uint8, device=q.device)
    rc = _L().ix_cache_attn(cache.ref, q.data_ptr(), qb, qh, out.data_ptr(), H, scale, w, sinks, accumulate, None if ws is None else ws.data_ptr(), need, s)
    if rc:
        _chk(rc, "ix_cache_attn")
    if accumulate:
        _written((cache._weight,))
    return out


def cache_select(weight, lens, budget, sinks=0, recent=0):
    """The tokens that stay when sequences shrink to `budget`: weight [B, kv_heads, capacity], lens int32 [B] -> (kept, left).

    kept int32 [B, kv_heads, budget], ascending: the first `sinks` tokens, the last `recent`, and of the rest those of the largest weight
    (a NaN counts less than any number; of equal weights the lowest index stays).  left int32 [B] = min(lens, budget); a sequence that
    is no longer than the budget keeps everything, and unused places of kept hold -1."""
    if weight.dim() != 3 or weight.dtype != torch.float32 or 0 in weight.shape or not weight.is_contiguous():
        raise ValueError("weight must be a contiguous float32 [batch, kv_heads, capacity], got %s %s" % (weight.dtype, list(weight.shape)))
    B, kv, cap = weight.shape
    if B > 65535 or cap >= 1 << 30:
        raise ValueError("weights of %d sequences of %d tokens are too large" % (B, cap))
    _whole(lens, "lens", torch.int32, (B,))
    budget, sinks, recent = _count(budget, "budget", 1), _count(sinks, "sinks"), _count(recent, "recent")
    if budget > cap or sinks + recent > budget:
        raise ValueError("a budget of %d tokens for a capacity of %d, of which %d first and %d last ones" % (budget, cap, sinks, recent))
    s = _here(("weight", "lens"), weight, lens)
    kept = torch.empty((B, kv, budget), dtype=torch.int32, device=weight.device)
    left = torch.empty(B, dtype=torch.int32, device=weight.device)
    _chk(_L().ix_cache_select(weight.data_ptr(), lens.data_ptr(), kept.data_ptr(), left.data_ptr(), B, kv, cap, budget, sinks, recent, s), "ix_cache_select")
    return kept, left


def cache_compact(cache, kept, left):
    """Moves the tokens kept[b, h, :left[b]] of every sequence and key head to its front, in place and in order, with their weights, and
    sets the lengths to left.  kept int32 [B, kv_heads, budget] ascends in every row (as cache_select returns it); the pages of a
    sequence must be its own: no other sequence's table may name them, and the pools must not share memory."""
    if kept.dim() != 3 or kept.shape[2] == 0:
        raise ValueError("kept must be [batch, kv_heads, budget], got %s" % list(kept.shape))
    _whole(kept, "kept", torch.int32, (cache.batch, cache.kv_heads, kept.shape[2]))
    _whole(left, "left", torch.int32, (cache.batch,))
    if kept.shape[2] > cache.capacity:
        raise ValueError("kept names %d tokens, the capacity is %d" % (kept.shape[2], cache.capacity))
    if abs(left.data_ptr() - cache.lens.data_ptr()) < 4 * cache.batch:
        raise ValueError("left must not be the cache's own lengths")
    s = _here(("kept", "left"), kept, left)
    _chk(_L().ix_cache_compact(cache.ref, kept.data_ptr(), left.data_ptr(), kept.shape[2], s), "ix_cache_compact")
    _written(cache._all)


def cache_evict(cache, budget, sinks=0, recent=0):
    """Cuts every sequence back to `budget` tokens by the cache's own accumulated weights (cache_select + cache_compact) -> kept."""
    if cache.weight is None:
        raise ValueError("cache_evict: the cache holds no weights")
    kept, left = cache_select(cache.weight, cache.lens, budget, sinks, recent)
    cache_compact(cache, kept, left)
    return kept
