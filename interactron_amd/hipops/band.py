"""hipops.band -- attention over a band around the diagonal and a few first keys, with its gradients (csrc/band.hip).

The sliding form of hipops.attention for sequences that are too long to attend to in full (reference models/gpt.py:39-57 and
models/detr_models/transformer.py:148-161 attend to everything): 16-bit or 32-bit rows as they are, shared key heads, padded batches.

It is no drop-in for hipops.attention inside the package's own models, and none of them calls it: the fusion transformer trains with dropout on
the weights, which this has not, and its inner gradient is differentiated again, which this refuses.
"""
import ctypes
import struct

import torch

from .. import _lib
from .cache import _DTYPES, _HEAD_DIMS, _count, _here, _scale
from .core import Function, _L, _NullCtx, _chk


# struct ix_band of include/interactron_hip.h: q, k, v, nine strides, q_lens, kv_lens, dtype .. causal, scale
_pack = struct.Struct("3P9q2P10if4x").pack


_NAMES = ("q", "k", "v", "q_lens", "kv_lens")
_LONGEST = 65535 * 64   # rows: blocks of 64 along one axis of a launch


def _dense_rows(t):
    """t, or a copy whose rows the kernels can read: last dimension dense, every row on 16 bytes and less than 2^24 bytes from the next"""
    per = 16 // t.element_size()
    sb, sl, sh, sd = t.stride()
    if sd != 1 or sb % per or sl % per or sh % per or t.data_ptr() & 15 or sl >= per << 20:
        t = t.clone(memory_format=torch.contiguous_format)
    return t


def _ptr(t):
    return None if t is None else t.data_ptr()


def _like(t):
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _band(q, k, v, q_lens, kv_lens, window, sinks, causal, scale):
    B, Lq, H, D = q.shape
    qb, ql, qh, _ = q.stride()
    kb, kl, kh, _ = k.stride()
    vb, vl, vh, _ = v.stride()
    return _pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), qb, ql, qh, kb, kl, kh, vb, vl, vh, 0 if q_lens is None else q_lens.data_ptr(),
                 0 if kv_lens is None else kv_lens.data_ptr(), _DTYPES[q.dtype], B, Lq, k.shape[1], H, k.shape[2], D, window, sinks, causal, scale)


class BandAttention(Function):
    """(q, k, v) -> out; see band_attention.  Differentiable once (the sliding form is not part of the adaptation step, whose inner gradient
    is differentiated again)."""
    b16 = "native"

    @staticmethod
    def forward(ctx, q, k, v, q_lens, kv_lens, window, sinks, causal, scale):
        s = _here(_NAMES, q, k, v, q_lens, kv_lens)
        recorded = not isinstance(ctx, _NullCtx) and any(ctx.needs_input_grad[:3])
        shape = q.shape
        ctx.empty = 0 in shape or k.shape[1] == 0
        if ctx.empty:   # nothing to see: zeros, and no gradient
            ctx.save_for_backward(q, k, v)
            return q.new_zeros(shape)
        q, k, v = _dense_rows(q), _dense_rows(k), _dense_rows(v)
        band = _band(q, k, v, q_lens, kv_lens, window, sinks, causal, scale)
        out, lse, rest = _like(q), None, None
        if recorded:   # for the gradients: the rows' normalisers and, with 16-bit types, behind them what rounding took from the output
            n = shape[0] * shape[2] * (-(-shape[1] // 128) * 512)
            kept = torch.empty(n if q.dtype is torch.float32 else n + 2 * q.numel(), dtype=torch.uint8, device=q.device)
            lse = kept.data_ptr()
            rest = None if q.dtype is torch.float32 else lse + n
            ctx.how = (window, sinks, causal, scale)
            ctx.save_for_backward(q, k, v, out, kept, q_lens, kv_lens)
        n, ws = ctypes.c_size_t(0), None
        _chk(_L().ix_workspace_bytes_band_attn_fwd(band, ctypes.byref(n)), "ix_workspace_bytes_band_attn_fwd")
        if n.value:
            ws = torch.empty(n.value, dtype=torch.uint8, device=q.device)
        _chk(_L().ix_band_attn_fwd(band, out.data_ptr(), lse, rest, _ptr(ws), n.value, s), "ix_band_attn_fwd")
        return out

    @staticmethod
    def backward(ctx, do):
        if torch.is_grad_enabled():   # (create_graph: a second derivative that silently left this node out would be a wrong one)
            raise _lib.HipLibraryError("band_attention is differentiable once: no gradient of its gradient (create_graph=True)")
        need = ctx.needs_input_grad
        if ctx.empty:
            return tuple([torch.zeros_like(t) if n else None for t, n in zip(ctx.saved_tensors, need)]) + (None,) * 6
        q, k, v, out, kept, q_lens, kv_lens = ctx.saved_tensors
        if do.dtype is not q.dtype:
            do = do.to(q.dtype)
        do = _dense_rows(do)
        s = _here(("the gradient",), do)
        band, n = _band(q, k, v, q_lens, kv_lens, *ctx.how), ctypes.c_size_t(0)
        _chk(_L().ix_workspace_bytes_band_attn_bwd(band, ctypes.byref(n)), "ix_workspace_bytes_band_attn_bwd")
        ws = torch.empty(n.value, dtype=torch.uint8, device=q.device)
        want = (1 if need[0] else 0) | (2 if need[1] or need[2] else 0)   # (dk and dv come together)
        if not want:
            return (None,) * 9
        dq, dk, dv = _like(q) if want & 1 else None, _like(k) if want & 2 else None, _like(v) if want & 2 else None
        lse, (gb, gl, gh, _) = kept.data_ptr(), do.stride()
        rest = None if q.dtype is torch.float32 else lse + kept.numel() - 2 * q.numel()
        _chk(_L().ix_band_attn_bwd_some(band, want, out.data_ptr(), rest, lse, do.data_ptr(), gb, gl, gh, _ptr(dq), _ptr(dk), _ptr(dv), ws.data_ptr(),
                                        n.value, s), "ix_band_attn_bwd_some")
        return dq if need[0] else None, dk if need[1] else None, dv if need[2] else None, None, None, None, None, None, None


def band_attention(q, k, v, window=None, sinks=0, causal=True, scale=None, q_lens=None, kv_lens=None):
    """Attention of q [B, Lq, heads, hd] over k, v [B, Lk, kv_heads, hd] -> [B, Lq, heads, hd].

    Query i of a sequence with m queries and n keys stands at p = i + n - m (the newest queries at the newest keys).  It sees the keys j
    with |p - j| < window (default: all) and the first `sinks` ones; with `causal` only those up to p.  heads is a multiple of kv_heads;
    head h reads key head h // (heads // kv_heads).  scale: default 1 / sqrt(hd).  q_lens, kv_lens: int32 [B], the lengths m and n of a
    padded batch; padding is never read and comes back as zeros.  A query that sees nothing gives zeros and has no gradient.

    float32, bfloat16 or float16, hd 32, 64 or 128, rows with any strides (a slice of a packed projection is taken as it is).  Sums and softmax
    are in 32 bits; 16-bit types carry weights and score gradients into the products as two terms of the type, so that results are off by their
    own rounding.  No dropout.  Differentiable once, computing only the gradients that are needed (those of k and v together).  Inside the lengths, values have to be finite also where a query does not see them, and for the
    gradients queries, keys and the gradient of the output too: there a weight of zero is multiplied with them.  A captured backward pass
    has leaves of its own: no eager graph of the same leaves may be alive."""
    for t, name in ((q, "q"), (k, "k"), (v, "v")):
        if t.dim() != 4 or t.dtype not in _DTYPES or t.dtype != q.dtype:
            raise ValueError("%s must be [batch, length, heads, hd] in float32, bfloat16 or float16 like q, got %s %s" % (name, t.dtype, list(t.shape)))
    B, Lq, H, D = q.shape
    if k.shape != v.shape or k.shape[0] != B or k.shape[3] != D:
        raise ValueError("k and v must be [%d, length, kv_heads, %d], got %s and %s" % (B, D, list(k.shape), list(v.shape)))
    if D not in _HEAD_DIMS:
        raise ValueError("a head dim of %d: %s are supported" % (D, _HEAD_DIMS))
    if k.shape[2] == 0 or H == 0 or H % k.shape[2]:
        raise ValueError("%d query heads over %d key heads" % (H, k.shape[2]))
    if max(Lq, k.shape[1]) > _LONGEST or B * H >= 1 << 24:
        raise ValueError("%d queries and %d keys of %d heads are too many" % (Lq, k.shape[1], B * H))
    for t, name in ((q_lens, "q_lens"), (kv_lens, "kv_lens")):
        if t is not None and (t.dtype != torch.int32 or tuple(t.shape) != (B,) or not t.is_contiguous()):
            raise ValueError("%s must be a contiguous int32 [%d], got %s %s" % (name, B, t.dtype, list(t.shape)))
    window, sinks = 0 if window is None else _count(window, "window", 1), _count(sinks, "sinks")
    return BandAttention.call(q, k, v, q_lens, kv_lens, window, sinks, 1 if causal else 0, _scale(scale, D))
