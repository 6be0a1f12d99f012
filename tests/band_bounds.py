"""Bounds of band attention's output and of dv where the weights are as good as 32-bit ones: what tests/sequence_reference.py allows
for weights of one 16-bit term is left out."""
import numpy as np
import torch

from tests import sequence_reference as ref


def close(got, want, err, name=""):
    """got is want after an error of at most err and the rounding to its type"""
    dtype = got.dtype
    got = ref.f64(got)
    assert np.isfinite(got).all(), name
    # half a step of the value before it; below fp16's normal range a step is absolute
    tol = err + ref.half_step(dtype) * (np.abs(want) + err) + (2.0 ** -25 if dtype == torch.float16 else 1e-38)
    off = np.abs(got - want)
    assert (off <= tol).all(), (name, float((off / tol).max()), np.unravel_index((off / tol).argmax(), off.shape), int((off > tol).sum()), off.size)


def band(q, k, v, window=None, sinks=0, causal=True, scale=None, q_lens=None, kv_lens=None, do=None, floor=0.0, floor_dv=None):
    """-> values and errors as sequence_reference.band_attention gives them, the errors of out and dv with weights as two terms of the
    type.  h: half a step; a term leaves h of what it rounds, two leave h^2 (2 h^2 allowed).  floor: the smallest step of the second
    term, absolute, as a share of the row's largest weight; floor_dv (default: the same): the same of a weight in dv (fp16)."""
    lens = {x: t.cpu() for x, t in (("q_lens", q_lens), ("kv_lens", kv_lens)) if t is not None}
    val, err = ref.band_attention(q, k, v, window, sinks, causal, scale, do=do, **lens)
    two = 0.0 if q.dtype == torch.float32 else 2 * ref.half_step(q.dtype) ** 2
    q, k, v, do = (ref.f64(t) if t is not None else None for t in (q, k, v, do))
    (B, Lq, H, D), Lk = q.shape, k.shape[1]
    G, scale = H // k.shape[2], (D ** -0.5 if scale is None else scale)
    for x in ("out",) if do is None else ("out", "dv"):
        err[x][:] = 0
    for b in range(B):
        m, n = (min(max(int(lens[x][b]), 0), L) if x in lens else L for x, L in (("q_lens", Lq), ("kv_lens", Lk)))
        if not m or not n:
            continue
        see = ref.visible(m, n, window, sinks, causal)
        for i in range(H):
            qq, kk, vv = q[b, :m, i], k[b, :n, i // G], v[b, :n, i // G]
            p = ref.softmax_rows(qq @ kk.T * scale, see)
            # scores, exp2, sums in 32 bits: the same terms as there
            worst = np.where(see, np.abs(qq) @ np.abs(kk).T, 0.0).max(1, keepdims=True) * abs(scale)
            rel = 2 * (D + 8) * ref.U * worst + (n / 16 + 64) * ref.U
            err["out"][b, :m, i] = (p * (rel + two) + floor * see * p.max(1, keepdims=True)) @ np.abs(vv)
            if do is not None:
                err["dv"][b, :n, i // G] += (p * (rel + two + (m / 16 + 64 + 8 * G) * ref.U) + (floor if floor_dv is None else floor_dv) * see).T @ np.abs(do[b, :m, i])
    return val, err


def check(q, k, v, do=None, floor=0.0, floor_dv=None, **how):
    """the call against the bounds above"""
    from interactron_amd import hipops
    want, err = band(q, k, v, do=do, floor=floor, floor_dv=floor_dv, **how)
    if do is None:
        out = hipops.band_attention(q, k, v, **how)
        close(out, want["out"], err["out"], "out")
        return dict(out=out)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = hipops.band_attention(*leaves, **how)
    got = dict(out=out.detach(), **dict(zip(("dq", "dk", "dv"), torch.autograd.grad(out, leaves, do))))
    for x in want:
        assert got[x].dtype == q.dtype and tuple(got[x].shape) == want[x].shape
        close(got[x], want[x], err[x], x)
    return got
