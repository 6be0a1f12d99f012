"""The sequence operators (band attention, paged cache) from their definitions, in 64 bits on the CPU: loops over sequences and heads.

Also the error bounds of their tests.  u = 2^-24 is the rounding of a 32-bit operation (half a step); h(t) that of a storage type."""
import math

import numpy as np
import torch

U = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def visible(m, n, window, sinks, causal):
    """[m, n] truth values: query i stands at i + n - m"""
    p, j = np.arange(m)[:, None] + n - m, np.arange(n)[None, :]
    see = np.ones((m, n), bool)
    if window is not None:
        see = (np.abs(p - j) < window) | (j < sinks)
    return see & (j <= p) if causal else see


def softmax_rows(z, see):
    z = np.where(see, z, -np.inf)
    top = z.max(1, keepdims=True) if z.shape[1] else np.full((z.shape[0], 1), -np.inf)
    e = np.where(see, np.exp(z - np.where(np.isfinite(top), top, 0.0)), 0.0)
    total = e.sum(1, keepdims=True)
    return e / np.where(total == 0, 1.0, total)


def f64(t):
    return t.detach().cpu().double().numpy()


class Pool:
    """The tokens of a paged cache as dense rows"""

    def __init__(self, cache):
        self.k, self.v, self.table, self.lens = (x.detach().cpu() for x in (cache.k, cache.v, cache.table, cache.lens))
        self.page = self.k.shape[2]

    def rows(self, which, b, h, n):
        t = torch.arange(n)
        pages = self.table[b].long()[t // self.page]
        ok = (pages >= 0) & (pages < self.k.shape[0])
        x = getattr(self, which)[torch.where(ok, pages, 0), h, t % self.page].double()
        return x.numpy(), ok.numpy()


def cache_attention(q, cache, scale=None, window=None, sinks=0):
    """-> out [B, H, D], weights by (b, key head) as arrays over the tokens, bound [B, H, D] of what 32-bit arithmetic may be off before the
    last rounding"""
    pool, qq = Pool(cache), f64(q)
    B, H, D = qq.shape
    kv = cache.kv_heads
    G, scale = H // kv, (D ** -0.5 if scale is None else scale)
    out, bound, weights = np.zeros((B, H, D)), np.zeros((B, H, D)), {}
    for b in range(B):
        n = int(np.clip(pool.lens[b].item(), 0, cache.capacity))
        for h in range(kv):
            k, ok = pool.rows("k", b, h, n)
            v, _ = pool.rows("v", b, h, n)
            see = visible(1, n, window, sinks, True) & ok[None, :] if n else np.zeros((1, 0), bool)
            k, v = np.where(see[0][:, None], k, 0.0), np.where(see[0][:, None], v, 0.0)
            w = np.zeros(n)
            for g in range(G):
                i = h * G + g
                p = softmax_rows((k @ qq[b, i])[None, :] * scale, see)[0] if n else np.zeros(0)
                out[b, i], w = p @ v, w + p
                # scores: D products and D sums in 32 bits, the scale and the base change: (D + 4) u of sum |q k| scale; a weight is
                # off by that much relatively, as is the normaliser; exp2, the carried maximum, the sums over tokens (64 per lane and
                # tile stride at most) and the two 16-bit terms of a weight (2^-17 of it) come on top; the output is a mean of values
                a = (np.abs(k) @ np.abs(qq[b, i])).max() * abs(scale) if n else 0.0
                rel = 2 * ((D + 4) * U * a + 4 * U * a) + (n / 64 + 64) * U + (2.0 ** -17 if q.dtype != torch.float32 else 0.0)
                bound[b, i] = rel * (np.abs(v).max(0) if n else 0.0)
            weights[b, h] = w
    return out, weights, bound


def select(weight, n, budget, sinks, recent):
    if n <= budget:
        return np.arange(n)
    middle = np.arange(sinks, n - recent)
    key = np.where(np.isnan(weight[middle]), -np.inf, weight[middle]).astype(np.float64)
    number = ~np.isnan(weight[middle])   # (every number before every NaN)
    best = middle[np.lexsort((middle, -key, ~number))[: budget - sinks - recent]]
    return np.sort(np.concatenate([np.arange(sinks), best, np.arange(n - recent, n)])).astype(np.int64)


def band_attention(q, k, v, window, sinks, causal, scale=None, q_lens=None, kv_lens=None, do=None):
    """-> dict of out (and dq, dk, dv) and of their bounds before the last rounding, arrays [B, L, heads, hd]"""
    dtype = q.dtype
    q, k, v, do = (f64(t) if t is not None else None for t in (q, k, v, do))
    B, Lq, H, D = q.shape
    Lk, kv = k.shape[1], k.shape[2]
    G, scale = H // kv, (D ** -0.5 if scale is None else scale)
    names = ("out",) if do is None else ("out", "dq", "dk", "dv")
    shapes = dict(out=q.shape, dq=q.shape, dk=k.shape, dv=k.shape)
    val, err = ({x: np.zeros(shapes[x]) for x in names} for _ in range(2))
    # 16-bit types: weights are rounded to the type (h), score gradients are carried as two of its terms (2 h^2), and the output that delta
    # comes from as two terms too (fp16: the second no finer than 2^-25)
    h = 0.0 if dtype == torch.float32 else half_step(dtype)
    h_out, floor = (U, 0.0) if dtype == torch.float32 else (2 * h * h, 2.0 ** -25 if dtype == torch.float16 else 0.0)
    for b in range(B):
        m = Lq if q_lens is None else min(max(int(q_lens[b]), 0), Lq)
        n = Lk if kv_lens is None else min(max(int(kv_lens[b]), 0), Lk)
        if not m or not n:
            continue
        see = visible(m, n, window, sinks, causal)
        for i in range(H):
            qq, kk, vv = q[b, :m, i], k[b, :n, i // G], v[b, :n, i // G]
            p = softmax_rows(qq @ kk.T * scale, see)
            o = p @ vv
            # a score is off by (D + 8) u of its absolute products, a weight by twice the row's worst of that (numerator and
            # normaliser), plus exp2 and log2, the sums over n and the maximum carried: relatively to the weight
            worst = np.where(see, np.abs(qq) @ np.abs(kk).T, 0.0).max(1, keepdims=True) * abs(scale)
            rel = 2 * (D + 8) * U * worst + (n / 16 + 64) * U
            val["out"][b, :m, i] = o
            err["out"][b, :m, i] = p * (rel + h) @ np.abs(vv)
            if dtype == torch.float16:   # below 2^-14 its steps are 2^-24: weights relative to the row's largest
                err["out"][b, :m, i] += 2.0 ** -25 * see @ np.abs(vv)
            if do is None:
                continue
            g = do[b, :m, i]
            dp, delta = g @ vv.T, (g * o).sum(1, keepdims=True)
            ds = p * (dp - delta)
            e_delta = (np.abs(g) * (h_out * np.abs(o) + floor + err["out"][b, :m, i] + (D + 2) * U * np.abs(o))).sum(1, keepdims=True)
            e_dp = (D + 2) * U * (np.abs(g) @ np.abs(vv).T)
            e_ds = np.abs(ds) * (rel + 2 * h * h + 4 * U) + p * (1 + rel) * (e_dp + e_delta)
            if dtype == torch.float16:   # ... and score gradients are carried up to 2^15, weights up to 2^10
                e_ds = e_ds + see * 2.0 ** -38 * np.abs(ds).max()
            val["dq"][b, :m, i] = scale * ds @ kk
            err["dq"][b, :m, i] = abs(scale) * ((e_ds + (n / 16 + 8) * U * np.abs(ds)) @ np.abs(kk))
            val["dk"][b, :n, i // G] += scale * ds.T @ qq
            err["dk"][b, :n, i // G] += abs(scale) * ((e_ds + (m / 16 + 64 + 8 * G) * U * np.abs(ds)).T @ np.abs(qq))
            val["dv"][b, :n, i // G] += p.T @ g
            err["dv"][b, :n, i // G] += (p * (rel + h + (m / 16 + 64 + 8 * G) * U) + (2.0 ** -35 * see if dtype == torch.float16 else 0.0)).T @ np.abs(g)
    return val, err
