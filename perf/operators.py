"""The operators of attention over long rollouts, as cases that can be timed and compared.

A case names an operator ("op"), its sizes and its type.  ``prepare`` makes what a program has in hand before the call, ``run``
makes one pass: with ``own`` false in elementary torch operations (32 bits inside, rounded once at the end), with ``own`` true
through ``interactron_amd.hipops``.  ``exact`` computes the same outputs from the definitions in 64 bits.

    train    band attention and the gradients of its three inputs (a training step's share)
    prompt   band attention alone (tokens of a prompt, or the newest part of one, against all keys so far)
    attend   one new token of every sequence over a paged cache, with or without the accumulated attention weights
    append   new keys and values into a paged cache
    evict    choose the tokens that stay by accumulated weight, and move them to the front of their pages

Band attention: query i of a sequence with n keys and m queries stands at p = i + n - m and sees the keys j < n with
|p - j| < window (all of them without a window) or j < sinks; where it is causal also j <= p.  A query that sees nothing gives
zeros.  o_i = sum_j P_ij v_j, P_ij = exp(scale q_i k_j) / sum_j' exp(scale q_i k_j').
"""
import math

import numpy as np
import torch

own = False

_T = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _bytes(case):
    return 4 if case["dtype"] == "fp32" else 2


def listed():
    return [
        # two 300 x 300 episodes through the fusion transformer (5 frames, 2 060 tokens, 8 heads of 64) in the 16-bit mode, each
        # token seeing about a frame's tokens on either side and the first five; the second episode is padded
        dict(name="train fusion 300", op="train", dtype="bf16", B=2, L=2060, Lk=2060, H=8, G=1, D=64, window=412, sinks=5, causal=False, ragged=True),
        # the detector's 19 x 19 memory, 16 images, 8 heads of 32, in 32 bits, a band of some rows of the map
        dict(name="train memory fp32", op="train", dtype="fp32", B=16, L=361, Lk=361, H=8, G=1, D=32, window=64, sinks=1, causal=False, ragged=False),
        # one 800 x 800 episode (12 755 tokens), causal over its frames, one frame's tokens back and the first sixteen
        dict(name="train fusion 800", op="train", dtype="bf16", B=1, L=12755, Lk=12755, H=8, G=1, D=64, window=2551, sinks=16, causal=True, ragged=False),
        # a prompt of 8 192 tokens with shared key heads, no gradients
        dict(name="prompt 8192", op="prompt", dtype="fp16", B=1, L=8192, Lk=8192, H=32, G=4, D=128, window=2048, sinks=4, causal=True, ragged=False),
        # the smallest decoding step: one sequence, a frame's tokens in the cache
        dict(name="attend one", op="attend", dtype="fp32", B=1, H=8, G=1, D=64, n=411, low=411, page=16, pages=32, window=None, sinks=0, weigh=False),
        # an ordinary decoding batch: 32 sequences of different lengths
        dict(name="attend batch", op="attend", dtype="bf16", B=32, H=32, G=4, D=128, n=8192, low=700, page=64, pages=128, window=None, sinks=0, weigh=False),
        # a decoding batch that keeps the attention weights for a later eviction
        dict(name="attend weigh", op="attend", dtype="fp16", B=16, H=16, G=4, D=64, n=4001, low=61, page=32, pages=128, window=None, sinks=0, weigh=True),
        # one long sequence
        dict(name="attend long", op="attend", dtype="bf16", B=1, H=32, G=4, D=128, n=131071, low=131071, page=64, pages=2048, window=None, sinks=0, weigh=False),
        # one token of every sequence of a batch
        dict(name="append token", op="append", dtype="bf16", B=32, T=1, Hkv=8, D=128, page=64, pages=128, ragged=False),
        # four prompts of the fusion sequence's length, of which three are padded
        dict(name="append prompt", op="append", dtype="bf16", B=4, T=2060, Hkv=8, D=64, page=32, pages=80, ragged=True),
        # every 256 tokens a batch is cut back to 4 096
        dict(name="evict page", op="evict", dtype="bf16", B=16, Hkv=8, D=128, n=4352, low=4200, page=64, pages=72, budget=4096, sinks=4, recent=1024),
        # two 800 x 800 rollouts cut back to the length of a 300 x 300 one
        dict(name="evict rollout", op="evict", dtype="fp32", B=2, Hkv=8, D=64, n=12755, low=12755, page=128, pages=100, budget=2060, sinks=16, recent=411),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["train", "train", "prompt", "attend", "attend", "append", "evict"])
    dtype, D = rng.choice(["bf16", "bf16", "fp16", "fp32"]), rng.choice([32, 64, 64, 128])
    if op in ("train", "prompt"):
        G, kv = rng.choice([1, 1, 2, 4, 8]), rng.choice([1, 2, 4, 8])
        B, Lk = rng.randint(1, 4), _log(rng, 1, 6000)
        L = Lk if op == "train" or rng.random() < 0.4 else _log(rng, 1, Lk)
        while B * G * kv * L * Lk > 1_000_000_000 or B * G * kv * Lk > 400_000:
            B, kv, G = max(1, B // 2), max(1, kv // 2) if B == 1 else kv, max(1, G // 2) if B == 1 and kv == 1 else G
        return dict(op=op, dtype=dtype, B=B, L=L, Lk=Lk, H=G * kv, G=G, D=D, window=None if rng.random() < 0.25 else _log(rng, 1, Lk),
                    sinks=rng.choice([0, 1, 4, rng.randint(0, 70)]), causal=rng.random() < 0.6, ragged=B > 1 and rng.random() < 0.5)
    page = rng.choice([16, 32, 64, 128])
    if op == "attend":
        G, kv, n = rng.choice([1, 2, 4, 5, 8]), rng.choice([1, 2, 4, 8]), _log(rng, 1, 60000)
        B = max(1, min(_log(rng, 1, 64), 200_000_000 // (n * kv * D)))
        return dict(op=op, dtype=dtype, B=B, H=G * kv, G=G, D=D, n=n, low=rng.randint(1, n), page=page, pages=-(-n // page) + rng.randint(0, 5),
                    window=None if rng.random() < 0.6 else _log(rng, 1, n), sinks=rng.choice([0, 4, 17]), weigh=rng.random() < 0.4)
    kv = rng.choice([1, 2, 4, 8])
    if op == "append":
        T = _log(rng, 1, 3000)
        B = max(1, min(_log(rng, 1, 64), 40_000_000 // (T * kv * D)))
        return dict(op=op, dtype=dtype, B=B, T=T, Hkv=kv, D=D, page=page, pages=-(-2 * T // page) + 2, ragged=rng.random() < 0.5)
    n = _log(rng, 40, 20000)
    B, budget = max(1, min(_log(rng, 1, 32), 60_000_000 // (n * kv * D))), rng.randint(20, n)
    sinks = rng.randint(0, 8)
    return dict(op=op, dtype=dtype, B=B, Hkv=kv, D=D, n=n, low=rng.randint(1, n), page=page, pages=-(-n // page) + rng.randint(0, 3), budget=budget,
                sinks=sinks, recent=rng.randint(0, budget - sinks))


# ---- lengths: fixed by the case (so that its work is), dealt out by the seed ------------------------------------------------------
def _spread(low, high, B):
    return [high - (high - low) * b // max(1, B - 1) for b in range(B)]


def _lens(case):
    """-> (queries, keys) of every sequence"""
    if not case["ragged"]:
        return [case["L"]] * case["B"], [case["Lk"]] * case["B"]
    return _spread(max(1, 2 * case["L"] // 3), case["L"], case["B"]), _spread(max(1, 3 * case["Lk"] // 4), case["Lk"], case["B"])


def _pairs(m, n, window, sinks, causal):
    """how many (query, key) pairs of one sequence see each other"""
    p = np.arange(m, dtype=np.int64) + n - m
    far = (window or n + m) - 1
    hi = np.minimum(n - 1, p if causal else p + far)
    lo = np.maximum(0, p - far)
    band = np.maximum(0, hi - lo + 1)
    first = np.minimum(sinks, np.minimum(n, p + 1) if causal else n)
    return int((band + np.maximum(0, np.minimum(first, np.where(band > 0, lo, first)))).sum())


def work(case):
    e, op = _bytes(case), case["op"]
    if op in ("train", "prompt"):
        m, n = _lens(case)
        pairs = sum(_pairs(a, b, case["window"], case["sinks"], case["causal"]) for a, b in zip(m, n)) * case["H"]
        q, k = sum(m) * case["H"] * case["D"] * e, sum(n) * case["H"] // case["G"] * case["D"] * e
        if op == "prompt":
            return {"bytes": 2 * q + 2 * k, "flops": 4 * case["D"] * pairs}
        return {"bytes": 4 * q + 4 * k, "flops": 12 * case["D"] * pairs}
    if op == "attend":
        kv, lens = case["H"] // case["G"], _spread(case["low"], case["n"], case["B"])
        seen = sum(_pairs(1, n, case["window"], case["sinks"], True) for n in lens)
        byt = 2 * seen * kv * case["D"] * e + 2 * case["B"] * case["H"] * case["D"] * e + (8 * seen * kv if case["weigh"] else 0)
        return {"bytes": byt, "flops": 4 * case["D"] * seen * case["H"]}
    if op == "append":
        rows = sum(_spread(max(1, case["T"] // 2), case["T"], case["B"]) if case["ragged"] else [case["T"]] * case["B"])
        return {"bytes": 4 * rows * case["Hkv"] * case["D"] * e, "flops": 0}
    lens = _spread(case["low"], case["n"], case["B"])
    stay = sum(min(n, case["budget"]) for n in lens)
    return {"bytes": case["Hkv"] * (4 * sum(lens) + stay * (4 * case["D"] * e + 8)), "flops": 0}


# ---- inputs -----------------------------------------------------------------------------------------------------------------------
def _randn(g, dtype, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(_T[dtype])


def _pool(case, g, kv):
    """keys, values and page table of a paged cache: the pages of a sequence lie anywhere in the pool"""
    B, pages = case["B"], case["pages"]
    shape = (B * pages + 3, kv, case["page"], case["D"])
    table = torch.randperm(shape[0], generator=g, device="cuda")[: B * pages].reshape(B, pages).to(torch.int32)
    return dict(k=_randn(g, case["dtype"], *shape), v=_randn(g, case["dtype"], *shape), table=table)


def _dealt(lens, seed):
    order = np.random.RandomState(seed % (1 << 32)).permutation(len(lens))
    return torch.tensor([lens[i] for i in order], dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, B, D = case["op"], case["B"], case["D"]
    s = {"case": case}
    if op in ("train", "prompt"):
        L, Lk, H, kv = case["L"], case["Lk"], case["H"], case["H"] // case["G"]
        s["q"] = _randn(g, case["dtype"], B, L, H, D).mul_(1.5)   # (scores a little wider than a unit normal's)
        s["k"], s["v"] = _randn(g, case["dtype"], B, Lk, kv, D), _randn(g, case["dtype"], B, Lk, kv, D)
        s["q_lens"] = s["kv_lens"] = None
        if case["ragged"]:
            m, n = _lens(case)
            s["q_lens"], s["kv_lens"] = _dealt(m, seed), _dealt(n, seed)
        if op == "train":
            s["do"] = _randn(g, case["dtype"], B, L, H, D)
            for t in ("q", "k", "v"):
                s[t].requires_grad_(True)
        return s
    if op == "attend":
        kv = case["H"] // case["G"]
        s.update(_pool(case, g, kv), q=_randn(g, case["dtype"], B, case["H"], D).mul_(1.5), lens=_dealt(_spread(case["low"], case["n"], B), seed))
        s["weight"] = torch.rand(B, kv, case["pages"] * case["page"], generator=g, device="cuda") if case["weigh"] else None
        return s
    if op == "append":
        kv, T = case["Hkv"], case["T"]
        s.update(_pool(case, g, kv), new_k=_randn(g, case["dtype"], B, T, kv, D), new_v=_randn(g, case["dtype"], B, T, kv, D), counts=None)
        s["at"] = torch.randint(0, case["pages"] * case["page"] - T + 1, (B,), generator=g, device="cuda").to(torch.int32)
        if case["ragged"]:
            s["counts"] = _dealt(_spread(max(1, T // 2), T, B), seed)
        s["lens"] = s["at"].clone()
        return s
    s.update(_pool(case, g, case["Hkv"]), lens=_dealt(_spread(case["low"], case["n"], B), seed))
    # accumulated attention: most tokens have had little, a few very much; tokens that nobody has looked at yet have none (ties)
    x = torch.randn(B, case["Hkv"], case["pages"] * case["page"], generator=g, device="cuda").mul_(2).exp_()
    s["score"] = torch.where(torch.rand(x.shape, generator=g, device="cuda") < 0.05, torch.zeros_like(x), x)
    s["weight"], s["cut"] = s["score"].clone(), s["lens"].clone()   # (the cache's own weights and lengths: the call rewrites them)
    return s


# ---- one pass ---------------------------------------------------------------------------------------------------------------------
def run(s):
    case = s["case"]
    return (_own if own else _plain)[case["op"]](s, case)


def _own_band(s, c):
    from interactron_amd import hipops
    return hipops.band_attention(s["q"], s["k"], s["v"], window=c["window"], sinks=c["sinks"], causal=c["causal"], q_lens=s["q_lens"], kv_lens=s["kv_lens"])


def _own_train(s, c):
    out = _own_band(s, c)
    return (out.detach(),) + torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["do"])


def _own_attend(s, c):
    from interactron_amd import hipops
    cache = hipops.PagedCache(s["k"], s["v"], s["table"], s["lens"], s["weight"])
    out = hipops.cache_attention(s["q"], cache, window=c["window"], sinks=c["sinks"], accumulate=c["weigh"])
    return (out, s["weight"]) if c["weigh"] else out


def _own_append(s, c):
    from interactron_amd import hipops
    cache = hipops.PagedCache(s["k"], s["v"], s["table"], s["lens"])
    hipops.cache_append(cache, s["new_k"], s["new_v"], counts=s["counts"], at=s["at"])
    return s["k"], s["v"], s["lens"]


def _own_evict(s, c):
    from interactron_amd import hipops
    cache = hipops.PagedCache(s["k"], s["v"], s["table"], s["cut"], s["weight"])
    kept, left = hipops.cache_select(s["score"], s["lens"], c["budget"], sinks=c["sinks"], recent=c["recent"])
    hipops.cache_compact(cache, kept, left)
    return kept, left, s["cut"], s["k"], s["v"], s["weight"]


_own = {"train": _own_train, "prompt": _own_band, "attend": _own_attend, "append": _own_append, "evict": _own_evict}


def _visible(p, j, n, c):
    """truth values [..., queries, keys] from positions p [..., queries, 1], keys j and lengths n that broadcast against them"""
    see = j < n
    if c["window"] is not None:
        see = see & (((p - j).abs() < c["window"]) | (j < c["sinks"]))
    return see & (j <= p) if c["causal"] else see


def _band_parts(s, c):
    B, L, Lk, H, G, D = (c[x] for x in ("B", "L", "Lk", "H", "G", "D"))
    kv, dev = H // G, s["q"].device
    m = s["q_lens"].long().view(B, 1, 1) if s["q_lens"] is not None else torch.full((B, 1, 1), L, device=dev)
    n = s["kv_lens"].long().view(B, 1, 1) if s["kv_lens"] is not None else torch.full((B, 1, 1), Lk, device=dev)
    i, j = torch.arange(L, device=dev).view(1, L, 1), torch.arange(Lk, device=dev).view(1, 1, Lk)
    see = (_visible(i + n - m, j, n, c) & (i < m)).view(B, 1, 1, L, Lk)
    heads = lambda t, rows, h: t.detach().float().view(B, rows, kv, h, D).permute(0, 2, 3, 1, 4).reshape(B, kv, h * rows, D)  # noqa: E731
    q, k, v = heads(s["q"], L, G), heads(s["k"], Lk, 1), heads(s["v"], Lk, 1)
    x = torch.matmul(q, k.transpose(2, 3)).view(B, kv, G, L, Lk).mul_(1 / math.sqrt(D)).masked_fill_(~see, -math.inf)
    top = x.amax(-1, keepdim=True)
    x.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
    total = x.sum(-1, keepdim=True)
    x.div_(torch.where(total == 0, torch.ones_like(total), total))
    return q, k, v, x.view(B, kv, G * L, Lk), lambda t, rows, h: t.view(B, kv, h, rows, D).permute(0, 3, 1, 2, 4).reshape(B, rows, kv * h, D).to(_T[c["dtype"]]), heads


def _plain_prompt(s, c):
    q, k, v, prob, back, _ = _band_parts(s, c)
    return back(torch.matmul(prob, v), c["L"], c["G"])


def _plain_train(s, c):
    q, k, v, prob, back, heads = _band_parts(s, c)
    scale = 1 / math.sqrt(c["D"])
    do = heads(s["do"], c["L"], c["G"])
    out, dv = torch.matmul(prob, v), torch.matmul(prob.transpose(2, 3), do)
    ds = torch.matmul(do, v.transpose(2, 3)).sub_((do * out).sum(-1, keepdim=True)).mul_(prob)
    dq, dk = torch.matmul(ds, k).mul_(scale), torch.matmul(ds.transpose(2, 3), q).mul_(scale)
    return back(out, c["L"], c["G"]), back(dq, c["L"], c["G"]), back(dk, c["Lk"], 1), back(dv, c["Lk"], 1)


def _plain_attend(s, c):
    B, H, G, D, C = c["B"], c["H"], c["G"], c["D"], c["page"] * c["pages"]
    kv, table = H // G, s["table"].long()
    k, v = (s[t][table].permute(0, 2, 1, 3, 4).reshape(B, kv, C, D).float() for t in ("k", "v"))
    n = s["lens"].long().view(B, 1, 1)
    see = _visible(n - 1, torch.arange(C, device=n.device).view(1, 1, C), n, dict(c, causal=True)).view(B, 1, 1, C)
    x = torch.matmul(s["q"].float().view(B, kv, G, D), k.transpose(2, 3)).mul_(1 / math.sqrt(D)).masked_fill_(~see, -math.inf)
    x.sub_(x.amax(-1, keepdim=True)).exp_()
    x.div_(x.sum(-1, keepdim=True))
    out = torch.matmul(x, v).reshape(B, H, D).to(s["q"].dtype)
    if not c["weigh"]:
        return out
    s["weight"].add_(x.sum(2))
    return out, s["weight"]


def _plain_append(s, c):
    B, T = c["B"], c["T"]
    at = s["at"].long()
    n = s["counts"].long() if s["counts"] is not None else torch.full_like(at, T)
    t = torch.arange(T, device=at.device).view(1, T)
    b, t = (t < n.view(B, 1)).nonzero(as_tuple=True) if s["counts"] is not None else (torch.arange(B, device=at.device).repeat_interleave(T), t.expand(B, T).reshape(-1))
    slot = at[b] + t
    page = s["table"].long()[b, slot // c["page"]]
    s["k"][page, :, slot % c["page"]] = s["new_k"][b, t]
    s["v"][page, :, slot % c["page"]] = s["new_v"][b, t]
    s["lens"].copy_(at + n)
    return s["k"], s["v"], s["lens"]


def _plain_evict(s, c):
    B, kv, page, C = c["B"], c["Hkv"], c["page"], c["page"] * c["pages"]
    n = s["lens"].long().view(B, 1, 1)
    left = n.clamp(max=c["budget"])
    j = torch.arange(C, device=n.device).view(1, 1, C)
    x = torch.where((j < c["sinks"]) | (j >= n - c["recent"]), math.inf, s["score"])
    x = torch.where(j < n, x, -math.inf)
    first = x.sort(dim=-1, descending=True, stable=True).indices[..., : c["budget"]]
    first = torch.where(torch.arange(c["budget"], device=n.device) < left, first, C).sort(-1).values   # (what is over sorts last)
    kept = torch.where(first < C, first, -1).to(torch.int32)
    b, h, t = (first < C).nonzero(as_tuple=True)
    slot, table = first[b, h, t], s["table"].long()
    old, new = (table[b, slot // page], h, slot % page), (table[b, t // page], h, t % page)
    s["k"][new], s["v"][new] = s["k"][old], s["v"][old]
    s["weight"][b, h, t] = s["weight"][b, h, slot]
    s["cut"].copy_(left.view(B))
    return kept, left.view(B).to(torch.int32), s["cut"], s["k"], s["v"], s["weight"]


_plain = {"train": _plain_train, "prompt": _plain_prompt, "attend": _plain_attend, "append": _plain_append, "evict": _plain_evict}


# ---- the definitions in 64 bits, sequence by sequence and head by head ------------------------------------------------------------
def _band_rows(m, n, c, dev):
    """which keys each of m queries sees among n, from the bounds of the band"""
    p = torch.arange(n - m, n, device=dev).unsqueeze(1)
    j = torch.arange(n, device=dev).unsqueeze(0)
    far = c["window"] if c["window"] is not None else n + m
    band = torch.logical_and(j > p - far, j < p + far)
    return torch.logical_and(torch.logical_or(band, j < c["sinks"]), j <= p if c["causal"] else j >= 0)


def _exact_band(s, c):
    B, H, G, D = c["B"], c["H"], c["G"], c["D"]
    m, n = ([x] * B if t is None else t.tolist() for x, t in ((c["L"], s["q_lens"]), (c["Lk"], s["kv_lens"])))
    q, k, v = (s[t].detach().double() for t in "qkv")
    out = torch.zeros_like(q)
    train = c["op"] == "train"
    if train:
        do, dq, dk, dv = s["do"].double(), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for b in range(B):
        unseen = ~_band_rows(m[b], n[b], c, q.device)
        for h in range(H):
            qq, kk, vv = q[b, : m[b], h], k[b, : n[b], h // G], v[b, : n[b], h // G]
            z = (qq @ kk.T) / math.sqrt(D)
            z[unseen] = -math.inf
            lse = torch.logsumexp(z, 1, keepdim=True)
            a = torch.exp(z - torch.where(torch.isinf(lse), torch.zeros_like(lse), lse))
            del z
            out[b, : m[b], h] = a @ vv
            if train:
                g = do[b, : m[b], h]
                dv[b, : n[b], h // G] += a.T @ g
                da = g @ vv.T
                dz = a * (da - (a * da).sum(1, keepdim=True)) / math.sqrt(D)
                dq[b, : m[b], h] = dz @ kk
                dk[b, : n[b], h // G] += dz.T @ qq
    return (out, dq, dk, dv) if train else out


def _exact_attend(s, c):
    G, page = c["G"], c["page"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    weight = s["weight"].double() if c["weigh"] else None
    for b, n in enumerate(s["lens"].tolist()):
        pages = s["table"][b].long()[: -(-n // page)]
        t = torch.arange(n, device="cuda")
        if c["window"] is not None:
            t = t[(t >= n - c["window"]) | (t < c["sinks"])]
        for h in range(c["H"] // G):
            k, v = (s[x][pages, h].double().flatten(0, 1)[t] for x in ("k", "v"))
            z = s["q"][b, h * G:(h + 1) * G].double() @ k.T / math.sqrt(c["D"])
            a = torch.exp(z - torch.logsumexp(z, 1, keepdim=True))
            out[b, h * G:(h + 1) * G] = a @ v
            if c["weigh"]:
                weight[b, h, t] += a.sum(0)
    return (out, weight) if c["weigh"] else out


def _exact_append(s, c):
    k, v, lens = s["k"].clone(), s["v"].clone(), s["lens"].clone()
    at, table = s["at"].tolist(), s["table"].tolist()
    n = [c["T"]] * c["B"] if s["counts"] is None else s["counts"].tolist()
    for b in range(c["B"]):
        done = 0
        while done < n[b]:   # page by page
            slot = at[b] + done
            here = min(n[b] - done, c["page"] - slot % c["page"])
            for pool, new in ((k, s["new_k"]), (v, s["new_v"])):
                pool[table[b][slot // c["page"]], :, slot % c["page"]: slot % c["page"] + here] = new[b, done: done + here].transpose(0, 1)
            done += here
        lens[b] = at[b] + n[b]
    return k.double(), v.double(), None


def _exact_evict(s, c):
    k, v, weight = s["k"].clone(), s["v"].clone(), s["weight"].clone()
    score, page = s["score"].double().cpu().numpy(), c["page"]
    for b, n in enumerate(s["lens"].tolist()):
        middle = np.arange(min(c["sinks"], n), max(min(c["sinks"], n), n - c["recent"]))
        pages = s["table"][b].long()
        for h in range(c["Hkv"]):
            stay = np.arange(n)
            if n > c["budget"]:
                room = c["budget"] - (n - len(middle))
                best = middle[np.lexsort((middle, -score[b, h, middle]))[:room]]
                stay = np.sort(np.concatenate([np.setdiff1d(stay, middle), best]))
            to, stay = torch.arange(len(stay), device="cuda"), torch.from_numpy(stay).cuda()
            for pool in (k, v):
                pool[pages[to // page], h, to % page] = pool[pages[stay // page], h, stay % page]
            weight[b, h, to] = weight[b, h, stay]
    return None, None, None, k.double(), v.double(), weight.double()


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op in ("train", "prompt"):
        return _exact_band(s, case)
    return {"attend": _exact_attend, "append": _exact_append, "evict": _exact_evict}[op](s, case)
