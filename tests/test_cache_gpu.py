"""The paged cache against its definitions in 64 bits (tests/sequence_reference.py)."""
import numpy as np
import pytest
import torch

from tests import sequence_reference as ref

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def make(lens, kv=2, page=16, hd=64, pages=None, dtype=BF16, weight=True, seed=0, spare=3, tail=None):
    """A cache with random rows whose pages lie anywhere in the pool; `tail`: what stands in every row behind a sequence's last token"""
    from interactron_amd import hipops
    g = torch.Generator().manual_seed(seed)
    B = len(lens)
    pages = pages or max(1, max(-(-n // page) for n in lens))
    total = B * pages + spare
    k, v = (torch.randn(total, kv, page, hd, generator=g) for _ in range(2))
    table = torch.randperm(total, generator=g)[: B * pages].reshape(B, pages).to(torch.int32)
    if tail is not None:
        live = torch.zeros(total, page, dtype=torch.bool)
        for b, n in enumerate(lens):
            t = torch.arange(min(n, pages * page))
            live[table[b].long()[t // page], t % page] = True
        for x in (k, v):
            x.permute(0, 2, 1, 3)[~live] = tail
    w = torch.rand(B, kv, pages * page, generator=g) if weight else None
    up = lambda t: t.cuda() if t is not None else None  # noqa: E731
    return hipops.PagedCache(up(k.to(dtype)), up(v.to(dtype)), up(table), torch.tensor(lens, dtype=torch.int32, device="cuda"), up(w))


def query(cache, heads, seed=1, scale=1.5):
    return (torch.randn(cache.batch, heads, cache.hd, generator=torch.Generator().manual_seed(seed)) * scale).to(cache.k.dtype).cuda()


def check_attention(cache, q, accumulate=False, **how):
    from interactron_amd import hipops
    want, weights, bound = ref.cache_attention(q, cache, **how)
    before = ref.f64(cache.weight) if cache.weight is not None else None
    k, v = cache.k.clone(), cache.v.clone()
    got = hipops.cache_attention(q, cache, accumulate=accumulate, **how)
    assert got.dtype == q.dtype and got.shape == q.shape
    # the last rounding: half a step of the result, and the result is off by `bound` before it (fp16: below 2^-14 a step is 2^-24)
    tol = bound + ref.half_step(q.dtype) * (np.abs(want) + bound) + (2.0 ** -25 if q.dtype == FP16 else 0.0)
    off = np.abs(ref.f64(got) - want)
    assert np.isfinite(ref.f64(got)).all() and (off <= tol).all(), (off / np.maximum(tol, 1e-300)).max()
    assert torch.equal(k.view(torch.uint8), cache.k.view(torch.uint8)) and torch.equal(v.view(torch.uint8), cache.v.view(torch.uint8))
    if accumulate:
        after, G = ref.f64(cache.weight), q.shape[1] // cache.kv_heads
        lens = cache.lens.tolist()
        for b in range(cache.batch):
            n = min(max(lens[b], 0), cache.capacity)
            for h in range(cache.kv_heads):
                add = weights[b, h]
                # a weight is off by 2 delta of itself (as in the bound of the outputs, without their values); the sum over G heads and
                # the old weight rounds G times
                rel = np.max([bound[b, h * G + i].max() / max(1e-30, np.abs(ref.Pool(cache).rows("v", b, h, n)[0]).max() if n else 1.0) for i in range(G)])
                tol = rel * add * 2 + (G + 2) * ref.U * (before[b, h, :n] + add) + 1e-30
                assert (np.abs(after[b, h, :n] - before[b, h, :n] - add) <= tol).all(), (b, h)
                assert (after[b, h, n:] == before[b, h, n:]).all()
    elif before is not None:
        assert (ref.f64(cache.weight) == before).all()
    return got


# ---- attention ----------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("heads, kv", [(2, 2), (8, 2), (5, 1), (40, 2)])
def test_attention_types_and_head_layouts(dtype, hd, heads, kv):
    cache = make([0, 1, 77, 200], kv=kv, hd=hd, dtype=dtype)
    out = check_attention(cache, query(cache, heads))
    assert (out[0] == 0).all()


@pytest.mark.parametrize("dtype", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("page", [16, 32, 128, 1024])
def test_attention_page_sizes_and_ragged_ends(dtype, page):
    lens = [1, 15, 16, 17, 31, 33, 127, 128, 129, 511, 513, 1500]
    cache = make(lens, page=page, dtype=dtype, tail=float("nan"))
    check_attention(cache, query(cache, 4))


@pytest.mark.parametrize("dtype", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("window, sinks", [(1, 0), (16, 0), (17, 3), (40, 33), (100, 200), (300, 5), (1 << 20, 1 << 20), (None, 7)])
def test_attention_window_and_first_tokens(dtype, window, sinks):
    cache = make([0, 1, 16, 17, 49, 130, 333, 700], dtype=dtype, tail=float("inf"))
    check_attention(cache, query(cache, 4), window=window, sinks=sinks)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("heads, kv, how", [(4, 4, {}), (12, 2, {}), (40, 1, dict(window=50, sinks=4)), (130, 1, {})])
def test_attention_accumulates_weights(dtype, heads, kv, how):
    cache = make([0, 3, 100, 1100, 2600], kv=kv, dtype=dtype, page=32)
    check_attention(cache, query(cache, heads), accumulate=True, **how)
    check_attention(cache, query(cache, heads, seed=2), accumulate=True, **how)


def test_attention_masked_values_do_not_matter():
    """NaN and infinities in tokens outside the window, in tokens behind the end and in pages nobody names"""
    from interactron_amd import hipops
    clean = make([60, 300], dtype=FP32, tail=0.0)
    q = query(clean, 4)
    want = hipops.cache_attention(q, clean, window=40, sinks=3)
    for value in (float("nan"), float("inf"), float("-inf"), torch.finfo(FP32).min):
        dirty = make([60, 300], dtype=FP32, tail=value)
        for b, n in enumerate([60, 300]):
            for t in range(3, n - 40):
                for x in (dirty.k, dirty.v):
                    x[dirty.table[b, t // 16].long(), :, t % 16] = value
        assert torch.equal(hipops.cache_attention(q, dirty, window=40, sinks=3), want)


@pytest.mark.parametrize("dtype", [BF16, FP32], ids=["bf16", "fp32"])
def test_attention_large_and_small_scores(dtype):
    cache = make([5, 400], dtype=dtype)
    check_attention(cache, query(cache, 4, scale=40.0))
    check_attention(cache, query(cache, 4), scale=0.0)
    check_attention(cache, query(cache, 4), scale=-0.3)


def test_attention_bad_pages_are_masked():
    cache = make([100, 100, 20], dtype=BF16, page=16)
    for b, i, bad in ((0, 2, -1), (0, 6, cache.k.shape[0]), (1, 0, 1 << 30), (2, 0, -(1 << 31)), (2, 1, 0x7fffffff)):
        cache.table[b, i] = bad
    out = check_attention(cache, query(cache, 4), accumulate=True)
    assert (out[2] == 0).all()


def test_attention_lengths_are_clamped():
    from interactron_amd import hipops
    cache = make([64, 64], page=16, pages=4)
    q = query(cache, 4)
    want = hipops.cache_attention(q, cache)
    cache.lens.copy_(torch.tensor([1 << 30, -5], dtype=torch.int32))
    got = hipops.cache_attention(q, cache)
    assert torch.equal(got[0], want[0]) and (got[1] == 0).all()


def test_attention_query_views_and_shared_pages():
    from interactron_amd import hipops
    cache = make([90, 90], dtype=BF16)
    cache.table[1] = cache.table[0]
    packed = torch.randn(2, 3, 8, 64, generator=torch.Generator().manual_seed(3)).to(BF16).cuda()
    q = packed[:, 1]
    assert torch.equal(hipops.cache_attention(q, cache), hipops.cache_attention(q.clone(), cache))
    odd = torch.zeros(2, 8, 65, dtype=BF16, device="cuda")[..., 1:]   # (rows off 16 bytes)
    odd.copy_(q)
    assert torch.equal(hipops.cache_attention(odd, cache), hipops.cache_attention(q, cache))
    same = hipops.cache_attention(q[:1].expand(2, 8, 64), cache)
    assert torch.equal(same[0], same[1])


def test_attention_beyond_32_bit_offsets():
    """The last pages of pools of more than 2^32 bytes each"""
    from interactron_amd import hipops
    kv, page, hd = 8, 1024, 128
    total = (1 << 32) // (kv * page * hd * 2) + 3
    k, v = (torch.empty(total, kv, page, hd, dtype=BF16, device="cuda") for _ in range(2))
    table = torch.tensor([[total - 1, 0]], dtype=torch.int32, device="cuda")
    for x in (k, v):
        for i in (0, total - 1):
            x[i] = torch.randn(kv, page, hd, generator=torch.Generator().manual_seed(i)).to(BF16).cuda()
    big = hipops.PagedCache(k, v, table, torch.zeros(1, dtype=torch.int32, device="cuda"))
    new = [torch.randn(1, 1100, kv, hd, generator=torch.Generator().manual_seed(5 + i)).to(BF16).cuda() for i in range(2)]
    hipops.cache_append(big, *new)
    assert big.lens.tolist() == [1100]
    assert torch.equal(k[total - 1].transpose(0, 1), new[0][0, :1024]) and torch.equal(v[0, :, :76].transpose(0, 1), new[1][0, 1024:])
    small = hipops.PagedCache(k[[total - 1, 0]].contiguous(), v[[total - 1, 0]].contiguous(), torch.tensor([[0, 1]], dtype=torch.int32, device="cuda"), big.lens)
    q = query(big, 8)
    assert torch.equal(hipops.cache_attention(q, big), hipops.cache_attention(q, small))


def test_attention_refuses():
    from interactron_amd import _lib, hipops
    cache = make([4, 4], weight=False)
    q = query(cache, 4)
    for bad, words in ((q[:1], "q must be"), (q[:, :3], "multiple"), (q.float(), "bfloat16"), (q[..., :32], "q must be"), (q[0], "q must be")):
        with pytest.raises(ValueError, match=words):
            hipops.cache_attention(bad, cache)
    for how, words in ((dict(window=0), "window"), (dict(window=2.0), "window"), (dict(sinks=-1), "sinks"), (dict(accumulate=True), "no weights")):
        with pytest.raises(ValueError, match=words):
            hipops.cache_attention(q, cache, **how)
    with pytest.raises(_lib.HipLibraryError, match="no backward"):
        hipops.cache_attention(q.clone().requires_grad_(True), cache)
    with pytest.raises(_lib.HipLibraryError, match="GPU"):
        hipops.cache_attention(q.cpu(), cache)
    with pytest.raises(ValueError, match="no weights"):
        hipops.cache_evict(cache, 4)


# ---- append -------------------------------------------------------------------------------------------------------------------------
def append_by_hand(cache, k, v, counts, at):
    """-> (k, v, weight, lens) after the call, token by token on the CPU"""
    pk, pv, table = cache.k.cpu().clone(), cache.v.cpu().clone(), cache.table.cpu()
    w, lens = cache.weight.cpu().clone() if cache.weight is not None else None, cache.lens.cpu().clone()
    for b in range(cache.batch):
        start = min(max(int((at if at is not None else lens)[b]), 0), cache.capacity)
        n = min(max(int(counts[b]), 0), k.shape[1]) if counts is not None else k.shape[1]
        for t in range(min(n, cache.capacity - start)):
            s = start + t
            if w is not None:
                w[b, :, s] = 0
            page = int(table[b, s // cache.page])
            if 0 <= page < pk.shape[0]:
                pk[page, :, s % cache.page], pv[page, :, s % cache.page] = k[b, t].cpu(), v[b, t].cpu()
        lens[b] = min(start + n, cache.capacity)
    return pk, pv, w, lens


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("hd, T, weight", [(32, 1, True), (64, 1, False), (128, 5, True), (64, 130, True), (32, 0, True)])
@pytest.mark.parametrize("form", ["plain", "counts", "at", "both"])
def test_append(dtype, hd, T, weight, form):
    from interactron_amd import hipops
    cache = make([0, 15, 16, 200, 64], kv=3, hd=hd, dtype=dtype, weight=weight, pages=15)
    g = torch.Generator().manual_seed(7)
    k, v = (torch.randn(5, T, 3, hd, generator=g).to(dtype).cuda() for _ in range(2))
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    counts = ints(T, 0, T // 2, 3 * T, -1) if form in ("counts", "both") else None
    at = ints(3, 0, 239, 100, 240) if form in ("at", "both") else None
    want = append_by_hand(cache, k, v, counts, at)
    hipops.cache_append(cache, k, v, counts=counts, at=at)
    for got, x in zip((cache.k, cache.v, cache.weight, cache.lens), want):
        assert x is None or torch.equal(got.cpu(), x)


def test_append_views_overflow_and_bad_pages():
    from interactron_amd import hipops
    cache = make([30, 47, 5], kv=2, page=16, pages=3, dtype=BF16)
    cache.table[2, 0], cache.table[2, 1] = -1, cache.k.shape[0]
    packed = torch.randn(3, 40, 3, 2, 64, generator=torch.Generator().manual_seed(8)).to(BF16).cuda()
    k, v = packed[:, :, 1], packed[:, :, 2]
    want = append_by_hand(cache, k, v, None, None)
    hipops.cache_append(cache, k, v)
    for got, x in zip((cache.k, cache.v, cache.weight, cache.lens), want):
        assert torch.equal(got.cpu(), x)
    assert cache.lens.tolist() == [48, 48, 45]
    # lengths as starts, passed by name: the call may not read what it has already changed
    again = make([30, 47, 5], kv=2, page=16, pages=3, dtype=BF16)
    want = append_by_hand(again, k, v, None, again.lens)
    hipops.cache_append(again, k, v, at=again.lens)
    for got, x in zip((again.k, again.v, again.weight, again.lens), want):
        assert torch.equal(got.cpu(), x)


def test_append_refuses():
    from interactron_amd import _lib, hipops
    cache = make([4, 4])
    k = torch.zeros(2, 3, 2, 64, dtype=BF16, device="cuda")
    ints = torch.zeros(2, dtype=torch.int32, device="cuda")
    for a, b in ((k[:1], k), (k.float(), k), (k, k[:, :2]), (k[:, :, :1], k), (k[..., :32], k), (k[0], k)):
        with pytest.raises(ValueError):
            hipops.cache_append(cache, a, b)
    for how in (dict(counts=ints.long()), dict(at=ints[:1]), dict(counts=ints.float())):
        with pytest.raises(ValueError):
            hipops.cache_append(cache, k, k, **how)
    with pytest.raises(_lib.HipLibraryError, match="GPU"):
        hipops.cache_append(cache, k, k.cpu())
    with pytest.raises(_lib.HipLibraryError, match="no backward"):
        hipops.cache_append(cache, k.clone().requires_grad_(True), k)
    base = torch.zeros(3, dtype=torch.int32, device="cuda")
    shared = hipops.PagedCache(cache.k, cache.v, cache.table, base[:2])
    for how in (dict(at=base[1:]), dict(counts=base[1:])):
        with pytest.raises(_lib.HipLibraryError, match="overlap"):
            hipops.cache_append(shared, k, k, **how)


def test_the_cache_keeps_its_tensors():
    cache = make([4, 4])
    for name in ("k", "v", "table", "lens", "weight"):
        with pytest.raises(AttributeError):
            setattr(cache, name, getattr(cache, name).clone())


# ---- select and compact -------------------------------------------------------------------------------------------------------------
def check_select(weight, lens, budget, sinks, recent):
    from interactron_amd import hipops
    kept, left = hipops.cache_select(weight, lens, budget, sinks=sinks, recent=recent)
    w, cap = weight.cpu().numpy(), weight.shape[2]
    for b in range(weight.shape[0]):
        n = min(max(int(lens[b]), 0), cap)
        assert int(left[b]) == min(n, budget)
        for h in range(weight.shape[1]):
            want = ref.select(w[b, h], n, budget, sinks, recent)
            got = kept[b, h].cpu().numpy()
            assert (got[: len(want)] == want).all() and (got[len(want):] == -1).all(), (b, h, n)
    return kept, left


@pytest.mark.parametrize("budget, sinks, recent", [(1, 0, 0), (1, 1, 0), (40, 0, 0), (40, 4, 30), (40, 40, 0), (40, 0, 40), (65, 3, 7), (300, 4, 100), (2000, 1, 1)])
def test_select(budget, sinks, recent):
    g = torch.Generator().manual_seed(budget)
    w = torch.randn(7, 3, 2000, generator=g).exp()
    w = torch.where(torch.rand(w.shape, generator=g) < 0.3, torch.zeros(()), w)
    lens = torch.tensor([0, 1, budget, min(budget + 1, 2000), 333, 1999, 1 << 29], dtype=torch.int32)
    check_select(w.cuda(), lens.cuda(), budget, sinks, recent)


@pytest.mark.parametrize("kind", ["equal", "few", "negative", "special", "steps", "groups"])
def test_select_ties_and_special_weights(kind):
    g = torch.Generator().manual_seed(3)
    shape = (3, 2, 5000)
    if kind == "equal":
        w = torch.full(shape, 0.25)
    elif kind == "few":
        w = torch.randint(0, 3, shape, generator=g).float()
    elif kind == "negative":
        w = torch.randn(shape, generator=g)
    elif kind == "special":
        pool = torch.tensor([float("nan"), float("inf"), float("-inf"), 0.0, -0.0, 1e-45, -1e-45, torch.finfo(FP32).max, torch.finfo(FP32).min, 1.0])
        w = pool[torch.randint(0, 10, shape, generator=g)]
    elif kind == "groups":   # all weights of a size stay or go: 2999 and 700 of the large ones, alike in their first or first two digits
        w = torch.rand(shape, generator=g) * 1e-3
        for first, count, base in ((100, 700, 1.5), (1000, 2299, 1.0 + 2.0 ** -8)):
            w[:, :, first: first + count] = base * (1 + torch.rand(3, 2, count, generator=g) * 2.0 ** -9)
        for budget in (700, 2999, 3000, 2998):
            check_select(w.cuda(), torch.tensor([5000, 4999, 3501], dtype=torch.int32, device="cuda"), budget, 0, 0)
    else:   # neighbours in the last bits
        w = (torch.randint(0, 1 << 12, shape, generator=g) + 0x3f800000).to(torch.int32).view(FP32)
    for budget, sinks, recent in ((700, 4, 100), (4999, 0, 0), (64, 0, 0), (3500, 10, 0)):
        check_select(w.cuda(), torch.tensor([5000, 4999, 3501], dtype=torch.int32, device="cuda"), budget, sinks, recent)


def test_select_long():
    w = torch.rand(1, 2, 140_001, generator=torch.Generator().manual_seed(1)).cuda()
    check_select(w, torch.tensor([140_001], dtype=torch.int32, device="cuda"), 70_003, 17, 1001)


@pytest.mark.parametrize("dtype", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("hd, kv, B, budget, weight", [(32, 1, 1, 30, True), (64, 2, 2, 900, True), (128, 3, 2, 1500, False), (64, 8, 40, 100, True), (128, 8, 1, 2100, True)])
def test_compact(dtype, hd, kv, B, budget, weight):
    from interactron_amd import hipops
    n = 2 * budget + 37
    lens = [max(0, n - 61 * b) for b in range(B)]
    cache = make(lens, kv=kv, hd=hd, page=64, dtype=dtype, weight=weight, pages=-(-n // 64) + 1)
    g = torch.Generator().manual_seed(11)
    score = torch.rand(B, kv, cache.capacity, generator=g).cuda()
    kept, left = check_select(score, cache.lens, budget, min(3, budget), budget // 4)
    k, v, w, table = cache.k.cpu(), cache.v.cpu(), cache.weight.cpu() if weight else None, cache.table.cpu().long()
    for b in range(B):
        m = int(left[b])
        to = torch.arange(m)
        old = kept[b, :, :m].cpu().long()
        for h in range(kv):
            for x in (k, v):
                x[table[b, to // 64], h, to % 64] = x[table[b, old[h] // 64], h, old[h] % 64].clone()
            if weight:
                w[b, h, :m] = w[b, h, old[h]].clone()
    hipops.cache_compact(cache, kept, left)
    assert torch.equal(cache.k.cpu(), k) and torch.equal(cache.v.cpu(), v) and torch.equal(cache.lens, left)
    assert not weight or torch.equal(cache.weight.cpu(), w)


def test_compact_skips_what_it_cannot_move():
    """indexes behind a row's own place, outside the capacity, and pages outside the pool are left alone"""
    from interactron_amd import hipops
    cache = make([64, 64], kv=1, page=16, pages=4, dtype=FP32)
    cache.table[1, 3] = -7
    k, w = cache.k.clone(), cache.weight.clone()
    kept = torch.tensor([[[0, 0, 2, 64, 1 << 30, -3]], [[0, 1, 2, 3, 50, 51]]], dtype=torch.int32, device="cuda")
    hipops.cache_compact(cache, kept, torch.tensor([6, 1 << 30], dtype=torch.int32, device="cuda"))
    assert torch.equal(cache.k, k) and cache.lens.tolist() == [6, 6]
    w[1, 0, 4:6] = w[1, 0, 50:52].clone()   # (weights are not in pages)
    assert torch.equal(cache.weight, w)


def test_compact_refuses():
    from interactron_amd import hipops
    cache = make([40, 40])
    kept, left = torch.zeros(2, 2, 8, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    for a, b in ((kept.long(), left), (kept[:, :1], left), (kept, left[:1]), (kept, left.long()), (kept[..., :0], left), (kept, cache.lens),
                 (torch.zeros(2, 2, 1000, dtype=torch.int32, device="cuda"), left), (kept.transpose(0, 1), left)):
        with pytest.raises(ValueError):
            hipops.cache_compact(cache, a, b)


# ---- together -----------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, FP32], ids=["bf16", "fp32"])
def test_a_rollout_with_evictions(dtype):
    """Prompt, then token by token, cut back whenever a sequence would pass 96 tokens; every step against the dense rows"""
    from interactron_amd import hipops
    cache = make([0, 0, 0], kv=2, page=16, pages=7, dtype=dtype)
    cache.weight.zero_()
    g = torch.Generator().manual_seed(5)
    rows = lambda T: [torch.randn(3, T, 2, 64, generator=g).to(dtype).cuda() for _ in range(2)]  # noqa: E731
    hipops.cache_append(cache, *rows(70), counts=torch.tensor([70, 33, 1], dtype=torch.int32, device="cuda"))
    evictions = 0
    for step in range(60):
        if step % 20 == 19:
            w, n = cache.weight.cpu().numpy(), cache.lens.tolist()
            want = [[ref.select(w[b, h], n[b], 60, 2, 20) for h in range(2)] for b in range(3)]
            dense = {(b, h): [ref.Pool(cache).rows(x, b, h, n[b])[0] for x in "kv"] for b in range(3) for h in range(2)}
            hipops.cache_evict(cache, 60, sinks=2, recent=20)
            for (b, h), (k, v) in dense.items():
                assert (ref.Pool(cache).rows("k", b, h, min(n[b], 60))[0] == k[want[b][h]]).all()
                assert (ref.Pool(cache).rows("v", b, h, min(n[b], 60))[0] == v[want[b][h]]).all()
                assert (cache.weight[b, h, : min(n[b], 60)].cpu().numpy() == w[b, h][want[b][h]]).all()
            evictions += sum(x > 60 for x in n)
        hipops.cache_append(cache, *rows(1))
        check_attention(cache, query(cache, 6, seed=100 + step), accumulate=True)
    assert evictions == 5 and max(cache.lens.tolist()) < 112


def test_captured_and_replayed():
    """A decoding step with its eviction as one graph: every replay like the eager calls, with eager work between them"""
    from interactron_amd import hipops

    def fresh():
        c = make([50, 30], kv=2, page=16, pages=6, dtype=BF16, seed=4)
        c.weight.zero_()
        return c

    def step(c, q, k, v):
        hipops.cache_append(c, k, v)
        out = hipops.cache_attention(q, c, accumulate=True)
        hipops.cache_evict(c, 56, sinks=1, recent=8)
        return out

    eager, caught = fresh(), fresh()
    q, k, v = query(eager, 4), torch.zeros(2, 3, 2, 64, dtype=BF16, device="cuda"), torch.zeros(2, 3, 2, 64, dtype=BF16, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(fresh(), q, k, v)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(caught, q, k, v)
    g = torch.Generator().manual_seed(9)
    for i in range(12):
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=g).to(BF16))
        graph.replay()
        want = step(eager, q, k, v)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(caught.lens, eager.lens) and torch.equal(caught.weight, eager.weight), i
        assert torch.equal(caught.k, eager.k) and torch.equal(caught.v, eager.v)
    assert eager.lens.tolist() == [56, 56]


def test_on_another_stream_and_two_at_once():
    from interactron_amd import hipops
    a, b = make([900, 1500], seed=1, page=64), make([1200, 7], seed=2, page=64)
    q = query(a, 8)
    want = [hipops.cache_attention(q, c) for c in (a, b)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(20):
        for i, c in enumerate((a, b)):
            with torch.cuda.stream(streams[i]):
                got[i].append(hipops.cache_attention(q, c))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


def test_the_same_call_gives_the_same_bits():
    from interactron_amd import hipops
    c = make([3000, 1234], kv=2, hd=128, page=64)
    q = query(c, 16)
    first = hipops.cache_attention(q, c, accumulate=True), c.weight.clone()
    for _ in range(5):
        c.weight.copy_(make([3000, 1234], kv=2, hd=128, page=64).weight)
        assert torch.equal(hipops.cache_attention(q, c, accumulate=True), first[0]) and torch.equal(c.weight, first[1])
