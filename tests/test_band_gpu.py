"""Band attention and its gradients against the definition in 64 bits (tests/sequence_reference.py)."""
import numpy as np
import pytest
import torch

from tests import sequence_reference as ref

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
TYPES = pytest.mark.parametrize("dtype", [BF16, FP16, FP32], ids=["bf16", "fp16", "fp32"])


def rows(B, L, H, D, dtype, seed, scale=1.0):
    return (torch.randn(B, L, H, D, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).cuda()


def inputs(B, Lq, Lk, H, kv, D, dtype, seed=0, scale=1.5):
    return rows(B, Lq, H, D, dtype, 4 * seed, scale), rows(B, Lk, kv, D, dtype, 4 * seed + 1), rows(B, Lk, kv, D, dtype, 4 * seed + 2), rows(B, Lq, H, D, dtype, 4 * seed + 3)


def close(got, want, err, name=""):
    dtype = got.dtype
    got = ref.f64(got)
    assert np.isfinite(got).all(), name
    # the last rounding: half a step of the value before it; below the type's normal range (fp16: 2^-14) a step is absolute
    tol = err + ref.half_step(dtype) * (np.abs(want) + err) + (2.0 ** -25 if dtype == FP16 else 1e-38)
    off = np.abs(got - want)
    assert (off <= tol).all(), (name, float((off / tol).max()), np.unravel_index((off / tol).argmax(), off.shape))


def check(q, k, v, do=None, **how):
    from interactron_amd import hipops
    lens = {x: how[x].cpu() for x in ("q_lens", "kv_lens") if how.get(x) is not None}
    want, err = ref.band_attention(q, k, v, how.get("window"), how.get("sinks", 0), how.get("causal", True), how.get("scale"), do=do, **lens)
    if do is None:
        out = hipops.band_attention(q, k, v, **how)
        close(out, want["out"], err["out"], "out")
        return out
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = hipops.band_attention(*leaves, **how)
    got = dict(out=out, **dict(zip(("dq", "dk", "dv"), torch.autograd.grad(out, leaves, do))))
    for x in want:
        assert got[x].dtype == q.dtype and tuple(got[x].shape) == want[x].shape
        close(got[x].detach(), want[x], err[x], x)
    return got


@TYPES
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("H, kv, causal", [(2, 2, True), (4, 1, False), (6, 2, True)])
def test_types_and_head_layouts(dtype, D, H, kv, causal):
    check(*inputs(2, 150, 150, H, kv, D, dtype), window=40, sinks=3, causal=causal)


@pytest.mark.parametrize("dtype, D", [(BF16, 64), (FP32, 32), (FP16, 128)])
@pytest.mark.parametrize("Lq, Lk", [(1, 1), (1, 200), (2, 3), (63, 63), (64, 64), (65, 65), (127, 129), (129, 127), (17, 300), (300, 17), (257, 257)])
@pytest.mark.parametrize("causal", [True, False])
def test_lengths(dtype, D, Lq, Lk, causal):
    check(*inputs(1, Lq, Lk, 2, 1, D, dtype), window=50, sinks=2, causal=causal)
    check(*inputs(1, Lq, Lk, 2, 1, D, dtype), causal=causal)


@pytest.mark.parametrize("dtype, D", [(BF16, 64), (FP32, 64), (FP16, 32), (BF16, 128)])
@pytest.mark.parametrize("window, sinks", [(1, 0), (2, 1), (16, 0), (17, 64), (64, 5), (65, 65), (128, 130), (400, 0), (1 << 29, 0), (None, 40), (3, 1 << 29)])
@pytest.mark.parametrize("causal", [True, False])
def test_windows_and_first_keys(dtype, D, window, sinks, causal):
    check(*inputs(1, 330, 330, 2, 2, D, dtype), window=window, sinks=sinks, causal=causal)


@TYPES
@pytest.mark.parametrize("causal", [True, False])
def test_padded_batches(dtype, causal):
    """padding may hold anything; rows that see nothing give zeros, in the middle of a batch and at the front of a sequence"""
    q, k, v, do = inputs(6, 140, 170, 2, 1, 64, dtype)
    m, n = [140, 100, 0, 1, 140, 64], [170, 100, 50, 170, 30, 0]
    for b in range(6):
        for t, x in ((q, m), (do, m), (k, n), (v, n)):
            t[b, x[b]:] = float("nan") if b % 2 else float("inf")
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    got = check(q, k, v, do, window=33, sinks=4, causal=causal, q_lens=ints(m), kv_lens=ints(n))
    for b in range(6):
        for x in ("out", "dq"):
            assert (got[x][b, m[b]:] == 0).all()
        for x in ("dk", "dv"):
            assert (got[x][b, n[b]:] == 0).all()
    if causal:   # 140 queries over 30 keys: the first 110 stand before the first key
        assert (got["out"][4, :110] == 0).all() and (got["dq"][4, :110] == 0).all() and (got["out"][4, 110:] != 0).any()
    assert (got["out"][5] == 0).all()
    # lengths beyond the tensors and below zero are clamped
    again = check(q, k, v, None, window=33, sinks=4, causal=causal, q_lens=ints([1 << 30, 100, -7, 1, 140, 64]), kv_lens=ints([1 << 30, 100, 50, 170, 30, -1]))
    assert torch.equal(again, got["out"])


def test_masked_keys_may_be_infinite():
    """keys outside every query's band: no score of them survives (their values have to be finite)"""
    from interactron_amd import hipops
    q, k, v, _ = inputs(1, 40, 200, 2, 1, 64, BF16)
    want = hipops.band_attention(q, k, v, window=30, sinks=2)
    for value in (float("nan"), float("inf"), float("-inf"), torch.finfo(BF16).min):
        k[:, 2:131] = value
        assert torch.equal(hipops.band_attention(q, k, v, window=30, sinks=2), want)


@pytest.mark.parametrize("dtype", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("scale", [0.0, -0.2, 2.0, 1e-6])
def test_scales(dtype, scale):
    check(*inputs(1, 100, 100, 2, 1, 64, dtype), window=30, sinks=1, scale=scale)


@TYPES
def test_large_scores(dtype):
    """rows whose maximum climbs from tile to tile, and weights that vanish"""
    q, k, v, do = inputs(1, 300, 300, 2, 2, 64, dtype)
    k *= torch.linspace(0.05, 6, 300, device="cuda").view(1, 300, 1, 1).to(dtype)
    check(q, k, v, None, causal=False)
    check(q, k, v, do, window=100, sinks=3, causal=True)


@pytest.mark.parametrize("size", [1e-6, 1e-3, 1e3, 3e4])
def test_gradients_of_any_size_in_fp16(size):
    q, k, v, do = inputs(1, 200, 200, 2, 1, 64, FP16)
    check(q, k, (v * 1e-2).to(FP16) if size > 1 else v, (do.float() * size / do.float().abs().max()).to(FP16), window=60, sinks=2)


@pytest.mark.parametrize("dtype", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("Lq, Lk, H, kv, window, sinks", [(1500, 1500, 2, 2, 100, 130), (1500, 1500, 8, 1, 64, 5), (700, 900, 8, 1, None, 0)])
def test_long_rows_and_blocks_cut_into_splits(dtype, Lq, Lk, H, kv, window, sinks):
    check(*inputs(1, Lq, Lk, H, kv, 64, dtype), window=window, sinks=sinks)
    check(*inputs(1, Lq, Lk, H, kv, 64, dtype), window=window, sinks=sinks, causal=False)


@TYPES
@pytest.mark.parametrize("Lq, Lk, how", [(1, 4000, {}), (3, 2500, dict(causal=False)), (70, 3000, dict(window=2000, sinks=130)), (40, 1200, dict(window=5, sinks=1000))])
def test_few_queries_over_many_keys(dtype, Lq, Lk, how):
    """pieces of the keys, joined; with gradients, and with a batch whose lengths leave pieces and rows empty"""
    q, k, v, do = inputs(1, Lq, Lk, 4, 2, 64, dtype)
    check(q, k, v, do, **how)
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    q, k, v, do = inputs(3, Lq, Lk, 2, 1, 128, dtype)
    check(q, k, v, do, q_lens=ints(Lq, Lq // 2, Lq), kv_lens=ints(Lk, 37, 0), **how)


@TYPES
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("Lq, Lk, H, kv, how", [(1100, 1100, 1, 1, {}), (400, 2000, 2, 1, dict(window=900, sinks=70)), (90, 1300, 3, 1, dict(causal=False, window=1000))])
def test_gradients_of_few_rows_in_pieces(dtype, D, Lq, Lk, H, kv, how):
    check(*inputs(1, Lq, Lk, H, kv, D, dtype), **how)


@TYPES
def test_views(dtype):
    """a packed projection in place, rows off 16 bytes, swapped axes, inputs that are one row many times"""
    from interactron_amd import hipops
    packed = rows(2, 90, 3 * 4, 64, dtype, 3).view(2, 90, 3, 4, 64).requires_grad_(True)
    do = rows(2, 90, 4, 64, dtype, 4)
    how = dict(window=20, sinks=1)
    parts = [packed[:, :, i] for i in range(3)]
    plain = [p.detach().clone().requires_grad_(True) for p in parts]
    a, b = hipops.band_attention(*parts, **how), hipops.band_attention(*plain, **how)
    assert torch.equal(a, b)
    (ga,), gb = torch.autograd.grad(a, packed, do), torch.autograd.grad(b, plain, do)
    assert all(torch.equal(ga[:, :, i], gb[i]) for i in range(3))
    odd = torch.empty(2, 90, 4, 65, dtype=dtype, device="cuda")[..., 1:].copy_(plain[0].detach())
    swapped = plain[1].detach().transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(hipops.band_attention(odd, swapped, plain[2], **how), a)
    (gc,) = torch.autograd.grad(hipops.band_attention(*plain, **how), plain[0], do.transpose(1, 2).contiguous().transpose(1, 2))
    assert torch.equal(gc, gb[0])
    # one key row for all: its gradient is the sum (in the type, by autograd) of the rows' gradients
    one = rows(2, 1, 4, 64, dtype, 9).requires_grad_(True)
    got = check(plain[0].detach(), one.detach().expand(2, 90, 4, 64), plain[2].detach(), do, **how)
    (g1,) = torch.autograd.grad(hipops.band_attention(plain[0], one.expand(2, 90, 4, 64), plain[2], **how), one, do)
    assert torch.allclose(g1, got["dk"].sum(1, keepdim=True), rtol=0.05, atol=0.05)
    # a gradient that is one number everywhere
    (gs,) = torch.autograd.grad(hipops.band_attention(*plain, **how).sum(), plain[2])
    assert torch.equal(gs, torch.autograd.grad(hipops.band_attention(*plain, **how), plain[2], torch.ones_like(do))[0])


def test_gradients_against_differences():
    """fp32, along random directions: (f(x + e d) - f(x - e d)) / 2 e, f = sum(out * do) in 64 bits; the error of the middle difference is
    e^2 / 6 of the third derivative, the rounding of out u sum|do out| / e: at e = 2^-7 both are below 2^-9 of |do| |out|"""
    from interactron_amd import hipops
    q, k, v, do = inputs(2, 70, 90, 4, 2, 64, FP32, scale=1.0)
    how = dict(window=25, sinks=3)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    grads = torch.autograd.grad(hipops.band_attention(*leaves, **how), leaves, do)
    f = lambda *x: float((hipops.band_attention(*x, **how).double() * do.double()).sum())  # noqa: E731
    for i, (t, g) in enumerate(zip((q, k, v), grads)):
        d = rows(*t.shape, FP32, 50 + i)
        x = [q, k, v]
        e = 2.0 ** -7
        x[i] = t + e * d
        up = f(*x)
        x[i] = t - e * d
        diff, dot = (up - f(*x)) / (2 * e), float((g.double() * d.double()).sum())
        assert abs(diff - dot) <= 2.0 ** -9 * float((g.double().abs() * d.double().abs()).sum()), (i, diff, dot)


def test_some_gradients_only():
    from interactron_amd import hipops
    q, k, v, do = inputs(1, 60, 60, 2, 1, 64, BF16)
    full = check(q, k, v, do, window=9)
    for i, name in enumerate(("dq", "dk", "dv")):
        t = [q, k, v]
        t[i] = t[i].clone().requires_grad_(True)
        out = hipops.band_attention(*t, window=9)
        out.backward(do)
        assert torch.equal(t[i].grad, full[name]) and torch.equal(out.detach(), full["out"])
    with torch.no_grad():
        assert torch.equal(hipops.band_attention(*[x.clone().requires_grad_(True) for x in (q, k, v)], window=9), full["out"])


def test_nothing_to_attend_to():
    from interactron_amd import hipops
    for B, Lq, Lk in ((0, 5, 5), (2, 0, 5), (2, 5, 0)):
        t = [torch.randn(B, L, 2, 64, device="cuda", requires_grad=True) for L in (Lq, Lk, Lk)]
        out = hipops.band_attention(*t, window=3)
        assert out.shape == t[0].shape and (out == 0).all()
        assert all((g == 0).all() and g.shape == x.shape for g, x in zip(torch.autograd.grad(out.sum(), t), t))


def test_not_differentiable_twice():
    from interactron_amd import _lib, hipops
    t = [x.requires_grad_(True) for x in inputs(1, 20, 20, 2, 1, 64, FP32)[:3]]
    with pytest.raises(_lib.HipLibraryError, match="differentiable once"):
        torch.autograd.grad(hipops.band_attention(*t).sum(), t[0], create_graph=True)


def test_inputs_changed_in_between_are_noticed():
    from interactron_amd import hipops
    q, k, v, do = inputs(1, 20, 20, 2, 1, 64, FP32)
    n = torch.tensor([20], dtype=torch.int32, device="cuda")
    out = hipops.band_attention(q.requires_grad_(True), k, v, kv_lens=n)
    n.fill_(3)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.backward(do)


@TYPES
def test_a_graph_kept_for_two_backward_passes(dtype):
    from interactron_amd import hipops
    q, k, v, do = inputs(1, 500, 500, 4, 2, 64, dtype)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    out = hipops.band_attention(*leaves, sinks=2)
    out.backward(do, retain_graph=True)
    once = [t.grad.clone() for t in leaves]
    out.backward(do)
    assert all(torch.equal(t.grad, 2 * g) for t, g in zip(leaves, once))


@TYPES
def test_saved_tensors_kept_elsewhere(dtype):
    """hooks that move what the forward pass saves: the gradients come from the tensors that come back"""
    from interactron_amd import hipops
    q, k, v, do = inputs(2, 150, 150, 4, 2, 64, dtype)
    n = torch.tensor([150, 90], dtype=torch.int32, device="cuda")

    def step():
        t = [x.detach().requires_grad_(True) for x in (q, k, v)]
        return hipops.band_attention(*t, window=40, sinks=3, q_lens=n, kv_lens=n), t

    out, t = step()
    want = torch.autograd.grad(out, t, do)
    with torch.autograd.graph.save_on_cpu():
        out, t = step()
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, t, do), want))


@pytest.mark.parametrize("D", [64, 128])
def test_the_same_call_gives_the_same_bits(D):
    q, k, v, do = inputs(2, 700, 700, 8, 2, D, BF16)
    from interactron_amd import hipops
    def once():
        t = [x.detach().requires_grad_(True) for x in (q, k, v)]
        out = hipops.band_attention(*t, window=100, sinks=9)
        return (out.detach(),) + torch.autograd.grad(out, t, do)
    first = once()
    for _ in range(4):
        assert all(torch.equal(a, b) for a, b in zip(first, once()))


@pytest.mark.parametrize("L", [300, 900])
def test_captured_and_replayed_with_gradients(L):
    """(900: all three gradients and the output in pieces)"""
    from interactron_amd import hipops
    q, k, v, do = inputs(2, L, L, 4, 2, 64, BF16)
    n = torch.tensor([L, L - 100], dtype=torch.int32, device="cuda")

    def step():
        t = [x.detach().requires_grad_(True) for x in (q, k, v)]
        out = hipops.band_attention(*t, window=70 if L == 300 else None, sinks=5, q_lens=n, kv_lens=n)
        return (out.detach(),) + torch.autograd.grad(out, t, do)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        caught = step()
    g = torch.Generator().manual_seed(1)
    for i in range(6):
        for t in (q, k, v, do):
            t.copy_(torch.randn(t.shape, generator=g).to(BF16))
        n.copy_(torch.tensor([L - 20 * i, 10 * i], dtype=torch.int32))
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(caught, want)), i


def test_two_streams_at_once():
    from interactron_amd import hipops
    sets = [inputs(1, 900, 900, 4, 4, 64, BF16, seed=s) for s in (1, 2)]

    def step(q, k, v, do):
        t = [x.detach().requires_grad_(True) for x in (q, k, v)]
        out = hipops.band_attention(*t, window=300, sinks=20)
        return (out.detach(),) + torch.autograd.grad(out, t, do)

    want = [step(*s) for s in sets]
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(8):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(step(*sets[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, b) for x in got[i] for a, b in zip(x, want[i]))


def test_beyond_32_bit_offsets():
    """keys of more than 2^32 bytes: the last 300 queries over their band and the first keys"""
    from interactron_amd import hipops
    L, kv, D = (1 << 21) + 77, 8, 128
    k, v = (torch.empty(1, L, kv, D, dtype=BF16, device="cuda") for _ in range(2))
    for t in (k, v):
        t.zero_()
        t[:, :8] = rows(1, 8, kv, D, BF16, 1)
        t[:, -900:] = rows(1, 900, kv, D, BF16, 2)
    q, do = rows(1, 300, kv, D, BF16, 3), rows(1, 300, kv, D, BF16, 4)
    near = [torch.cat([t[:, :8], t[:, -900:]], 1).contiguous() for t in (k, v)]
    leaves, small = [x.requires_grad_(True) for x in (q, k, v)], [x.detach().clone().requires_grad_(True) for x in (q, *near)]
    a, b = hipops.band_attention(*leaves, window=500, sinks=8), hipops.band_attention(*small, window=500, sinks=8)
    # (the same keys for every query; tiles start elsewhere, so sums differ in their order)
    assert torch.allclose(a.float(), b.float(), rtol=2 ** -7, atol=2 ** -9)
    ga, gb = torch.autograd.grad(a, leaves, do), torch.autograd.grad(b, small, do)
    assert torch.allclose(ga[0].float(), gb[0].float(), rtol=2 ** -6, atol=2 ** -7)
    for x, y in zip(ga[1:], gb[1:]):
        assert torch.allclose(x[:, -900:].float(), y[:, 8:].float(), rtol=2 ** -6, atol=2 ** -6)
        assert torch.allclose(x[:, :8].float(), y[:, :8].float(), rtol=2 ** -6, atol=2 ** -6)
        assert (x[:, 8:-900] == 0).all()


def test_prompt_then_tokens():
    """A prompt by band attention, then token by token over a paged cache with the same window and first keys: like one long prompt"""
    from interactron_amd import hipops
    B, L, T, H, kv, D, how = 2, 130, 40, 4, 2, 64, dict(window=48, sinks=3)
    q, k, v, _ = inputs(B, L + T, L + T, H, kv, D, FP32)
    want, err = ref.band_attention(q, k, v, causal=True, **how)
    pool = [torch.zeros(30, kv, 16, D, device="cuda") for _ in range(2)]
    table = torch.randperm(30, generator=torch.Generator().manual_seed(1))[:22].reshape(2, 11).to(torch.int32).cuda()
    cache = hipops.PagedCache(*pool, table, torch.zeros(B, dtype=torch.int32, device="cuda"))
    hipops.cache_append(cache, k[:, :L], v[:, :L])
    close(hipops.band_attention(q[:, :L], k[:, :L], v[:, :L], **how), want["out"][:, :L], err["out"][:, :L])
    for t in range(L, L + T):
        hipops.cache_append(cache, k[:, t:t + 1], v[:, t:t + 1])
        close(hipops.cache_attention(q[:, t], cache, **how), want["out"][:, t], err["out"][:, t] + 1e-30)
    # ... and its last tokens once more as the newest part of the prompt
    close(hipops.band_attention(q[:, L:], k, v, **how), want["out"][:, L:], err["out"][:, L:])
