"""Band attention with as many blocks of rows as large calls have: owner blocks of 128 rows, and blocks in pieces where the launch has one or
two of them a compute unit.  Many short sequences, lengths off the blocks' size (tests/band_bounds.py)."""
import ctypes

import pytest
import torch

from tests import band_bounds as bounds
from tests.test_band_weights_gpu import BF16, FP16, FP32, inputs

pytestmark = pytest.mark.gpu

FLOOR = {BF16: 0.0, FP16: 2.0 ** -32, FP32: 0.0}
TYPES16 = pytest.mark.parametrize("dtype", [BF16, FP16], ids=["bf16", "fp16"])


def lengths(B, most, least):
    """from nothing to `most`"""
    x = [most - (most - least) * b // (B - 1) for b in range(B)]
    x[1], x[2] = 0, 1
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@TYPES16
@pytest.mark.parametrize("D", [32, 64])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("Lq, Lk, how", [(70, 70, dict(window=21, sinks=2)), (129, 129, {}), (129, 75, dict(window=40, sinks=9)), (75, 150, dict(sinks=3, window=64))],
                         ids=["70", "129", "more queries", "more keys"])
def test_128_rows_a_block_with_gradients(dtype, D, causal, Lq, Lk, how):
    """38 x 16 blocks or more: from 600 on"""
    bounds.check(*inputs(38, Lq, Lk, 16, 16, D, dtype, seed=Lq + D), causal=causal, floor=FLOOR[dtype], **how)


@TYPES16
@pytest.mark.parametrize("D", [32, 64])
@pytest.mark.parametrize("causal", [True, False])
def test_128_rows_a_block_padded(dtype, D, causal):
    """sequences of nothing, one token and parts of a block; three blocks a head, shared key heads; padding is never read"""
    B, L = 20, 290
    q, k, v, do = inputs(B, L, L, 16, 4, D, dtype, seed=D)
    m, n = lengths(B, L, 100), lengths(B, L, 60)
    n[3], m[4] = 0, 129
    for b in range(B):
        for t, x in ((q, m), (do, m), (k, n), (v, n)):
            t[b, int(x[b]):] = float("nan")
    got = bounds.check(q, k, v, do, window=77, sinks=5, causal=causal, q_lens=m, kv_lens=n, floor=FLOOR[dtype])
    for b in range(B):
        assert (got["out"][b, int(m[b]):] == 0).all() and (got["dq"][b, int(m[b]):] == 0).all()
        assert (got["dk"][b, int(n[b]):] == 0).all() and (got["dv"][b, int(n[b]):] == 0).all()


@TYPES16
@pytest.mark.parametrize("B, Lq, Lk, how", [(24, 70, 70, dict(causal=False)), (24, 129, 140, dict(window=50, sinks=3)), (33, 90, 90, {}), (25, 127, 300, dict(window=33, sinks=20, causal=False))])
def test_128_rows_a_block_of_head_dim_128(dtype, B, Lq, Lk, how):
    """the forward pass: from 384 blocks on, 512 with causal rows and no window"""
    q, k, v, _ = inputs(B, Lq, Lk, 16, 4, 128, dtype, seed=B)
    bounds.check(q, k, v, None, floor=FLOOR[dtype], **how)
    bounds.check(q, k, v, None, floor=FLOOR[dtype], q_lens=lengths(B, Lq, 5), kv_lens=lengths(B, Lk, 40), **how)


def pieces(q, k, **how):
    """of the forward pass, from its workspace"""
    from interactron_amd import hipops
    n = ctypes.c_size_t(0)
    c = hipops.band._band(q, k, k, None, None, how.get("window", 0), how.get("sinks", 0), 1 if how.get("causal", True) else 0, 0.125)
    assert hipops._L().ix_workspace_bytes_band_attn_fwd(c, ctypes.byref(n)) == 0
    return n.value // (q.shape[0] * q.shape[2] * q.shape[1] * (q.shape[3] + 2) * 4)


@pytest.mark.parametrize("dtype, D", [(BF16, 64), (FP16, 128), (FP32, 64), (BF16, 32)])
@pytest.mark.parametrize("how", [dict(causal=False), dict(sinks=7), dict(window=1050, sinks=3)], ids=["full", "causal", "window"])
def test_pieces_of_129_to_511_blocks(dtype, D, how):
    q, k, v, _ = inputs(2, 590, 1150, 8, 4, D, dtype, seed=D)
    assert pieces(q, k, **how) in (2, 3, 4)   # 160 blocks of 64 queries over 18 tiles of 64 keys (36 of 32)
    lens = torch.tensor([590, 333], dtype=torch.int32, device="cuda"), torch.tensor([1111, 70], dtype=torch.int32, device="cuda")
    bounds.check(q, k, v, None, floor=FLOOR[dtype], **how)
    bounds.check(q, k, v, None, floor=FLOOR[dtype], q_lens=lens[0], kv_lens=lens[1], **how)


@pytest.mark.parametrize("dtype, D", [(BF16, 128), (FP32, 32)])
def test_two_pieces_of_the_gradients(dtype, D):
    """416 blocks of 64 queries that stream 3 200 keys, 400 of keys that stream 4 x 800 queries: two pieces each"""
    q, k, v, do = inputs(2, 800, 3200, 16, 4, D, dtype, seed=D)
    m, n = torch.tensor([800, 130], dtype=torch.int32, device="cuda"), torch.tensor([3190, 200], dtype=torch.int32, device="cuda")
    bounds.check(q, k, v, do, sinks=3, causal=D == 128, q_lens=m, kv_lens=n, floor=FLOOR[dtype])
