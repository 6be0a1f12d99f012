"""What the gradients of band attention ask for as workspace: -delta of every row and the partial sums of the blocks that are cut, no more."""
import ctypes

import pytest

from interactron_amd import _lib
from tests.test_band_cpu import c_band


def need(**how):
    f = dict(dict(batch=1, window=0, sinks=0, causal=1, dtype=1), **how)
    for t, L, h in (("q", "Lq", "heads"), ("k", "Lk", "kv_heads"), ("v", "Lk", "kv_heads")):
        f.update({t + "_sb": f[L] * f[h] * f["hd"], t + "_sl": f[h] * f["hd"], t + "_sh": f["hd"]})
    n = ctypes.c_size_t(0)
    assert _lib.load().ix_workspace_bytes_band_attn_bwd(ctypes.byref(c_band(**f)), ctypes.byref(n)) == 0
    return n.value - f["batch"] * f["heads"] * (-(-f["Lq"] // 128) * 128) * 4


def test_only_the_blocks_of_the_first_keys_are_cut():
    # 12 755 tokens: one block of 128 keys has first keys; it streams 200 tiles of queries where the others stream 43: three pieces
    assert need(Lq=12755, Lk=12755, heads=8, kv_heads=8, hd=64, window=2551, sinks=16) == 8 * 3 * 2 * 128 * 64 * 4


@pytest.mark.parametrize("L", [131072, 1 << 20])
def test_long_sequences(L):
    grads = 2 * L * 8 * 128 * 2   # dk and dv
    assert 0 < need(Lq=L, Lk=L, heads=32, kv_heads=8, hd=128, window=4096, sinks=4) <= grads // 16


def test_nothing_is_cut():
    for sinks in (0, 200):
        assert need(Lq=4096, Lk=4096, heads=32, kv_heads=32, hd=64, sinks=sinks) == 0
    assert need(Lq=12755, Lk=12755, heads=8, kv_heads=8, hd=64, window=2551) == 0


def test_all_blocks_are_cut():
    # one head of 1 100 rows: 18 blocks of 64 keys and 18 of queries, each in more than one piece and in no more than make 384 of 18
    n = need(Lq=1100, Lk=1100, heads=1, kv_heads=1, hd=128)
    assert n % (64 * 128 * 4) == 0 and 18 * 2 * 64 * 128 * 4 < n <= (18 * 2 * 22 + 18 * 22) * 64 * 128 * 4
