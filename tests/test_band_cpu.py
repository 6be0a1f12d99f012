"""Refusals of band attention, at the Python entry point and at the C boundary."""
import ctypes

import pytest
import torch

from interactron_amd import _lib, hipops

BF16 = torch.bfloat16


def qkv(B=2, Lq=5, Lk=7, H=4, kv=2, D=64, dtype=BF16):
    return torch.zeros(B, Lq, H, D, dtype=dtype), torch.zeros(B, Lk, kv, D, dtype=dtype), torch.zeros(B, Lk, kv, D, dtype=dtype)


def test_cpu_tensors_are_refused():
    with pytest.raises(_lib.HipLibraryError, match="GPU"):
        hipops.band_attention(*qkv())


@pytest.mark.parametrize("shape, how, words", [
    (dict(D=48), {}, "head dim of 48"), (dict(H=3), {}, "3 query heads"), (dict(kv=0), {}, "key heads"), (dict(dtype=torch.float64), {}, "q must be"),
    ({}, dict(window=0), "window"), ({}, dict(window=-3), "window"), ({}, dict(window=1.5), "window"), ({}, dict(window=1 << 30), "window"),
    ({}, dict(sinks=-1), "sinks"), ({}, dict(sinks=None), "sinks"), ({}, dict(scale=float("nan")), "scale"), ({}, dict(scale=float("inf")), "scale"), ({}, dict(scale=-1e39), "scale"),
    ({}, dict(q_lens=torch.zeros(2)), "q_lens"), ({}, dict(kv_lens=torch.zeros(3, dtype=torch.int32)), "kv_lens"),
    ({}, dict(kv_lens=torch.zeros(4, dtype=torch.int32)[::2]), "kv_lens"), ({}, dict(q_lens=torch.zeros(2, dtype=torch.int64)), "q_lens"),
])
def test_wrong_arguments_are_refused(shape, how, words):
    with pytest.raises(ValueError, match=words):
        hipops.band_attention(*qkv(**shape), **how)


def test_too_many_heads_for_a_launch_are_refused():
    q, k = torch.zeros(1, 1, 1, 64, dtype=BF16).expand(1 << 22, 1, 4, 64), torch.zeros(1, 1, 1, 64, dtype=BF16).expand(1 << 22, 1, 1, 64)
    with pytest.raises(ValueError, match="too many"):
        hipops.band_attention(q, k, k)


@pytest.mark.parametrize("change", [lambda q, k, v: (q[0], k, v), lambda q, k, v: (q, k.float(), v), lambda q, k, v: (q, k, v[:, :3]),
                                    lambda q, k, v: (q[:1], k, v), lambda q, k, v: (q[..., :32], k, v), lambda q, k, v: (q, k[:, :, :1], v)])
def test_tensors_that_do_not_fit_are_refused(change):
    with pytest.raises(ValueError):
        hipops.band_attention(*change(*qkv()))


class BandC(ctypes.Structure):   # struct ix_band of include/interactron_hip.h
    _fields_ = ([(n, ctypes.c_void_p) for n in ("q", "k", "v")] + [("%s_s%s" % (t, d), ctypes.c_int64) for t in "qkv" for d in "blh"] +
                [("q_lens", ctypes.c_void_p), ("kv_lens", ctypes.c_void_p)] +
                [(n, ctypes.c_int) for n in ("dtype", "batch", "Lq", "Lk", "heads", "kv_heads", "hd", "window", "sinks", "causal")] +
                [("scale", ctypes.c_float)])


def c_band(**change):
    """A description whose pointers are never followed"""
    f = dict(q=4096, k=4096, v=4096, q_sb=1280, q_sl=256, q_sh=64, k_sb=896, k_sl=128, k_sh=64, v_sb=896, v_sl=128, v_sh=64, q_lens=None, kv_lens=None,
             dtype=1, batch=2, Lq=5, Lk=7, heads=4, kv_heads=2, hd=64, window=0, sinks=0, causal=1, scale=0.125)
    f.update(change)
    return BandC(*[f[n] for n, _ in BandC._fields_])


def test_the_description_is_packed_as_the_header_lays_it_out():
    q, k, v = torch.zeros(2, 5, 4, 64, dtype=BF16), torch.zeros(2, 7, 2, 64, dtype=BF16), torch.zeros(2, 7, 4, 64, dtype=BF16)[:, :, :2]
    n = torch.zeros(2, dtype=torch.int32)
    for lens in (None, n):
        c = BandC.from_buffer_copy(hipops.band._band(q, k, v, n, lens, 3, 9, 1, -0.25))
        want = dict(q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), q_sb=1280, q_sl=256, q_sh=64, k_sb=896, k_sl=128, k_sh=64, v_sb=1792, v_sl=256, v_sh=64,
                    q_lens=n.data_ptr(), kv_lens=None if lens is None else n.data_ptr(), dtype=1, batch=2, Lq=5, Lk=7, heads=4, kv_heads=2, hd=64, window=3,
                    sinks=9, causal=1, scale=-0.25)
        assert {f: getattr(c, f) for f, _ in BandC._fields_} == want


@pytest.mark.parametrize("change", [dict(q=None), dict(k=None), dict(v=4100), dict(dtype=3), dict(hd=80), dict(batch=0), dict(Lq=0), dict(Lk=0), dict(Lq=65535 * 64 + 1), dict(Lk=65535 * 64 + 1),
                                    dict(heads=3), dict(kv_heads=0), dict(heads=0), dict(window=-1), dict(sinks=-1), dict(scale=float("nan")),
                                    dict(scale=float("inf")), dict(q_sl=252), dict(v_sh=33), dict(batch=1 << 29), dict(batch=1 << 22)], ids=str)
def test_c_entries_refuse_a_bad_description(change):
    L, c, n = _lib.load(), c_band(**change), ctypes.c_size_t(0)
    for rc in (L.ix_band_attn_fwd(ctypes.byref(c), 4096, 4096, 4096, 4096, 1 << 30, None), L.ix_workspace_bytes_band_attn_fwd(ctypes.byref(c), ctypes.byref(n)), L.ix_workspace_bytes_band_attn_bwd(ctypes.byref(c), ctypes.byref(n)),
               L.ix_band_attn_bwd(ctypes.byref(c), 4096, 4096, 4096, 4096, 1280, 256, 64, 4096, 4096, 4096, 4096, 1 << 30, None)):
        assert rc == -1 and L.ix_last_error()


def test_c_entries_refuse_bad_buffers():
    L, c, n = _lib.load(), c_band(), ctypes.c_size_t(0)
    ref = ctypes.byref(c)
    assert L.ix_band_attn_fwd(ref, None, None, None, None, 0, None) == -1 and L.ix_band_attn_fwd(ref, 4104, None, None, None, 0, None) == -1
    assert L.ix_band_attn_fwd(ref, 4096, 4096, 4104, None, 0, None) == -1
    assert L.ix_workspace_bytes_band_attn_bwd(ref, ctypes.byref(n)) == 0 and n.value >= 2 * 4 * 128 * 4
    good = [ref, 4096, 4096, 4096, 4096, 1280, 256, 64, 4096, 4096, 4096, 4096, n.value, None]
    for place, value, code in ((1, None, -1), (2, None, -1), (3, None, -1), (4, 4104, -1), (6, 100, -1), (8, None, -1), (9, 4104, -1), (11, None, -3), (11, 4100, -3), (12, n.value - 1, -3)):
        args = list(good)
        args[place] = value
        assert L.ix_band_attn_bwd(*args) == code, (place, L.ix_last_error())
    few = c_band(Lq=3, Lk=5000, q_sb=768, k_sb=640000, v_sb=640000)   # few rows over many keys: pieces
    assert L.ix_workspace_bytes_band_attn_fwd(ctypes.byref(few), ctypes.byref(n)) == 0 and n.value >= 2 * 2 * 4 * 3 * 66 * 4
    for ws, size in ((None, n.value), (4100, n.value), (4096, n.value - 1)):
        assert L.ix_band_attn_fwd(ctypes.byref(few), 4096, None, None, ws, size, None) == -3
    p = ctypes.c_int64(0)
    assert L.ix_band_attn_lse_pitch(0, ctypes.byref(p)) == -1 and L.ix_band_attn_lse_pitch(129, ctypes.byref(p)) == 0 and p.value == 256


def test_c_gradients_refuse_more_rows_than_a_launch_has():
    L, c = _lib.load(), c_band(batch=1 << 12, Lq=65535 * 64)
    assert L.ix_band_attn_bwd(ctypes.byref(c), 4096, 4096, 4096, 4096, 1280, 256, 64, 4096, 4096, 4096, 4096, 1 << 62, None) == -1
    assert b"too many rows" in L.ix_last_error()
