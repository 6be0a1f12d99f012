"""The softmax weights of band attention in its products with v and do (tests/band_bounds.py)."""
import pytest
import torch

from tests import band_bounds as bounds

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def inputs(B, Lq, Lk, H, kv, D, dtype, seed=0, scale=1.5):
    g = torch.Generator().manual_seed(seed)
    make = lambda L, h, s=1.0: (torch.randn(B, L, h, D, generator=g) * s).to(dtype).cuda()  # noqa: E731
    return make(Lq, H, scale), make(Lk, kv), make(Lk, kv), make(Lq, H)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("Lq, Lk, how", [(200, 200, dict(window=60, sinks=3)), (200, 200, dict(causal=False)), (5, 1500, {}), (700, 700, dict(sinks=70, window=30))],
                         ids=["band", "full", "pieces", "first keys"])
def test_weights_are_as_good_as_32_bit_ones(dtype, D, Lq, Lk, how):
    """out and dv are off by their own rounding and what 32-bit arithmetic leaves, not by a rounding of the weights"""
    # (fp16: steps below 2^-14 are 2^-24, half of one off; a row's largest weight is 1 in the forward pass)
    bounds.check(*inputs(2, Lq, Lk, 4, 2, D, dtype, seed=D), floor=2.0 ** -25 if dtype is FP16 else 0.0, **how)


@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("Lq, Lk, how", [(200, 200, dict(window=60, sinks=3)), (300, 300, dict(window=40, sinks=1)), (7, 2000, dict(window=90, sinks=1))], ids=["band", "first key", "pieces"])
@pytest.mark.parametrize("lead", [0.0, 12.0, 17.0, 24.0])
def test_small_weights_in_fp16(D, Lq, Lk, how, lead):
    """the first key stands `lead` above the others and its value is zero: outputs and dv are made of the small weights alone.  Half the type's
    smallest step, 2^-25, is 2^-32 of the row's largest weight (carried 2^7 times as large, or more), and 2^-35 in dv (2^10 times)"""
    q, k, v, do = inputs(2, Lq, Lk, 4, 2, D, FP16, seed=int(lead), scale=0.5)
    if lead:
        q[..., 0], k[..., 0] = 4.0, 0.0
        k[:, 0] = 0.0
        k[:, 0, :, 0] = lead * D ** 0.5 / 4
        v *= 1e4
        v[:, 0] = 0.0
        do *= 1e4
    bounds.check(q, k, v, None, floor=2.0 ** -32, **how)
    # (gradients: values and do that keep do v within the type's range)
    got = bounds.check(q, k, v * 1e-4, do * 1e-2, floor=2.0 ** -32, floor_dv=2.0 ** -35, **how)
    assert lead == 0 or float(got["dv"][:, 1:].abs().max()) > 0


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("size", [20, 23, 25, 27, 29])
def test_scores_that_a_float32_does_not_hold_exactly(dtype, D, size):
    """exponents of up to 2^size: every query's largest score is millions above the next and its value is the output, though an exponent's own step
    is larger than what a weight can grow by in fp16"""
    from interactron_amd import hipops
    for B, Lq, Lk, H in ((2, 100, 300, 2), (1, 5, 2000, 2), (24, 129, 140, 16)):   # (one piece, several, blocks of 128 rows)
        q, k, v, _ = inputs(B, Lq, Lk, H, H, D, dtype, seed=size, scale=1.0)
        z = torch.einsum("bihd,bjhd->bhij", q.double().cpu(), k.double().cpu())
        scale = 2.0 ** size / float(z.abs().max()) / 1.4427
        best = z.topk(2, -1)
        clear = (best.values[..., 0] - best.values[..., 1]) * scale > max(40.0, 2.0 ** (size - 12))   # (2^-12 of the largest: the score's own error)
        assert clear.double().mean() >= 0.8   # (most rows tell)
        want = torch.gather(v.cpu().permute(0, 2, 1, 3), 2, best.indices[..., :1].expand(-1, -1, -1, D)).permute(0, 2, 1, 3)
        got = hipops.band_attention(q, k, v, causal=False, scale=scale).cpu()
        assert torch.isfinite(got).all()
        clear = clear.permute(0, 2, 1)
        assert torch.allclose(got[clear].float(), want[clear].float(), rtol=2.0 ** -7, atol=1e-6)
