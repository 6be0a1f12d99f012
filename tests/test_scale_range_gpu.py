"""The largest scales that are taken: scores of zero stay zero."""
import pytest
import torch

from interactron_amd import hipops
from tests.test_cache_gpu import make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("scale", [2.34e38, -2.34e38])
def test_scores_of_zero(dtype, scale):
    q = torch.zeros(2, 50, 2, 64, device="cuda", dtype=dtype, requires_grad=True)
    k, v = (torch.randn(2, 50, 2, 64, device="cuda").to(dtype) for _ in range(2))
    out = hipops.band_attention(q, k, v, causal=False, scale=scale)
    assert torch.allclose(out.float(), v.float().mean(1, keepdim=True).expand_as(out), atol=1e-2)
    cache = make([50, 700], dtype=dtype)
    got = hipops.cache_attention(torch.zeros(2, 2, 64, device="cuda", dtype=dtype), cache, scale=scale)
    assert torch.isfinite(got).all()
    assert torch.equal(got, hipops.cache_attention(torch.zeros(2, 2, 64, device="cuda", dtype=dtype), cache, scale=1.0))
    with pytest.raises(ValueError, match="scale"):
        hipops.cache_attention(torch.zeros(2, 2, 64, device="cuda", dtype=dtype), cache, scale=2.36e38)
