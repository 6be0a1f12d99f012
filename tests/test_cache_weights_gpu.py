"""The softmax weights of attention over a paged cache in their product with the values."""
import numpy as np
import pytest
import torch

from tests import sequence_reference as ref
from tests.test_cache_gpu import FP16, make, query

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("n", [40, 700, 5000])   # (one piece and several)
@pytest.mark.parametrize("lead", [0.0, 12.0, 17.0, 24.0])
def test_small_weights_in_fp16(hd, n, lead):
    """the first token stands `lead` above the others and its value is zero: the output is made of the small weights alone.  A weight carries 2 h^2
    of itself (two terms) and 2^-25, half of the type's smallest step, where the row's largest is 2^15: 2^-40 of that"""
    from interactron_amd import hipops
    cache, q = make([n, n // 2], kv=2, hd=hd, dtype=FP16, seed=n), query(make([1, 1], hd=hd, dtype=FP16), 4, scale=0.5)
    q[..., 0] = 4.0
    cache.k[..., 0] = 0.0
    first = cache.table[:, 0].long()
    cache.k[first, :, 0] = 0.0
    cache.k[first, :, 0, 0] = lead * hd ** 0.5 / 4
    cache.v.mul_(1e4)
    cache.v[first, :, 0] = 0.0
    got = ref.f64(hipops.cache_attention(q, cache))
    assert np.isfinite(got).all()
    pool, qq = ref.Pool(cache), ref.f64(q)
    for b in range(2):
        m = int(cache.lens[b])
        for h in range(4):
            (k, _), (v, _) = (pool.rows(x, b, h // 2, m) for x in "kv")
            z = (k @ qq[b, h]) * hd ** -0.5
            p = np.exp(z - z.max())
            p /= p.sum()
            worst = (np.abs(k) @ np.abs(qq[b, h])).max() * hd ** -0.5
            rel = 2 * (hd + 8) * ref.U * worst + (m / 64 + 64) * ref.U + 2.0 ** -21
            want, err = p @ v, (p * rel + 2.0 ** -40) @ np.abs(v)
            off, tol = np.abs(got[b, h] - want), err + 2.0 ** -11 * (np.abs(want) + err) + 2.0 ** -25
            assert (off <= tol).all(), (b, h, float((off / tol).max()))
