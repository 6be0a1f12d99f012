"""Band attention where only some inputs need a gradient: the others' are not computed."""
import itertools

import pytest
import torch

from tests.test_band_weights_gpu import BF16, FP16, FP32, inputs

pytestmark = pytest.mark.gpu


def grads(x, do, need, **how):
    from interactron_amd import hipops
    t = [a.detach().requires_grad_(n) for a, n in zip(x, need)]
    out = hipops.band_attention(*t, **how)
    got = iter(torch.autograd.grad(out, [a for a in t if a.requires_grad], do))
    return [next(got) if n else None for n in need]


# nothing cut; both sides cut; first keys' blocks cut alone; blocks of 128 rows
@pytest.mark.parametrize("B, Lq, Lk, H, kv, D, dtype, how", [(2, 90, 130, 4, 2, 64, BF16, dict(window=33, sinks=2)), (1, 700, 900, 4, 1, 128, FP16, {}),
                                                             (4, 1100, 1100, 8, 8, 32, FP32, dict(window=30, sinks=5)), (5, 1100, 1100, 8, 8, 32, BF16, dict(window=30, sinks=5))])
def test_the_same_bits_as_all_three(B, Lq, Lk, H, kv, D, dtype, how):
    *x, do = inputs(B, Lq, Lk, H, kv, D, dtype, seed=D)
    want = grads(x, do, (True, True, True), **how)
    for need in itertools.product((True, False), repeat=3):
        if any(need):
            for a, b in zip(grads(x, do, need, **how), want):
                assert a is None or torch.equal(a, b), need


@pytest.mark.parametrize("need, least", [((True, False, False), 0), ((False, True, False), 2), ((False, False, True), 2)])
def test_memory(need, least):
    """few queries over many keys: dk and dv are 64 MB each"""
    *x, do = inputs(1, 64, 65536, 8, 8, 64, BF16)
    grads(x, do, need)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    grads(x, do, need)
    used = (torch.cuda.max_memory_allocated() - before) >> 26
    assert (used >= least) if least else used == 0
