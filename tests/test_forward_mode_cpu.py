"""Inputs that carry a forward-mode derivative are refused, recorded or not: no op here has one."""
import pytest
import torch
import torch.autograd.forward_ad as fwd_ad

from interactron_amd import _lib, hipops
from interactron_amd.hipops.core import Function


def qkv(L=4):
    return [torch.randn(1, L, 2, 64) for _ in range(3)]


@pytest.mark.parametrize("which", [0, 1, 2])
def test_band_attention_without_recording(which):
    x = qkv()
    with fwd_ad.dual_level(), torch.no_grad():
        with pytest.raises(_lib.HipLibraryError, match="GPU"):   # (a dual level alone is nothing)
            hipops.band_attention(*x)
        x[which] = fwd_ad.make_dual(x[which], torch.ones_like(x[which]))
        with pytest.raises(_lib.HipLibraryError, match="forward-mode"):
            hipops.band_attention(*x)


def test_band_attention_recorded():
    x = qkv()
    with fwd_ad.dual_level():
        x[1] = fwd_ad.make_dual(x[1], torch.ones_like(x[1]))
        with pytest.raises((NotImplementedError, _lib.HipLibraryError)):
            hipops.band_attention(*x)


def test_every_function():
    class Twice(Function):
        @staticmethod
        def forward(ctx, x, by):
            return x * by

        @staticmethod
        def backward(ctx, g):
            return g * 2, None

    x = torch.arange(3.0)
    with fwd_ad.dual_level():
        dual = fwd_ad.make_dual(x, torch.ones(3))
        with torch.no_grad():
            assert torch.equal(Twice.call(x, 2), 2 * x)
            with pytest.raises(_lib.HipLibraryError, match="Twice"):
                Twice.call(dual, 2)
        with pytest.raises(NotImplementedError):
            Twice.call(dual, 2)
    with torch.no_grad():
        assert torch.equal(Twice.call(x, 2), 2 * x)
