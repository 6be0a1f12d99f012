"""Gradients of band attention where only the blocks with first keys are cut into pieces (the others write dk and dv directly)."""
import pytest
import torch

from tests import band_bounds as bounds
from tests.test_band_weights_gpu import BF16, FP16, FP32, inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B, dtype", [(4, BF16), (4, FP16), (4, FP32), (5, BF16), (5, FP16)])   # blocks of 64 rows, of 128
def test_pieces_of_the_first_keys_alone(B, dtype):
    q, k, v, do = inputs(B, 1100, 1100, 8, 8, 32, dtype, seed=B)
    bounds.check(q, k, v, do, window=30, sinks=5, floor=2.0 ** -32 if dtype is FP16 else 0.0)
