"""How exact the products with packed weights are, in norm: the elementwise bounds of the other tests grow with the
length of a row, and what a row's error norm is does not."""

import pytest
import torch

from hi2_b200 import linear
from hi2_b200.format import dequantize_stored
from tests.stored_helpers import packed, turned

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _relative(got, want):
    return ((got.double() - want).norm() / want.norm()).item()


@pytest.mark.parametrize("tokens", [4, 600, 3001])
@pytest.mark.parametrize("size", [1.0, 1e-28, 1e-33, 1e-35, 1e-36, 1e-37])
def test_small_fp32_activations_keep_their_bits(tokens, size):
    """Two fp16 parts of a value leave 2^-22 of it, the rotation's steps in fp32 2^-21 at most, sums of up to 128 columns that
    are truncated at 8 steps 8 * 2^-24 of it: together below 2^-20, for any power of two that a row is divided by."""
    t = packed(140, 1024, 3)
    x = size * torch.randn(tokens, 1024, generator=torch.Generator(device=DEV).manual_seed(tokens), device=DEV)
    want = turned(x.double(), t) @ dequantize_stored(t, DEV).T
    assert _relative(linear.stored_linear(x, linear.lay_out(t, DEV)), want) < 2.0**-20
