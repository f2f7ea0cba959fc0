"""No GPU needed: what the kernels of the products with packed weights are launched with, and what the calls refuse."""

import ctypes as C

import pytest
import torch
from torch.autograd import forward_ad

from hi2_b200 import _lib
from hi2_b200._args import no_gradient


@pytest.mark.parametrize("exact,widest", [(False, 192), (True, 128)])
def test_wide_tiles_have_a_width_that_a_pair_multiplies(exact, widest):
    """With the A operand in tensor memory a pair of blocks multiplies 32, 64, .. columns at once, nothing between."""
    wide_width = getattr(_lib.load(), "_ZN3hi26stored10wide_widthElb")
    wide_width.argtypes, wide_width.restype = [C.c_int64, C.c_bool], C.c_int
    for rows in [*range(1, 2000), 4096, 32768, 1 << 20, (1 << 30) - 1]:
        width = wide_width(rows, exact)
        assert width % 32 == 0 and 32 <= width <= widest, (rows, width)
        tiles = -(-rows // width)
        assert tiles == -(-rows // widest)  # as few as there can be
        assert width < -(-rows // tiles) + 32  # and no wider than that asks for


def test_dual_tensors_are_refused():
    x = torch.zeros(3)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones(3))
        no_gradient("op", x, None)
        no_gradient("op", forward_ad.unpack_dual(dual).primal)
        with pytest.raises(ValueError, match="no derivative"):
            no_gradient("op", None, dual)
        with torch.no_grad(), pytest.raises(ValueError, match="no derivative"):
            no_gradient("op", x, dual)
    with pytest.raises(ValueError, match="no derivative"):
        torch.func.jvp(lambda v: no_gradient("op", v), (x,), (torch.ones(3),))
