"""No GPU needed: what the kernels of the products with packed weights are launched with, and what the calls refuse."""

import ctypes as C

import pytest

from hi2_b200 import _lib


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
