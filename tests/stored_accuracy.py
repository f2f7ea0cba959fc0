"""What the errors of the products with packed weights may be in size, not at worst: limits that do not grow with the length
of a row, so that a lost chunk of columns, a lost part or a truncated sum shows at every size."""

import ctypes as C

import torch

from hi2_b200 import _lib, linear
from tests.stored_helpers import half_step

# rows, columns, tokens: enough of each kernel and split for every type
SIZES = [(33, 64, 2), (128, 128, 1), (257, 1088, 16), (1000, 4096, 4), (700, 9024, 16), (96, 34816, 2), (64, 65536, 8), (4096, 4096, 1),
         (500, 4224, 40), (96, 4160, 600), (640, 4096, 90), (1000, 8192, 200), (130, 16448, 300), (4096, 11008, 32), (2000, 8192, 60),
         (300, 64, 5003), (257, 1088, 2600), (2000, 4096, 3001), (11008, 4096, 600), (11008, 4096, 1500)]
NUMBER = {torch.float32: _lib.F32, torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}


def form_of(rows, k, tokens, dtype):
    """Which form a product takes, from its workspace: none (tiles of few rows); the prepared activations (whole columns); and
    the sums of slices behind them."""
    w = linear._Struct(256, 256, 256, 256, None, 256, 1, rows, -(-rows // 128) * 4, k)
    need = _lib.load().hi2_stored_linear_workspace_bytes(C.byref(w), NUMBER[dtype], tokens)
    prepared = tokens * k * 2 * (1 if dtype == torch.bfloat16 else 2) + tokens * 4
    return "few" if need == 0 else "whole" if need < prepared + 1024 else "sliced"


def linear_limits(dtype):
    """``(norm, bias)`` of a product's error relative to ``y``, besides the result's own rounding.

    fp32: an activation is off by 2^-23.2 (root mean square: two fp16 parts 2^-24.5, division 2^-24.3, four additions of a
    rotation 2^-23.8), the fp32 additions of n sums of 128 columns by 0.6 sqrt(n) 2^-24.8 (n = 128: 2^-22), and a sum of 128
    columns is truncated at 16 steps, 2^-23.2 together and towards zero: 2^-21.4, here with a factor of 2.6.  Columns of a
    whole row truncated at every step take off 1e-9 a column (2e-6 at 2048).
    fp16 results: the same parts, whole rows truncated, up to 16384 columns.  bf16: one part, 2^-12.3 an activation."""
    if dtype == torch.float32:
        return 2.0**-20, 2.0**-21
    if dtype == torch.float16:
        return 2.0**-15, 2.0**-15
    return 2.0**-11, 2.0**-12


def check_product(got, want, size, dtype):
    """``size``: the root of the sum of the squares of an element's terms.  An element's error is a sum of many small
    ones that go by it: eight times their root mean square at most."""
    norm, bias = linear_limits(dtype)
    off = got.double() - want
    total, own = want.norm(), half_step(dtype)
    assert off.norm() <= (norm + own) * total, f"norm of the error {(off.norm() / total).item():.3g}"
    # rounding the results is not biased: over n of them what is left of it goes with sqrt(n)
    slope = ((off * want).sum() / total**2).abs()
    assert slope <= bias + 4 * own / want.numel() ** 0.5, f"errors along the result {slope.item():.3g}"
    each = 8 * norm * size + own * (want.abs() + 8 * norm * size) + 2.0**-24 * (dtype == torch.float16)
    assert bool((off.abs() <= each).all()), f"an element at {(off.abs() / each).max().item():.3g} of its limit"
