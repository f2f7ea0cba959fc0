"""No GPU needed: what the kernels of the products with packed weights are launched with, and what the calls refuse."""

import ctypes as C

import pytest
import torch
from torch.autograd import forward_ad

from hi2_b200 import _lib, moe
from hi2_b200._args import no_gradient
from tests.stored_accuracy import SIZES, check_product, form_of
from tests.stored_helpers import DTYPES, packed, turned


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


@pytest.mark.parametrize("rows,k,tokens", [(64, 65536, 8), (96, 34816, 2), (200, 1024, 33), (96, 4160, 70)])
def test_error_limits_reject_what_is_lost(rows, k, tokens):
    """The limits that the products are held to on the device, met by a rounded result and not by one with a defect."""
    t = packed(rows, k, rows + tokens)
    g = torch.Generator().manual_seed(tokens)
    v = 0.05 * torch.randn(rows, k, generator=g, dtype=torch.float64)
    x = turned(torch.randn(tokens, k, generator=g).double() * torch.exp(0.5 * torch.randn(k, generator=g)), t)
    want, size = x @ v.T, ((x * x) @ (v * v).T).sqrt()
    for dtype in DTYPES.values():
        check_product(want.to(dtype), want, size, dtype)
        without = x.clone()
        without[:, -64:] = 0  # a chunk of columns
        with pytest.raises(AssertionError):
            check_product((without @ v.T).to(dtype), want, size, dtype)
        with pytest.raises(AssertionError):
            check_product(torch.zeros_like(want).to(dtype), want, size, dtype)
    one_part = x.half().double()
    check_product((one_part @ v.T).bfloat16(), want, size, torch.bfloat16)
    with pytest.raises(AssertionError):
        check_product((one_part @ v.T).float(), want, size, torch.float32)
    with pytest.raises(AssertionError):  # truncated towards zero all along 2048 columns
        check_product((want * (1 - 2e-6)).float(), want, size, torch.float32)


@pytest.mark.parametrize("dtype", sorted(DTYPES))
def test_sizes_cover_every_form(dtype):
    forms = [(form_of(*size, DTYPES[dtype]), size[1]) for size in SIZES]
    for form in ("few", "sliced", "whole"):
        assert sum(f == form and k >= 4096 for f, k in forms) >= 2, (form, forms)


class _Fused(torch.nn.Module):
    def __init__(self, experts, hidden, inner):
        super().__init__()
        g = torch.Generator().manual_seed(0)
        self.gate_up_proj = torch.nn.Parameter(torch.randn(experts, 2 * inner, hidden, generator=g))
        self.down_proj = torch.nn.Parameter(torch.randn(experts, hidden, inner, generator=g))
        self.act_fn = torch.nn.SiLU()


@pytest.mark.parametrize("unused", [[], [3], [0, 1, 2, 3], list(range(10))])
def test_expert_views_pass_over_unused_slots(unused):
    """Routing leaves -1 in slots that no expert is open for; the experts over unpacked weights take its outputs too."""
    fused, g = _Fused(3, 6, 4), torch.Generator().manual_seed(1)
    x, weight = torch.randn(5, 6, generator=g), torch.rand(5, 2, generator=g)
    index = torch.randint(0, 3, (5, 2), generator=g)
    index.view(-1)[unused] = -1
    index[4, 1] = 3 if unused else index[4, 1]  # behind the last expert
    want = torch.zeros(5, 6, dtype=torch.float64)
    for t, j in ((t, j) for t in range(5) for j in range(2)):
        e = int(index[t, j])
        if 0 <= e < 3:
            z = fused.gate_up_proj[e].double() @ x[t].double()
            want[t] += weight[t, j].double() * (fused.down_proj[e].double() @ (fused.act_fn(z[:4]) * z[4:]))
    with torch.no_grad():
        y = moe.ExpertViews(fused)(x, index, weight)
    assert (y - want).abs().max() <= 2.0**-20 * max(want.abs().max().item(), 1.0) * 8  # fp32 sums of 6, 4 and 2 terms
