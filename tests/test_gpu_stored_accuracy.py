"""How exact the products with packed weights are, in norm: the elementwise bounds of the other tests grow with the
length of a row, and what a row's error norm is does not."""

import pytest
import torch

from hi2_b200 import linear, moe
from hi2_b200.format import dequantize_stored
from tests.stored_accuracy import SIZES, check_product
from tests.stored_helpers import DTYPES, act64, packed, turned
from tests.test_gpu_stored import _stacks, _x

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


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("rows,k,tokens", SIZES)
def test_linear_errors_in_size(rows, k, tokens, dtype):
    dt = DTYPES[dtype]
    t = packed(rows, k, rows + tokens)
    w = linear.lay_out(t, DEV)
    x = _x(tokens, k, dt, 3, 0.5)
    z, v = turned(x.double(), t), dequantize_stored(t, DEV)
    want, size = z @ v.T, ((z * z) @ (v * v).T).sqrt()
    del z, v
    check_product(linear.stored_linear(x, w), want, size, dt)


@pytest.mark.parametrize("tokens", [3, 40, 1500])
def test_fp32_experts_errors_in_size(tokens):
    """Two products, each with the errors of a linear one (2^-22), the first one's twice in act(gate) * up: 1.8 * 2^-22 in norm and
    3.1 * 2^-23.2 along the result, with a factor of four and of three."""
    gu, dn, gate_up, down = _stacks(4, 2048, 1024, 60)
    g = torch.Generator(device=DEV).manual_seed(tokens)
    index = torch.rand(tokens, 4, generator=g, device=DEV).argsort(1)[:, :2].contiguous()
    weight = torch.rand(tokens, 2, generator=g, device=DEV)
    x = _x(tokens, 2048, torch.float32, 5, 0.5)
    want = torch.zeros(tokens, 2048, dtype=torch.float64, device=DEV)
    for e, ((tu, vu), (td, vd)) in enumerate(zip(gate_up, down)):
        token, slot = (index == e).nonzero(as_tuple=True)
        z = turned(x[token].double(), tu) @ vu.T
        y = turned(act64(z[:, :1024], "silu") * z[:, 1024:], td) @ vd.T
        want.index_add_(0, token, y * weight[token, slot, None].double())
    off = moe.stored_experts(x, index, weight, gu, dn).double() - want
    assert off.norm() / want.norm() < 2.0**-19
    assert ((off * want).sum() / want.norm() ** 2).abs() < 2.0**-20
