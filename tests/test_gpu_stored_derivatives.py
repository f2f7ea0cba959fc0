"""The calls over packed weights have no derivatives: every operand that carries one is refused, forward mode too."""

import pytest
import torch
from torch.autograd import forward_ad

from hi2_b200 import linear, moe
from tests.stored_helpers import packed
from tests.test_gpu_stored import _stacks

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("grad_mode", [True, False])
def test_dual_operands(grad_mode):
    w = linear.lay_out(packed(64, 128, 2), DEV)
    gu, dn, _, _ = _stacks(2, 128, 64, 30)
    x, bias, residual = torch.zeros(3, 128, device=DEV), torch.zeros(64, device=DEV), torch.zeros(3, 64, device=DEV)
    index, weight = torch.zeros(3, 2, dtype=torch.int64, device=DEV), torch.zeros(3, 2, device=DEV)
    balance = torch.zeros(128, device=DEV)
    calls = {
        "x": lambda v: linear.stored_linear(v(x), w),
        "bias": lambda v: linear.stored_linear(x, w, bias=v(bias)),
        "residual": lambda v: linear.stored_linear(x, w, residual=v(residual)),
        "activations of experts": lambda v: moe.stored_experts(v(x), index, weight, gu, dn),
        "weights of experts": lambda v: moe.stored_experts(x, index, v(weight), gu, dn),
        "logits": lambda v: moe.route(v(x), 2),
        "balance": lambda v: moe.route(x, 2, bias=v(balance)),
    }
    with forward_ad.dual_level(), torch.set_grad_enabled(grad_mode):
        for name, call in calls.items():
            call(lambda t: t)
            call(lambda t: forward_ad.unpack_dual(forward_ad.make_dual(t, torch.ones_like(t))).primal)
            with pytest.raises(ValueError, match="no derivative"):
                call(lambda t: forward_ad.make_dual(t, torch.ones_like(t)))
                pytest.fail(name)
