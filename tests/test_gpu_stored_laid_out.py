"""What a laid-out weight keeps, and what it shares with nobody."""

import dataclasses

import pytest
import torch

from hi2_b200 import _lib, linear, moe, stack
from tests.stored_helpers import packed

pytestmark = pytest.mark.gpu
DEV = "cuda"
FIELDS = ("codes", "code_off", "blk_params", "param_off", "row_consts", "row_nbits", "row_block", "had", "col_scale")


def _overwrite(t):
    t.copy_(torch.where(t == 0, torch.ones_like(t), torch.zeros_like(t)))


def test_a_laid_out_tensor_keeps_nothing_of_its_source():
    t = packed(150, 192, 3)
    t = dataclasses.replace(t, **{f: getattr(t, f).to(DEV) for f in FIELDS})
    w = linear.lay_out(t)
    x = torch.randn(5, 192, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV)
    want = linear.stored_linear(x, w)
    for f in FIELDS:
        _overwrite(getattr(t, f))
        assert torch.equal(linear.stored_linear(x, w), want), f


def test_a_laid_out_stack_keeps_nothing_of_its_source():
    def part(like, rows, k, seed):
        t = packed(rows, k, seed)
        if like is not None:
            t.had, t.col_scale = like.had, like.col_scale
        return t

    gates = [part(None, 64, 128, e) for e in range(3)]
    arrays = (stack.build_stack([[g, part(g, 64, 128, 10 + e)] for e, g in enumerate(gates)]),
              stack.build_stack([[part(None, 128, 64, 20 + e)] for e in range(3)]))
    arrays = [{name: t.to(DEV) for name, t in a.items()} for a in arrays]
    gu, dn = linear.lay_out_stack(arrays[0], 2), linear.lay_out_stack(arrays[1], 1)
    g = torch.Generator(device=DEV).manual_seed(2)
    x, index = torch.randn(7, 128, generator=g, device=DEV), torch.randint(0, 3, (7, 2), generator=g, device=DEV)
    weight = torch.rand(7, 2, generator=g, device=DEV)
    want = moe.stored_experts(x, index, weight, gu, dn)
    for a in arrays:
        for name, t in a.items():
            _overwrite(t)
            assert torch.equal(moe.stored_experts(x, index, weight, gu, dn), want), name


def test_memory_of_a_weight_in_use_on_another_stream():
    w = linear.lay_out(packed(4096, 1024, 5, [(8, 16)]), DEV)
    x = torch.randn(4, 1024, generator=torch.Generator(device=DEV).manual_seed(3), device=DEV)
    want = linear.stored_linear(x, w)
    torch.cuda.synchronize()
    tensors = [t for t in w._tensors.values() if t is not None]
    ranges = [(t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()) for t in tensors]
    del tensors
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(400_000_000)  # some 0.2 s
        y = linear.stored_linear(x, w)
    w.record_stream(side)
    del w
    try:
        new = [torch.empty(hi - lo, dtype=torch.uint8, device=DEV) for lo, hi in ranges for _ in range(3)]
        waiting = not side.query()
    finally:
        side.synchronize()  # before anything else is allocated: a product must not meet tables that somebody wrote over
    assert waiting
    for t in new:  # nothing of it was handed out while the call waited
        for lo, hi in ranges:
            assert t.data_ptr() >= hi or t.data_ptr() + t.numel() <= lo
    assert torch.equal(y, want)


def test_check_reports_a_wait_that_ran_out():
    """The status word as a kernel raises it, set from the host: nothing on the device has to wait for it."""
    gu = linear.lay_out_stack(stack.build_stack([[packed(64, 64, e), packed(64, 64, e)] for e in range(2)]), 2, DEV)
    for w in (linear.lay_out(packed(70, 64, 1), DEV), gu):
        w.check()
        w._status.fill_(_lib.ERR_TIMEOUT)
        for _ in range(2):  # nothing clears it
            with pytest.raises(RuntimeError, match="ran out"):
                w.check()


def test_check_waits_for_every_stream():
    w = linear.lay_out(packed(70, 64, 1), DEV)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(400_000_000)  # some 0.2 s
        w._status.fill_(_lib.ERR_TIMEOUT)
    try:
        with pytest.raises(RuntimeError, match="ran out"):
            w.check()
    finally:
        side.synchronize()
