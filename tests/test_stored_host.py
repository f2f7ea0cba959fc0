"""No GPU needed: what the products with packed weights and the routing refuse before anything is launched."""

import ctypes as C
import math

import pytest
import torch

from hi2_b200 import _lib, linear, moe
from tests.stored_helpers import packed


def _struct(**kw):
    base = dict(data=256, groups=256, rows=256, had=256, inv_scale=None, status=256, experts=1, rows_per_expert=64,
                groups_per_expert=4, k=128)
    return linear._Struct(*(base | kw).values())


def test_stored_linear_arguments():
    lib = _lib.load()

    def call(s, x=256, dtype=_lib.BF16, tokens=4, act=0, out=256, ws=256, size=1 << 20):
        return lib.hi2_stored_linear(C.byref(s), x, dtype, tokens, 128, None, act, None, 0, out, 64, ws, size, None)

    ok = _struct()
    assert lib.hi2_stored_linear_workspace_bytes(C.byref(ok), _lib.BF16, 4) == 0  # a few rows need none
    assert linear.FEW_TOKENS == 16
    long = _struct(rows_per_expert=1 << 20, groups_per_expert=1 << 15, k=1 << 16)
    for dtype in (_lib.BF16, _lib.F16, _lib.F32):
        assert lib.hi2_stored_linear_workspace_bytes(C.byref(long), dtype, 16) == 0
        assert lib.hi2_stored_linear_workspace_bytes(C.byref(long), dtype, 17) >= 17 * (1 << 16) * 2
    need = lib.hi2_stored_linear_workspace_bytes(C.byref(ok), _lib.BF16, 4000)
    assert need >= 4000 * 128 * 2 + 4000 * 4
    assert lib.hi2_stored_linear_workspace_bytes(C.byref(ok), _lib.F32, 4000) >= 2 * 4000 * 128 * 2
    assert call(ok, tokens=0) == _lib.OK
    for bad in (_struct(k=100), _struct(experts=2), _struct(data=None), _struct(groups_per_expert=3),
                _struct(rows_per_expert=129), _struct(experts=0), _struct(k=0)):
        assert call(bad) == _lib.ERR_ARG
    for kw in (dict(dtype=_lib.F64), dict(act=5), dict(act=-1), dict(tokens=-1), dict(tokens=1 << 31), dict(x=None), dict(out=None)):
        assert call(ok, **kw) == _lib.ERR_ARG
    for kw in (dict(ws=None), dict(size=need - 1), dict(ws=264)):
        assert call(ok, tokens=4000, **kw) == _lib.ERR_WORKSPACE


def test_stored_experts_arguments():
    lib = _lib.load()
    up, down = _struct(experts=4, rows_per_expert=128, groups_per_expert=4, k=128), _struct(experts=4, rows_per_expert=128, k=64)

    def call(a, b, tokens=3, top_k=2, dtype=_lib.F32, act=2, index=256, ws=256, size=1 << 24):
        return lib.hi2_stored_experts(C.byref(a), C.byref(b), 256, dtype, tokens, 128, index, 256, top_k, act, 256, 128, ws, size, None)

    assert call(up, down, tokens=0) == _lib.OK
    for a, b in ((up, _struct(experts=3, rows_per_expert=128, k=64)), (up, _struct(experts=4, rows_per_expert=64, k=64)),
                 (up, _struct(experts=4, rows_per_expert=128, k=128)), (_struct(experts=4, k=100), down)):
        assert call(a, b) == _lib.ERR_ARG
    big = [_struct(experts=1025, rows_per_expert=128, k=128), _struct(experts=1025, rows_per_expert=128, k=64)]
    assert call(*big) == _lib.ERR_ARG
    for kw in (dict(top_k=0), dict(tokens=-1), dict(tokens=1 << 29, top_k=2), dict(dtype=_lib.F64), dict(act=9), dict(index=None)):
        assert call(up, down, **kw) == _lib.ERR_ARG
    need = lib.hi2_stored_experts_workspace_bytes(C.byref(up), _lib.F32, 3, 2)
    assert need > 0
    for kw in (dict(ws=None), dict(size=need - 1), dict(ws=260)):
        assert call(up, down, **kw) == _lib.ERR_WORKSPACE


def test_route_arguments():
    lib = _lib.load()

    def call(dtype=_lib.F32, tokens=4, experts=64, top_k=8, groups=1, top_groups=1, logits=256):
        return lib.hi2_route(logits, dtype, tokens, experts, 64, top_k, 0, None, groups, top_groups, 0, 1.0, 256, 256, None)

    assert call(tokens=0) == _lib.OK
    for kw in (dict(dtype=_lib.F64), dict(experts=0), dict(experts=1025), dict(top_k=0), dict(top_k=33), dict(experts=4, top_k=5),
               dict(groups=0), dict(groups=7), dict(experts=66, groups=33), dict(groups=8, top_groups=9), dict(groups=8, top_groups=0),
               dict(tokens=-1), dict(tokens=1 << 31), dict(logits=None)):
        assert call(**kw) == _lib.ERR_ARG


def test_lay_out_arguments():
    lib = _lib.load()
    assert lib.hi2_lay_out_rows(C.byref(_struct(k=96)), 256, 256, 256, 256, 256, 256, None) == _lib.ERR_ARG
    assert lib.hi2_lay_out_rows(C.byref(_struct()), None, 256, 256, 256, 256, 256, None) == _lib.ERR_ARG
    t = packed(8, 64, 1)
    with pytest.raises(RuntimeError, match="CUDA"):
        linear.lay_out(t, "cpu")
    odd = packed(8, 64, 1)
    odd.shape = (8, 80)
    with pytest.raises((ValueError, RuntimeError)):
        linear.lay_out(odd, "cuda")


def test_cpu_tensors_are_refused():
    with pytest.raises(RuntimeError):
        moe.route(torch.zeros(2, 8), 2)
    with pytest.raises(ValueError):
        moe.route(torch.zeros(2, 8), 2, scores="tanh")
    with pytest.raises(ValueError):
        moe.route(torch.zeros(2, 8, dtype=torch.float64), 2)
    with pytest.raises(ValueError):
        moe.route(torch.full((), math.inf), 1)
