"""Argument checks and buffers that the products with packed weights and the routing share."""

from __future__ import annotations

import torch
from torch.autograd import forward_ad

from . import _lib

ACTIVATIONS = {None: 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}
DTYPES = {torch.float32: _lib.F32, torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}


def activation_number(name) -> int:
    try:
        return ACTIVATIONS[name]
    except (KeyError, TypeError):
        raise ValueError(f"activation {name!r} is not one of {', '.join(map(str, ACTIVATIONS))}") from None


def no_gradient(what: str, *tensors) -> None:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise ValueError(f"{what}: there is no gradient; call it under torch.no_grad()")
    if forward_ad._current_level >= 0:  # inside a dual level, which no_grad() does not end
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise ValueError(f"{what}: there is no derivative; give it the primal of a dual tensor")


def on_device(what: str, dev: torch.device, *tensors) -> None:
    for t in tensors:
        if t is not None and t.device != dev:
            if not t.is_cuda:
                raise RuntimeError(f"hi2_b200 runs on CUDA devices only (got a tensor on {t.device}); there is no CPU path")
            raise RuntimeError(f"{what}: tensors on different devices: {t.device} and {dev}")


def rows_of(x: torch.Tensor, k: int, what: str):
    """``(x as [tokens, k] with unit column stride, its row stride, its dtype's number)``; a copy only where the strides
    ask for one."""
    dtype = DTYPES.get(x.dtype)
    if dtype is None:
        raise ValueError(f"{what}: unsupported dtype {x.dtype}")
    if x.dim() != 2 or x.shape[1] != k:
        if x.dim() < 1 or x.shape[-1] != k:
            raise ValueError(f"{what}: the last dimension must be {k}, got shape {tuple(x.shape)}")
        x = x.reshape(-1, k)
    ld, unit = x.stride()
    return (x, ld, dtype) if unit == 1 else (x.contiguous(), k, dtype)


def output_rows(out, shape, like: torch.Tensor, what: str):
    """The caller's ``out`` as rows ``[tokens, n]``."""
    if out.shape != shape or out.dtype != like.dtype:
        raise ValueError(f"{what}: out must have shape {tuple(shape)} and the dtype of the activations")
    if out.numel() and out.stride(-1) != 1 and out.shape[-1] != 1:
        raise ValueError(f"{what}: out must have unit column stride")
    try:
        rows = out.view(-1, shape[-1])
    except RuntimeError:
        raise ValueError(f"{what}: the rows of out must lie at one stride") from None
    if rows.shape[0] > 1 and rows.stride(0) < shape[-1]:
        raise ValueError(f"{what}: the rows of out overlap")
    return rows


def apart(what: str, name: str, t, out) -> None:
    """Refuse an ``out`` whose rows share memory with those of the operand ``t`` (``[tokens, n]`` or ``[n]``, unit column stride)."""
    size, o_size = t.element_size(), out.element_size()
    a, o = t.data_ptr(), out.data_ptr()
    rows = t if t.dim() == 2 else t[None]
    if not rows.numel() or not out.numel():
        return
    step, o_step = rows.stride(0) * size, out.stride(0) * o_size
    width, o_width = rows.shape[1] * size, out.shape[1] * o_size
    if a + (rows.shape[0] - 1) * step + width <= o or o + (out.shape[0] - 1) * o_step + o_width <= a:
        return
    if rows.shape[0] > 1 and out.shape[0] > 1 and step == o_step:  # columns of one buffer
        off = (o - a) % step
        if off >= width and off + o_width <= step:
            return
    raise ValueError(f"{what}: out shares memory with {name}")


def workspace(need: int, dev: torch.device):
    """``(tensor, address)``: fresh for every call, so that calls on several streams or in several graphs share nothing."""
    if need == 0:
        return None, None
    t = torch.empty(need, dtype=torch.uint8, device=dev)
    return t, t.data_ptr()
