"""Products of activations with packed weights on the tensor cores (the product of hi2/format.py:242-249
``reference_linear``, for evaluating and serving what was encoded).

A packed tensor (or a stack of routed experts) is laid out once with :func:`lay_out` /
:func:`lay_out_stack`; the layout keeps the packed size but for a few groups (codes and ladder parameters are re-ordered).
:func:`stored_linear` then multiplies activations with the fp16 reconstruction, decoded on the fly, and
applies bias, activation and residual as it stores the sums (behind the sum of the slices, where the columns of a product
are split); :func:`hi2_b200.moe.stored_experts` is the
same for a mixture layer.  bf16 activations are taken to 11 bits in the stored basis, fp16 and fp32 ones to
22; sums are held in fp32.  Inference only: activations that require a gradient are refused.
"""

from __future__ import annotations

import ctypes as C

import torch

from . import _lib
from ._args import ACTIVATIONS, activation_number, apart, no_gradient, on_device, output_rows, rows_of, workspace
from .format import GROUP, HI2Tensor
from .stack import MARK, stack_dims

CHUNK = 64  # columns that a row's codes are dealt out by
FEW_TOKENS = 16  # up to here a product never needs a workspace
_GROUP_ROWS, _TILE_GROUPS = 32, 4


class _Struct(C.Structure):  # hi2_stored_weight
    _fields_ = [("data", C.c_void_p), ("groups", C.c_void_p), ("rows", C.c_void_p), ("had", C.c_void_p),
                ("inv_scale", C.c_void_p), ("status", C.c_void_p), ("experts", C.c_int64), ("rows_per_expert", C.c_int64),
                ("groups_per_expert", C.c_int64), ("k", C.c_int64)]


class StoredWeight:
    """Packed rows laid out for products: ``shape`` is ``(rows, K)``, or ``(experts, rows, K)`` for a stack.
    Made by :func:`lay_out` or :func:`lay_out_stack`; read-only, and usable on any stream of its device.  Its memory
    belongs to the stream that was current then: before the last reference goes while calls on OTHER streams may still
    be queued, :meth:`record_stream` them (as for a tensor) or wait for them.  A captured graph does not keep it alive."""

    def __init__(self, shape, stacked: bool, tensors: dict):
        experts, rows, k = shape
        self.shape = tuple(shape) if stacked else (rows, k)
        self.experts, self.rows, self.k = experts, rows, k
        self.device = tensors["data"].device
        self._tensors = tensors
        self._status = tensors["status"]
        self._struct = _Struct(*(None if tensors[f] is None else tensors[f].data_ptr()
                                 for f in ("data", "groups", "rows", "had", "inv_scale", "status")),
                               experts, rows, tensors["groups"].shape[0] // experts, k)
        self.arg = C.byref(self._struct)

    @property
    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in self._tensors.values() if t is not None)

    def record_stream(self, stream: torch.cuda.Stream) -> None:
        """Keep the memory from being handed out again before what is queued on ``stream`` by the time the weight goes has run."""
        for t in self._tensors.values():
            if t is not None:
                t.record_stream(stream)

    def check(self) -> None:
        """Raise ``RuntimeError`` if a device-side wait of a product with this weight ever ran out (waits
        for the device; products themselves never wait)."""
        torch.cuda.synchronize(self.device)  # calls on every stream
        if int(self._status.item()):
            raise RuntimeError("stored product: a bounded device-side wait ran out; results since then are not valid")


def _lay_out(f: dict, experts: int, rows: int, k: int, stacked: bool, device) -> StoredWeight:
    codes = f["codes"]
    dev = torch.device(device) if device is not None else (
        codes.device if codes.is_cuda else torch.device("cuda", torch.cuda.current_device()))
    if dev.type != "cuda":
        raise RuntimeError("hi2_b200 runs on CUDA devices only; there is no CPU path")
    if dev.index is None:
        dev = torch.device("cuda", torch.cuda.current_device())
    if rows < 1 or k < 1 or k % CHUNK:
        raise ValueError(f"lay_out: K={k} must be a positive multiple of {CHUNK}, with at least one row")
    with torch.cuda.device(dev):
        return _lay_out_on(f, experts, rows, k, stacked, dev)


def _lay_out_on(f: dict, experts: int, rows: int, k: int, stacked: bool, dev: torch.device) -> StoredWeight:
    def up(name, dtype):
        return _lib.upload(f[name], dev, dtype).reshape(-1)

    codes, params = up("codes", torch.int32), up("blk_params", torch.uint8)
    code_off, param_off = up("code_off", torch.int32), up("param_off", torch.int32)
    nbits, block = up("row_nbits", torch.int64), up("row_block", torch.int64)
    consts = _lib.upload(f["row_consts"], dev, torch.float16).reshape(-1, 3)
    had = up("had", torch.uint8).clone()  # (every other field is made anew below)
    total = experts * rows
    for name, t, n in (("row_nbits", nbits, total), ("row_block", block, total), ("row_consts", consts, 3 * total),
                       ("code_off", code_off, total + 1), ("param_off", param_off, total + 1),
                       ("had", had, experts * (k // GROUP))):
        if t.numel() != n:
            raise ValueError(f"lay_out: {name} has {t.numel()} entries, expected {n}")
    scale = None
    if f.get("col_scale") is not None:
        scale = up("col_scale", torch.float32)
        if scale.numel() != experts * k:
            raise ValueError(f"lay_out: col_scale has {scale.numel()} entries, expected {experts * k}")
    # everything the copies rely on, read back once
    known = ((nbits == 2) | (nbits == 4) | (nbits == 8)) & ((block == 16) | (block == 32) | (block == 64))
    co, po = code_off.long(), param_off.long()
    fits = (co[1:] - co[:-1] == k * nbits // 32) & (po[1:] - po[:-1] == k // block.clamp_min(1))
    good = torch.stack([known.all(), fits.all(), (co[0] >= 0) & (co[-1] <= codes.numel()),
                        (po[0] >= 0) & (2 * po[-1] <= params.numel())]).tolist()
    if not good[0]:
        raise ValueError("lay_out: a row's code width or block size is not one of the format's")
    if not all(good[1:]):
        raise ValueError("lay_out: the row offsets do not fit the buffers")

    # Rows by width and falling block, a stable order, cut into groups of 32 and filled up to whole tiles.  A group has
    # the widest codes and the shortest blocks of its rows.
    shift = torch.log2(block.double()).round().long() - 4       # 0, 1, 2
    width = torch.log2(nbits.double()).round().long()           # 1, 2, 3
    order = torch.sort((3 * width - shift).view(experts, rows), dim=1, stable=True).indices
    tile_rows = _GROUP_ROWS * _TILE_GROUPS
    src = torch.full((experts, -(-rows // tile_rows) * tile_rows), -1, dtype=torch.int64, device=dev)
    src[:, :rows] = order + rows * torch.arange(experts, device=dev)[:, None]
    src = src.reshape(-1)
    real, at = src >= 0, src.clamp_min(0)

    def of_groups(t):
        return t.view(-1, _GROUP_ROWS)

    live = of_groups(real)[:, 0]  # the others have padding rows only
    widest = of_groups(torch.where(real, width[at], 0)).amax(1)
    shortest = of_groups(torch.where(real, shift[at], 2)).amin(1)
    # groups whose largest step, times the power of two that their codes are read with, is still an fp16 number
    limit = 65504.0 / 2.0 ** (16 + 2 * widest)[:, None]  # 2^18, 2^20, 2^22
    step = of_groups(255 * consts[:, 2].float()[at])
    small = (((step >= 0) & (step <= limit)) | ~of_groups(real)).all(1).long()
    form = torch.where(live, widest | shortest << 2 | small << 4, 0)
    units = torch.where(live, (16 << widest) + (16 >> shortest), 0)  # of 16 bytes, per chunk
    base = (units * (k // CHUNK)).cumsum(0)
    total_units = int(base[-1].item())
    if total_units >= 2**32:
        raise ValueError("lay_out: more than 64 GiB of packed rows")
    base = base - units * (k // CHUNK)
    half = consts.view(torch.int16).long() & 0xFFFF
    rows_t = torch.stack([torch.where(real, at % rows, 2**32 - 1),
                          (half[:, 0] | half[:, 1] << 16)[at], half[:, 2][at], torch.zeros_like(at)], 1)

    def words(t):  # the low 32 bits
        return torch.where(t >= 2**31, t - 2**32, t).to(torch.int32).contiguous()

    tensors = dict(data=torch.zeros(max(total_units, 1) * 16, dtype=torch.uint8, device=dev),
                   groups=words(torch.stack([base, form], 1)), rows=words(rows_t), had=had,
                   inv_scale=None if scale is None else scale.reciprocal(),
                   status=torch.zeros(1, dtype=torch.int32, device=dev))
    w = StoredWeight((experts, rows, k), stacked, tensors)
    src = src.to(torch.int32)
    _lib.call("hi2_lay_out_rows", w.arg, _lib.ptr(src), _lib.ptr(codes), _lib.ptr(code_off), _lib.ptr(params),
              _lib.ptr(param_off), _lib.ptr(tensors["data"]), _lib.stream(dev))
    torch.cuda.current_stream(dev).synchronize()  # complete for every stream that uses it later
    return w


def lay_out(t: HI2Tensor, device=None) -> StoredWeight:
    """The packed tensor laid out for :func:`stored_linear` on ``device`` (default: where its codes are,
    else the current device).  Waits for the device."""
    fields = {name: getattr(t, name) for name in ("codes", "code_off", "blk_params", "param_off", "row_consts", "row_nbits",
                                                  "row_block", "had", "col_scale")}
    return _lay_out(fields, 1, int(t.shape[0]), int(t.shape[1]), False, device)


def lay_out_stack(arrays: dict, parts: int, device=None) -> StoredWeight:
    """The arrays of :func:`hi2_b200.stack.build_stack` with ``parts`` parts per expert (2: gate and up,
    1: down) laid out for :func:`hi2_b200.moe.stored_experts`.  The parts of all experts must have the same
    number of rows.  Waits for the device."""
    experts, k = stack_dims(arrays, parts)
    ends = arrays[MARK].to("cpu", torch.int64)
    rows = ends[1:] - ends[:-1]
    if experts == 0 or int(ends[0]) != 0 or not bool((rows == rows[0]).all()):
        raise ValueError("lay_out_stack: the parts of the stack differ in their number of rows")
    return _lay_out(arrays, experts, parts * int(rows[0]), k, True, device)


def stored_linear(x: torch.Tensor, w: StoredWeight, bias: torch.Tensor | None = None, activation: str | None = None,
                  residual: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """``activation(x @ W^T + bias) + residual`` with the packed weight ``w`` (``[rows, K]``), as ``[..., rows]`` in
    the dtype of ``x [..., K]`` (bf16, fp16 or fp32, any strides).  ``activation`` is None, ``"relu"``, ``"silu"``,
    ``"gelu"`` or ``"gelu_tanh"``; ``bias [rows]`` and ``residual [..., rows]`` have the dtype of ``x``.
    ``out`` may be given, and may be ``residual`` itself, but share no memory with the other operands.  Queued on the current stream of the weight's device; a token with a
    non-finite activation gets non-finite sums and leaves the others alone."""
    if len(w.shape) != 2:
        raise ValueError("stored_linear: a stack of experts goes through moe.stored_experts")
    act = activation_number(activation)
    rows, ldx, dtype = rows_of(x, w.k, "stored_linear")
    dev = w.device
    on_device("stored_linear", dev, x, bias, residual, out)
    no_gradient("stored_linear", x, bias, residual, out)
    n, tokens = w.rows, rows.shape[0]
    shape = (tokens, n) if x.dim() == 2 else (*x.shape[:-1], n)
    if bias is not None:
        if bias.shape != (n,) or bias.dtype != x.dtype:
            raise ValueError(f"stored_linear: bias must have shape {(n,)} and dtype {x.dtype}")
        bias = bias.contiguous()
    res, res_ptr, ld_res = None, None, 0
    if residual is not None:
        if residual.shape != shape or residual.dtype != x.dtype:
            raise ValueError(f"stored_linear: residual must have shape {shape} and dtype {x.dtype}")
        res = residual if len(shape) == 2 else residual.reshape(-1, n)
        ld_res, unit = res.stride()
        if unit != 1:
            res, ld_res = res.contiguous(), n
        res_ptr = res.data_ptr()
    if out is None:
        out = x.new_empty(shape)
        ld_out = n
    else:
        y = output_rows(out, shape, x, "stored_linear")
        ld_out = y.stride(0)
        apart("stored_linear", "x", rows, y)
        if bias is not None:
            apart("stored_linear", "bias", bias, y)
        if res is not None and (res_ptr != y.data_ptr() or (ld_res != ld_out and tokens > 1)):
            apart("stored_linear", "residual", res, y)
    if tokens == 0:
        return out
    need = 0
    space = at = None
    if tokens > FEW_TOKENS:
        need = _lib.load().hi2_stored_linear_workspace_bytes(w.arg, dtype, tokens)
        space, at = workspace(need, dev)
    _lib.launch("hi2_stored_linear", dev.index, w.arg, rows.data_ptr(), dtype, tokens, ldx,
                None if bias is None else bias.data_ptr(), act, res_ptr, ld_res, out.data_ptr(), ld_out, at, need)
    return out


__all__ = ["ACTIVATIONS", "StoredWeight", "lay_out", "lay_out_stack", "stored_linear"]
