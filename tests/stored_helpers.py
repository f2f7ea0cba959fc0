"""Random packed tensors and the 64-bit forms of the products with them, with the error bounds that follow
from the number formats."""

import torch

from hi2_b200.format import HI2Tensor, hadamard16

FORMATS = [(2, 16), (2, 32), (2, 64), (4, 16), (4, 32), (4, 64), (8, 16), (8, 32), (8, 64)]
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def packed(rows, k, seed, formats=None, scaled=True, flags=0.7):
    """A packed tensor (host buffers, as an encode leaves them) with a random format per row."""
    g = torch.Generator().manual_seed(seed)
    formats = torch.tensor(formats or FORMATS)
    pick = torch.randint(len(formats), (rows,), generator=g)
    nbits, block = formats[pick, 0], formats[pick, 1]
    zero = torch.zeros(1, dtype=torch.int64)
    code_off = torch.cat([zero, torch.cumsum(k * nbits // 32, 0)])
    param_off = torch.cat([zero, torch.cumsum(k // block, 0)])
    reach = 0.05 * torch.exp(0.5 * torch.randn(rows, generator=g))
    consts = torch.stack([-1.3 * reach, reach / 255, 2.2 * reach / (2.0**nbits - 1) / 200], 1).half()
    return HI2Tensor(
        codes=torch.randint(-(2**31), 2**31, (int(code_off[-1]),), generator=g).to(torch.int32),
        code_off=code_off.to(torch.int32), blk_params=torch.randint(0, 256, (2 * int(param_off[-1]),), generator=g).to(torch.uint8),
        param_off=param_off.to(torch.int32), row_consts=consts, row_nbits=nbits.to(torch.uint8), row_block=block.to(torch.uint8),
        had=(torch.rand(k // 16, generator=g) < flags).to(torch.uint8), shape=(rows, k),
        col_scale=torch.exp(0.5 * torch.randn(k, generator=g)).half() if scaled else None)


def turned(x, t, magnitude=False):
    """fp64 activations in the stored basis; ``magnitude``: with every term of a rotation counted positive."""
    if t.col_scale is not None:
        x = x / t.col_scale.to(x.device, torch.float64)
    h = hadamard16(device=x.device)
    y = x.reshape(*x.shape[:-1], -1, 16)
    flag = t.had.to(x.device).bool()[:, None]
    return torch.where(flag, y @ (h.abs() if magnitude else h), y).reshape(x.shape)


def act64(v, name):
    if name == "relu":
        return v.clamp_min(0)
    if name == "silu":
        return v * torch.sigmoid(v)
    if name == "gelu":
        return 0.5 * v * torch.erfc(-v * 0.5**0.5)
    if name == "gelu_tanh":
        return torch.nn.functional.gelu(v, approximate="tanh")
    return v


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def product_bound(x, x_err, t, v, dtype):
    """``(x' V^T, its error bound)`` in fp64 for activations ``x`` known to ``x_err``: the rotation's fp32 steps
    (division, four additions, a multiplication by 1/4), the rounding of x' (one fp16 part for bf16, else two:
    the second is rounded relative to what the first left, and both are fp16 numbers down to 2^-24 of a row whose largest
    value is at least 2^14), and an fp32 sum of ``k`` exact products, each step truncated (2^-23)."""
    k = x.shape[-1]
    xt, big = turned(x, t), turned(x.abs(), t, True)
    part = 2.0**-11 if dtype == torch.bfloat16 else 2.0**-22
    top = xt.abs().amax(-1, keepdim=True)
    err = turned(x_err, t, True) + 8 * 2.0**-24 * big + part * (xt.abs() + 8 * 2.0**-24 * big) + 2.0**-39 * top
    parts = 1 if dtype == torch.bfloat16 else 2
    size = xt.abs() @ v.abs().T
    return xt @ v.T, err @ v.abs().T + parts * (k + 64) * 2.0**-23 * (size + err @ v.abs().T)


def linear64(x, t, v, bias, activation, residual, dtype):
    """``(y, bound)`` of the stored product with its epilogue; ``v`` is the fp64 reconstruction."""
    y, err = product_bound(x.double(), torch.zeros_like(x, dtype=torch.float64), t, v, dtype)
    if bias is not None:
        y = y + bias.double()
        err = err + 2.0**-24 * y.abs()
    z = act64(y, activation)
    if activation in ("silu", "gelu", "gelu_tanh"):  # slope below 1.13, and some steps of fp32
        err = 1.13 * err + 2.0**-20 * (z.abs() + 2.0**-20)
        if activation == "gelu_tanh":  # the cubic argument of the exponential, relative to its size
            err = err + 2.0**-20 * y.abs() * (1 + y.abs()).clamp_max(12)
    if residual is not None:
        z = z + residual.double()
        err = err + 2.0**-24 * z.abs()
    return z, err + half_step(dtype) * (z.abs() + err) + 2.0**-24 * (dtype == torch.float16)


def experts64(x, index, weight, gate_up, down, dtype, activation="silu"):
    """``(y, bound)`` of the routed experts; ``gate_up[e]`` and ``down[e]`` are ``(HI2Tensor with the transform,
    fp64 reconstruction)``."""
    y, err = torch.zeros_like(x, dtype=torch.float64), torch.zeros_like(x, dtype=torch.float64)
    for e, ((tu, vu), (td, vd)) in enumerate(zip(gate_up, down)):
        token, slot = (index == e).nonzero(as_tuple=True)
        if token.numel() == 0:
            continue
        xe = x[token].double()
        z, ze = product_bound(xe, torch.zeros_like(xe), tu, vu, dtype)
        inner = vd.shape[1]
        g, u, ge, ue = z[:, :inner], z[:, inner:], ze[:, :inner], ze[:, inner:]
        a = act64(g, activation)
        ae = 1.13 * ge + 2.0**-20 * (a.abs() + 2.0**-20)
        he = ae * u.abs() + a.abs() * ue + ae * ue + 2.0**-23 * (a * u).abs()
        o, oe = product_bound(a * u, he, td, vd, dtype)
        w = weight[token, slot, None].double()
        y.index_add_(0, token, o * w)
        err.index_add_(0, token, oe * w.abs() + 2.0**-22 * (o * w).abs())
    err = err + index.shape[1] * 2.0**-23 * (y.abs() + err)
    return y, err + half_step(dtype) * (y.abs() + err) + 2.0**-24 * (dtype == torch.float16)


def within(got, want, bound):
    """Whether every element is inside its bound; says how far the worst one is."""
    off = (got.double() - want).abs()
    worst = (off / bound.clamp_min(1e-300)).max().item() if off.numel() else 0.0
    assert bool((off <= bound).all()), f"worst element at {worst:.3g} of its bound"
    return worst
