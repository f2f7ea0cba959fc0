"""Dispatch of many (token, slot) pairs and many experts: passes of the counting loop, sums over many warps of experts,
experts without pairs and experts with nearly all of them."""

from types import SimpleNamespace

import pytest
import torch

from hi2_b200 import linear, moe
from hi2_b200.format import dequantize_stored
from tests.stored_helpers import DTYPES, experts64, packed, within

pytestmark = pytest.mark.gpu
DEV = "cuda"
HIDDEN = INNER = 64


def _stack(experts, rows, k, parts, seed):
    """A stack cut out of one packed tensor, with a transform for every expert."""
    t = packed(experts * rows, k, seed)
    g = torch.Generator().manual_seed(seed)
    arrays = {f: getattr(t, f) for f in ("codes", "code_off", "blk_params", "param_off", "row_consts", "row_nbits", "row_block")}
    arrays["had"] = (torch.rand(experts, k // 16, generator=g) < 0.7).to(torch.uint8)
    arrays["col_scale"] = torch.exp(0.5 * torch.randn(experts, k, generator=g)).half()
    arrays["part_off"] = rows // parts * torch.arange(parts * experts + 1, dtype=torch.int32)
    values = dequantize_stored(t, DEV).view(experts, rows, k)
    had, scale = arrays["had"].to(DEV), arrays["col_scale"].to(DEV)
    return linear.lay_out_stack(arrays, parts, DEV), [(SimpleNamespace(had=had[e], col_scale=scale[e]), values[e]) for e in range(experts)]


def _choice(kind, tokens, experts, top_k, g):
    if kind == "spread":
        return torch.stack([torch.randperm(experts, generator=g, device=DEV)[:top_k] for _ in range(tokens)])
    index = torch.randint(0, experts, (tokens, top_k), generator=g, device=DEV)
    if kind == "one":  # nearly everybody takes the last expert
        index[torch.rand(index.shape, generator=g, device=DEV) < 0.95] = experts - 1
    else:  # few experts with pairs, and most slots without one
        index = index // 97 * 97
        index[torch.rand(index.shape, generator=g, device=DEV) < 0.8] = -1
    return index


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("experts,top_k,tokens,kind", [(64, 8, 1024, "spread"), (64, 8, 1025, "spread"), (64, 8, 2500, "spread"), (200, 8, 300, "spread"),
                                                       (1024, 8, 64, "spread"), (1024, 8, 3000, "spread"), (1024, 1, 1, "spread"),
                                                       (64, 2, 10000, "one"), (1000, 4, 3000, "one"), (1024, 8, 5000, "holes"), (33, 8, 700, "holes")])
def test_many_pairs_and_many_experts(experts, top_k, tokens, kind, dtype):
    dt = DTYPES[dtype]
    gu, gate_up = _stack(experts, 2 * INNER, HIDDEN, 2, 7)
    dn, down = _stack(experts, HIDDEN, INNER, 1, 8)
    g = torch.Generator(device=DEV).manual_seed(tokens)
    index = _choice(kind, tokens, experts, top_k, g)
    weight = torch.rand(index.shape, generator=g, device=DEV)
    x = torch.randn(tokens, HIDDEN, generator=g, device=DEV).to(dt)
    y = moe.stored_experts(x, index, weight, gu, dn)
    want, bound = experts64(x, index, weight, gate_up, down, dt)
    within(y, want, bound)
    if dt == torch.float32:
        assert (y - want).norm() < 2.0**-19 * want.norm()
    assert torch.equal(y, moe.stored_experts(x, index, weight, gu, dn))
    gu.check(), dn.check()


@pytest.mark.parametrize("tokens", [3, 40, 700])
@pytest.mark.parametrize("before", ["copy", "fill", "join", "nothing"])
def test_first_calls_of_a_graph(before, tokens):
    """A captured call behind a copy from the host, a fill, a kernel on each of two streams, or as the graph's root; with a
    call on another stream beside it."""
    gu, _ = _stack(4, 2 * INNER, HIDDEN, 2, 9)
    dn, _ = _stack(4, HIDDEN, INNER, 1, 10)
    w = linear.lay_out(packed(HIDDEN, HIDDEN, 11), DEV)
    g = torch.Generator(device=DEV).manual_seed(tokens)
    index = torch.randint(0, 4, (tokens, 2), generator=g, device=DEV)
    weight = torch.rand(tokens, 2, generator=g, device=DEV)
    host = torch.randn(tokens, HIDDEN, generator=torch.Generator().manual_seed(tokens)).bfloat16().pin_memory()
    x, residual = host.to(DEV), torch.zeros(tokens, HIDDEN, dtype=torch.bfloat16, device=DEV)
    linear.stored_linear(x, w, residual=residual), moe.stored_experts(x, index, weight, gu, dn)
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph):
        here = torch.cuda.current_stream()
        if before == "copy":
            x.copy_(host, non_blocking=True)
        elif before == "fill":
            residual.zero_()
        elif before == "join":
            side.wait_stream(here)
            with torch.cuda.stream(side):
                residual.add_(1)
            x.mul_(1)
            here.wait_stream(side)
        y = linear.stored_linear(x, w, residual=residual)
        side.wait_stream(here)
        with torch.cuda.stream(side):
            beside = linear.stored_linear(x, w)
        z = moe.stored_experts(x, index, weight, gu, dn)
        here.wait_stream(side)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, linear.stored_linear(x, w, residual=residual)) and torch.equal(beside, linear.stored_linear(x, w))
    assert torch.equal(z, moe.stored_experts(x, index, weight, gu, dn))


def test_offsets_beyond_32_bits():
    """More than 2^31 results, and more than 2^31 intermediate values of the routed experts."""
    g = torch.Generator(device=DEV).manual_seed(0)
    w = linear.lay_out(packed(28672, 64, 12), DEV)
    x = torch.randn(80000, 64, generator=g, device=DEV).bfloat16()
    y = linear.stored_linear(x, w)
    assert y.numel() > 2**31
    for rows in (slice(0, 3001), slice(74000, 77001), slice(76999, 80000)):
        assert torch.equal(y[rows], linear.stored_linear(x[rows], w))
    del y
    inner, tokens = 512, 270_000
    gu, _ = _stack(4, 2 * inner, HIDDEN, 2, 13)
    dn, _ = _stack(4, HIDDEN, inner, 1, 14)
    index = torch.randint(0, 4, (tokens, 8), generator=g, device=DEV)
    weight = torch.rand(tokens, 8, generator=g, device=DEV)
    assert tokens * 8 * 2 * inner > 2**31
    x = torch.randn(tokens, HIDDEN, generator=g, device=DEV).bfloat16()
    y = moe.stored_experts(x, index, weight, gu, dn)
    for rows in (slice(0, 5000), slice(131_072, 136_000), slice(265_000, 270_000)):
        assert torch.equal(y[rows], moe.stored_experts(x[rows], index[rows], weight[rows], gu, dn))
