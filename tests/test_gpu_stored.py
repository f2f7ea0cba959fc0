"""Products with packed weights and the routed experts over stacks of them, against the 64-bit
reconstruction (``format.dequantize_stored``) and elementwise bounds from the number formats."""

import threading

import pytest
import torch

from hi2_b200 import _lib, linear, moe, stack
from hi2_b200.format import dequantize_stored, reference_linear
from tests.stored_helpers import DTYPES, FORMATS, experts64, linear64, packed, within

pytestmark = pytest.mark.gpu
DEV = "cuda"
NUMBER = {torch.float32: _lib.F32, torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _x(tokens, k, dtype, seed, spread=1.0):
    g = _gen(seed)
    x = torch.randn(tokens, k, generator=g, device=DEV) * torch.exp(spread * torch.randn(k, generator=g, device=DEV))
    return x.to(dtype)


def _check(t, x, dtype, bias=None, activation=None, residual=None, out=None):
    w = linear.lay_out(t, DEV)
    if x.numel() // x.shape[-1] > 2000:  # sizes that are meant for the wide tiles
        assert _lib.load().hi2_stored_linear_workspace_bytes(w.arg, NUMBER[dtype], x.numel() // x.shape[-1]) > 0
    keep = None if residual is None else residual.clone()
    y = linear.stored_linear(x, w, bias=bias, activation=activation, residual=residual, out=out)
    flat = x.reshape(-1, x.shape[-1])
    want, bound = linear64(flat, t, dequantize_stored(t, DEV), bias, activation,
                           None if keep is None else keep.reshape(-1, keep.shape[-1]), dtype)
    assert y.dtype == dtype and y.shape == (*x.shape[:-1], t.shape[0])
    within(y.reshape(want.shape), want, bound)
    w.check()
    return y


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("rows,k,tokens", [(1, 64, 1), (33, 64, 2), (128, 128, 1), (129, 192, 7), (257, 1088, 16),
                                           (500, 320, 17), (640, 2048, 33), (96, 4160, 70), (1000, 576, 129), (300, 64, 300),
                                           (1, 64, 2501), (33, 64, 2600), (129, 192, 2501), (257, 1088, 701), (257, 1088, 1101),
                                           (500, 320, 2400),
                                           (640, 2048, 333), (96, 4160, 600), (1000, 576, 1300), (300, 64, 5003)])
def test_linear_sizes_and_types(rows, k, tokens, dtype):
    t = packed(rows, k, rows + k)
    _check(t, _x(tokens, k, DTYPES[dtype], tokens), DTYPES[dtype])


@pytest.mark.parametrize("form", FORMATS)
def test_every_row_format_alone(form):
    t = packed(160, 256, 7, [form])
    _check(t, _x(5, 256, torch.float32, 3), torch.float32)
    _check(t, _x(40, 256, torch.bfloat16, 4), torch.bfloat16)
    _check(t, _x(2501, 256, torch.float32, 5), torch.float32)


@pytest.mark.parametrize("activation", [None, "relu", "silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("tokens", [1, 50, 1500, 3001])
def test_epilogue(activation, dtype, tokens):
    dt = DTYPES[dtype]
    t = packed(200, 320, 11)
    bias, residual = _x(1, 200, dt, 1)[0], _x(tokens, 200, dt, 2)
    x = _x(tokens, 320, dt, 5)
    _check(t, x, dt, bias, activation, residual)
    _check(t, x, dt, bias, activation, None)
    _check(t, x, dt, None, activation, residual)


@pytest.mark.parametrize("rows,k,tokens,dtype", [(40000, 128, 1, "bf16"), (40000, 192, 5, "f32"), (39000, 64, 8, "f16"), (20000, 1088, 9, "bf16"),
                                                 (96, 34816, 2, "bf16"), (64, 65536, 8, "f32"), (64, 65536, 8, "bf16"), (130, 16448, 20, "bf16"),
                                                 (40000, 64, 200, "bf16"), (700, 9024, 16, "f16")])
def test_many_rows_and_many_columns(rows, k, tokens, dtype):
    t = packed(rows, k, rows + tokens)
    _check(t, _x(tokens, k, DTYPES[dtype], 1), DTYPES[dtype])


@pytest.mark.parametrize("tokens", [8, 17, 40, 400])
@pytest.mark.parametrize("dtype", sorted(DTYPES))
def test_epilogue_behind_a_sum_of_slices(tokens, dtype):
    dt = DTYPES[dtype]
    t = packed(200, 4224, 13)
    bias, buf = _x(1, 200, dt, 1)[0], _x(tokens, 210, dt, 2)
    x = _x(tokens, 4224, dt, 5, 0.3)
    before = buf.clone()
    _check(t, x, dt, bias, "silu", buf[:, 3:203], out=buf[:, 3:203])
    assert torch.equal(buf[:, :3], before[:, :3]) and torch.equal(buf[:, 203:], before[:, 203:])


@pytest.mark.parametrize("scale", [1.0, 2.0, 5.0, 20.0, 3e3])
def test_steps_on_both_sides_of_the_short_decoding(scale):
    """Groups whose steps (times a power of two) are fp16 numbers are decoded by one operation, others by two."""
    t = packed(400, 192, 17)
    t.row_consts = (t.row_consts.float() * torch.where(torch.arange(400) % 3 == 0, scale, 1.0)[:, None]).half()
    for tokens in (2, 50, 1500, 3001):
        _check(t, _x(tokens, 192, torch.float32, 3), torch.float32)
    # every weight of a one-hot product is the stored one, to the bit
    eye = torch.eye(192, device=DEV)
    t.had.zero_()
    t.col_scale = None
    w = linear.lay_out(t, DEV)
    v = dequantize_stored(t, DEV, torch.float32)
    for lo in range(0, 192, 8):
        assert torch.equal(linear.stored_linear(eye[lo : lo + 8], w), v[:, lo : lo + 8].T)
    assert torch.equal(linear.stored_linear(eye, w), v.T)
    assert torch.equal(linear.stored_linear(eye.repeat(15, 1), w), v.T.repeat(15, 1))


@pytest.mark.parametrize("tokens", [9, 1501, 3001])
def test_agrees_with_the_reference_product(tokens):
    t = packed(300, 512, 21)
    x = _x(tokens, 512, torch.float32, 8)
    y = linear.stored_linear(x, linear.lay_out(t, DEV))
    want = reference_linear(x, t)
    assert (y.double() - want).norm() / want.norm() < 2e-6


@pytest.mark.parametrize("scaled,flags", [(False, 0.0), (False, 1.0), (True, 0.0)])
def test_without_smoothing_or_rotation(scaled, flags):
    t = packed(130, 192, 5, scaled=scaled, flags=flags)
    for tokens in (3, 65, 2501):
        _check(t, _x(tokens, 192, torch.float16, tokens), torch.float16)


@pytest.mark.parametrize("tokens", [4, 66, 1501, 3001])
def test_strides_offsets_and_out(tokens):
    dt = torch.bfloat16
    t = packed(190, 256, 31)
    wide = _x(2 * tokens, 600, dt, 1)
    for x in (wide[::2, 3:259], wide[:tokens, 1:513:2], wide[:1, 8:264].expand(tokens, 256),
              wide.t()[7 : 7 + tokens].contiguous().t()[:tokens, :tokens].repeat(1, 256)[:, :256]):
        _check(t, x, dt)
    x3 = wide[: 2 * (tokens // 2), :256].reshape(2, tokens // 2, 256)
    _check(t, x3, dt)
    # rows of a wider buffer, in place of the residual; what lies around them stays
    buf = _x(tokens, 400, dt, 9)
    before = buf.clone()
    y = _check(t, wide[:tokens, :256], dt, residual=buf[:, 5:195], out=buf[:, 5:195])
    assert y.data_ptr() == buf[:, 5:195].data_ptr()
    assert torch.equal(buf[:, :5], before[:, :5]) and torch.equal(buf[:, 195:], before[:, 195:])
    bias = _x(2, 190, dt, 4).t()[:, 1]  # strided
    _check(t, wide[:tokens, :256], dt, bias=bias)


@pytest.mark.parametrize("tokens", [20, 2501])
def test_range_of_the_activations(tokens):
    t = packed(140, 128, 3)
    for dt, sizes in ((torch.bfloat16, (1e30, 1e-30, 1e-36)), (torch.float32, (1e30, 1e-28)), (torch.float16, (6e4, 1e-6))):
        for size in sizes:
            x = _x(tokens, 128, torch.float32, 2, 0.0).clamp(-1, 1)
            if dt == torch.float16 and size > 1:
                t1 = packed(140, 128, 3, scaled=False, flags=0.0)
                y = linear.stored_linear((x * size / 128).to(dt), linear.lay_out(t1, DEV))
                want, bound = linear64((x * size / 128).to(dt), t1, dequantize_stored(t1, DEV), None, None, None, dt)
            else:
                y = linear.stored_linear((x * size).to(dt), linear.lay_out(t, DEV))
                want, bound = linear64((x * size).to(dt), t, dequantize_stored(t, DEV), None, None, None, dt)
            within(y, want, bound + 2.0**-133)
    w = linear.lay_out(t, DEV)
    assert not linear.stored_linear(torch.zeros(3, 128, dtype=torch.bfloat16, device=DEV), w).any()


@pytest.mark.parametrize("tokens", [5, 130, 1501, 3001])
def test_non_finite_activations_stay_in_their_row(tokens):
    t = packed(150, 192, 41)
    x = _x(tokens, 192, torch.bfloat16, 6)
    w = linear.lay_out(t, DEV)
    clean = linear.stored_linear(x, w)
    bad = x.clone()
    bad[1, 7], bad[3, 100] = float("nan"), float("inf")
    y = linear.stored_linear(bad, w)
    assert not torch.isfinite(y[1]).any() and not torch.isfinite(y[3]).any()
    rest = [i for i in range(tokens) if i not in (1, 3)]
    assert torch.equal(y[rest], clean[rest])


def test_no_tokens_and_one_row():
    w = linear.lay_out(packed(70, 64, 1), DEV)
    assert linear.stored_linear(torch.zeros(0, 64, device=DEV), w).shape == (0, 70)
    assert linear.stored_linear(torch.zeros(2, 0, 64, device=DEV), w).shape == (2, 0, 70)
    y = linear.stored_linear(_x(1, 64, torch.float32, 1)[0], w)
    assert y.shape == (70,)


@pytest.mark.parametrize("tokens", [16, 200, 1500, 3001])
def test_equal_inputs_give_equal_bits(tokens):
    t = packed(260, 640, 51)
    w = linear.lay_out(t, DEV)
    x = _x(tokens, 640, torch.bfloat16, 7)
    whole = linear.stored_linear(x, w)
    again = linear.stored_linear(x, w)
    assert torch.equal(whole, again)


# ---- stacks -----------------------------------------------------------------------------------------
def _stacks(experts, hidden, inner, seed, formats=None):
    def with_transform(t, like):
        t.had, t.col_scale = like.had, like.col_scale
        return t

    ups, downs = [], []
    for e in range(experts):
        gate = packed(inner, hidden, seed + 10 * e, formats)
        ups.append([gate, with_transform(packed(inner, hidden, seed + 10 * e + 1, formats), gate)])
        downs.append([packed(hidden, inner, seed + 10 * e + 2, formats)])
    gu, dn = linear.lay_out_stack(stack.build_stack(ups), 2, DEV), linear.lay_out_stack(stack.build_stack(downs), 1, DEV)
    gate_up = [(a, torch.cat([dequantize_stored(a, DEV), dequantize_stored(b, DEV)])) for a, b in ups]
    down = [(a, dequantize_stored(a, DEV)) for (a,) in downs]
    return gu, dn, gate_up, down


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("experts,top_k,hidden,inner,tokens", [(1, 1, 64, 64, 1), (5, 3, 128, 192, 1), (5, 3, 320, 64, 37),
                                                               (8, 2, 256, 128, 300), (40, 8, 64, 64, 64), (3, 3, 192, 320, 130),
                                                               (24, 2, 1088, 576, 96), (6, 2, 2112, 64, 3),
                                                               (1, 1, 64, 64, 2501), (5, 3, 320, 64, 900), (8, 2, 256, 128, 1501),
                                                               (40, 8, 64, 64, 1024), (3, 3, 192, 320, 1300), (24, 2, 1088, 576, 400)])
def test_experts_sizes_and_types(experts, top_k, hidden, inner, tokens, dtype):
    dt = DTYPES[dtype]
    gu, dn, gate_up, down = _stacks(experts, hidden, inner, 100 * experts + tokens)
    g = _gen(tokens)
    logits = torch.randn(tokens, experts, generator=g, device=DEV)
    logits[:, 0] += 1.0  # a popular expert
    index, weight = moe.route(logits, top_k, renormalise=True)
    index = index.masked_fill(torch.rand(index.shape, generator=g, device=DEV) < 0.15, -1)
    weight[index < 0] = float("nan")  # an unused slot's weight is not looked at
    x = _x(tokens, hidden, dt, 3, 0.5)
    y = moe.stored_experts(x, index, weight, gu, dn)
    want, bound = experts64(x, index, weight, gate_up, down, dt)
    within(y, want, bound)
    assert torch.equal(y, moe.stored_experts(x, index, weight, gu, dn))
    gu.check(), dn.check()


@pytest.mark.parametrize("n", [90, 1700, 3001])
def test_experts_extremes(n):
    gu, dn, gate_up, down = _stacks(4, 128, 64, 900)
    x = _x(n, 128, torch.float32, 4, 0.5)
    index = torch.full((n, 2), 2, device=DEV)  # one expert for everybody, twice
    weight = torch.rand(n, 2, generator=_gen(1), device=DEV)
    want, bound = experts64(x, index, weight, gate_up, down, torch.float32)
    within(moe.stored_experts(x, index, weight, gu, dn), want, bound)
    # indices that no expert has, of either sign, and int32
    far = torch.full((n, 2), 4, device=DEV, dtype=torch.int32)
    far[::2] = -7
    assert not moe.stored_experts(x, far, weight, gu, dn).any()
    far[3, 1] = 1
    y = moe.stored_experts(x, far, weight, gu, dn)
    want, bound = experts64(x, far, weight, gate_up, down, torch.float32)
    within(y, want, bound)
    assert not y[4:].any() and y[3].any()
    assert moe.stored_experts(x[:0], index[:0], weight[:0], gu, dn).shape == (0, 128)
    # strided activations and a given output; other activations
    wide = _x(n, 300, torch.bfloat16, 5, 0.5)
    buf = torch.ones(n, 200, dtype=torch.bfloat16, device=DEV)
    y = moe.stored_experts(wide[:, 3:131], index, weight.bfloat16(), gu, dn, activation="gelu", out=buf[:, 7:135])
    want, bound = experts64(wide[:, 3:131], index, weight.bfloat16().float(), gate_up, down, torch.bfloat16, "gelu")
    within(y, want, bound)
    assert bool((buf[:, :7] == 1).all()) and bool((buf[:, 135:] == 1).all())
    # in place of the activations
    y = moe.stored_experts(x, index, weight, gu, dn)
    same = x.clone()
    assert torch.equal(moe.stored_experts(same, index, weight, gu, dn, out=same), y) and torch.equal(same, y)


def test_mixture_layer_one_token_and_a_batch():
    """The operators as a mixture layer uses them: a projection added to the residual stream, routing,
    experts through the module, and the sum; against the same steps in 64 bits with the same choice."""
    hidden, experts, top_k = 256, 16, 4
    gu, dn, gate_up, down = _stacks(experts, hidden, 128, 5000)
    t = packed(hidden, 320, 77)
    proj = linear.lay_out(t, DEV)
    router = torch.randn(experts, hidden, generator=_gen(3), device=DEV) * 0.1
    module = moe.StoredExperts(gu, dn)
    assert len(module) == experts
    for tokens in (1, 48, 1500, 3001):
        a, stream = _x(tokens, 320, torch.float32, 1, 0.5), _x(tokens, hidden, torch.float32, 2, 0.2)
        h = linear.stored_linear(a, proj, residual=stream)
        index, weight = moe.route(h @ router.T, top_k, scores="sigmoid", bias=torch.zeros(experts, device=DEV), groups=4,
                                  top_groups=2, renormalise=True)
        y = linear.stored_linear(a, proj, residual=module(h[None], index, weight)[0])
        h64, _ = linear64(a, t, dequantize_stored(t, DEV), None, None, stream, torch.float32)
        assert (h - h64).norm() / h64.norm() < 1e-5
        e64, bound = experts64(h, index, weight, gate_up, down, torch.float32)
        p64, p_bound = linear64(a, t, dequantize_stored(t, DEV), None, None, None, torch.float32)
        within(y, e64 + p64, bound + p_bound + 2.0**-23 * (e64 + p64).abs())


def test_captured_graphs_and_side_streams():
    """Two graphs of the same weights, replayed beside each other and beside eager calls."""
    gu, dn, _, _ = _stacks(6, 128, 64, 700)
    w = linear.lay_out(packed(128, 128, 70), DEV)
    xs = [_x(n, 128, torch.bfloat16, n) for n in (1, 40, 2501)]

    def step(x):
        index, weight = moe.route(x[:, :6].contiguous(), 2)
        return linear.stored_linear(moe.stored_experts(x, index, weight, gu, dn), w, activation="silu", residual=x)

    want = [step(x) for x in xs]
    fixed = [x.clone() for x in xs]
    graphs, outs = [], []
    for x in fixed:
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            step(x)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(x))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in xs]
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        eager = [step(x) for x in xs]
    torch.cuda.synchronize()
    for o, e, y in zip(outs, eager, want):
        assert torch.equal(o, y) and torch.equal(e, y)
    for x, g, o in zip(fixed, graphs, outs):  # new inputs in the same buffers
        x.copy_(x.flip(0) * 0.5)
        g.replay()
        assert torch.equal(o, step(x))


def test_threads_with_streams_of_their_own():
    gu, dn, _, _ = _stacks(6, 128, 64, 700)
    w = linear.lay_out(packed(128, 128, 70), DEV)
    xs = [_x(n, 128, torch.float32, n) for n in (3, 2501, 60, 2501)]

    def step(x):
        index, weight = moe.route(x[:, :6], 2, scores="sigmoid")
        return linear.stored_linear(moe.stored_experts(x, index, weight, gu, dn), w, activation="gelu")

    want = [step(x) for x in xs]
    torch.cuda.synchronize()
    got = [[] for _ in xs]

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            got[i] = [step(xs[i]) for _ in range(10)]
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(xs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for ys, y in zip(got, want):
        assert len(ys) == 10 and all(torch.equal(v, y) for v in ys)
    w.check(), gu.check(), dn.check()


@pytest.mark.parametrize("tokens", [5, 1500, 3001])
def test_operands_and_results_in_one_buffer(tokens):
    t = packed(190, 128, 61)
    w = linear.lay_out(t, DEV)
    buf = _x(tokens, 400, torch.bfloat16, 3)
    want = linear.stored_linear(buf[:, :128].clone(), w, residual=buf[:, 200:390].clone())
    y = linear.stored_linear(buf[:, :128], w, residual=buf[:, 200:390], out=buf[:, 200:390])  # other columns: allowed
    assert torch.equal(y, want)
    flat = buf.reshape(-1)
    for call in (
        lambda: linear.stored_linear(buf[:, :128], w, out=buf[:, 100:290]),
        lambda: linear.stored_linear(buf[:, :128], w, residual=buf[:, 201:391], out=buf[:, 200:390]),
        lambda: linear.stored_linear(buf[:, :128], w, bias=buf[0, 200:390], out=buf[:, 200:390]),
        lambda: linear.stored_linear(flat[: 128 * tokens].view(tokens, 128), w, out=flat[: 190 * tokens].view(tokens, 190)),
    ):
        with pytest.raises(ValueError, match="shares memory"):
            call()


def test_refusals_on_the_device():
    t = packed(64, 128, 2)
    w = linear.lay_out(t, DEV)
    gu, dn, _, _ = _stacks(2, 128, 64, 30)
    x = torch.zeros(3, 128, device=DEV)
    i2, w2 = torch.zeros(3, 2, dtype=torch.int64, device=DEV), torch.zeros(3, 2, device=DEV)
    for call in (
        lambda: linear.stored_linear(x[:, :64], w),
        lambda: linear.stored_linear(x.double(), w),
        lambda: linear.stored_linear(x, w, activation="tanh"),
        lambda: linear.stored_linear(x, w, bias=torch.zeros(63, device=DEV)),
        lambda: linear.stored_linear(x, w, bias=torch.zeros(64, device=DEV, dtype=torch.float16)),
        lambda: linear.stored_linear(x, w, residual=torch.zeros(1, 64, device=DEV)),
        lambda: linear.stored_linear(x, w, out=torch.zeros(3, 65, device=DEV)),
        lambda: linear.stored_linear(x, w, out=torch.zeros(64, 3, device=DEV).t()),
        lambda: linear.stored_linear(x, w, out=torch.zeros(1, 64, device=DEV).expand(3, 64)),
        lambda: linear.stored_linear(x.clone().requires_grad_(), w),
        lambda: linear.stored_linear(x, gu),
        lambda: moe.stored_experts(x, i2, w2, dn, gu),
        lambda: moe.stored_experts(x, i2, w2, w, w),
        lambda: moe.stored_experts(x, i2[:2], w2[:2], gu, dn),
        lambda: moe.stored_experts(x, i2, w2[:, :1], gu, dn),
        lambda: moe.stored_experts(x, w2, w2, gu, dn),
        lambda: moe.stored_experts(x, i2, w2.clone().requires_grad_(), gu, dn),
        lambda: moe.stored_experts(x[:, :64], i2, w2, gu, dn),
    ):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(RuntimeError):
        linear.stored_linear(x.cpu(), w)
    with torch.no_grad():
        linear.stored_linear(x.clone().requires_grad_(), w)
    bad = packed(64, 128, 2)
    bad.row_nbits[5] = 3
    with pytest.raises(ValueError, match="code width"):
        linear.lay_out(bad, DEV)
    bad = packed(64, 128, 2)
    bad.code_off[7] += 1
    with pytest.raises(ValueError, match="offsets"):
        linear.lay_out(bad, DEV)
    bad = packed(64, 128, 2)
    bad.codes = bad.codes[:-1]
    with pytest.raises(ValueError, match="offsets"):
        linear.lay_out(bad, DEV)
    bad = packed(64, 128, 2)
    bad.had = bad.had[:-1]
    with pytest.raises(ValueError):
        linear.lay_out(bad, DEV)
