"""Cases for the forward pass over packed weights: the product of activations with a packed tensor and its
epilogue, the routing of tokens to experts, and the routed experts' products over stacked packed tensors.

``run`` computes an operator in its plain form (elementary tensor operations in 32 bits, in 64 where a
comparison may hang on the last bits), or with ``own`` through the package's entry points.  ``exact`` is
the operator's definition in 64 bits, written apart.  The packed tensors are random codes and ladder
parameters of the format's own types and ranges, with a mix of row formats as the allocation leaves it."""

import math

import torch

own = False  # the package's kernels instead of the plain forms

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
# share of the rows by (code width, block): a 3 bits/weight allocation, one with sensitive rows kept in
# INT8, the two-bit floor, and all-INT4
MIXES = {
    "flex": (((2, 16), 0.60), ((2, 32), 0.25), ((4, 64), 0.10), ((4, 32), 0.03), ((4, 16), 0.02)),
    "flex8": (((2, 16), 0.45), ((2, 64), 0.25), ((4, 32), 0.20), ((8, 64), 0.06), ((8, 32), 0.04)),
    "int2": (((2, 16), 0.40), ((2, 32), 0.35), ((2, 64), 0.25)),
    "int4": (((4, 32), 0.50), ((4, 64), 0.50)),
}


def listed():
    return [
        # one new token through an attention output projection of a 4096-wide layer, added to the residual stream
        dict(name="linear one token", op="linear", rows=4096, k=4096, tokens=1, mix="flex", dtype="bf16",
             bias=False, act="", residual=True),
        # one new token through the widest projection of an 8192-wide layer: bound by the packed weights' bytes
        dict(name="linear one token, wide", op="linear", rows=28672, k=8192, tokens=1, mix="int2", dtype="bf16",
             bias=False, act="silu", residual=False),
        # a decode batch through a down projection, fp16 activations
        dict(name="linear batch", op="linear", rows=4096, k=11008, tokens=32, mix="flex", dtype="f16",
             bias=False, act="", residual=True),
        # odd everything in fp32: a small encoder's projection with bias and activation
        dict(name="linear odd", op="linear", rows=1001, k=1088, tokens=77, mix="flex8", dtype="f32",
             bias=True, act="gelu", residual=True),
        # a calibration window (2048 tokens) through a gate projection
        dict(name="linear prompt", op="linear", rows=11008, k=4096, tokens=2048, mix="flex", dtype="bf16",
             bias=False, act="silu", residual=False),
        # routing of one new token: latency
        dict(name="route one token", op="route", tokens=1, experts=64, top_k=8, dtype="f32", scores="softmax",
             bias=False, groups=1, top_groups=1, renormalise=False, masked=False),
        # routing of a long prompt batch with balanced, grouped sigmoid scores; padding tokens have no expert
        dict(name="route grouped", op="route", tokens=16384, experts=128, top_k=6, dtype="f32", scores="sigmoid",
             bias=True, groups=8, top_groups=3, renormalise=True, masked=True),
        # routing of a calibration window from bf16 logits, where equal logits are common
        dict(name="route ties", op="route", tokens=2048, experts=64, top_k=8, dtype="bf16", scores="softmax",
             bias=False, groups=1, top_groups=1, renormalise=True, masked=False),
        # one new token through 64 experts, eight of them chosen
        dict(name="experts one token", op="experts", tokens=1, experts=64, top_k=8, hidden=2048, inner=1024,
             mix="flex", dtype="bf16", unused=False),
        # a decode batch: every expert is read, few tokens each
        dict(name="experts batch", op="experts", tokens=64, experts=64, top_k=8, hidden=2048, inner=1024,
             mix="flex", dtype="bf16", unused=False),
        # few small experts in fp16, slots left unused by a padded batch
        dict(name="experts odd", op="experts", tokens=37, experts=5, top_k=3, hidden=320, inner=192,
             mix="flex8", dtype="f16", unused=True),
        # a calibration window's prompt through all experts
        dict(name="experts prompt", op="experts", tokens=4096, experts=64, top_k=8, hidden=2048, inner=1024,
             mix="flex", dtype="bf16", unused=False),
    ]


def _spread(rng, lo, hi, step=1):
    """A multiple of ``step`` in [lo, hi], uniform in its logarithm."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(v / step)) * step))


def draw(rng):
    op = rng.choice(["linear", "linear", "route", "experts", "experts"])
    if op == "linear":
        case = dict(op=op, rows=_spread(rng, 65, 16000), k=_spread(rng, 64, 16384, 64), tokens=_spread(rng, 1, 4096),
                    mix=rng.choice(sorted(MIXES)), dtype=rng.choice(sorted(DTYPES)), bias=rng.random() < 0.5,
                    act=rng.choice(["", "relu", "silu", "gelu", "gelu_tanh"]), residual=rng.random() < 0.5)
        case["rows"] = min(case["rows"], 28672 * 8192 // case["k"])
        case["tokens"] = max(1, min(case["tokens"], 11008 * 4096 * 2048 // (case["rows"] * case["k"])))
        return case
    if op == "route":
        groups = rng.choice([1, 1, 2, 4, 8])
        per = _spread(rng, 2, 256 // groups)
        top_groups = rng.randint(1, groups)
        return dict(op=op, tokens=_spread(rng, 1, 16384), experts=groups * per, top_k=rng.randint(1, min(8, per * top_groups)),
                    dtype=rng.choice(sorted(DTYPES)), scores=rng.choice(["softmax", "sigmoid"]), bias=rng.random() < 0.5,
                    groups=groups, top_groups=top_groups, renormalise=rng.random() < 0.5, masked=rng.random() < 0.5)
    experts = _spread(rng, 2, 64)
    return dict(op=op, tokens=_spread(rng, 1, 4096), experts=experts, top_k=rng.randint(1, min(8, experts)),
                hidden=_spread(rng, 64, 2048, 64), inner=_spread(rng, 64, 1024, 64), mix=rng.choice(sorted(MIXES)),
                dtype=rng.choice(sorted(DTYPES)), unused=rng.random() < 0.3)


def work(case):
    if case["op"] == "route":
        t, e, k = case["tokens"], case["experts"], case["top_k"]
        size = 4 if case["dtype"] == "f32" else 2
        return {"bytes": t * e * size + t * k * 12 + (4 * e if case["bias"] else 0), "flops": 4 * t * e}
    size = 4 if case["dtype"] == "f32" else 2
    per_weight = sum(share * (nbits / 8 + 2 / block) for (nbits, block), share in MIXES[case["mix"]])
    if case["op"] == "linear":
        n, k, m = case["rows"], case["k"], case["tokens"]
        moved = m * (k + n * (2 if case["residual"] else 1)) * size + (n * size if case["bias"] else 0)
        return {"bytes": int(n * k * per_weight) + 6 * n + moved, "flops": 2 * m * n * k}
    t, e, top, h, i = case["tokens"], case["experts"], case["top_k"], case["hidden"], case["inner"]
    named = e * (1 - (1 - top / e) ** t)
    return {"bytes": int(named * (3 * h * i * per_weight + 6 * (2 * i + h))) + 2 * t * h * size + 12 * t * top,
            "flops": 6 * t * top * h * i}


# ---- inputs ---------------------------------------------------------------------------------------
def _packed(rows, k, mix, experts, g):
    """The flat buffers of ``experts`` tensors of ``rows`` rows one after the other: random codes, block
    ladders that reach from about -2 to 2 standard deviations of weights around 0.02."""
    dev, total = "cuda", rows * experts
    formats = torch.tensor([f for f, _ in MIXES[mix]], device=dev)
    shares = torch.tensor([s for _, s in MIXES[mix]], device=dev)
    pick = torch.multinomial(shares, total, replacement=True, generator=g)
    nbits, block = formats[pick, 0], formats[pick, 1]
    code_off = torch.cat([nbits.new_zeros(1), torch.cumsum(k * nbits // 32, 0)])
    param_off = torch.cat([nbits.new_zeros(1), torch.cumsum(k // block, 0)])
    n_words, n_blocks = torch.stack([code_off[-1], param_off[-1]]).tolist()
    codes = torch.randint(-(2**31), 2**31, (n_words,), generator=g, device=dev, dtype=torch.int32)
    params = torch.randint(0, 256, (n_blocks, 2), generator=g, device=dev, dtype=torch.uint8)
    params[:, 1] = 128 + params[:, 1] // 2
    reach = 0.03 * torch.exp(0.3 * torch.randn(total, generator=g, device=dev))
    consts = torch.stack([-1.4 * reach, 0.8 * reach / 255, 2 * reach / (2.0**nbits - 1) / 192], 1).half()
    had = (torch.rand(experts, k // 16, generator=g, device=dev) < 0.8).to(torch.uint8)
    scale = torch.exp(0.5 * torch.randn(experts, k, generator=g, device=dev)).half()
    return dict(codes=codes, code_off=code_off.int(), blk_params=params.reshape(-1), param_off=param_off.int(),
                row_consts=consts, row_nbits=nbits.to(torch.uint8), row_block=block.to(torch.uint8), had=had,
                col_scale=scale)


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    if case["op"] == "route":
        t, e = case["tokens"], case["experts"]
        logits = 1.5 * normal(t, e) + 0.7 * normal(e)
        if case["masked"]:  # experts that a token may not take, and padding tokens
            logits[torch.rand(t, e, generator=g, device="cuda") < 0.05] = -math.inf
            logits[torch.rand(t, generator=g, device="cuda") < 0.1] = -math.inf
        return dict(logits=logits.to(DTYPES[case["dtype"]]), bias=0.1 * normal(e) if case["bias"] else None)
    dtype = DTYPES[case["dtype"]]
    if case["op"] == "linear":
        n, k, m = case["rows"], case["k"], case["tokens"]
        x = normal(m, k) * torch.exp(normal(k))
        return dict(x=x.to(dtype), w=_packed(n, k, case["mix"], 1, g), bias=normal(n).to(dtype) if case["bias"] else None,
                    residual=normal(m, n).to(dtype) if case["residual"] else None)
    t, e, h, i = case["tokens"], case["experts"], case["hidden"], case["inner"]
    x = (normal(t, h) * torch.exp(0.5 * normal(h))).to(dtype)
    chosen = torch.topk(normal(t, e) + 0.7 * normal(e), case["top_k"], dim=1)
    index, weight = chosen.indices, torch.softmax(chosen.values, 1)
    if case["unused"]:  # a padded batch: slots without an expert
        index = index.masked_fill(torch.rand(t, case["top_k"], generator=g, device="cuda") < 0.2, -1)
    return dict(x=x, index=index, weight=weight, gate_up=_packed(2 * i, h, case["mix"], e, g),
                down=_packed(h, i, case["mix"], e, g))


def prepare(case, seed):
    state = dict(case=case, **_inputs(case, seed))
    if own:
        from hi2_b200 import linear
        from hi2_b200.format import FIELDS, HI2Tensor

        if case["op"] == "linear":
            w = state["w"]
            flat = {f: w[f] for f in FIELDS} | {"had": w["had"][0], "col_scale": w["col_scale"][0]}
            state["w"] = linear.lay_out(HI2Tensor(shape=(case["rows"], case["k"]), **flat))
        elif case["op"] == "experts":
            for name, parts, rows in (("gate_up", 2, case["inner"]), ("down", 1, case["hidden"])):
                part_off = rows * torch.arange(parts * case["experts"] + 1, dtype=torch.int32)
                state[name] = linear.lay_out_stack(state[name] | {"part_off": part_off}, parts)
    return state


# ---- the plain forms --------------------------------------------------------------------------------
def _weights(p, rows, k):
    """The fp16 values of the given rows of the flat buffers, as fp32 ``[*rows.shape, k]``."""
    col = torch.arange(k, device=rows.device)
    nbits, block = p["row_nbits"].long()[rows], p["row_block"].long()[rows]
    bit = col * nbits[..., None]
    word = p["codes"][p["code_off"].long()[rows][..., None] + bit // 32]
    code = (word >> (bit % 32).int()) & ((1 << nbits) - 1).int()[..., None]
    pair = p["blk_params"].view(-1, 2)[p["param_off"].long()[rows][..., None] + col // block[..., None]].float()
    const = p["row_consts"].float()[rows][..., None, :]
    lo = (pair[..., 0].double() * const[..., 1].double() + const[..., 0].double()).float().half()
    step = (pair[..., 1] * const[..., 2]).half()
    return (lo.double() + code.double() * step.double()).half().float()  # in 64 bits: one rounding, next to borders too


def _hadamard(dtype):
    i = torch.arange(16, device="cuda")
    both = i[:, None] & i
    ones = sum((both >> b) & 1 for b in range(4))
    return (1.0 - 2.0 * (ones % 2)).to(dtype) / 4


def _stored_basis(x, scale, had):
    """``x [..., k]`` divided by the smoothing vector and rotated in the flagged groups of 16 columns."""
    z = (x / scale.float()).unflatten(-1, (-1, 16))
    z = torch.where(had[..., None] != 0, z @ _hadamard(z.dtype), z)
    return z.flatten(-2)


def _activate(v, act):
    if act == "relu":
        return torch.where(v < 0, torch.zeros_like(v), v)
    if act == "silu":
        return v / (1 + torch.exp(-v))
    if act == "gelu":
        return 0.5 * v * (1 + torch.erf(v / math.sqrt(2)))
    if act == "gelu_tanh":
        z = math.sqrt(2 / math.pi) * (v + 0.044715 * v * v * v)
        return v / (1 + torch.exp(-2 * z))
    return v


def _linear(s):
    case, p = s["case"], s["w"]
    w = _weights(p, torch.arange(case["rows"], device="cuda"), case["k"])
    y = _stored_basis(s["x"].float(), p["col_scale"][0], p["had"][0]) @ w.T
    if s["bias"] is not None:
        y = y + s["bias"].float()
    y = _activate(y, case["act"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(s["x"].dtype)


def _route(s):
    case = s["case"]
    logits = s["logits"].double()  # in 64 bits: keys that nearly agree must not change places
    open_ = logits > -math.inf
    top = torch.where(open_, logits, torch.full_like(logits, -1e300)).amax(1, keepdim=True)
    if case["scores"] == "softmax":
        z = torch.where(open_, torch.exp(logits - top), torch.zeros_like(logits))
        score = z / z.sum(1, keepdim=True).clamp_min(1e-300)
    else:
        score = torch.where(open_, 1 / (1 + torch.exp(-logits)), torch.zeros_like(logits))
    key = logits if s["bias"] is None else score + s["bias"].double()
    key = key.masked_fill(~open_, -math.inf)
    if case["groups"] > 1:  # a group counts with the sum of its two best biased scores
        value = (score if s["bias"] is None else score + s["bias"].double()).masked_fill(~open_, -math.inf)
        best = value.unflatten(1, (case["groups"], -1)).sort(dim=2, descending=True).values[..., :2]
        total = torch.where(best > -math.inf, best, torch.zeros_like(best)).sum(2)
        total = torch.where(best[..., 0] > -math.inf, total, torch.full_like(total, -math.inf))
        rank = total.sort(dim=1, descending=True, stable=True).indices.argsort(1)
        key = torch.where((rank < case["top_groups"])[..., None], key.unflatten(1, (case["groups"], -1)), -math.inf).flatten(1)
    best = key.sort(dim=1, descending=True, stable=True)
    key, index = best.values[:, : case["top_k"]], best.indices[:, : case["top_k"]]
    weight = torch.where(key > -math.inf, score.gather(1, index), torch.zeros_like(key))
    index = index.masked_fill(~(key > -math.inf), -1)
    if case["renormalise"]:
        weight = weight / weight.sum(1, keepdim=True).clamp_min(1e-20)
    return index, (weight * 1.5).float()


def _pair_products(p, expert, z, rows, k):
    """One product per (token, slot) pair with its own expert's weights."""
    at = expert[:, None] * rows + torch.arange(rows, device=z.device)
    return (_weights(p, at, k) @ z[..., None]).squeeze(-1)


def _experts(s):
    case = s["case"]
    t, top = s["index"].shape
    h, i, e = case["hidden"], case["inner"], case["experts"]
    used = s["index"] >= 0
    expert = s["index"].clamp_min(0).reshape(-1)
    x = s["x"].float().repeat_interleave(top, 0)
    gu, dn = s["gate_up"], s["down"]
    if t * top <= e:  # few pairs: only the rows of their experts are decoded
        z = _pair_products(gu, expert, _stored_basis(x, gu["col_scale"][expert], gu["had"][expert]), 2 * i, h)
        a = _activate(z[:, :i], "silu") * z[:, i:]
        y = _pair_products(dn, expert, _stored_basis(a, dn["col_scale"][expert], dn["had"][expert]), h, i)
    else:  # every expert's pairs in one padded batch
        order = torch.argsort(expert, stable=True)
        counts = torch.zeros(e, dtype=torch.long, device=x.device).index_add_(0, expert, torch.ones_like(expert))
        slot = torch.arange(expert.numel(), device=x.device) - (torch.cumsum(counts, 0) - counts)[expert[order]]
        batch = x.new_zeros(e, int(counts.max()), h)
        batch[expert[order], slot] = x[order]
        every = torch.arange(e, device=x.device)[:, None]
        w = _weights(gu, every * 2 * i + torch.arange(2 * i, device=x.device), h)
        z = torch.bmm(_stored_basis(batch, gu["col_scale"][:, None], gu["had"][:, None]), w.transpose(1, 2))
        a = _activate(z[..., :i], "silu") * z[..., i:]
        w = _weights(dn, every * h + torch.arange(h, device=x.device), i)
        z = torch.bmm(_stored_basis(a, dn["col_scale"][:, None], dn["had"][:, None]), w.transpose(1, 2))
        y = torch.empty_like(x)
        y[order] = z[expert[order], slot]
    share = torch.where(used, s["weight"], torch.zeros_like(s["weight"]))
    return (y.view(t, top, h) * share[..., None]).sum(1).to(s["x"].dtype)


def run(state):
    case = state["case"]
    if own:
        from hi2_b200 import linear, moe

        if case["op"] == "linear":
            return linear.stored_linear(state["x"], state["w"], bias=state["bias"], activation=case["act"] or None,
                                        residual=state["residual"])
        if case["op"] == "route":
            return moe.route(state["logits"], case["top_k"], scores=case["scores"], bias=state["bias"], groups=case["groups"],
                             top_groups=case["top_groups"], renormalise=case["renormalise"], scale=1.5)
        return moe.stored_experts(state["x"], state["index"], state["weight"], state["gate_up"], state["down"])
    return {"linear": _linear, "route": _route, "experts": _experts}[case["op"]](state)


# ---- the definitions in 64 bits ---------------------------------------------------------------------
def _decoded(p, k):
    """All rows in fp64, one row format after the other."""
    out = torch.empty(p["row_nbits"].numel(), k, dtype=torch.float64, device="cuda")
    for nbits in (2, 4, 8):
        for block in (16, 32, 64):
            rows = ((p["row_nbits"] == nbits) & (p["row_block"] == block)).nonzero().squeeze(1)
            if rows.numel() == 0:
                continue
            n_words = k * nbits // 32
            words = p["codes"][p["code_off"][rows].long()[:, None] + torch.arange(n_words, device="cuda")]
            fields = torch.arange(0, 32, nbits, device="cuda")
            codes = ((words.long()[..., None] >> fields) & (2**nbits - 1)).reshape(rows.numel(), k // block, block).double()
            at = p["param_off"][rows].long()[:, None] + torch.arange(k // block, device="cuda")
            u = p["blk_params"].view(-1, 2)[at].double()
            c = p["row_consts"][rows].double()
            lo = (u[..., 0] * c[:, 1:2] + c[:, 0:1]).float().half().double()
            step = (u[..., 1] * c[:, 2:3]).float().half().double()
            out[rows] = (lo[..., None] + codes * step[..., None]).half().double().reshape(rows.numel(), k)
    return out


def _turned(x, scale, had):
    """fp64 activations in the basis of the stored rows."""
    x = x / scale.double()
    sign = torch.ones(1, 1, dtype=torch.float64, device="cuda")
    for _ in range(4):
        sign = torch.cat([torch.cat([sign, sign], 1), torch.cat([sign, -sign], 1)], 0)
    groups = x.reshape(x.shape[0], -1, 16)
    flag = had.bool()[None, :, None]
    return torch.where(flag, torch.einsum("tgi,ij->tgj", groups, sign / 4), groups).reshape(x.shape)


def _smooth(v, act):
    if act == "relu":
        return v.clamp_min(0)
    if act == "silu":
        return v * torch.sigmoid(v)
    if act == "gelu":
        return v * 0.5 * torch.erfc(-v / math.sqrt(2))
    if act == "gelu_tanh":
        return 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v**3)))
    return v


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "linear":
        y = _turned(s["x"].double(), s["w"]["col_scale"][0], s["w"]["had"][0]) @ _decoded(s["w"], case["k"]).T
        y = _smooth(y if s["bias"] is None else y + s["bias"].double(), case["act"])
        return y if s["residual"] is None else y + s["residual"].double()
    if case["op"] == "route":
        logits = s["logits"].double().cpu()
        bias = None if s["bias"] is None else s["bias"].double().cpu()
        open_ = logits != -math.inf
        score = torch.softmax(logits, 1) if case["scores"] == "softmax" else torch.sigmoid(logits)
        score = score.nan_to_num(0.0)
        biased = torch.where(open_, score if bias is None else score + bias, -math.inf)
        key = torch.where(open_, logits, -math.inf) if bias is None else biased.clone()
        if case["groups"] > 1:
            per = case["experts"] // case["groups"]
            value = torch.full((len(key), case["groups"]), -math.inf, dtype=torch.float64)
            for q in range(case["groups"]):
                part = biased[:, q * per : (q + 1) * per]
                first = part.amax(1)
                at = part.argmax(1, keepdim=True)
                second = part.scatter(1, at, -math.inf).amax(1)
                value[:, q] = first + torch.where(second > -math.inf, second, 0.0)
            keep = torch.zeros_like(key, dtype=torch.bool)
            for _ in range(case["top_groups"]):
                q = value.argmax(1, keepdim=True)
                live = value.gather(1, q) > -math.inf
                keep |= (torch.arange(case["experts"]) // per == q) & live
                value.scatter_(1, q, -math.inf)
            key = torch.where(keep, key, -math.inf)
        index, weight = [], []
        for _ in range(case["top_k"]):
            best = key.amax(1, keepdim=True)
            at = (key == best).to(torch.uint8).argmax(1, keepdim=True)  # the first of equal keys
            live = best > -math.inf
            index.append(torch.where(live, at, -1))
            weight.append(torch.where(live, score.gather(1, at), 0.0))
            key = key.scatter(1, at, -math.inf)
        weight = torch.cat(weight, 1)
        if case["renormalise"]:
            weight = weight / weight.sum(1, keepdim=True).clamp_min(1e-20)
        return torch.cat(index, 1).cuda(), (1.5 * weight).cuda()
    h, i = case["hidden"], case["inner"]
    x = s["x"].double()
    y = torch.zeros_like(x)
    up, dn = _decoded(s["gate_up"], h).view(-1, 2 * i, h), _decoded(s["down"], i).view(-1, h, i)
    for e in range(case["experts"]):
        token, slot = (s["index"] == e).nonzero(as_tuple=True)
        if token.numel() == 0:
            continue
        z = _turned(x[token], s["gate_up"]["col_scale"][e], s["gate_up"]["had"][e]) @ up[e].T
        a = _smooth(z[:, :i], "silu") * z[:, i:]
        z = _turned(a, s["down"]["col_scale"][e], s["down"]["had"][e]) @ dn[e].T
        y.index_add_(0, token, z * s["weight"][token, slot, None].double())
    return y
