"""Routing against a row-by-row restatement in 64 bits: choices equal, weights to fp32 rounding."""

import math

import pytest
import torch

from hi2_b200 import moe

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _oracle(logits, top_k, scores, bias, groups, top_groups, renormalise, scale):
    rows, experts = logits.shape
    index, weight = [], []
    b = [0.0] * experts if bias is None else bias.double().tolist()
    for row in logits.double().tolist():
        row = [min(v, 3.4028234663852886e38) if v == v else v for v in row]
        live = [v > -math.inf and c > -math.inf for v, c in zip(row, b)]
        top = max([v for v, ok in zip(row, live) if ok], default=0.0)
        if scores == "softmax":
            z = [math.exp(max(v - top, -745.0)) if ok and v - top > -745 else 0.0 for v, ok in zip(row, live)]
            total = sum(z) or 1.0
            s = [v / total for v in z]
        else:
            s = [(1 / (1 + math.exp(-v)) if v > -700 else 0.0) if ok else 0.0 for v, ok in zip(row, live)]
        biased = [a + c for a, c in zip(s, b)]
        opened = [e for e in range(experts) if live[e]]
        if groups > 1:
            per = experts // groups
            totals = []
            for q in range(groups):
                best = sorted((biased[e] for e in opened if e // per == q), reverse=True)[:2]
                if best:
                    totals.append((-sum(best), q))
            kept = {q for _, q in sorted(totals)[:top_groups]}
            opened = [e for e in opened if e // per in kept]
        key = (lambda e: (-row[e], e)) if bias is None else (lambda e: (-biased[e], e))
        chosen = sorted(opened, key=key)[:top_k]
        w = [s[e] for e in chosen]
        if renormalise:
            w = [v / max(sum(w), 1e-20) for v in w]
        index.append(chosen + [-1] * (top_k - len(chosen)))
        weight.append([v * scale for v in w] + [0.0] * (top_k - len(chosen)))
    return torch.tensor(index), torch.tensor(weight, dtype=torch.float64)


def _check(logits, top_k, scores="softmax", bias=None, groups=1, top_groups=None, renormalise=False, scale=1.0):
    i, w = moe.route(logits.to(DEV), top_k, scores=scores, bias=None if bias is None else bias.to(DEV), groups=groups,
                     top_groups=top_groups, renormalise=renormalise, scale=scale)
    wi, ww = _oracle(logits.reshape(-1, logits.shape[-1]), top_k, scores, bias, groups, top_groups or groups, renormalise, scale)
    assert i.dtype == torch.int64 and w.dtype == torch.float32 and i.shape == w.shape == (*logits.shape[:-1], top_k)
    assert torch.equal(i.cpu().reshape(wi.shape), wi)
    # fp32: an exponential to 2 steps and its argument, a sum of up to `experts` terms, two quotients, a product
    rel = (2 * logits.shape[-1] + 32) * 2.0**-24 + 2 * logits.float().nan_to_num(0, 0, 0).abs().max().item() * 2.0**-24
    assert bool(((w.cpu().double().reshape(ww.shape) - ww).abs() <= rel * ww.abs() + 1e-37).all())


def _logits(rows, experts, seed, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return (2 * torch.randn(rows, experts, generator=g)).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("experts,top_k", [(1, 1), (5, 5), (32, 4), (33, 8), (64, 8), (100, 1), (200, 32), (300, 6), (600, 8), (1024, 32)])
def test_sizes_and_types(experts, top_k, dtype):
    x = _logits(23, experts, experts, dtype)
    bias = 0.3 * torch.randn(experts, generator=torch.Generator().manual_seed(1))
    for scores in ("softmax", "sigmoid"):
        for b in (None, bias):
            for renormalise in (False, True):
                _check(x, top_k, scores, b, renormalise=renormalise, scale=2.5)


@pytest.mark.parametrize("experts,groups,top_groups,top_k", [(8, 8, 3, 2), (64, 8, 4, 8), (96, 3, 1, 6), (128, 32, 5, 8), (256, 8, 8, 8),
                                                             (36, 4, 2, 18), (10, 5, 2, 6)])
def test_groups(experts, groups, top_groups, top_k):
    x = _logits(40, experts, groups)
    bias = 0.3 * torch.randn(experts, generator=torch.Generator().manual_seed(2))
    for scores in ("softmax", "sigmoid"):
        for b in (None, bias):
            _check(x, top_k, scores, b, groups, top_groups, renormalise=True)


def test_ties_go_to_the_lowest_index():
    x = torch.randint(-2, 3, (200, 64), generator=torch.Generator().manual_seed(0)).float()
    x[0] = 0.0
    x[1, ::2] = -0.0
    for b in (None, torch.zeros(64)):
        _check(x, 8, bias=b)
        _check(x.bfloat16(), 9, "sigmoid", bias=b, groups=4, top_groups=2)


def test_closed_experts_and_empty_rows():
    inf, nan = math.inf, math.nan
    x = _logits(30, 48, 5)
    x[torch.rand(30, 48, generator=torch.Generator().manual_seed(3)) < 0.6] = -inf
    x[3] = -inf
    x[4, :] = nan
    x[5, 1:] = -inf
    x[6, 7] = nan
    x[7, 5] = inf
    x[8, :] = torch.finfo(torch.float32).min
    bias = 0.2 * torch.randn(48, generator=torch.Generator().manual_seed(4))
    closed = bias.clone()
    closed[3], closed[9] = -inf, nan
    for b in (None, bias, closed):
        for groups, top_groups in ((1, 1), (6, 2), (16, 16)):
            for scores in ("softmax", "sigmoid"):
                for renormalise in (False, True):
                    _check(x, 10, scores, b, groups, top_groups, renormalise)


def test_far_logits():
    x = torch.tensor([[1e4, 0.0, -1e4, 9.9e3], [-100.0, -101.0, -102.0, -300.0], [80.0, 81.0, 79.0, 60.0]])
    for b in (None, torch.tensor([0.0, 0.5, 1e6, -1e6])):
        for scores in ("softmax", "sigmoid"):
            _check(x, 3, scores, b)


def test_strides_shapes_and_no_tokens():
    wide = _logits(12, 100, 9)
    dev = wide.to(DEV)
    want = moe.route(dev[:, 10:74].contiguous(), 4)
    for view in (dev[:, 10:74], dev.t().contiguous().t()[:, 10:74]):
        got = moe.route(view, 4)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    i, w = moe.route(dev[:, :64].reshape(3, 4, 64), 2)
    assert i.shape == w.shape == (3, 4, 2)
    i, w = moe.route(dev[0, :64], 2)
    assert i.shape == (2,)
    i, w = moe.route(dev[:0, :64], 2)
    assert i.shape == w.shape == (0, 2)


def test_refusals():
    x = torch.zeros(2, 64, device=DEV)
    for kw in (dict(top_k=0), dict(top_k=65), dict(top_k=33), dict(top_k=2, scores="relu"), dict(top_k=2, groups=7),
               dict(top_k=2, groups=64), dict(top_k=2, groups=8, top_groups=9), dict(top_k=2, groups=8, top_groups=0),
               dict(top_k=2, bias=torch.zeros(63, device=DEV)), dict(top_k=2, bias=torch.zeros(64, device=DEV).half())):
        with pytest.raises(ValueError):
            moe.route(x, **kw)
    with pytest.raises(ValueError):
        moe.route(x.double(), 2)
    with pytest.raises(ValueError):
        moe.route(torch.zeros(2, 1025, device=DEV), 2)
    with pytest.raises(ValueError):
        moe.route(x.clone().requires_grad_(), 2)
    with pytest.raises(RuntimeError):
        moe.route(x.cpu(), 2)
