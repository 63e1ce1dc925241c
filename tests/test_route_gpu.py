"""The router against its definition in 64 bits: choices equal, weights and gradients within roundings.

Tolerances.  Choices: equal.  Weights: the kernel has them to 2^-36 relative (a softmax over all experts adds
in fp32: every term to 2^-22 and the sum of E <= 4096 of them, at most 64 + 6 additions deep, to 70 * 2^-24,
under 2^-17 together), then rounds once, half a step of the type.  Gradients are fp32 sums of k <= 64 products
of such numbers: (k + 8) * 2^-24 of the sum of the terms' sizes, plus the shares' own 2^-17, and one rounding.
"""
from __future__ import annotations

import pytest
import torch

import fastmoe_amd as fm
from tests import route_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.float32, torch.bfloat16, torch.float16]
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}


def _logits(T, E, dtype, seed=0, masked=0.0):
    gen = torch.Generator().manual_seed(seed)
    l = 1.5 * torch.randn(T, E, generator=gen) + 0.5 * torch.randn(E, generator=gen)
    if masked:
        l[torch.rand(T, E, generator=gen) < masked] = float("-inf")
    return l.to(dtype)


def _half(dtype):
    return torch.finfo(dtype).eps / 2


def _check_weights(got, want, dtype, whole):
    err = (got.double().cpu() - want).abs()
    tol = want.abs() * (_half(dtype) + (2.0 ** -17 if whole else 2.0 ** -30)) + TINY[dtype]
    assert bool((err <= tol).all()), float((err / tol).max())


def _run(logits, k, r, bias=None, out=None):
    got = fm.route_tokens(logits.to(DEV), k, r, bias=None if bias is None else bias.to(DEV), out_dtype=out)
    ids = ref.choose(logits, k, r, bias)
    assert got.topk_indices.dtype == torch.int64
    assert torch.equal(got.topk_indices.cpu(), ids)
    want = ref.shares(logits, ids, r) * r.scale
    assert got.topk_weights.dtype == (out or logits.dtype)
    _check_weights(got.topk_weights, want, out or logits.dtype, r.score == "softmax" and not r.renormalize)
    return got


SIZES = [  # T, E, k, groups, top_groups
    (1, 1, 1, 1, 1), (1, 8, 2, 1, 1), (3, 7, 7, 1, 1), (130, 64, 6, 1, 1), (5000, 64, 6, 1, 1),
    (5001, 60, 5, 6, 3), (65, 60, 5, 6, 3), (4100, 256, 8, 8, 4), (9, 256, 8, 8, 4), (17, 333, 9, 1, 1),
    (5, 1024, 64, 1, 1), (4099, 1023, 3, 3, 2), (6, 4096, 8, 1, 1), (3, 4001, 33, 1, 1), (7, 64, 4, 64, 5),
    (21, 1024, 16, 64, 4), (4097, 1024, 4, 5 - 1, 2), (11, 48, 3, 2, 2), (2, 130, 64, 2, 1), (4098, 3, 2, 3, 2),
    (8193, 64, 6, 1, 1), (8192, 61, 3, 1, 1), (2049, 256, 8, 8, 4), (2048, 256, 5, 1, 1), (2050, 192, 6, 3, 2)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("T,E,k,G,tg", SIZES)
def test_choices_and_weights(T, E, k, G, tg, dtype):
    logits = _logits(T, E, dtype, seed=T + E)
    bias = 0.05 * torch.randn(E, generator=torch.Generator().manual_seed(E))
    for score in ("softmax", "sigmoid"):
        for group_score in ("max", "top2") if G > 1 else ("max",):
            for b in (None, bias):
                r = fm.Routing(score, G, tg, group_score, renormalize=b is None, scale=2.5)
                _run(logits[:300], k, r, b) if T > 300 and E > 500 else _run(logits, k, r, b)
    _run(logits, k, fm.Routing(groups=G, top_groups=tg, renormalize=False))
    _run(logits, k, fm.Routing("sigmoid", groups=G, top_groups=tg), bias, out=torch.float32)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [True, False])
def test_masked_experts_and_rows(score, renormalize, dtype):
    logits = _logits(300, 24, dtype, seed=3, masked=0.7)
    logits[5] = logits[77] = float("-inf")
    logits[6, 1:] = float("-inf")
    bias = 0.2 * torch.randn(24, generator=torch.Generator().manual_seed(1))
    for r in (fm.Routing(score, renormalize=renormalize), fm.Routing(score, 4, 2, "top2", renormalize),
              fm.Routing(score, 4, 2, "max", renormalize)):
        for b in (None, bias):
            got = _run(logits, 4, r, b)
            assert torch.isfinite(got.topk_weights).all()
            assert not got.topk_weights[5].any() and not got.topk_weights[77].any()
            for row in got.topk_indices.cpu():
                assert len(set(row.tolist())) == 4


@pytest.mark.parametrize("T", [3, 4100])
def test_ties_go_to_the_lowest_index(T):
    logits = torch.zeros(T, 40)
    logits[:, 1::2] = -0.0  # equal to 0
    for r in (fm.Routing(), fm.Routing("sigmoid", 4, 2, "top2"), fm.Routing("softmax", 5, 3)):
        got = _run(logits, 7, r)
        assert torch.equal(got.topk_indices.cpu(), torch.arange(7).expand(T, 7))
    # a few values only, so that most choices are ties
    gen = torch.Generator().manual_seed(2)
    logits = torch.randint(0, 3, (T, 40), generator=gen).float()
    for G, tg in ((1, 1), (8, 3)):
        for gs in ("max", "top2"):
            _run(logits, 6, fm.Routing("sigmoid", G, tg, gs))
            _run(logits, 6, fm.Routing("softmax", G, tg, gs), torch.zeros(40))


def test_nan_and_infinities():
    logits = _logits(4, 16, torch.float32)
    logits[0, 9] = float("nan")
    logits[1, 3] = logits[1, 12] = float("inf")
    logits[2, 4] = -float("nan")
    got = fm.route_tokens(logits.to(DEV), 3, fm.Routing("sigmoid", renormalize=False))
    assert got.topk_indices[0, 0] == 9 and got.topk_indices[2, 0] == 4
    assert got.topk_indices[1, :2].tolist() == [3, 12]
    assert got.topk_weights[1, :2].tolist() == [1.0, 1.0]
    assert got.topk_weights[0, 0].isnan() and not got.topk_weights[0, 1:].isnan().any()
    for r in (fm.Routing(), fm.Routing("sigmoid")):  # what hangs on it is NaN; the ids are experts
        got = fm.route_tokens(logits.to(DEV), 3, r)
        assert got.topk_weights[0].isnan().all()
        assert int(got.topk_indices.min()) >= 0 and int(got.topk_indices.max()) < 16


@pytest.mark.parametrize("shift", [-200.0, 90.0])
def test_far_logits_keep_their_shares(shift):
    """Scores below fp32's range: the weights are of the logits' differences."""
    logits = _logits(50, 12, torch.float32) + shift
    _run(logits, 4, fm.Routing("sigmoid"))
    _run(logits, 4, fm.Routing("softmax"))
    _run(logits, 4, fm.Routing("softmax", renormalize=False))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_strided_rows_at_any_alignment(dtype):
    flat = _logits(1, 37 * 90 + 1, dtype, seed=4).view(-1)
    for start in (0, 1):
        logits = flat[start:start + 37 * 90].view(37, 90)[:, 3:80]
        r = fm.Routing("sigmoid", 7, 3, "top2")
        got = fm.route_tokens(flat.to(DEV)[start:start + 37 * 90].view(37, 90)[:, 3:80], 5, r)
        ids = ref.choose(logits, 5, r)
        assert torch.equal(got.topk_indices.cpu(), ids)
    one = flat.to(DEV)[:90].view(1, 90).expand(6, 90)  # every row the same memory
    assert torch.equal(fm.route_tokens(one, 3).topk_indices.cpu(), ref.choose(one.cpu(), 3, fm.Routing()))


def test_no_tokens():
    w, ids = fm.route_tokens(torch.empty(0, 8, device=DEV, requires_grad=True), 2)
    assert w.shape == ids.shape == (0, 2)
    (g,) = torch.autograd.grad(w.sum(), w.grad_fn.next_functions[0][0].variable)
    assert g.shape == (0, 8)


GRADS = [(1, 1, 1, 1, 1), (33, 8, 2, 1, 1), (300, 60, 5, 6, 3), (70, 256, 8, 8, 4), (5, 1001, 64, 1, 1), (4200, 33, 3, 1, 1)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("T,E,k,G,tg", GRADS)
def test_gradient_of_the_logits(T, E, k, G, tg, renormalize, score, dtype):
    logits = _logits(T, E, dtype, seed=E, masked=0.2 if E > 8 else 0.0)
    bias = 0.05 * torch.randn(E, generator=torch.Generator().manual_seed(2)) if G > 1 else None
    r = fm.Routing(score, G, tg, "top2", renormalize, scale=2.5)
    g = torch.randn(T, k, generator=torch.Generator().manual_seed(7)).to(dtype)
    x = logits.to(DEV).requires_grad_(True)
    w, ids = fm.route_tokens(x, k, r, bias=None if bias is None else bias.to(DEV))
    assert w.requires_grad and not ids.requires_grad
    (got,) = torch.autograd.grad(w, x, g.to(DEV))
    assert got.dtype == dtype and got.shape == (T, E)
    l = logits.double().requires_grad_(True)
    share = ref.shares(l, ref.choose(logits, k, r, bias), r)
    (want,) = torch.autograd.grad(share * 2.5, l, g.double())
    want = want.nan_to_num(0.0)
    # the sizes of what is added: scale * share * (|g| + sum |share g|), of every expert's share
    every = torch.softmax(logits.double(), -1) if score == "softmax" else torch.ones(T, E, dtype=torch.double)
    size = (share.detach() * g.double().abs()).sum(-1, keepdim=True)
    u = torch.zeros(T, E, dtype=torch.double).scatter_(1, ids.cpu(), share.detach())
    ga = torch.zeros(T, E, dtype=torch.double).scatter_(1, ids.cpu(), g.double().abs())
    # renormalised, a chosen expert's share of a masked rest may be 1; over all experts it is `every`
    terms = 2.5 * (u * (ga + size) + (0 if renormalize else every.nan_to_num(0.0) * size))
    tol = want.abs() * _half(dtype) + terms * ((k + 8) * 2.0 ** -24 + 2.0 ** -17) + TINY[dtype]
    err = (got.double().cpu() - want).abs()
    assert bool((err <= tol).all()), float((err / tol).max())


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [True, False])
def test_gradient_against_differences(score, renormalize):
    """Along random directions, the change of sum(g * w) of the definition in 64 bits: central differences
    with a step of 2^-12 are off by the third derivative's h^2 / 6 (the scores' derivatives are below 1, the
    directions' size below 6, so below 1e-4 of the terms' size), the kernel by 2^-16."""
    T, E, k = 20, 30, 4
    logits = _logits(T, E, torch.float32, seed=9)
    r = fm.Routing(score, renormalize=renormalize)
    g = torch.randn(T, k, generator=torch.Generator().manual_seed(7))
    x = logits.to(DEV).requires_grad_(True)
    w, ids = fm.route_tokens(x, k, r)
    (got,) = torch.autograd.grad(w, x, g.to(DEV))
    ids, got = ids.cpu(), got.double().cpu()
    h = 2.0 ** -12
    for seed in range(4):
        d = torch.randn(T, E, generator=torch.Generator().manual_seed(seed), dtype=torch.double)
        def f(s):
            return (ref.shares(logits.double() + s * h * d, ids, r) * g.double()).sum(-1)
        slope = (f(1) - f(-1)) / (2 * h)
        size = (g.double().abs().sum(-1) + 1) * d.abs().amax(-1)
        assert bool(((got * d).sum(-1) - slope).abs().le(2e-4 * size).all())


def test_gradient_is_refused_twice_and_survives_strides():
    x = _logits(6, 10, torch.float32).to(DEV).requires_grad_(True)
    w, _ = fm.route_tokens(x, 3)
    g = torch.randn(3, 6, device=DEV).t()  # columns first
    (a,) = torch.autograd.grad(w, x, g, retain_graph=True)
    (b,) = torch.autograd.grad(w, x, g.contiguous(), retain_graph=True)
    assert torch.equal(a, b)
    (c,) = torch.autograd.grad(w.sum(), x, retain_graph=True)  # an expanded gradient
    assert c.abs().max() < 1e-6
    (d,) = torch.autograd.grad(w, x, g.contiguous(), create_graph=True)
    assert torch.equal(b, d)
    with pytest.raises(RuntimeError, match="no gradient of its own"):
        d.sum().backward()


def test_graph_replays_on_other_logits():
    r = fm.Routing("sigmoid", 8, 4, "top2", scale=2.5)
    x = torch.empty(16, 64, device=DEV)
    bias = 0.1 * torch.randn(64, device=DEV)
    with torch.no_grad():
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            x.copy_(_logits(16, 64, torch.float32).to(DEV))
            fm.route_tokens(x, 6, r, bias=bias)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = fm.route_tokens(x, 6, r, bias=bias)
        for seed in range(4):
            x.copy_(_logits(16, 64, torch.float32, seed=seed).to(DEV))
            graph.replay()
            torch.cuda.synchronize()
            want = fm.route_tokens(x, 6, r, bias=bias)
            assert torch.equal(held.topk_indices, want.topk_indices)
            assert torch.equal(held.topk_weights, want.topk_weights)


def test_capture_of_the_autograd_call_is_refused():
    x = torch.randn(8, 16, device=DEV, requires_grad=True)
    fm.route_tokens(x, 2)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="capture"):
            fm.route_tokens(x, 2)
        torch.zeros(1, device=DEV)  # a graph with something in it


def test_refusals_of_gpu_tensors():
    x = torch.randn(4, 8, device=DEV)
    bias = torch.zeros(8, device=DEV)
    with pytest.raises(ValueError, match="top_k"):
        fm.route_tokens(x, 9)
    with pytest.raises(ValueError, match="top_k"):
        fm.route_tokens(x, 0)
    with pytest.raises(ValueError, match="columns|unit"):
        fm.route_tokens(x.t(), 2)
    with pytest.raises(TypeError, match="dtype"):
        fm.route_tokens(x.double(), 2)
    with pytest.raises(TypeError, match="out_dtype"):
        fm.route_tokens(x, 2, out_dtype=torch.int32)
    with pytest.raises(ValueError, match="bias"):
        fm.route_tokens(x, 2, bias=bias.half())
    with pytest.raises(ValueError, match="bias"):
        fm.route_tokens(x, 2, bias=bias[:7])
    with pytest.raises(RuntimeError, match="no gradient"):
        fm.route_tokens(x, 2, bias=bias.clone().requires_grad_(True))
    with pytest.raises(ValueError, match="groups"):
        fm.route_tokens(x, 2, fm.Routing(groups=3, top_groups=1))
    with pytest.raises(ValueError, match="top_k"):
        fm.route_tokens(x, 3, fm.Routing(groups=4, top_groups=1))
    with pytest.raises(OverflowError):
        fm.route_tokens(torch.zeros(2, 100, device=DEV), 65)
    with pytest.raises(OverflowError):
        fm.route_tokens(torch.zeros(2, 4097, device=DEV), 2)
    with pytest.raises(OverflowError):
        fm.route_tokens(torch.zeros(2, 2048, device=DEV), 2, fm.Routing(groups=2))
    with pytest.raises(RuntimeError, match="functorch|tracing"):
        torch.func.grad(lambda t: fm.route_tokens(t, 2).topk_weights.sum())(x)
