"""Uses of the router beside its values: masks with a bias, logits changed in place, autograd's own tools."""
from __future__ import annotations

import pytest
import torch

import fastmoe_amd as fm

from . import route_ref as ref
from .test_route_gpu import DEV, TYPES, _logits, _run

pytestmark = pytest.mark.gpu
INF = float("inf")


@pytest.mark.parametrize("renormalize", [True, False])
def test_a_bias_chooses_among_masked_experts_too(renormalize):
    """Where s + bias chooses, a masked expert's choice is its bias; it has no weight.  -inf leaves it out."""
    logits = torch.tensor([[-INF, 0.0, -1.0, -INF]])
    r = fm.Routing("sigmoid", renormalize=renormalize)
    got = _run(logits, 1, r, torch.tensor([0.5, -0.1, -0.1, 0.0]))
    assert got.topk_indices.tolist() == [[0]] and got.topk_weights.tolist() == [[0.0]]
    got = _run(logits, 2, r, torch.tensor([0.5, -0.1, -0.1, 0.0]))
    assert got.topk_indices.tolist() == [[0, 1]]
    assert got.topk_weights.tolist() == [[0.0, 1.0 if renormalize else 0.5]]
    got = _run(logits, 2, r, torch.tensor([-INF, -0.1, -0.1, -INF]))
    assert got.topk_indices.tolist() == [[1, 2]]
    got = _run(logits, 2, r)  # no bias: the logits choose, and masked experts come last
    assert got.topk_indices.tolist() == [[1, 2]]
    assert _run(logits, 4, r).topk_indices.tolist() == [[1, 2, 0, 3]]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("T", [5, 4200])
def test_experts_left_out_by_their_bias(T, dtype):
    logits = _logits(T, 48, dtype, seed=T, masked=0.2)
    bias = 0.2 * torch.randn(48, generator=torch.Generator().manual_seed(1))
    bias[::3] = -INF
    for score in ("softmax", "sigmoid"):
        for r in (fm.Routing(score), fm.Routing(score, 4, 2, "top2"), fm.Routing(score, 4, 2, "max")):
            got = _run(logits, 5, r, bias)
            assert bool((got.topk_indices % 3 != 0).all())
        got = _run(logits, 40, fm.Routing(score), bias)  # 32 are left
        assert bool((got.topk_indices[:, :32] % 3 != 0).all()) and bool((got.topk_indices[:, 32:] % 3 == 0).all())


def test_balance_leaves_a_bias_of_minus_infinity():
    moe = fm.MoEFeedForward(32, 16, 6, 2, routing=fm.Routing("sigmoid"), balance=True).cuda().bfloat16()
    moe.balance_bias[2] = -INF
    for seed in range(3):
        moe(torch.randn(1, 40, 32, device=DEV, generator=torch.Generator(DEV).manual_seed(seed)).bfloat16())
        assert int(moe.expert_load[2]) == 0 and int(moe.expert_load.sum()) == 80
        moe.update_balance(0.25)
    assert moe.balance_bias[2] == -INF and torch.isfinite(moe.balance_bias).sum() == 5


RULES = [fm.Routing(), fm.Routing("sigmoid"), fm.Routing("sigmoid", renormalize=False), fm.Routing(renormalize=False)]


@pytest.mark.parametrize("r", RULES, ids=str)
@pytest.mark.parametrize("leaf", [True, False])
def test_logits_changed_before_the_backward(r, leaf):
    """Only the gradient of a softmax over all experts reads the logits again; it says so."""
    x = _logits(40, 24, torch.float32).to(DEV).requires_grad_(True)
    g = torch.randn(40, 3, device=DEV, generator=torch.Generator(DEV).manual_seed(1))
    logits = x if leaf else x * 1
    w, _ = fm.route_tokens(logits, 3, r)
    (want,) = torch.autograd.grad(w, x, g, retain_graph=True)
    with torch.no_grad():
        logits.zero_()
    if r.score == "softmax" and not r.renormalize:
        with pytest.raises(RuntimeError, match="modified"):
            torch.autograd.grad(w, x, g)
    else:
        assert torch.equal(torch.autograd.grad(w, x, g)[0], want)


def test_logits_are_not_held_for_a_gradient_that_does_not_read_them():
    x = torch.zeros(1 << 14, 1 << 10, device=DEV, requires_grad=True)  # 64 MiB
    for r, held in ((RULES[0], False), (RULES[1], False), (RULES[3], True)):
        before = torch.cuda.memory_allocated()
        w, _ = fm.route_tokens(x * 1, 2, r)
        assert (torch.cuda.memory_allocated() - before > 1 << 25) == held
        assert torch.autograd.grad(w.sum(), x)[0].shape == x.shape
        del w, _


@pytest.mark.parametrize("r", RULES, ids=str)
@pytest.mark.parametrize("leaf", [True, False])
def test_a_second_derivative_is_refused_by_every_rule(r, leaf):
    x = _logits(6, 10, torch.float32).to(DEV).requires_grad_(True)
    w, _ = fm.route_tokens(x if leaf else x * 1, 3, r)
    (d,) = torch.autograd.grad(w, x, torch.randn(6, 3, device=DEV), create_graph=True)
    assert d.requires_grad
    with pytest.raises(RuntimeError, match="no gradient of its own"):
        d.square().sum().backward()
    g = torch.randn(6, 3, device=DEV, requires_grad=True)
    with pytest.raises(RuntimeError, match="no gradient of its own"):
        torch.autograd.grad(w, x, g, create_graph=True)
