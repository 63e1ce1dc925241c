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
