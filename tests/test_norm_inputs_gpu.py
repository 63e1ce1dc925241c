"""The norm where its inputs are shared, broadcast, empty or computed again."""
from __future__ import annotations

import pytest
import torch
from torch.utils.checkpoint import checkpoint

import fastmoe_amd as fm

from .test_norm_quantize_gpu import U, close, rand

pytestmark = pytest.mark.gpu


def plain(x, w, r=None, eps=1e-6):
    h = x if r is None else x + r
    return h / torch.sqrt((h * h).mean(-1, keepdim=True) + eps) * w, h


def against_64_bits(call, leaves, outs_of):
    """Gradients of sum(c * out) through the kernels in fp32 and through the formula in 64 bits."""
    got_out = outs_of(call, leaves)
    wide = [t.detach().double().requires_grad_(True) for t in leaves]
    want_out = outs_of(plain, wide)
    cs = [rand(*o.shape, seed=30 + i) for i, o in enumerate(got_out)]
    got = torch.autograd.grad(got_out, leaves, cs)
    want = torch.autograd.grad(want_out, wide, [c.double() for c in cs])
    for a, b in zip(got, want):
        assert a.shape == b.shape
        # sums of up to some thousand terms whose sizes are like the result's norm
        assert (a - b).norm() <= 256 * U * b.norm() and (a - b).abs().max() <= 4096 * U * b.abs().max()


def test_x_is_its_own_residual():
    x, w = rand(300, 200).requires_grad_(True), rand(200, seed=1).requires_grad_(True)
    against_64_bits(fm.add_rms_norm, [x, w], lambda f, t: f(t[0], t[1], t[0]))


def test_a_broadcast_row_and_a_broadcast_residual():
    x, w = rand(1, 200).requires_grad_(True), rand(200, seed=1).requires_grad_(True)
    r = rand(40, 200, seed=2).requires_grad_(True)
    against_64_bits(fm.add_rms_norm, [x, w, r], lambda f, t: f(t[0].expand(40, 200), t[1], t[2]))
    against_64_bits(fm.add_rms_norm, [x, w, r], lambda f, t: f(t[2], t[1], t[0].expand(40, 200)))


def test_two_norms_in_a_row_share_the_stream():
    """h of the first is the residual of the second, as in a stack of blocks, and its gradient has two parts."""
    x, w, r = (rand(*s, seed=i).requires_grad_(True) for i, s in enumerate([(70, 300), (300,), (70, 300)]))

    def blocks(f, t):
        y, h = f(t[0], t[1], t[2])
        y2, h2 = f(torch.tanh(y), t[1], h)
        return y2, h2 * 1

    against_64_bits(fm.add_rms_norm, [x, w, r], blocks)


def test_no_rows_have_gradients():
    x, w = torch.empty(0, 64, device="cuda").requires_grad_(True), rand(64).requires_grad_(True)
    r = torch.empty(0, 64, device="cuda").requires_grad_(True)
    for res in (None, r):
        y, h = fm.add_rms_norm(x, w, res)
        gx, gw = torch.autograd.grad(y.sum() + h.sum(), [x, w])
        assert gx.shape == (0, 64) and gw.shape == (64,) and not gw.any()


@pytest.mark.parametrize("reentrant", [False, True])
def test_under_activation_checkpointing(reentrant):
    x, w, r = (rand(*s, seed=i).requires_grad_(True) for i, s in enumerate([(50, 96), (96,), (50, 96)]))
    g = rand(50, 96, seed=9)
    want = torch.autograd.grad(fm.add_rms_norm(x, w, r)[0], [x, w, r], g)
    y, _ = checkpoint(lambda *a: fm.add_rms_norm(*a), x, w, r, use_reentrant=reentrant)
    y.backward(g)
    for t, b in zip((x, w, r), want):
        assert torch.equal(t.grad, b)


def test_held_experts_under_activation_checkpointing():
    moe = fm.MoEFeedForward(64, 96, 2, 1).cuda()
    x, g = rand(8, 64).requires_grad_(True), rand(8, 64, seed=1)
    run = lambda t: torch.cat(fm.compute_experts(moe.experts, t, [3, 5], checkpoint="int8"))
    want = torch.autograd.grad(run(x), [x, *moe.experts.parameters()], g)
    checkpoint(run, x, use_reentrant=False).backward(g)
    for t, b in zip((x, *moe.experts.parameters()), want):
        assert torch.equal(t.grad, b)


def test_a_changed_stream_is_noticed():
    """The backward reads h: changing it in place before is an error, not a wrong gradient."""
    x, w, r = (rand(*s, seed=i).requires_grad_(True) for i, s in enumerate([(4, 32), (32,), (4, 32)]))
    y, h = fm.add_rms_norm(x, w, r)
    with torch.no_grad():
        h.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    y, _ = fm.add_rms_norm(x, w, r)
    with torch.no_grad():
        w.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
