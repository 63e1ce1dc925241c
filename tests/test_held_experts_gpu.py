"""What the experts with held activations keep in memory, and what they compute without a backward."""
from __future__ import annotations

import pytest
import torch

import fastmoe_amd as fm

pytestmark = pytest.mark.gpu


def rand(*shape, dtype=torch.float32, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def peak_of(call):
    """(the call's result, the largest memory in use during it beyond what was before)"""
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    out = call()
    return out, torch.cuda.max_memory_allocated() - before


def test_intermediate_results_are_released():
    """Forward: the first product and GELU's output (2 H bytes each) with the 8-bit rows (H and scales),
    then without the first product, but with the outputs (2 D) and the rows in 8 bits (D and scales).
    Backward: GELU's output, its gradient and the gradient that it reads; then the first two with the
    rows, their gradient (2 D each) and the weights' gradients."""
    D, H, N = 1024, 2048, 16384
    moe = fm.MoEFeedForward(D, H, 4, 1).cuda().bfloat16()
    x = rand(N, D, dtype=torch.bfloat16).requires_grad_(True)
    warm = fm.compute_experts(moe.experts, x, [N // 4] * 4, checkpoint="int8")  # the library's workspace
    torch.autograd.grad(warm, x, [torch.ones_like(o) for o in warm])
    del warm
    outs, peak = peak_of(lambda: fm.compute_experts(moe.experts, x, [N // 4] * 4, checkpoint="int8"))
    held = N * (H + D) * (1 + 4 / 128)
    assert peak <= 1.01 * max(N * 5 * H + N * H * 4 / 128, held + N * (2 * H + 2 * D)), peak / N / H
    grads = [torch.ones_like(o) for o in outs]
    leaves = [x, *moe.experts.parameters()]
    weights = sum(2 * p.numel() for p in moe.experts.parameters())
    got, peak = peak_of(lambda: torch.autograd.grad(outs, leaves, grads))
    assert all(g is not None for g in got)
    assert peak <= 1.01 * max(N * 6 * H, N * 4 * H + N * 4 * D + weights), peak / N / H
