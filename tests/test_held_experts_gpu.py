"""What the experts with held activations keep in memory, and what they compute without a backward."""
from __future__ import annotations

import pytest
import torch

import fastmoe_amd as fm
from fastmoe_amd import _abi
from fastmoe_amd.ops import _stream_handle

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


@pytest.mark.parametrize("frozen", [False, True])
def test_nothing_is_held_without_a_backward(frozen):
    """The largest memory in use is that of the first product and GELU's output, 4 H bytes a row; H more
    would be the 8-bit rows."""
    D, H, N = 1024, 2048, 16384
    moe = fm.MoEFeedForward(D, H, 4, 1).cuda().bfloat16()
    x, counts = rand(N, D, dtype=torch.bfloat16), [N // 4] * 4
    want = fm.compute_experts(moe.experts, x, counts, checkpoint="int8")
    assert want[0].requires_grad
    want = [o.detach() for o in want]
    if frozen:
        moe.requires_grad_(False)
    with torch.set_grad_enabled(frozen):
        got, peak = peak_of(lambda: fm.compute_experts(moe.experts, x, counts, checkpoint="int8"))
    assert peak <= 4.04 * N * H, peak / (N * H)
    for a, b in zip(got, want):
        assert torch.equal(a, b) and not a.requires_grad
    with torch.inference_mode():
        for a, b in zip(fm.compute_experts(moe.experts, x, counts, checkpoint="int8"), want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("R,C", [(1, 1), (33, 200), (5, 2049), (300, 384)])
def test_gelu_alone_has_the_same_bits(R, C, dtype):
    x = rand(R, C, dtype=dtype) * 2
    want, _ = fm.gelu_compress(x)
    code = {torch.float32: _abi.F32, torch.bfloat16: _abi.BF16, torch.float16: _abi.F16}[dtype]
    got = torch.full_like(x, 7)
    assert _abi.lib().fmoe_compress_rows(x.data_ptr(), C, R, C, code, None, 0, None, got.data_ptr(),
                                         _stream_handle(x.device)) == 0
    assert torch.equal(got, want)


def test_a_call_after_one_without_a_backward_records():
    moe = fm.MoEFeedForward(64, 96, 2, 1).cuda()
    x = rand(8, 64).requires_grad_(True)
    with torch.no_grad():
        free = fm.compute_experts(moe.experts, x, [4, 4], checkpoint="int8")
    outs = fm.compute_experts(moe.experts, x, [4, 4], checkpoint="int8")
    assert all(torch.equal(a, b) for a, b in zip(free, outs))
    torch.cat(outs).sum().backward()
    assert x.grad.isfinite().all() and all(p.grad is not None for p in moe.experts.parameters())
