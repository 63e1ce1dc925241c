"""Uses of the layers on the router, the 4-bit products and the norms around a block: parameters of other types, empty
batches, routers in place."""
from __future__ import annotations

import pytest
import torch
import torch.nn as nn

import fastmoe_amd as fm

from .test_block_layers_gpu import DEV, layer, rand

pytestmark = pytest.mark.gpu


def fp32_parameters(block, seed):
    """The block's own parameters in float32, with values that 16 bits do not hold."""
    for i, (name, p) in enumerate(list(block.named_parameters(recurse=False))):
        setattr(block, name, nn.Parameter(1 + 0.1 * rand(*p.shape, seed=seed + i)))
    return block


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_norms_in_fp32_stay_so_in_4_bits(dtype):
    D, eps = 128, 1e-6
    x, r = rand(2, 9, D, dtype=dtype, seed=1), rand(2, 9, D, dtype=dtype, seed=2)
    flat, rows = x.view(-1, D), r.view(-1, D)
    block = fp32_parameters(fm.NormedMoEFeedForward(layer(D, 64, 4, 2, dtype)).cuda(), 3)
    served = block.fp4()
    assert served.norm_weight.dtype == torch.float32 and torch.equal(served.norm_weight, block.norm_weight)
    assert served.norm_weight.data_ptr() != block.norm_weight.data_ptr() and not served.norm_weight.requires_grad
    with torch.no_grad():
        out, stream = served(x, r)
        y, h = fm.add_rms_norm(flat, block.norm_weight, rows, eps=eps)
        assert torch.equal(stream.view(-1, D), h) and torch.equal(out, block.moe.fp4()(y.view(x.shape)))
    for gated in (False, True):
        block = fp32_parameters(fm.SandwichMoEFeedForward(layer(D, 64, 4, 2, dtype), scale=0.5, gated=gated).cuda(), 5)
        served = block.fp4()
        own, kept = dict(block.named_parameters(recurse=False)), dict(served.named_parameters(recurse=False))
        assert own.keys() == kept.keys() == {"norm_weight", "post_weight"} | ({"gate"} if gated else set())
        for name, p in own.items():
            assert kept[name].dtype == torch.float32 and torch.equal(kept[name], p) and not kept[name].requires_grad
        with torch.no_grad():
            h, y = served(x, next_weight=block.norm_weight)
            normed = fm.add_rms_norm(flat, block.norm_weight, eps=eps)[0]
            out = block.moe.fp4()(normed.view(x.shape)).view(-1, D)
            want_y, want_h = fm.sandwich_norm(out, block.post_weight, flat, block.norm_weight, gate=block.gate, scale=0.5,
                                              eps=eps)
            assert torch.equal(h.view(-1, D), want_h) and torch.equal(y.view(-1, D), want_y)


def test_a_parameter_used_twice_is_copied_twice():
    block = fm.SandwichMoEFeedForward(layer(64, 32, 4, 2)).cuda()
    block.post_weight = block.norm_weight
    with torch.no_grad():
        block.norm_weight.copy_(rand(64))
    served = block.fp4()
    assert torch.equal(served.post_weight, block.norm_weight) and torch.equal(served.norm_weight, block.norm_weight)


@pytest.mark.parametrize("B,T", [(0, 5), (3, 0)])
def test_an_empty_batch_with_a_gate_for_each_sequence(B, T):
    D = 64
    block = fm.SandwichMoEFeedForward(layer(D, 32, 4, 2)).cuda()
    gate = rand(B, D, dtype=torch.bfloat16).requires_grad_(True)
    x = rand(B, T, D, dtype=torch.bfloat16).requires_grad_(True)
    h, y = block(x, gate=gate, next_weight=block.norm_weight)
    assert h.shape == y.shape == (B, T, D)
    leaves = [x, gate, block.post_weight, block.norm_weight]
    for t, g in zip(leaves, torch.autograd.grad([h, y], leaves, [torch.zeros_like(h), torch.zeros_like(y)])):
        assert g.shape == t.shape and g.dtype == t.dtype and not g.any()
    many = rand(4, D, dtype=torch.bfloat16)
    with torch.no_grad():
        h, y = block.fp4()(x, gate=many[:B], next_weight=block.norm_weight)
    assert h.shape == y.shape == (B, T, D)
    with pytest.raises(ValueError, match="gate"):  # no gate for the rows that there are
        fm.sandwich_norm(rand(6, D), rand(D), rand(6, D), gate=rand(0, D))
