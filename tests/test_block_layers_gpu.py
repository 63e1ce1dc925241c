"""The router, the 4-bit products and the norms around a block run together: layers, blocks, graphs."""
from __future__ import annotations

import copy

import pytest
import torch
import torch.nn as nn

import fastmoe_amd as fm
from tests import route_ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
GROUPED = fm.Routing("sigmoid", 4, 2, "top2", scale=2.5)


def layer(dim, ff, E, k, dtype=torch.bfloat16, seed=0, bias=False, **kw):
    torch.manual_seed(seed)
    moe = fm.MoEFeedForward(dim, ff, E, k, **kw)
    if bias:
        for e in moe.experts:
            e[0].bias = nn.Parameter(torch.randn(ff) * 0.1)
            e[2].bias = nn.Parameter(torch.randn(dim) * 0.1)
    return moe.cuda().to(dtype)


def rand(*shape, dtype=torch.float32, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def plain_layer(moe, x, routing, bias=None):
    """The layer by torch's operators alone; experts chosen by the definition."""
    flat = x.reshape(-1, x.shape[-1])
    logits = moe.router(flat)
    ids = route_ref.choose(logits.detach().cpu(), moe.top_k, routing, bias).to(DEV)
    w = (route_ref.shares(logits, ids, routing) * routing.scale).to(flat.dtype)
    out = torch.zeros_like(flat)
    for e, expert in enumerate(moe.experts):
        token, slot = (ids == e).nonzero(as_tuple=True)
        if len(token):
            out = out.index_add(0, token, expert(flat[token]) * w[token, slot].unsqueeze(1))
    return out.view(x.shape)


@pytest.mark.parametrize("routing", [fm.Routing(), fm.Routing("softmax", renormalize=False), GROUPED], ids=str)
def test_layer_trains_with_a_routing(routing):
    """fp32: values and gradients are those of torch's operators up to the order of sums of at most 64 terms
    through two products (1e-4 of sizes near 1)."""
    moe = layer(48, 32, 8, 3, torch.float32, routing=routing, balance=routing is GROUPED)
    if moe.balance_bias is not None:
        moe.balance_bias.copy_(0.05 * rand(8, seed=4))
    x = rand(2, 30, 48, seed=1).requires_grad_(True)
    out = moe(x)
    want = plain_layer(moe, x, routing, None if moe.balance_bias is None else moe.balance_bias.cpu())
    assert (out - want).abs().max() < 1e-4
    g = rand(2, 30, 48, seed=2)
    leaves = [x, *moe.parameters()]
    got = torch.autograd.grad(out, leaves, g, allow_unused=True)
    ref = torch.autograd.grad(want, leaves, g, allow_unused=True)
    for a, b in zip(got, ref):
        if b is not None:
            assert (a - b).abs().max() < 1e-3 * (1 + float(b.abs().max()))
    if moe.balance_bias is not None:
        assert int(moe.expert_load.sum()) == 60 * 3
        # int8-held activations take the same route
        held = copy.deepcopy(moe)
        held.checkpoint = "int8"
        assert (held(x) - out).abs().max() < 1e-4


def test_default_rule_is_as_it_was():
    """No routing: the chosen are those of torch.topk, as before, and Routing() chooses and weighs alike."""
    moe = layer(64, 32, 8, 2, torch.float32)
    x = rand(1, 50, 64)
    flat = x.view(-1, 64)
    logits = moe.router(flat)
    top, ids = torch.topk(logits, 2, dim=-1)
    six = fm.gate_and_sort(x, moe.router, 2, 8)
    p = fm.permute_tokens(flat, ids, torch.softmax(top, -1, dtype=torch.float32), 8)
    assert torch.equal(six[3], p.reverse_map_indices) and torch.equal(six[4], p.sorted_weights)
    routed = fm.gate_and_sort(x, moe.router, 2, 8, routing=fm.Routing())
    assert torch.equal(routed[3], p.reverse_map_indices)
    assert (routed[4] - p.sorted_weights).abs().max() < 2.0 ** -21
    with pytest.raises(ValueError, match="routing"):
        fm.gate_and_sort(x, moe.router, 2, 8, bias=torch.zeros(8, device=DEV))


def test_balance_moves_the_bias_against_the_load():
    moe = layer(32, 16, 6, 2, routing=fm.Routing("sigmoid"), balance=True)
    assert moe.balance_bias.dtype == torch.float32  # through .to(bfloat16)
    with torch.no_grad():
        moe.router.weight.zero_()
        moe.router.weight[1] = 0.01
    x = torch.ones(1, 40, 32, device=DEV, dtype=torch.bfloat16)
    moe(x)
    assert moe.expert_load.tolist() == [40, 40, 0, 0, 0, 0]  # equal scores go to the lowest index
    moe.update_balance(0.25)
    assert moe.balance_bias.tolist() == [-0.25, -0.25, 0.25, 0.25, 0.25, 0.25]
    assert not moe.expert_load.any()
    moe.eval()
    moe(x)
    assert not moe.expert_load.any()
    assert fm.gate_and_sort(x, moe.router, 2, 6, routing=moe.routing, bias=moe.balance_bias)[2].tolist() == \
        [[0, 0, 40, 40, 0, 0]]
    kept = copy.deepcopy(moe).half()
    assert torch.equal(kept.balance_bias, moe.balance_bias) and kept.balance_bias.dtype == torch.float32
    with pytest.raises(ValueError, match="without balance"):
        layer(32, 16, 6, 2).update_balance()


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,T,dim,ff,E,k,routing", [
    (1, 1, 64, 32, 4, 2, None), (2, 33, 200, 72, 8, 3, GROUPED), (4, 300, 256, 512, 8, 2, fm.Routing()),
    (1, 2048, 128, 256, 16, 4, GROUPED)])
def test_fp4_layer_is_its_calls(B, T, dim, ff, E, k, routing, dtype, bias):
    moe = layer(dim, ff, E, k, dtype, bias=bias, routing=routing, balance=routing is GROUPED)
    if moe.balance_bias is not None:
        moe.balance_bias.copy_(0.05 * rand(E, seed=4))
    x = rand(B, T, dim, dtype=dtype, seed=1)
    flat = x.view(-1, dim)
    with torch.no_grad():
        logits = moe.router(flat)
        if routing is None:
            top, ids = torch.topk(logits, k, dim=-1)
            gates = torch.softmax(top, -1, dtype=torch.float32).to(dtype)
        else:
            gates, ids = fm.route_tokens(logits, k, routing, bias=moe.balance_bias)
        p = fm.permute_tokens(flat, ids, gates, E)
        w1, w2 = (fm.quantize_weights_fp4([e[i].weight for e in moe.experts]) for i in (0, 2))
        b1, b2 = ([e[i].bias for e in moe.experts] for i in (0, 2))
        b1, b2 = (None if b[0] is None else torch.stack(b) for b in (b1, b2))
        h = fm.fp4_linear(flat, w1, p.expert_offsets, rows=p.reverse_map_indices, bias=b1, activation="gelu")
        y = fm.fp4_linear(h, w2, p.expert_offsets, bias=b2)
        want = fm.weighted_scatter_add(y, p.reverse_map_indices, p.sorted_weights, flat.shape).view(x.shape)
        served = moe.fp4()
        got = served(x)
    assert torch.equal(got, want) and not got.requires_grad
    again = copy.deepcopy(served)
    again.load_state_dict(served.state_dict())
    assert torch.equal(again(x), want)
    assert served(x[:, :0]).shape == (B, 0, dim)


def test_fp4_layer_against_the_layer_it_was_made_of():
    """With weights that 4 bits hold exactly, the two differ by roundings alone: the hidden row and the
    expert's output are each rounded to bf16 once in both, the plain layer's GELU once more."""
    dim, ff, E, k = 128, 96, 6, 2
    moe = layer(dim, ff, E, k, routing=fm.Routing())
    with torch.no_grad():
        for e in moe.experts:
            for i in (0, 2):
                e[i].weight.copy_(fm.quantize_weights_fp4(e[i].weight).dequantize(torch.bfloat16)[0])
    x = rand(1, 100, dim, dtype=torch.bfloat16, seed=3)
    with torch.no_grad():
        got, want = moe.fp4()(x).double(), moe(x).double()
    assert float((got - want).norm() / want.norm()) < 2.0 ** -7


@pytest.mark.parametrize("routing", [None, GROUPED])
def test_int8_layer_keeps_the_routing(routing):
    moe = layer(128, 64, 8, 2, routing=routing, balance=routing is not None)
    if routing is not None:
        moe.balance_bias.copy_(0.5 * rand(8, seed=4))
    x = rand(1, 64, 128, dtype=torch.bfloat16, seed=3)
    with torch.no_grad():
        served = moe.int8()
        got, want = served(x).double(), moe(x).double()
    assert float((got - want).norm() / want.norm()) < 0.05


def block_by_formula(b, stream, gate, next_weight):
    rms = lambda v: v * torch.rsqrt(v.square().mean(-1, keepdim=True) + b.eps)
    out = b.moe(rms(stream) * b.norm_weight)
    term = b.scale * rms(out) * b.post_weight
    if gate is not None:
        term = term * (gate if gate.dim() == 1 else gate.unsqueeze(1))
    h = stream + term
    return h, None if next_weight is None else rms(h) * next_weight


@pytest.mark.parametrize("gated", ["none", "parameter", "sequence"])
def test_blocks_train_in_a_row(gated):
    """Two blocks, the second reading what the first made for it; fp32, to 1e-4 of sizes near 1 (5e-3 of the gradients')."""
    B, T, dim = 3, 20, 96
    blocks = [fm.SandwichMoEFeedForward(layer(dim, 64, 5, 2, torch.float32, seed=i, routing=fm.Routing()), scale=0.5,
                                        gated=gated == "parameter") for i in range(2)]
    with torch.no_grad():
        for i, b in enumerate(blocks):
            for j, p in enumerate(b.parameters(recurse=False)):
                p.copy_(1 + 0.1 * rand(dim, seed=10 * i + j))
    x = rand(B, T, dim, seed=1).requires_grad_(True)
    gate = rand(B, dim, seed=9).requires_grad_(True) if gated == "sequence" else None
    h, y = blocks[0](x, gate=gate, next_weight=blocks[1].norm_weight)
    h2, y2 = blocks[1](h, y, gate=gate)
    assert y2 is None
    w1, wy = block_by_formula(blocks[0], x, gate if gate is not None else blocks[0].gate, blocks[1].norm_weight)
    w2, _ = block_by_formula(blocks[1], w1, gate if gate is not None else blocks[1].gate, None)
    assert (h - w1).abs().max() < 1e-4 and (y - wy).abs().max() < 1e-4 and (h2 - w2).abs().max() < 1e-4
    leaves = [t for t in (x, gate) if t is not None] + [p for b in blocks for p in b.parameters()]
    g = rand(B, T, dim, seed=5)
    got = torch.autograd.grad(h2, leaves, g, allow_unused=True)
    ref = torch.autograd.grad(w2, leaves, g, allow_unused=True)
    for a, b in zip(got, ref):
        assert (a is None) == (b is None)
        if b is not None:
            assert (a - b).abs().max() < 5e-3 * (1 + float(b.abs().max()))
    with pytest.raises(ValueError, match="gate"):
        blocks[0](x, gate=rand(B + 1, dim))
    with pytest.raises(ValueError, match="residual"):
        blocks[0](x, y[:, :5])


def test_served_blocks_in_a_graph():
    """A decoding step of two blocks in 4 bits, captured once and replayed on other tokens."""
    dim, B, T = 256, 4, 1
    blocks = []
    for i in range(2):
        b = fm.SandwichMoEFeedForward(layer(dim, 128, 16, 4, seed=i, routing=GROUPED, balance=True), gated=True)
        b.moe.balance_bias.copy_(0.05 * rand(16, seed=i))
        blocks.append(b.fp4())
        assert not any(p.requires_grad for p in blocks[-1].parameters())

    def run(x):
        h, y = blocks[0](x, next_weight=blocks[1].norm_weight)
        return blocks[1](h, y)[0]

    x = torch.empty(B, T, dim, device=DEV, dtype=torch.bfloat16)
    with torch.no_grad():
        x.copy_(rand(B, T, dim, dtype=torch.bfloat16))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run(x)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run(x)
        for seed in range(4):
            x.copy_(rand(B, T, dim, dtype=torch.bfloat16, seed=seed))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, run(x))


def test_normed_layer_in_4_bits():
    block = fm.NormedMoEFeedForward(layer(128, 64, 4, 2)).cuda()
    with torch.no_grad():
        block.norm_weight.copy_(1 + 0.1 * rand(128))
    x, r = rand(2, 9, 128, dtype=torch.bfloat16, seed=1), rand(2, 9, 128, dtype=torch.bfloat16, seed=2)
    with torch.no_grad():
        out, stream = block.fp4()(x, r)
        y, h = fm.add_rms_norm(x.view(-1, 128), block.norm_weight, r.view(-1, 128))
        assert torch.equal(stream.view(-1, 128), h)
        assert torch.equal(out, block.moe.fp4()(y.view(x.shape)))


def test_layers_that_would_lose_something_are_refused():
    moe = layer(64, 32, 4, 2)
    with pytest.raises(TypeError, match="bfloat16 or float16"):
        layer(64, 32, 4, 2, torch.float32).fp4()

    class Own(fm.MoEFeedForward):
        def forward(self, x):
            return super().forward(x) * 2

    with pytest.raises(TypeError, match="lose"):
        Own(64, 32, 4, 2).cuda().bfloat16().fp4()
    moe.experts[0].register_forward_hook(lambda *a: None)
    with pytest.raises(ValueError, match="hooks"):
        moe.fp4()
    block = fm.SandwichMoEFeedForward(layer(64, 32, 4, 2))
    block.register_forward_hook(lambda *a: None)
    with pytest.raises(ValueError, match="hooks"):
        block.fp4()
    with pytest.raises(ValueError, match="x must be"):
        layer(64, 32, 4, 2).fp4()(torch.zeros(2, 64, device=DEV, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="balance needs"):
        fm.MoEFeedForward(8, 8, 2, 1, balance=True)


def test_layers_without_gradients_say_so():
    x = rand(2, 5, 64, dtype=torch.bfloat16).requires_grad_(True)
    with pytest.raises(RuntimeError, match="no gradient"):
        layer(64, 32, 4, 2).fp4()(x)
    with pytest.raises(RuntimeError, match="no gradient"):
        fm.NormedMoEFeedForward(layer(64, 32, 4, 2)).cuda().fp4()(x)
    for serving in (layer(64, 32, 4, 2).fp4(), layer(64, 32, 4, 2).int8()):
        block = fm.SandwichMoEFeedForward(serving).cuda()
        with pytest.raises(RuntimeError, match="no gradient"):
            block(x)
        with torch.no_grad():
            h, _ = block(x)
        assert not h.requires_grad
        assert torch.equal(h, block.requires_grad_(False)(x.detach())[0])


def test_layers_pickled_without_a_routing():
    moe = layer(64, 32, 4, 2)
    state = {k: v for k, v in moe.__dict__.items() if k != "routing"}
    state["_buffers"] = {}
    old = fm.MoEFeedForward.__new__(fm.MoEFeedForward)
    old.__setstate__(copy.deepcopy(state))
    x = rand(1, 9, 64, dtype=torch.bfloat16)
    assert torch.equal(old(x), moe(x)) and old.state_dict().keys() == moe.state_dict().keys()
    for form in ("int8", "fp4"):
        assert torch.equal(getattr(old, form)()(x), getattr(moe, form)()(x))


def test_an_empty_batch_between_norms():
    block = fm.SandwichMoEFeedForward(layer(64, 32, 4, 2)).cuda()
    h, y = block(rand(0, 5, 64, dtype=torch.bfloat16).requires_grad_(True), next_weight=block.norm_weight)
    assert h.shape == y.shape == (0, 5, 64)
