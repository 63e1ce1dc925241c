"""Uses of the 8-bit layer and operators together: captured, on several streams, under autocast, with more
experts than rows and with rows behind the last expert's."""
from __future__ import annotations

import pytest
import torch

import fastmoe_amd as fm

from .test_int8_linear_gpu import check, make, reference, route
from .test_norm_quantize_gpu import rand

pytestmark = pytest.mark.gpu


def capture(call):
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = call()
    return g, out


def test_held_rows_in_a_graph():
    """Every call on held activations, captured without a backward, replayed on new rows."""
    moe = fm.MoEFeedForward(200, 96, 3, 1).cuda().bfloat16()
    x = rand(50, 200, dtype=torch.bfloat16)

    def call():
        with torch.no_grad():
            a, held = fm.gelu_compress(x)
            again, grad = fm.gelu_compressed_backward(held, x)
            return [a, held.data, held.scales, again, grad, fm.restore_rows(fm.compress_rows(x), torch.float32),
                    *fm.compute_experts(moe.experts, x, [20, 0, 30], checkpoint="int8")]

    g, out = capture(call)
    for seed in (3, 4, 5):
        x.copy_(rand(50, 200, dtype=torch.bfloat16, seed=seed))
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, call()):
            assert torch.equal(a, b)


def test_two_graphs_of_one_layer_replayed_in_turn():
    """Two batch sizes of one serving layer, each in its graph, with eager calls between them."""
    torch.manual_seed(0)
    block = fm.NormedMoEFeedForward(fm.MoEFeedForward(128, 64, 8, 2)).cuda().bfloat16().int8()
    xs = [rand(1, n, 128, dtype=torch.bfloat16, seed=n) for n in (3, 70)]
    graphs = [capture(lambda x=x: block(x, x)) for x in xs]
    for seed in range(3):
        for x in xs:
            x.copy_(rand(*x.shape, dtype=torch.bfloat16, seed=20 + seed))
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for (_, (out, stream)), x in zip(graphs, xs):
            want, want_stream = block(x, x)
            assert torch.equal(out, want) and torch.equal(stream, want_stream)


def test_one_layer_on_two_streams():
    torch.manual_seed(0)
    layer = fm.MoEFeedForward(256, 128, 8, 2).cuda().bfloat16().int8()
    xs = [rand(2, n, 256, dtype=torch.bfloat16, seed=n) for n in (5, 300)]
    want = [layer(x) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        got = []
        for s, x in zip(streams, xs):
            with torch.cuda.stream(s):
                got.append(layer(x))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_a_single_token_of_many_experts_and_every_token_to_one():
    torch.manual_seed(0)
    moe = fm.MoEFeedForward(64, 32, 300, 8).cuda().bfloat16()
    layer = moe.int8()
    x = rand(1, 1, 64, dtype=torch.bfloat16)
    with torch.no_grad():
        ref = moe(x).float()
        assert (layer(x).float() - ref).norm() <= 0.05 * ref.norm()
    moe = fm.MoEFeedForward(64, 32, 5, 1).cuda().bfloat16()
    with torch.no_grad():
        moe.router.weight.zero_()
        moe.router.weight[3] = 1
        x = rand(1, 200, 64, dtype=torch.bfloat16).abs()
        ref = moe(x).float()
        assert (moe.int8()(x).float() - ref).norm() <= 0.05 * ref.norm()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_under_autocast(dtype):
    """fp32 layers under autocast: the router's logits come in the autocast type, rows stay in theirs."""
    torch.manual_seed(0)
    block = fm.NormedMoEFeedForward(fm.MoEFeedForward(128, 96, 4, 2)).cuda()
    layer, x = block.int8(), rand(2, 30, 128)
    with torch.no_grad(), torch.autocast("cuda", dtype=dtype):
        out, stream = layer(x)
        want, _ = block(x)
    assert out.dtype == torch.float32 and torch.equal(stream, x)
    # a token whose second and third logits tie in 16 bits may go elsewhere; most do not
    off = (out - want.float()).norm(dim=-1) / want.float().norm(dim=-1)
    assert off.median() <= 0.05


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("K,N", [(64, 33), (300, 257)])
def test_rows_behind_the_last_of_many_experts(K, N, dtype):
    """More experts than one scan takes (256), rows of none behind them, and indices outside."""
    counts = [(5 * e) % 7 if e % 3 else 0 for e in range(1000)] + [0] * 25 + [40]
    R = sum(counts) + 333
    x, w = make(90, K, len(counts), N)
    rows = torch.arange(R, device="cuda") * 7 % 94 - 2
    bias = torch.randn(len(counts), N, device="cuda")
    got = fm.int8_linear(x, w, route(counts), rows=rows, bias=bias, out_dtype=dtype)
    check(got, *reference(x, w, counts, rows, bias), dtype)
    assert not got[sum(counts):].any()


def test_a_captured_product_whose_rows_come_and_go():
    """Replays with all rows to one expert, with none to any, and even: each as the eager call gives it."""
    x, w = make(64, 512, 6, 300)
    off = route([64, 0, 0, 0, 0, 0])
    g, out = capture(lambda: fm.int8_linear(x, w, off))
    for counts in ([0] * 6, [10, 11, 10, 11, 11, 11], [0, 0, 0, 0, 0, 64], [1, 0, 0, 0, 0, 2]):
        off.copy_(route(counts))
        out.fill_(7)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, fm.int8_linear(x, w, off))
        assert not out[sum(counts):].any()
