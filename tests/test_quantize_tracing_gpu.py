"""Recording a program does not turn the 8-bit operators' results into constants: the calls refuse."""
from __future__ import annotations

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

import fastmoe_amd as fm

pytestmark = pytest.mark.gpu


def rand(*shape, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda")


def calls():
    """Every operator as a function of one tensor [4, 256] and its example."""
    x, w = rand(4, 256), rand(256, seed=1)
    q, held, weights = fm.quantize_rows(x), fm.compress_rows(x), fm.quantize_weights(rand(8, 256, seed=2))
    return x, {
        "add_rms_norm": lambda t: fm.add_rms_norm(t, w)[0],
        "add_rms_norm_int8": lambda t: fm.add_rms_norm_int8(t, w).normed,
        "quantize_rows": lambda t: fm.quantize_rows(t).data,
        "dequantize": lambda t: q._replace(scales=t[:, 0].contiguous()).dequantize(),
        "int8_linear": lambda t: fm.int8_linear(q._replace(scales=t[:, 0].contiguous()), weights),
        "compress_rows": lambda t: fm.compress_rows(t).data,
        "restore_rows": lambda t: fm.restore_rows(held._replace(scales=t[:, :2].contiguous()),
                                                  torch.float32),
        "gelu_compress": lambda t: fm.gelu_compress(t)[0],
        "gelu_compressed_backward": lambda t: fm.gelu_compressed_backward(held, t)[1],
    }


NAMES = ["add_rms_norm", "add_rms_norm_int8", "quantize_rows", "dequantize", "int8_linear", "compress_rows",
         "restore_rows", "gelu_compress", "gelu_compressed_backward"]


@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("name", NAMES)
def test_an_operator_is_not_recorded(name):
    x, every = calls()
    assert sorted(every) == sorted(NAMES)
    call = every[name]
    want = call(x)
    with pytest.raises(RuntimeError, match="tracing"):
        torch.jit.trace(call, (x,))
    with pytest.raises(RuntimeError, match="tracing"):
        make_fx(call)(x)
    assert torch.equal(call(x), want)


@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("normed", [False, True])
def test_the_serving_layer_is_not_recorded(normed):
    moe = fm.MoEFeedForward(128, 64, 4, 2).cuda()
    layer = (fm.NormedMoEFeedForward(moe) if normed else moe).int8()
    x = rand(1, 6, 128)
    with pytest.raises(RuntimeError, match="tracing"):
        torch.jit.trace(layer, (x,))
    with torch.no_grad(), pytest.raises(RuntimeError, match="tracing"):
        make_fx(layer)(x)


@pytest.mark.filterwarnings("ignore")
def test_held_experts_are_not_recorded():
    class Held(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.experts = fm.MoEFeedForward(128, 64, 2, 1).cuda().experts

        def forward(self, t):
            return fm.compute_experts(self.experts, t, [3, 3], checkpoint="int8")[0]

    with pytest.raises(RuntimeError, match="tracing"):
        torch.jit.trace(Held(), (rand(6, 128),))


def test_compiled_calls_run():
    """The compiler breaks its graph at the calls and runs them as they are."""
    w = rand(256, seed=1)
    f = torch.compile(lambda t: fm.quantize_rows(fm.add_rms_norm(t * 2, w)[0]).dequantize() + 1,
                      backend="eager")
    for seed in (0, 5):
        x = rand(4, 256, seed=seed)
        assert torch.equal(f(x), fm.quantize_rows(fm.add_rms_norm(x * 2, w)[0]).dequantize() + 1)
