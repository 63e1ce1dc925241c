"""The norm and the held experts under autograd's own tools: hooks on saved tensors, anomaly detection,
retained graphs, several threads, compiled training steps."""
from __future__ import annotations

import threading

import pytest
import torch

import fastmoe_amd as fm

from .test_norm_quantize_gpu import rand

pytestmark = pytest.mark.gpu


def leaves_of(dtype=torch.float32):
    return [rand(*s, dtype=dtype, seed=i).requires_grad_(True) for i, s in enumerate([(70, 200), (200,), (70, 200)])]


def step(x, w, r, moe):
    y, h = fm.add_rms_norm(x, w, r)
    outs = fm.compute_experts(moe.experts, y, [30, 40], checkpoint="int8")
    return torch.cat(outs) + h


@pytest.fixture(scope="module")
def moe():
    torch.manual_seed(0)
    return fm.MoEFeedForward(200, 96, 2, 1).cuda()


def test_saved_tensors_on_the_host_and_anomaly_detection(moe):
    leaves, g = leaves_of(), rand(70, 200, seed=7)
    want = torch.autograd.grad(step(*leaves, moe), leaves, g)
    with torch.autograd.graph.save_on_cpu():
        out = step(*leaves, moe)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, leaves, g), want))
    with torch.autograd.detect_anomaly(check_nan=True):
        got = torch.autograd.grad(step(*leaves, moe), leaves, g)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_a_hook_that_raises_is_heard():
    x, w, r = leaves_of()

    def refuse(t):
        raise KeyError("from the hook")

    with torch.autograd.graph.saved_tensors_hooks(refuse, lambda t: t):
        with pytest.raises(KeyError, match="from the hook"):
            fm.add_rms_norm(x, w, r)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, refuse):
        y, _ = fm.add_rms_norm(x, w, r)
    with pytest.raises(KeyError, match="from the hook"):
        y.sum().backward()
    y, _ = fm.add_rms_norm(x, w, r)  # and leaves nothing behind
    assert torch.autograd.grad(y.sum(), x)[0].isfinite().all()


def test_a_retained_graph_gives_the_same_again(moe):
    leaves, g = leaves_of(), rand(70, 200, seed=7)
    out = step(*leaves, moe)
    a = torch.autograd.grad(out, leaves, g, retain_graph=True)
    b = torch.autograd.grad(out, leaves, g)
    assert all(torch.equal(u, v) for u, v in zip(a, b))


def test_several_threads(moe):
    """Each on its own stream, forward and backward."""
    want = torch.autograd.grad(step(*(ls := leaves_of()), moe), ls, rand(70, 200, seed=7))
    torch.cuda.synchronize()
    got, errors = {}, []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(5):
                    ls = leaves_of()
                    got[i] = torch.autograd.grad(step(*ls, moe), ls, rand(70, 200, seed=7))
                    fm.quantize_rows(ls[0].detach(), activation="gelu").dequantize()
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert not errors and len(got) == 4
    for grads in got.values():
        assert all(torch.equal(a, b) for a, b in zip(grads, want))


@pytest.mark.filterwarnings("ignore")
def test_a_compiled_training_step():
    """The compiler breaks its graph at the norm and differentiates around it."""
    x, w, r = leaves_of()
    f = lambda a, b, c: torch.tanh(fm.add_rms_norm(a * 2, b, c)[0]).sum()  # noqa: E731
    want = torch.autograd.grad(f(x, w, r), [x, w, r])
    got = torch.autograd.grad(torch.compile(f, backend="eager")(x, w, r), [x, w, r])
    assert all(torch.equal(a, b) for a, b in zip(got, want))
