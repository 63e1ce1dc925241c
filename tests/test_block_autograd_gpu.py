"""The router and the norms around a block under autograd's own tools (hooks on saved tensors, anomaly detection, activation
checkpointing, threads, autocast, the compiler), and all of a block's operators under tracing and transforms."""
from __future__ import annotations

import threading

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils.checkpoint import checkpoint

import fastmoe_amd as fm

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
T, D, E, G = 60, 200, 24, 3
RULES = [fm.Routing("sigmoid", 4, 2, "top2", scale=2.5), fm.Routing(renormalize=False)]


def rand(*shape, dtype=torch.float32, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def leaves_of(dtype=torch.float32):
    shapes = [(T, D), (D,), (T, D), (D,), (G, D), (T, E)]  # x, post, residual, pre, gate, logits
    return [rand(*s, dtype=dtype, seed=i).requires_grad_(True) for i, s in enumerate(shapes)]


def step(x, post, residual, pre, gate, logits, rule):
    y, h = fm.sandwich_norm(x, post, residual, pre, gate=gate, scale=0.5)
    w, ids = fm.route_tokens(logits, 3, rule)
    return (y * w.sum(-1, keepdim=True) + h * w[:, :1]).float()


def grads_of(rule, seed=7, around=None, dtype=torch.float32):
    leaves = leaves_of(dtype)
    out = around(leaves) if around else step(*leaves, rule)
    return torch.autograd.grad(out, leaves, rand(T, D, seed=seed))


def same(a, b):
    return all(torch.equal(p, q) for p, q in zip(a, b)) and len(a) == len(b)


@pytest.mark.parametrize("rule", RULES, ids=str)
def test_saved_tensors_on_the_host_anomaly_detection_and_checkpointing(rule):
    want = grads_of(rule)

    def on_host(leaves):
        with torch.autograd.graph.save_on_cpu():
            return step(*leaves, rule)

    assert same(grads_of(rule, around=on_host), want)
    with torch.autograd.detect_anomaly(check_nan=True):
        assert same(grads_of(rule), want)
    assert same(grads_of(rule, around=lambda ls: checkpoint(step, *ls, rule, use_reentrant=False)), want)
    leaves = leaves_of()
    checkpoint(step, *leaves, rule, use_reentrant=True).backward(rand(T, D, seed=7))
    assert same([t.grad for t in leaves], want)


@pytest.mark.parametrize("rule", RULES, ids=str)
def test_a_retained_graph_gives_the_same_again(rule):
    leaves, g = leaves_of(), rand(T, D, seed=7)
    out = step(*leaves, rule)
    a = torch.autograd.grad(out, leaves, g, retain_graph=True)
    assert same(a, torch.autograd.grad(out, leaves, g))
    with pytest.raises(RuntimeError, match="second time|freed"):
        torch.autograd.grad(out, leaves, g)


@pytest.mark.parametrize("call", ["route", "sandwich"])
def test_a_hook_that_raises_is_heard(call):
    x, post, residual, pre, gate, logits = leaves_of()

    def run():
        if call == "route":
            return fm.route_tokens(logits, 3, RULES[1])[0]
        return fm.sandwich_norm(x, post, residual, pre, gate=gate)[0]

    def refuse(t):
        raise KeyError("from the hook")

    with torch.autograd.graph.saved_tensors_hooks(refuse, lambda t: t):
        with pytest.raises(KeyError, match="from the hook"):
            run()
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, refuse):
        out = run()
    with pytest.raises(KeyError, match="from the hook"):
        out.sum().backward()
    leaf = logits if call == "route" else x
    assert torch.autograd.grad(run().sum(), leaf)[0].isfinite().all()  # and leaves nothing behind


def test_several_threads():
    """Each on its own stream, forward and backward."""
    want = [grads_of(r) for r in RULES]
    torch.cuda.synchronize()
    got, errors = {}, []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(5):
                    got[i] = grads_of(RULES[i % 2])
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert not errors and len(got) == 4
    assert all(same(got[i], want[i % 2]) for i in got)


@pytest.mark.parametrize("rule", RULES, ids=str)
def test_autocast_leaves_the_operators_alone(rule):
    """They have no casts of their own: under autocast they run in their inputs' types."""
    want = grads_of(rule, dtype=torch.bfloat16)

    def cast(leaves):
        with torch.autocast("cuda", torch.bfloat16):
            y, h = fm.sandwich_norm(*leaves[:4], gate=leaves[4], scale=0.5)
            w, _ = fm.route_tokens(leaves[5], 3, rule)
            assert y.dtype == h.dtype == w.dtype == torch.bfloat16
            with torch.autocast("cuda", enabled=False):
                return step(*leaves, rule)

    assert same(grads_of(rule, around=cast, dtype=torch.bfloat16), want)


@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("rule", RULES, ids=str)
def test_a_layer_under_autocast(rule):
    """Products in bfloat16, the router's logits with them; the layer's own parameters are float32."""
    torch.manual_seed(0)
    moe = fm.MoEFeedForward(64, 32, 8, 2, routing=fm.Routing("sigmoid") if rule is RULES[0] else rule).cuda()
    x = rand(2, 30, 64).requires_grad_(True)
    with torch.autocast("cuda", torch.bfloat16):
        out = moe(x)
    grads = torch.autograd.grad(out.float().square().sum(), [x, moe.router.weight])
    assert all(g.isfinite().all() and g.any() for g in grads)
    plain = moe(x)
    assert float((out - plain).norm() / plain.norm()) < 0.1


@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("rule", RULES, ids=str)
def test_a_compiled_training_step(rule):
    """The compiler breaks its graph at the operators and differentiates around them."""
    leaves = leaves_of()
    f = lambda *ls: torch.tanh(step(*(t * 2 for t in ls), rule)).sum()  # noqa: E731
    want = torch.autograd.grad(f(*leaves), leaves)
    got = torch.autograd.grad(torch.compile(f, backend="eager")(*leaves), leaves)
    assert same(got, want)


def calls():
    """Every operator as a function of one float tensor [8, 256], and that tensor."""
    x, w = rand(8, 256, dtype=torch.bfloat16), rand(256, seed=1, dtype=torch.bfloat16)
    q = fm.quantize_weights_fp4(rand(16, 256, seed=2))
    return x, {
        "route_tokens": lambda t: fm.route_tokens(t, 3)[0],
        "sandwich_norm": lambda t: fm.sandwich_norm(t, w, x, w)[0],
        "quantize_weights_fp4": lambda t: fm.quantize_weights_fp4(t).data,
        "dequantize": lambda t: q._replace(scales=q.scales + 0 * t[0, 0].to(torch.uint8)).dequantize(),
        "fp4_linear": lambda t: fm.fp4_linear(t, q),
    }


NAMES = ["route_tokens", "sandwich_norm", "quantize_weights_fp4", "dequantize", "fp4_linear"]


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
@pytest.mark.parametrize("name", NAMES)
def test_transforms_are_refused(name):
    x, every = calls()
    call = every[name]
    several = torch.stack([x, x])
    for transform in (lambda: torch.func.vmap(call)(several), lambda: torch.func.jvp(call, (x,), (x,)),
                      lambda: torch.func.grad(lambda t: call(t).float().sum())(x)):
        with pytest.raises((RuntimeError, ValueError)):
            transform()
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, x)
        if name == "quantize_weights_fp4":  # gradients stay out of it, as they do in a backward
            assert torch.equal(call(dual), call(x))
        elif name != "dequantize":  # whole numbers, which have no tangent
            with pytest.raises((RuntimeError, ValueError), match="fastmoe_amd"):
                call(dual)
    assert call(x).shape  # and leaves nothing behind


@pytest.mark.filterwarnings("ignore")
def test_compiled_serving_calls_run():
    x, every = calls()
    for name in NAMES:
        if name == "dequantize":
            continue
        with torch.no_grad():
            assert torch.equal(torch.compile(every[name], backend="eager")(x), every[name](x)), name
