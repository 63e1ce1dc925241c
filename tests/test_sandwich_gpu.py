"""The norms around a block against their definition in 64 bits.

Tolerances.  A row's sum of squares in fp32 is off by less than 2^-18 of itself (a thread adds at most 32
terms, the rest is a tree), so the norms' factors and what is multiplied by them by less than 2^-18; a
result then has that of the sizes of its terms, and one rounding.  Gradients of rows go through two such
factors and two more sums: 2^-16 of the sizes of their terms.  Column sums add T products in fp32: (T + 64) * 2^-24
more.  y and the gradients are held to the definition at the stream as it is stored.
"""
from __future__ import annotations

import pytest
import torch

import fastmoe_amd as fm

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.float32, torch.bfloat16, torch.float16]
TINY = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -24}
EPS = 1e-6


def _half(dtype):
    return torch.finfo(dtype).eps / 2


def _inputs(T, D, dtype, gates=0, wdtype=None, gdtype=None, pre=True, seed=0):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=gen)
    d = {"x": r(T, D).to(dtype), "residual": r(T, D).to(dtype), "post": (1 + 0.1 * r(D)).to(wdtype or dtype)}
    if pre:
        d["pre"] = (1 + 0.1 * r(D)).to(wdtype or dtype)
    if gates:
        d["gate"] = (0.5 + 0.2 * r(gates, D)).to(gdtype or dtype)
    return d, r(T, D).to(dtype), r(T, D).to(dtype)


def _call(d, scale):
    return fm.sandwich_norm(d["x"], d["post"], d["residual"], d.get("pre"), gate=d.get("gate"), scale=scale, eps=EPS)


def _rms(v):
    return 1 / torch.sqrt((v * v).mean(-1, keepdim=True) + EPS)


def _weights(d, scale):
    T = d["x"].shape[0]
    w = scale * d["post"].double().expand_as(d["x"])
    if "gate" in d:
        gate = d["gate"].double().view(-1, w.shape[1])
        w = w * gate.repeat_interleave(T // gate.shape[0], 0)
    return w


def _check(name, got, want, terms, dtype, more=0.0):
    got = got.double().cpu()
    tol = want.abs() * _half(dtype) + terms * (2.0 ** -16 + more) + TINY[dtype]
    err = (got - want).abs()
    assert bool((err <= tol).all()), (name, float((err / tol).max()))


def _forward(d, scale, y, h):
    x, r = d["x"].double(), d["residual"].double()
    a = x * _rms(x) * _weights(d, scale)
    _check("h", h, r + a, a.abs() / 4 + r.abs() * 2.0 ** -8, d["x"].dtype)
    if y is not None:
        s = h.double().cpu()
        n = s * _rms(s) * d["pre"].double()
        _check("y", y, n, n.abs() / 4, d["x"].dtype)


def _backward(d, scale, h, gy, gh, grads):
    """Every gradient from the formulas, with the sizes of what is added."""
    dt = d["x"].dtype
    T, D = d["x"].shape
    x, s = d["x"].double(), h.double().cpu()
    cx, ch, w = _rms(x), _rms(s), _weights(d, scale)
    gate = w / d["post"].double()
    zero = torch.zeros(T, D, dtype=torch.double)
    gy = zero if gy is None else gy.double()
    gh = zero if gh is None else gh.double()
    t = gy * d["pre"].double() if "pre" in d else zero
    xh, hh = x * cx, s * ch
    R = gh + ch * (t - hh * (t * hh).mean(-1, keepdim=True))
    RA = gh.abs() + ch * (t.abs() + hh.abs() * (t * hh).abs().mean(-1, keepdim=True))
    gx = cx * (R * w - xh * (R * w * xh).mean(-1, keepdim=True))
    GA = cx * (RA * w.abs() + xh.abs() * (RA * (w * xh).abs()).mean(-1, keepdim=True))
    more = (T + 64) * 2.0 ** -24
    if "residual" in grads:
        _check("residual", grads["residual"], R, RA, dt)
    if "x" in grads:
        _check("x", grads["x"], gx, GA, dt)
    if "pre" in grads:
        _check("pre", grads["pre"], (gy * hh).sum(0), (gy * hh).abs().sum(0), d["pre"].dtype, more)
    if "post" in grads:
        _check("post", grads["post"], (R * gate * xh).sum(0), (RA * gate.abs() * xh.abs()).sum(0), d["post"].dtype, more)
    if "gate" in grads:
        G = d["gate"].numel() // D
        p = scale * d["post"].double()
        fold = lambda v: (v * p.abs()).view(G, -1, D).sum(1)
        want = (R * xh * p).view(G, -1, D).sum(1)
        _check("gate", grads["gate"].view(G, D), want, fold((RA * xh.abs())), d["gate"].dtype, more)


def _whole(d, gy, gh, scale, use=("y", "h")):
    on = {n: t.to(DEV).requires_grad_(True) for n, t in d.items()}
    y, h = _call(on, scale)
    _forward(d, scale, None if y is None else y.detach(), h.detach())
    outs, given = [], []
    if "y" in use and y is not None:
        outs, given = outs + [y], given + [gy.to(DEV)]
    if "h" in use:
        outs, given = outs + [h], given + [gh.to(DEV)]
    got = torch.autograd.grad(outs, list(on.values()), given, allow_unused="y" not in use)
    grads = {n: g for n, g in zip(on, got) if g is not None}
    _backward(d, scale, h.detach(), gy if "y" in use and y is not None else None, gh if "h" in use else None, grads)
    return on, y, h, grads


SHAPES = [(1, 8, 0), (5, 1, 1), (3, 100, 3), (70, 520, 1), (37, 1001, 0), (1, 1024, 1), (130, 1024, 2), (9, 2048, 3),
          (600, 136, 600), (1200, 72, 600), (11, 4096, 1), (8, 5000, 4), (700, 1030, 700), (7, 7168, 1),
          (3, 8192, 0), (6, 9000, 2), (300, 8200, 300), (5, 16384, 1), (4, 16392, 2), (5, 20001, 0), (515, 17000, 515)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("T,D,gates", SHAPES)
def test_values_and_gradients(T, D, gates, dtype):
    d, gy, gh = _inputs(T, D, dtype, gates, seed=T + D)
    _whole(d, gy, gh, 0.5)


@pytest.mark.parametrize("dtype", TYPES[1:], ids=str)
@pytest.mark.parametrize("T,D,gates", [(33, 264, 0), (20, 1500, 4), (520, 64, 520), (6, 8200, 1)])
def test_parameters_in_fp32(T, D, gates, dtype):
    d, gy, gh = _inputs(T, D, dtype, gates, wdtype=torch.float32)
    _whole(d, gy, gh, 1.5)
    d, gy, gh = _inputs(T, D, dtype, gates, gdtype=torch.float32)
    _whole(d, gy, gh, -1.5)


@pytest.mark.parametrize("D", [100, 3000, 16384, 16400])
def test_one_output_used_or_there(D):
    d, gy, gh = _inputs(12, D, torch.bfloat16, 3)
    _whole(d, gy, gh, 1.0, use=("y",))
    _whole(d, gy, gh, 1.0, use=("h",))
    d.pop("pre")
    on, y, h, grads = _whole(d, gy, gh, 1.0, use=("h",))
    assert y is None and set(grads) == {"x", "residual", "post", "gate"}


@pytest.mark.parametrize("wanted", ["x", "residual", "post", "pre", "gate"])
def test_each_gradient_alone(wanted):
    d, gy, gh = _inputs(40, 300, torch.bfloat16, 2)
    on = {n: t.to(DEV) for n, t in d.items()}
    on[wanted].requires_grad_(True)
    y, h = _call(on, 2.0)
    (g,) = torch.autograd.grad([y, h], [on[wanted]], [gy.to(DEV), gh.to(DEV)])
    _backward(d, 2.0, h.detach(), gy, gh, {wanted: g})


def test_gradients_against_differences():
    """fp32, along random directions: central differences of the definition in 64 bits with a step of 2^-14 of values
    near 1 are off by under 1e-7 of the slope's terms; the kernel's by its own 2^-16."""
    d, gy, gh = _inputs(6, 96, torch.float32, 2)
    on, y, h, grads = _whole(d, gy, gh, 0.5)

    def value(v):
        x = v["x"]
        s = v["residual"] + x * _rms(x) * 0.5 * v["post"] * v["gate"].repeat_interleave(3, 0)
        return (s * _rms(s) * v["pre"] * gy.double()).sum() + (s * gh.double()).sum()

    base = {n: t.double() for n, t in d.items()}
    for seed, name in enumerate(base):
        g = torch.randn(base[name].shape, generator=torch.Generator().manual_seed(seed), dtype=torch.double)
        f = [value({**base, name: base[name] + k * 2.0 ** -14 * g}) for k in (1, -1)]
        slope = (f[0] - f[1]) / 2.0 ** -13
        got = grads[name].double().cpu()
        size = (got * g).abs().sum() + g.abs().sum()
        assert abs(float((got * g).sum() - slope)) < 1e-4 * float(size)


@pytest.mark.parametrize("D", [96, 1000, 12000])
def test_strides_and_alignment(D):
    d, gy, gh = _inputs(10, D, torch.bfloat16, 1)
    wide = lambda t, at: torch.empty(10, D + 7, dtype=t.dtype, device=DEV)[:, at:at + D].copy_(t)
    on = {n: t.to(DEV) for n, t in d.items()}
    plain_y, plain_h = _call(on, 1.0)
    on["x"], on["residual"] = wide(d["x"], 1).requires_grad_(True), wide(d["residual"], 3).requires_grad_(True)
    y, h = _call(on, 1.0)
    assert torch.equal(y, plain_y) and torch.equal(h, plain_h)
    a = torch.autograd.grad([y, h], [on["x"], on["residual"]], [wide(gy, 5), wide(gh, 2)], retain_graph=True)
    b = torch.autograd.grad([y, h], [on["x"], on["residual"]], [gy.to(DEV), gh.to(DEV)], retain_graph=True)
    c = torch.autograd.grad([y, h], [on["x"], on["residual"]],
                            [gy.t().contiguous().to(DEV).t(), gh.to(DEV)], retain_graph=True)
    for p, q, s in zip(a, b, c):
        assert torch.equal(p, q) and torch.equal(p, s)
    one = d["x"][:1].to(DEV).expand(10, D)  # rows that share their memory, as a broadcast tensor's
    y, h = fm.sandwich_norm(one, on["post"], on["residual"].detach(), on["pre"])
    y2, h2 = fm.sandwich_norm(one.contiguous(), on["post"], on["residual"].detach(), on["pre"])
    assert torch.equal(y, y2) and torch.equal(h, h2)


def test_zero_rows_and_no_rows():
    d, gy, gh = _inputs(4, 64, torch.float32, 2)
    d["x"][1] = 0
    d["residual"][2] = 0
    d["x"][2] = 0
    _whole(d, gy, gh, 1.0)
    for gates in (1, 2):
        d, gy, gh = _inputs(0, 64, torch.bfloat16, gates)
        on = {n: t.to(DEV).requires_grad_(True) for n, t in d.items()}
        y, h = _call(on, 1.0)
        got = torch.autograd.grad([y, h], list(on.values()), [gy.to(DEV), gh.to(DEV)])
        assert all(g.shape == t.shape and not g.any() for g, t in zip(got, on.values()))


def test_repeats_bit_for_bit_and_in_a_graph():
    d, gy, gh = _inputs(300, 1024, torch.bfloat16, 3)
    on = {n: t.to(DEV).requires_grad_(True) for n, t in d.items()}
    runs = []
    for _ in range(2):
        y, h = _call(on, 1.0)
        runs.append((y, h, *torch.autograd.grad([y, h], list(on.values()), [gy.to(DEV), gh.to(DEV)])))
    assert all(torch.equal(a, b) for a, b in zip(*runs))
    held = {n: t.detach().clone() for n, t in on.items()}
    with torch.no_grad():
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            _call(held, 1.0)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = _call(held, 1.0)
        for seed in range(3):
            new, _, _ = _inputs(300, 1024, torch.bfloat16, 3, seed=seed + 5)
            for n in held:
                held[n].copy_(new[n])
            graph.replay()
            torch.cuda.synchronize()
            want = _call(held, 1.0)
            assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="capture"):
            _call(on, 1.0)
        torch.zeros(1, device=DEV)


def test_second_derivative_and_changed_inputs_are_refused():
    d, gy, gh = _inputs(4, 32, torch.float32, 1)
    on = {n: t.to(DEV).requires_grad_(True) for n, t in d.items()}
    y, h = _call(on, 1.0)
    (g,) = torch.autograd.grad(y, on["x"], gy.to(DEV), create_graph=True)
    with pytest.raises(RuntimeError, match="no gradient of its own"):
        g.sum().backward()
    y, h = _call(on, 1.0)
    with torch.no_grad():
        on["gate"].add_(1)
    with pytest.raises(RuntimeError, match="modified"):
        y.sum().backward()


def test_refusals():
    d, _, _ = _inputs(6, 32, torch.bfloat16, 2)
    on = {n: t.to(DEV) for n, t in d.items()}
    with pytest.raises(ValueError, match="residual"):
        _call({**on, "residual": on["residual"][:5]}, 1.0)
    with pytest.raises(ValueError, match="residual"):
        _call({**on, "residual": on["residual"].float()}, 1.0)
    with pytest.raises(ValueError, match="post_weight"):
        _call({**on, "post": on["post"][:31]}, 1.0)
    with pytest.raises(TypeError, match="post_weight"):
        _call({**on, "post": on["post"].half()}, 1.0)
    with pytest.raises(TypeError, match="share"):
        _call({**on, "pre": on["pre"].float()}, 1.0)
    with pytest.raises(ValueError, match="gate"):
        _call({**on, "gate": on["gate"].repeat(2, 1)}, 1.0)  # 4 rows for 6
    with pytest.raises(ValueError, match="gate"):
        _call({**on, "gate": on["gate"][:0]}, 1.0)
    with pytest.raises(ValueError, match="gate"):
        _call({**on, "gate": torch.ones(6, 1, device=DEV, dtype=torch.bfloat16)}, 1.0)
    with pytest.raises(ValueError, match="scale"):
        _call(on, float("nan"))
    with pytest.raises(ValueError, match="eps"):
        fm.sandwich_norm(on["x"], on["post"], on["residual"], eps=-1.0)
    with pytest.raises(ValueError, match="unit column stride"):
        _call({**on, "x": on["x"].t().contiguous().t()}, 1.0)
    with pytest.raises(RuntimeError, match="only on the GPU"):
        _call({**on, "gate": d["gate"]}, 1.0)
    with pytest.raises(TypeError, match="tensor"):
        fm.sandwich_norm(on["x"], on["post"], None)


def test_gates_that_are_slices_or_broadcast():
    """As a copy of them; the gradient comes back through the copy, a broadcast one's as the sum over its rows."""
    d, gy, gh = _inputs(12, 40, torch.bfloat16, gates=3)
    on = {k: v.to(DEV) for k, v in d.items()}
    many = torch.randn(3, 120, device=DEV).bfloat16().requires_grad_(True)
    one = torch.randn(1, 40, device=DEV).requires_grad_(True)
    for leaf, view in ((many, lambda t: t[:, 40:80]), (many, lambda t: t.chunk(3, -1)[2]), (one, lambda t: t.expand(3, 40)),
                       (many, lambda t: t.t()[:3, 0].expand(40, 3).t())):
        copy = view(leaf).detach().contiguous().requires_grad_(True)
        got = _call({**on, "gate": view(leaf)}, 0.5)
        want = _call({**on, "gate": copy}, 0.5)
        for g, w in zip(got, want):
            assert torch.equal(g, w)
        up = [gy.to(DEV), gh.to(DEV)]
        g, = torch.autograd.grad(got, leaf, up)
        w, = torch.autograd.grad(want, copy, up)
        assert torch.equal(g, torch.autograd.grad(view(leaf), leaf, w)[0])


def test_numbers_beyond_fp32_are_refused():
    d, *_ = _inputs(4, 16, torch.float32)
    on = {k: v.to(DEV) for k, v in d.items()}
    with pytest.raises(ValueError, match="finite"):
        _call(on, 1e39)
    with pytest.raises(ValueError, match="finite"):
        fm.sandwich_norm(on["x"], on["post"], on["residual"], eps=1e39)
    with pytest.raises(ValueError, match="finite"):
        fm.route_tokens(on["x"], 2, fm.Routing(scale=1e39))


def test_rows_beyond_32_bits_of_elements():
    """2^31 elements are passed: the last rows hold to the definition, forward and backward.  (A call on them alone may
    differ by roundings: few rows are given more threads.)"""
    T, D = (1 << 18) + 3, 8192
    gen = torch.Generator(device=DEV).manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=gen, device=DEV, dtype=torch.bfloat16)
    on = {"x": r(T, D), "residual": r(T, D), "post": r(D), "pre": r(D), "gate": r(D)}
    for t in on.values():
        t.requires_grad_(True)
    y, h = _call(on, 0.5)
    gx, gr = torch.autograd.grad([y, h], [on["x"], on["residual"]], [y.detach(), h.detach()])
    last = lambda t: t.detach()[-5:].cpu()
    d = {k: last(v) if v.dim() == 2 else v.detach().cpu() for k, v in on.items()}
    _forward(d, 0.5, y.detach()[-5:], h.detach()[-5:])
    _backward(d, 0.5, last(h), last(y), last(h), {"x": gx[-5:], "residual": gr[-5:]})
