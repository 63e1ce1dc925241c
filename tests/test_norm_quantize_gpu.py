"""The norm, its gradients and the rows in 8 bits against the formulas in 64 bits.

Bounds: u = 2^-24 is fp32's half step, h = finfo(type).eps / 2 the type's.  A thread adds at most 40
squares and a tree of at most 16 levels joins them; with the square root (which halves it), the
division and the products, a value of y carries at most 64 u before its own rounding."""
from __future__ import annotations

import pytest
import torch

import fastmoe_amd as fm

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
# one column; less than, exactly and more than a vector; every width class and one beyond registers
WIDTHS = [1, 7, 8, 129, 512, 513, 1001, 2048, 2056, 4096, 7168, 8200, 16384, 16392, 20011]


def half(dtype):
    return torch.finfo(dtype).eps / 2


def close(got, want, rel, absolute):
    err = (got.double() - want).abs()
    bound = rel * want.abs() + absolute
    bad = ~(err <= bound)
    assert not bad.any(), (f"{int(bad.sum())} of {bad.numel()} off, worst {float(err[bad].max())} "
                           f"where {float(bound[bad].min())} is allowed")


def rand(*shape, dtype=torch.float32, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def norm64(x, w, r, eps):
    h = (x if r is None else x + r).double()  # the sum is rounded to the tensors' type
    c = 1 / torch.sqrt((h * h).mean(-1, keepdim=True) + eps)
    return h, c, h * c * w.double()


def check_rows8(q, v, slack):
    """q holds the float64 values v, computed with a relative slack: whole numbers within half a step."""
    top = v.abs().amax(-1)
    close(q.scales, top / 127, slack + 2 * U, 0)
    step = q.scales.double().unsqueeze(-1)
    ideal = torch.where(step > 0, v / step, torch.zeros_like(v))
    got = q.data[:, :q.features].double()
    assert ((got - ideal).abs() <= 0.5 + 127 * (2 * slack + 8 * U)).all()
    assert (q.data[:, q.features:] == 0).all()
    assert q.data.shape[1] == -(-q.features // 128) * 128


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", WIDTHS)
def test_norm_and_its_8_bit_rows(D, dtype):
    T = 5
    x, r = rand(T, D, dtype=dtype, seed=D), rand(T, D, dtype=dtype, seed=D + 1)
    for w in (rand(D, dtype=dtype, seed=2), rand(D, seed=2)):
        for res in (r, None):
            h, _, want = norm64(x, w, res, 1e-6)
            y, stream = fm.add_rms_norm(x, w, res)
            assert torch.equal(stream.double(), h)
            assert y.dtype == dtype
            close(y, want, half(dtype) + 64 * U, 2.0 ** -25)
            got = fm.add_rms_norm_int8(x, w, res)
            assert torch.equal(got.normed, y) and torch.equal(got.residual, stream)
            check_rows8(got.rows, want, 64 * U)
            only = fm.add_rms_norm_int8(x, w, res, keep_normed=False)
            assert only.normed is None and torch.equal(only.rows.data, got.rows.data)


@pytest.mark.parametrize("T", [0, 1, 3, 4, 9, 700])
def test_norm_row_counts(T):
    x, w = rand(T, 200, dtype=torch.bfloat16), rand(200, dtype=torch.bfloat16, seed=1)
    got = fm.add_rms_norm_int8(x, w, x)
    assert got.rows.data.shape == (T, 256) and got.normed.shape == (T, 200)
    if T:
        close(got.normed, norm64(x, w, x, 1e-6)[2], half(torch.bfloat16) + 64 * U, 0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,D", [(1, 1), (3, 7), (9, 513), (700, 129), (1300, 1001), (33, 2048),
                                 (17, 4096), (520, 8200), (7, 16384), (5, 16391)])
def test_norm_gradients(T, D, dtype):
    x, r, w = rand(T, D, dtype=dtype, seed=1), rand(T, D, dtype=dtype, seed=2), rand(D, dtype=dtype, seed=3)
    gy, gh = rand(T, D, dtype=dtype, seed=4), rand(T, D, dtype=dtype, seed=5)
    leaves = [t.requires_grad_(True) for t in (x, r, w)]
    y, h = fm.add_rms_norm(x, w, r)
    gx, gr, gw = torch.autograd.grad([y, h], leaves, [gy, gh])
    assert torch.equal(gx, gr) and gw.dtype == dtype
    with torch.no_grad():
        h64, c, _ = norm64(x, w, r, 1e-6)
        t, hat = gy.double() * w.double(), h64 * c
        mean, size = (t * hat).mean(-1, keepdim=True), (t * hat).abs().mean(-1, keepdim=True)
        want = gh.double() + c * (t - hat * mean)
        # the mean of up to 48 terms a thread and their tree, then five rounded operations
        scale = gh.double().abs() + c * (t.abs() + hat.abs() * size)
        close(gx, want, half(dtype), 128 * U * scale + 2.0 ** -25)
        terms = gy.double() * hat
        units = min(T, 512)
        steps = -(-T // units) + units // 4 + 64
        close(gw, terms.sum(0), half(dtype), steps * U * terms.abs().sum(0) + 2.0 ** -25)
    # without a gradient through the stream, and through the stream alone
    y, h = fm.add_rms_norm(x, w, r)
    only = torch.autograd.grad(y, x, gy)[0]
    with torch.no_grad():
        close(only, c * (t - hat * mean), half(dtype), 128 * U * scale + 2.0 ** -25)
    y, h = fm.add_rms_norm(x, w, r)
    gx, gw = torch.autograd.grad(h, [x, w], gh, allow_unused=True)
    assert torch.equal(gx, gh) and (gw is None or not gw.any())


def test_norm_gradient_against_differences():
    """Central differences of sum(gy * y + gh * h) in fp32 along random directions.  Their error: the
    sum's rounding over the step (64 u * sum|gy y| / 0.01), and the cubic term of the step."""
    T, D = 4, 24
    x, r, w = (rand(*s, seed=i) for i, s in enumerate([(T, D), (T, D), (D,)]))
    gy, gh = rand(T, D, seed=8), rand(T, D, seed=9)
    leaves = [t.requires_grad_(True) for t in (x, r, w)]
    y, h = fm.add_rms_norm(x, w, r)
    grads = torch.autograd.grad([y, h], leaves, [gy, gh])
    with torch.no_grad():
        for i, leaf in enumerate(leaves):
            d = rand(*leaf.shape, seed=20 + i)
            vals = []
            for sign in (1, -1):
                args = [t + sign * 0.01 * d if j == i else t for j, t in enumerate(leaves)]
                y, h = fm.add_rms_norm(args[0], args[2], args[1])
                vals.append((gy.double() * y.double() + gh.double() * h.double()).sum())
            slope = (vals[0] - vals[1]) / 0.02
            want = (grads[i].double() * d.double()).sum()
            assert abs(float(slope - want)) <= 5e-3 * (1 + abs(float(want))) + 64 * U * 200 / 0.01


def test_no_residual_gradient_and_frozen_weight():
    x, w = rand(6, 40).requires_grad_(True), rand(40, seed=1)
    y, h = fm.add_rms_norm(x, w)
    assert h is x
    gx = torch.autograd.grad(y.sum(), x)[0]
    x64 = x.detach().double().requires_grad_(True)
    ref = (x64 / torch.sqrt((x64 * x64).mean(-1, keepdim=True) + 1e-6) * w.double()).sum()
    want = torch.autograd.grad(ref, x64)[0]
    close(gx, want, 0, 128 * U * 40)


def test_strided_rows_and_odd_starts():
    """Rows of a wider tensor, starting at every offset within 16 bytes, and a broadcast row."""
    for dtype in TYPES:
        wide = rand(6, 300, dtype=dtype)
        w = rand(77, dtype=dtype, seed=1)
        for start in range(9):
            x = wide[:, start:start + 77]
            y, h = fm.add_rms_norm(x, w, x)
            want, _ = fm.add_rms_norm(x.contiguous(), w, x.contiguous())
            assert torch.equal(y, want)
            a, b = fm.quantize_rows(x), fm.quantize_rows(x.contiguous())
            assert torch.equal(a.data, b.data) and torch.equal(a.scales, b.scales)
        x = wide[:1, :77].expand(6, 77)
        assert torch.equal(fm.add_rms_norm(x, w, wide[:, :77])[0],
                           fm.add_rms_norm(x.contiguous(), w, wide[:, :77])[0])
    gy = rand(1, 1).expand(6, 77)  # what a sum's backward hands on
    x, w = rand(6, 77).requires_grad_(True), rand(77, seed=1)
    a = torch.autograd.grad(fm.add_rms_norm(x, w)[0], x, gy)[0]
    b = torch.autograd.grad(fm.add_rms_norm(x, w)[0], x, gy.contiguous())[0]
    assert torch.equal(a, b)


# GELU's error beside rounding, as the kernels state it: fp32 erfc; polynomials for 16-bit types (bf16's
# degree also serves every 16-bit type whose result has 8 bits)
ERROR = {torch.float32: (16 * U, 1e-7), torch.float16: (2e-5, 4e-7), torch.bfloat16: (2.4e-4, 3e-6)}
ERROR8 = {torch.float32: 1e-7, torch.float16: 3e-6, torch.bfloat16: 3e-6}


def cdf64(x):
    return 0.5 * torch.erfc(-x * 0.5 ** 0.5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("C", WIDTHS)
def test_quantize_rows(C, dtype):
    x = rand(5, C, dtype=dtype, seed=C) * 3
    q = fm.quantize_rows(x)
    check_rows8(q, x.double(), 0)
    back = q.dequantize(dtype)
    close(back, q.data[:, :C].double() * q.scales.double().unsqueeze(1), half(dtype) + U, 2.0 ** -25)
    # GELU is within e of the value: the scale within e / 127, so 127 steps within e, and the value itself
    e = ERROR8[dtype] + 16 * U * float(x.double().abs().max())
    v = x.double() * cdf64(x.double())
    g = fm.quantize_rows(x, activation="gelu")
    top = v.abs().amax(-1)
    close(g.scales, top / 127, 8 * U, e / 127)
    step = g.scales.double().unsqueeze(-1)
    err = (g.data[:, :C].double() * step - v).abs()
    assert (err <= 0.5 * step + 2 * e + 64 * U * v.abs()).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_of_zeros_infinities_and_nan(dtype):
    x = rand(6, 200, dtype=dtype)
    x[1] = 0
    x[2, 7] = float("inf")
    x[3, 199] = float("-inf")
    x[4, 100] = float("nan")
    x[5] = torch.finfo(dtype).max if dtype is not torch.float32 else 1e30
    q = fm.quantize_rows(x)
    assert q.scales[1] == 0 and not q.data[1:5].any()
    assert q.scales[2:5].isnan().all() and q.scales[0].isfinite()
    back = q.dequantize()
    assert back[2:5].isnan().all() and not back[1].any()
    assert (q.data[5, :200] == 127).all()
    w = torch.ones(200, dtype=dtype, device="cuda")
    y = fm.add_rms_norm_int8(x, w)
    assert y.rows.scales[1] == 0 and not y.rows.data[1].any() and not y.normed[1].any()
    assert y.rows.scales[2:5].isnan().all()
    # GELU takes -inf to 0 and keeps inf and NaN
    g = fm.quantize_rows(x, activation="gelu")
    assert g.scales[2].isnan() and g.scales[4].isnan() and g.scales[3].isfinite()
    assert g.data[3, 199] == 0
    tiny = torch.full((1, 8), 2.0 ** -119, device="cuda")
    assert fm.quantize_rows(tiny).scales[0] == 0
    assert (fm.quantize_rows(tiny * 2).data[0, :8] == 127).all()


def test_gelu_of_half_precision_rows():
    """GELU's error moves values near a border to the next whole number: for fp16 it is the one that its
    own results have, 4e-7, not the larger one that bf16's rounding covers."""
    x = rand(64, 2048, dtype=torch.float16, seed=9) * 3
    v = x.double() * cdf64(x.double())
    e = 4e-7 + 16 * U * float(x.double().abs().max())
    g = fm.quantize_rows(x, activation="gelu")
    close(g.scales, v.abs().amax(-1) / 127, 8 * U, e / 127)
    step = g.scales.double().unsqueeze(-1)
    err = (g.data[:, :2048].double() * step - v).abs()
    assert (err <= 0.5 * step + 2 * e + 64 * U * v.abs()).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_the_largest_numbers_stay_finite(dtype):
    top = torch.finfo(dtype).max
    x = torch.tensor([[top, -top, top / 2, 0.0]], dtype=dtype, device="cuda")
    # 127 steps are within the scale's rounding (one fp32 step, 2 u) of the largest value
    for back in (fm.quantize_rows(x).dequantize(), fm.restore_rows(fm.compress_rows(x), torch.float32)):
        close(back[:, :2], x[:, :2].double(), 3 * U, 0)
        close(back[:, 2:], x[:, 2:].double(), 0, top / 127 * (0.5 + 127 * 8 * U))
    again, _ = fm.gelu_compressed_backward(fm.compress_rows(x.float()), torch.ones(1, 4, device="cuda"))
    assert again.isfinite().all()


def test_rows_into_a_wider_buffer_leave_its_rest():
    """The C entry points write a row's own 128-column pieces and nothing of a wider pitch."""
    from fastmoe_amd import _abi
    from fastmoe_amd.ops import _stream_handle

    x = rand(3, 130, dtype=torch.bfloat16)
    q = torch.full((3, 512), 9, dtype=torch.int8, device="cuda")
    s = torch.empty(3, device="cuda")
    for call in ("quantize", "compress"):
        q.fill_(9)
        if call == "quantize":
            rc = _abi.lib().fmoe_quantize_rows(x.data_ptr(), 130, 3, 130, _abi.BF16, 0, q.data_ptr(),
                                               512, s.data_ptr(), _stream_handle(x.device))
        else:
            s2 = torch.empty(3, 2, device="cuda")
            rc = _abi.lib().fmoe_compress_rows(x.data_ptr(), 130, 3, 130, _abi.BF16, q.data_ptr(), 512,
                                               s2.data_ptr(), None, _stream_handle(x.device))
        assert rc == 0
        assert not q[:, 130:256].any() and (q[:, 256:] == 9).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R,C", [(1, 1), (3, 7), (5, 128), (2, 129), (33, 200), (17, 1001),
                                 (3, 2048), (5, 2049), (2, 5000), (300, 384)])
def test_held_rows_and_gelu(R, C, dtype):
    x, ga = rand(R, C, dtype=dtype, seed=C) * 2, rand(R, C, dtype=dtype, seed=C + 1)
    held = fm.compress_rows(x)
    blocks = -(-C // 128)
    assert held.scales.shape == (R, blocks)
    padded = torch.zeros(R, blocks * 128, dtype=torch.float64, device="cuda")
    padded[:, :C] = x.double()
    v = padded.view(R * blocks, 128)
    check_rows8(fm.QuantizedRows(held.data.view(-1, 128), held.scales.view(-1), 128), v, 0)
    value = (held.data.double().view(R, blocks, 128) * held.scales.double().unsqueeze(-1)).view(R, -1)[:, :C]
    close(fm.restore_rows(held, dtype), value, half(dtype) + U, 2.0 ** -25)
    a, again_held = fm.gelu_compress(x)
    assert torch.equal(again_held.data, held.data) and torch.equal(again_held.scales, held.scales)
    x64 = x.double()
    _, absolute = ERROR[dtype]
    close(a, x64 * cdf64(x64), half(dtype) + 16 * U, absolute + 2.0 ** -25)
    again, grad = fm.gelu_compressed_backward(held, ga)
    value = value.float().double()  # q * s is rounded once to fp32
    close(again, value * cdf64(value), half(dtype) + 16 * U, absolute + 2.0 ** -25)
    slope = cdf64(value) + value * torch.exp(-value ** 2 / 2) * 0.3989422804014327
    # Phi = (x * Phi) / x: where |x| is small its log-odds' error, at most the relative one, counts a
    # quarter; phi and the sums add a few u
    rel, _ = ERROR[dtype]
    close(grad, ga.double() * slope, half(dtype),
          (min(rel / 4, 10 * absolute) + 64 * U) * ga.double().abs() + 2.0 ** -25)
    none, grad2 = fm.gelu_compressed_backward(held, ga, again=False)
    assert none is None and torch.equal(grad, grad2)


def test_held_rows_of_none():
    x = torch.empty(0, 40, device="cuda")
    a, held = fm.gelu_compress(x)
    assert a.shape == (0, 40) and fm.restore_rows(held, torch.float32).shape == (0, 40)
    assert fm.gelu_compressed_backward(held, x)[1].shape == (0, 40)


@pytest.mark.parametrize("dtype", TYPES)
def test_gelu_over_its_whole_range(dtype):
    """Every magnitude and both signs, to the values that overflow or vanish."""
    x = torch.cat([torch.linspace(-12, 12, 100001), torch.tensor([1e-30, -1e-30, 300., -300., 6e4, -6e4])])
    x = x.cuda().to(dtype).view(1, -1)
    a, _ = fm.gelu_compress(x)
    x64 = x.double()
    want = x64 * cdf64(x64)
    rel, absolute = ERROR[dtype]
    close(a, want, half(dtype) + 16 * U, absolute + 2.0 ** -25)
    at = (x64 < -0.01) & (x64 > -3.5)  # and relatively, where 1 + erf would have lost its bits
    close(a[at], want[at], half(dtype) + rel + 16 * U, 2.0 ** -25)


def test_another_stream():
    x, w = rand(64, 4096, dtype=torch.bfloat16), rand(4096, dtype=torch.bfloat16, seed=1)
    want = fm.add_rms_norm_int8(x, w, x)
    a, held = fm.gelu_compress(x)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = fm.add_rms_norm_int8(x, w, x)
        b, held2 = fm.gelu_compress(x)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got.rows.data, want.rows.data) and torch.equal(got.normed, want.normed)
    assert torch.equal(a, b) and torch.equal(held.data, held2.data)


def test_captured_rows_replay():
    """The serving calls in one graph, replayed on new inputs between eager calls."""
    x, w = rand(9, 1001, dtype=torch.float16), rand(1001, dtype=torch.float16, seed=1)
    for _ in range(2):
        fm.add_rms_norm_int8(x, w, x)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        n = fm.add_rms_norm_int8(x, w, x)
        q = fm.quantize_rows(n.normed, activation="gelu")
        back = q.dequantize(torch.float16)
    for seed in (3, 4, 5):
        x.copy_(rand(9, 1001, dtype=torch.float16, seed=seed))
        g.replay()
        torch.cuda.synchronize()
        want = fm.add_rms_norm_int8(x, w, x)
        assert torch.equal(n.rows.data, want.rows.data) and torch.equal(n.rows.scales, want.rows.scales)
        assert torch.equal(back, fm.quantize_rows(want.normed, activation="gelu").dequantize(torch.float16))


def test_recorded_norm_is_refused_under_capture():
    x, w = rand(4, 64), rand(64, seed=1)
    fm.add_rms_norm(x, w, x)
    leaf = x.clone().requires_grad_(True)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y, _ = fm.add_rms_norm(x, w, x)
        with pytest.raises(RuntimeError, match="graph capture"):
            fm.add_rms_norm(leaf, w, x)


def test_refusals():
    x, w = rand(4, 64), rand(64, seed=1)
    with pytest.raises(ValueError, match="unit column stride"):
        fm.add_rms_norm(x.t().contiguous().t(), w)
    with pytest.raises(ValueError, match="weight"):
        fm.add_rms_norm(x, w[:32])
    with pytest.raises(TypeError, match="weight"):
        fm.add_rms_norm(x, w.half())
    with pytest.raises(ValueError, match="residual"):
        fm.add_rms_norm(x, w, x.half())
    with pytest.raises(ValueError, match="eps"):
        fm.add_rms_norm(x, w, eps=float("nan"))
    with pytest.raises(TypeError, match="dtype"):
        fm.quantize_rows(x.double())
    with pytest.raises(ValueError, match="activation"):
        fm.quantize_rows(x, activation="relu")
    leaf = x.clone().requires_grad_(True)
    for call in (lambda: fm.quantize_rows(leaf), lambda: fm.add_rms_norm_int8(leaf, w),
                 lambda: fm.compress_rows(leaf), lambda: fm.gelu_compress(leaf)):
        with pytest.raises(RuntimeError, match="no gradient"):
            call()
        with torch.no_grad():
            call()
    held = fm.compress_rows(x)
    with pytest.raises(ValueError, match="grad must be"):
        fm.gelu_compressed_backward(held, x[:2])
    with pytest.raises(ValueError, match="features"):
        fm.restore_rows(held._replace(features=200), torch.float32)


def test_gradients_and_views_that_would_be_lost_are_refused():
    x, w = rand(4, 64), rand(64, seed=1)
    q, held = fm.quantize_rows(x), fm.compress_rows(x)
    weights = fm.quantize_weights(rand(8, 64, seed=2))
    grown = lambda t: t._replace(scales=t.scales.clone().requires_grad_(True))
    for call in (lambda: grown(q).dequantize(), lambda: fm.restore_rows(grown(held), torch.float32),
                 lambda: fm.gelu_compressed_backward(grown(held), x),
                 lambda: fm.int8_linear(grown(q), weights), lambda: fm.int8_linear(q, grown(weights))):
        with pytest.raises(RuntimeError, match="no gradient"):
            call()
        with torch.no_grad():
            call()
    negated = torch._neg_view(x)
    grads = []
    for hook in (torch.neg, torch._neg_view):
        leaf = x.clone().requires_grad_(True)
        y, _ = fm.add_rms_norm(leaf, w)
        y.register_hook(hook)
        y.backward(rand(4, 64, seed=3))
        grads.append(leaf.grad)
    assert torch.equal(*grads)
    for call in (lambda t: fm.quantize_rows(t), lambda t: fm.add_rms_norm(t, w),
                 lambda t: fm.add_rms_norm_int8(t, w), lambda t: fm.add_rms_norm(x, w, t),
                 lambda t: fm.gelu_compress(t), lambda t: fm.gelu_compressed_backward(held, t)):
        with pytest.raises(ValueError, match="negated"):
            call(negated)
        with torch.autograd.forward_ad.dual_level():
            with pytest.raises((ValueError, RuntimeError), match="forward-mode"):
                call(torch.autograd.forward_ad.make_dual(x, torch.ones_like(x)))


def test_outputs_past_the_caches_and_beyond_32_bits():
    """Arrays above 4 GiB (their last rows lie beyond 32-bit offsets), whose y is also large enough to be
    stored past the caches: each row is what the row alone gives."""
    T, D = 140_000, 16384
    x = torch.zeros(T, D, dtype=torch.bfloat16, device="cuda")
    at = [0, 1, 65_536, T - 2, T - 1]
    x[at] = rand(len(at), D, dtype=torch.bfloat16, seed=3)
    w = rand(D, dtype=torch.bfloat16, seed=4)
    got = fm.add_rms_norm_int8(x, w)
    want = fm.add_rms_norm_int8(x[at], w)
    assert torch.equal(got.normed[at], want.normed)
    assert torch.equal(got.rows.data[at], want.rows.data)
    assert torch.equal(got.rows.scales[at], want.rows.scales)
    assert not got.normed[2].any() and got.rows.scales[2] == 0
    del got
    held, some = fm.compress_rows(x), fm.compress_rows(x[at])
    assert torch.equal(held.data[at], some.data) and torch.equal(held.scales[at], some.scales)
    assert torch.equal(fm.restore_rows(held, torch.bfloat16)[at], fm.restore_rows(some, torch.bfloat16))
    q = fm.quantize_rows(x, activation="gelu")
    assert torch.equal(q.data[at], fm.quantize_rows(x[at], activation="gelu").data)


@pytest.mark.parametrize("dtype", TYPES)
def test_held_outputs_past_the_caches(dtype):
    """Outputs above 96 MiB, of rows that start anywhere: bit for bit what the rows give in small calls."""
    C = 1001
    R = 100 * 2 ** 20 // (C * dtype.itemsize) + 5
    x, g = rand(R, C, dtype=dtype), rand(R, C, dtype=dtype, seed=1)
    a, held = fm.gelu_compress(x)
    back, (again, grad) = fm.restore_rows(held, dtype), fm.gelu_compressed_backward(held, g)
    for at in (slice(0, 3), slice(R // 2, R // 2 + 129), slice(R - 70, R)):
        a1, h1 = fm.gelu_compress(x[at])
        b1, (g1, d1) = fm.restore_rows(h1, dtype), fm.gelu_compressed_backward(h1, g[at])
        for got, want in ((a, a1), (held.data, h1.data), (held.scales, h1.scales), (back, b1),
                          (again, g1), (grad, d1)):
            assert torch.equal(got[at], want)


def test_two_streams_at_once():
    """No workspace is shared: interleaved calls on two streams give what each gives alone."""
    sizes = [(700, 1001), (300, 4096)]
    inputs = [(rand(T, D, dtype=torch.bfloat16, seed=T), rand(D, dtype=torch.bfloat16, seed=D),
               rand(T, D, dtype=torch.bfloat16, seed=9)) for T, D in sizes]

    def step(x, w, g):
        leaves = [x.clone().requires_grad_(True), w.clone().requires_grad_(True)]
        y, _ = fm.add_rms_norm(leaves[0], leaves[1])
        grads = torch.autograd.grad(y, leaves, g)
        a, held = fm.gelu_compress(x)
        return [*grads, a, *fm.gelu_compressed_backward(held, g), fm.quantize_rows(x).data]

    want = [step(*i) for i in inputs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        got = []
        for s, i in zip(streams, inputs):
            with torch.cuda.stream(s):
                got.append(step(*i))
        torch.cuda.synchronize()
        for u, v in zip(want, got):
            assert all(torch.equal(a, b) for a, b in zip(u, v))


def test_the_norms_gradient_has_none():
    x, w = rand(4, 32).requires_grad_(True), rand(32, seed=1).requires_grad_(True)
    y, _ = fm.add_rms_norm(x, w)
    seed = torch.ones_like(y, requires_grad=True)
    with pytest.raises(RuntimeError, match="no gradient of its own"):
        torch.autograd.grad(y, x, seed, create_graph=True)
    y, _ = fm.add_rms_norm(x, w)
    y.sum().backward()
    with pytest.raises(RuntimeError):
        y.sum().backward()  # freed, as with any node
    with pytest.raises(RuntimeError, match="transforms"):
        torch.func.vmap(lambda t: fm.add_rms_norm(t, w)[0])(rand(2, 4, 32))


def test_inference_mode_and_parameters():
    w = torch.nn.Parameter(rand(64, seed=1))
    with torch.inference_mode():
        x = rand(3, 64)
        y, h = fm.add_rms_norm(x, w, x)
        r = fm.add_rms_norm_int8(x, w, x)
        assert torch.equal(r.normed, y) and not y.requires_grad
        assert fm.quantize_rows(x).dequantize().shape == (3, 64)
