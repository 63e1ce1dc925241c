"""int8_linear against whole-number sums in 64 bits.

The sums are exact, so the only roundings are the sum's conversion to fp32, the two scales' products
and the bias' addition, half a step u = 2^-24 each, and the output's own."""
from __future__ import annotations

import pytest
import torch

import fastmoe_amd as fm
from fastmoe_amd import _abi

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def make(T, K, E, N, seed=0, full=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    pad = -(-K // 128) * 128

    def whole(*shape):
        lo = -128 if full else -127
        return torch.randint(lo, 128, shape, generator=g, device="cuda", dtype=torch.int8)

    x = torch.zeros(T, pad, dtype=torch.int8, device="cuda")
    x[:, :K] = whole(T, K)
    w = torch.zeros(E, N, pad, dtype=torch.int8, device="cuda")
    w[:, :, :K] = whole(E, N, K)
    sx = torch.rand(T, generator=g, device="cuda") + 0.1
    sw = torch.rand(E, N, generator=g, device="cuda") * 1e-3 + 1e-4
    return fm.QuantizedRows(x, sx, K), fm.Int8Weights(w, sw, K)


def route(counts):
    c = torch.tensor([0, *counts], dtype=torch.int64)
    return c.cumsum(0).cuda()


def reference(x, w, counts, rows=None, bias=None, total=None):
    """float64 [R, N]; rows of no expert are zero, and so is the product of a row outside x."""
    N = w.data.shape[1]
    R = (x.data.shape[0] if rows is None else rows.shape[0]) if total is None else total
    out = torch.zeros(R, N, dtype=torch.float64, device="cuda")
    mag = torch.zeros_like(out)
    at = 0
    for e, n in enumerate(counts):
        if n:
            i = torch.arange(at, at + n, device="cuda") if rows is None else rows[at:at + n].long()
            ok = (i >= 0) & (i < x.data.shape[0])
            j = i.clamp(0, x.data.shape[0] - 1)
            y = x.data[j].double() @ w.data[e].double().t().contiguous()
            y = y * torch.where(ok, x.scales[j], 0.0).double().unsqueeze(1) * w.scales[e].double()
            mag[at:at + n] = y.abs()
            if bias is not None:
                y = y + bias[e].double()
                mag[at:at + n] += bias[e].double().abs()
            out[at:at + n] = y
        at += n
    return out, mag


def check(got, want, mag, dtype):
    assert got.dtype == dtype and got.shape == want.shape
    err = (got.double() - want).abs()
    bound = torch.finfo(dtype).eps / 2 * want.abs() + 6 * U * mag
    if dtype is torch.float16:
        bound = bound + 2.0 ** -25
    bad = ~(err <= bound)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()}, worst {float(err[bad].max())}"


COUNTS = {
    "one row": [1],
    "one expert": [77],
    "decode": [1, 0, 2, 0, 0, 1, 1, 3, 0, 1],
    "empty ends": [0, 0, 5, 0, 16, 17, 0],
    "skewed": [300, 0, 1, 64, 63, 65, 2, 129],
    "many experts": [(7 * e) % 5 for e in range(150)],
    "large": [257, 256, 511, 0, 130],
}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("K,N", [(128, 64), (1, 1), (100, 17), (129, 130), (384, 256), (1001, 515)])
@pytest.mark.parametrize("name", list(COUNTS))
def test_against_whole_numbers(name, K, N, dtype):
    counts = COUNTS[name]
    R, E = sum(counts), len(counts)
    x, w = make(R, K, E, N, seed=K + N)
    got = fm.int8_linear(x, w, route(counts), out_dtype=dtype)
    check(got, *reference(x, w, counts), dtype)


def ragged(E, mean, seed=0):
    """Rows of E experts: none, one, around the tile sizes, the rest to reach the mean."""
    special = [0, 1, 31, 32, 33, 63, 65, 127, 128, 129, 255, 256, 257, 0]
    counts = [min(special[(e + seed) % len(special)], 2 * mean) for e in range(E)]
    short = E * mean - sum(counts)
    for e in range(0, E, 3):
        if short > 0:
            counts[e] += min(short, 2 * mean)
            short -= min(short, 2 * mean)
    return counts


# (tile, experts, mean rows, columns): the sizes that the choice by size sends to each tile
TILES = [(256256, 50, 130, 1000), (128256, 40, 40, 1000), (128128, 16, 60, 1024), (32064, 30, 5, 300),
         (16016, 3, 4, 130)]


KS = [1, 130, 300, 500, 641, 1100]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("tile,E,mean,N,K", [(*t, K) for t in TILES for K in KS] +
                         [(32064, 130, 5, 500, K) for K in (4000, 4097, 4225)] +
                         [(32128, 30, 5, 2000, K) for K in (1, 130, 300, 500, 1100, 4000, 4097, 4225)])
def test_every_tile(tile, E, mean, N, K, dtype):
    """Every tile, with rings of every remainder of pieces, ragged experts and column ends."""
    counts = ragged(E, mean, seed=K)
    R = sum(counts)
    assert _abi.lib().fmoe_int8_linear_tile(R, E, N, K) == tile
    x, w = make(R, K, E, N, seed=K)
    bias = torch.randn(E, N, device="cuda")
    got = fm.int8_linear(x, w, route(counts), bias=bias, out_dtype=dtype)
    check(got, *reference(x, w, counts, bias=bias), dtype)
    g = torch.Generator(device="cuda").manual_seed(K)
    rows = torch.randint(-2, R + 2, (R + 37,), generator=g, device="cuda")
    got = fm.int8_linear(x, w, route(counts), rows=rows, out_dtype=dtype)
    check(got, *reference(x, w, counts, rows), dtype)


def test_more_experts_than_one_scan_and_offsets_that_are_none():
    counts = [(5 * e) % 7 if e % 3 else 0 for e in range(1000)]
    R = sum(counts)
    x, w = make(R, 64, 1000, 33)
    check(fm.int8_linear(x, w, route(counts)), *reference(x, w, counts), torch.bfloat16)
    zigzag = torch.tensor([0, R] * 500 + [0], device="cuda")
    fm.int8_linear(x, w, zigzag)  # bounded: each workgroup's tile lies within the rows
    torch.cuda.synchronize()


@pytest.mark.parametrize("index", [torch.int64, torch.int32])
@pytest.mark.parametrize("biased", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("name", list(COUNTS))
def test_rows_read_through_an_index_with_a_bias(name, index, biased):
    counts = COUNTS[name]
    R, E, T = sum(counts), len(counts), 13
    x, w = make(T, 300, E, 200)
    g = torch.Generator(device="cuda").manual_seed(5)
    rows = torch.randint(0, T, (R,), generator=g, device="cuda").to(index)
    bias = torch.randn(E, 200, generator=g, device="cuda").to(biased)
    got = fm.int8_linear(x, w, route(counts), rows=rows, bias=bias, out_dtype=torch.float32)
    check(got, *reference(x, w, counts, rows, bias), torch.float32)


@pytest.mark.parametrize("R,K,N", [(1, 128, 128), (3, 7168, 64), (40, 256, 1000), (300, 640, 384),
                                   (1000, 512, 272)])
def test_one_expert_without_offsets(R, K, N):
    x, w = make(R, K, 1, N)
    want = reference(x, w, [R])
    flat = fm.Int8Weights(w.data[0], w.scales[0], K)
    for weights in (w, flat):
        check(fm.int8_linear(x, weights, out_dtype=torch.float32), *want, torch.float32)
    b = torch.randn(N, device="cuda")
    got = fm.int8_linear(x, flat, bias=b, out_dtype=torch.float32)
    check(got, *reference(x, w, [R], bias=b.view(1, N)), torch.float32)


@pytest.mark.parametrize("rows_per", [1, 100])
def test_largest_sums_stay_exact(rows_per):
    """K at its limit with every value at -128: the sum is 2^31 - 16384."""
    K = 131071
    x = torch.full((rows_per, 131072), -128, dtype=torch.int8, device="cuda")
    x[:, K:] = 0
    w = torch.full((1, 16, 131072), -128, dtype=torch.int8, device="cuda")
    w[:, :, K:] = 0
    got = fm.int8_linear(fm.QuantizedRows(x, torch.ones(rows_per, device="cuda"), K),
                         fm.Int8Weights(w, torch.ones(1, 16, device="cuda"), K),
                         out_dtype=torch.float32)
    assert (got == float(16384 * K)).all()


@pytest.mark.parametrize("per", [1, 40, 200])
def test_rows_of_no_expert_and_indices_outside(per):
    counts = [per, 0, per + 3]
    R, T = sum(counts) + 70, 9
    x, w = make(T, 200, 3, 40)
    rows = torch.arange(R, device="cuda") % T
    rows[0], rows[per], rows[per + 1] = -1, T, 1 << 40
    got = fm.int8_linear(x, w, route(counts), rows=rows, out_dtype=torch.float32)
    want, mag = reference(x, w, counts, rows)
    check(got, want, mag, torch.float32)
    assert not got[0].any() and not got[per].any() and not got[per + 1].any()
    assert not got[sum(counts):].any()
    with pytest.raises(IndexError):
        fm.int8_linear(x, w, route(counts), rows=rows, validate=True)
    # offsets that fall, or end outside the rows: bounded on the device, refused with validate
    for off in ([0, 5, 2, 30], [0, 5, 9, R + 1], [3, 5, 9, 12], [0, -4, 1 << 50, 7]):
        off = torch.tensor(off, device="cuda")
        fm.int8_linear(x, w, off, rows=rows)
        torch.cuda.synchronize()
        with pytest.raises(IndexError):
            fm.int8_linear(x, w, off, rows=rows.clamp(0, T - 1), validate=True)
    fm.int8_linear(x, w, route(counts), rows=rows.clamp(0, T - 1), validate=True)


def test_bad_scales_show():
    """A row whose scale is NaN (it held an infinity) gives NaN, and only that row."""
    x, w = make(40, 256, 2, 33)
    x.scales[7] = float("nan")
    got = fm.int8_linear(x, w, route([20, 20]))
    assert got[7].isnan().all()
    assert torch.cat([got[:7], got[8:]]).isfinite().all()


def test_rows_of_a_wider_buffer_and_no_rows():
    x, w = make(50, 256, 2, 48)
    want = fm.int8_linear(x, w, route([20, 30]))
    wide = torch.full((50, 512), 77, dtype=torch.int8, device="cuda")
    wide[:, 128:384] = x.data
    got = fm.int8_linear(fm.QuantizedRows(wide[:, 128:384], x.scales, 256), w, route([20, 30]))
    assert torch.equal(got, want)
    none = fm.int8_linear(fm.QuantizedRows(x.data[:0], x.scales[:0], 256), w, route([0, 0]))
    assert none.shape == (0, 48)
    none = fm.int8_linear(x, w, route([0, 0]), rows=torch.empty(0, dtype=torch.int64, device="cuda"))
    assert none.shape == (0, 48)
    assert not fm.int8_linear(x, w, route([0, 0])).any()


def test_graph_and_stream():
    x, w = make(12, 512, 20, 128)
    rows = torch.arange(96, device="cuda") % 12
    off = route([5] * 16 + [4] * 4)
    s = torch.cuda.Stream()
    want = fm.int8_linear(x, w, off, rows=rows)
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = fm.int8_linear(x, w, off, rows=rows)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = fm.int8_linear(x, w, off, rows=rows)
    for shift in (1, 2, 3):  # new routing in the same buffers
        rows.copy_((torch.arange(96, device="cuda") + shift) % 12)
        off.copy_(route([5 - shift] * 16 + [4 + 4 * shift] * 4))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, fm.int8_linear(x, w, off, rows=rows))


def test_weights_from_modules_and_tensors():
    g = torch.Generator(device="cuda").manual_seed(1)
    w = torch.randn(3, 20, 150, generator=g, device="cuda")
    a = fm.quantize_weights(w)
    b = fm.quantize_weights([w[e] for e in range(3)])
    c = fm.quantize_weights(w[1])
    assert torch.equal(a.data, b.data) and torch.equal(a.scales, b.scales)
    assert torch.equal(a.data[1], c.data[0]) and a.data.shape == (3, 20, 256) and a.features == 150
    back = a.data[:, :, :150].double() * a.scales.double().unsqueeze(-1)
    assert ((back - w.double()).abs() <= a.scales.double().unsqueeze(-1) * 0.5001).all()


def test_refusals():
    x, w = make(8, 256, 2, 16)
    off = route([4, 4])
    with pytest.raises(ValueError, match="need expert_offsets"):
        fm.int8_linear(x, w)
    with pytest.raises(ValueError, match="expert_offsets"):
        fm.int8_linear(x, w, off[:2])
    with pytest.raises(ValueError, match="expert_offsets"):
        fm.int8_linear(x, w, off.int())
    with pytest.raises(ValueError, match="features"):
        fm.int8_linear(x, fm.Int8Weights(w.data[:, :, :128].contiguous(), w.scales, 128), off)
    with pytest.raises(ValueError, match="columns"):
        fm.int8_linear(x._replace(features=100), w, off)
    with pytest.raises(TypeError, match="int8"):
        fm.int8_linear(x._replace(data=x.data.float()), w, off)
    with pytest.raises(ValueError, match="16 bytes"):
        shifted = torch.zeros(8 * 256 + 8, dtype=torch.int8, device="cuda")[8:].view(8, 256)
        fm.int8_linear(x._replace(data=shifted), w, off)
    with pytest.raises(ValueError, match="scales"):
        fm.int8_linear(x._replace(scales=x.scales[:3]), w, off)
    with pytest.raises(TypeError, match="rows"):
        fm.int8_linear(x, w, off, rows=torch.zeros(8, device="cuda"))
    with pytest.raises(ValueError, match="bias"):
        fm.int8_linear(x, w, off, bias=torch.zeros(16, device="cuda"))
    with pytest.raises(RuntimeError, match="no gradient"):
        fm.int8_linear(x, w, off, bias=torch.zeros(2, 16, device="cuda", requires_grad=True))
    with pytest.raises(TypeError, match="out_dtype"):
        fm.int8_linear(x, w, off, out_dtype=torch.int32)
    with pytest.raises(ValueError, match="not empty"):
        fm.int8_linear(fm.QuantizedRows(x.data[:0], x.scales[:0], 256), w, off,
                       rows=torch.zeros(8, dtype=torch.int64, device="cuda"))


def test_arrays_beyond_32_bits():
    """Rows, weights and results whose offsets pass 4 GiB."""
    K, N = 16384, 2048
    x, w = make(4, K, 2, N)
    want = reference(x, w, [2, 2])[0]
    big = torch.zeros(270_000, K, dtype=torch.int8, device="cuda")  # 4.4e9 bytes
    last = torch.arange(270_000 - 4, 270_000, device="cuda")
    big[last] = x.data
    scales = torch.zeros(270_000, device="cuda")
    scales[last] = x.scales
    heavy = torch.zeros(140, N, K, dtype=torch.int8, device="cuda")  # 4.7e9 bytes
    heavy[-2:] = w.data
    heavy_scales = torch.zeros(140, N, device="cuda")
    heavy_scales[-2:] = w.scales
    got = fm.int8_linear(fm.QuantizedRows(big, scales, K), fm.Int8Weights(heavy, heavy_scales, K),
                         route([0] * 138 + [2, 2]), rows=last, out_dtype=torch.float32)
    assert ((got.double() - want).abs() <= 6 * U * want.abs()).all()
    del big, heavy
    R, wide = 80_000, 32768
    x, w = make(R, 128, 1, wide)
    got = fm.int8_linear(x, w)  # 5.2e9 bytes
    for at in (slice(0, 3), slice(R - 3, R)):
        part = fm.QuantizedRows(x.data[at], x.scales[at], 128)
        check(got[at], *reference(part, w, [3]), torch.bfloat16)


def test_two_streams_at_once():
    cases = []
    for seed, counts in enumerate(([1, 0, 5], [300, 200, 77], [3000])):
        x, w = make(sum(counts), 640, len(counts), 512, seed=seed)
        cases.append((x, w, route(counts)))
    want = [fm.int8_linear(*c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(10):
        got = []
        for s, c in zip(streams, cases):
            with torch.cuda.stream(s):
                got.append(fm.int8_linear(*c))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_indices_and_offsets_with_gaps():
    """Every second element of a longer tensor is taken as it is."""
    x, w = make(9, 200, 3, 40)
    counts = [4, 0, 7]
    rows, off = torch.randint(0, 9, (11,), device="cuda"), route(counts)
    bias = torch.randn(3, 40, device="cuda")
    gaps = [torch.stack([t, torch.full_like(t, 7)], -1)[..., 0] for t in (rows, off, bias)]
    assert not any(t.is_contiguous() for t in gaps)
    got = fm.int8_linear(x, w, gaps[1], rows=gaps[0], bias=gaps[2])
    assert torch.equal(got, fm.int8_linear(x, w, off, rows=rows, bias=bias))
