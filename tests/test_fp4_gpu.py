"""Weights in 4 bits and the products with them against their definition in 64 bits.

Tolerances.  Codes, scales and restored values: equal.  A product's sum in fp32: every weight and every single
product is exact, a matrix unit adds up to 32 of them and a chain of at most K / 16 such sums (and eight parts) follows, each
addition off by at most 2^-23 of the sizes added: (K / 16 + 40) * 2^-23 of sum |x w|; one rounding to the
output's type.  GELU has a slope below 1.13 and its own error: 2^-12 relative and 2^-18 absolute for bf16, 2^-15 and 2^-21
for the others (fp32 output: erfc, (x^2 + 2) * 2^-23 relative for |x| below 8).
"""
from __future__ import annotations

import pytest
import torch

import fastmoe_amd as fm
from tests import fp4_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
B, H, F = torch.bfloat16, torch.float16, torch.float32
TINY = {F: 2.0 ** -126, B: 2.0 ** -126, H: 2.0 ** -24}


def offsets_of(counts):
    return torch.cat([torch.zeros(1, dtype=torch.int64), torch.tensor(counts).cumsum(0)])


def check(got, want, size, K, gelu=False):
    dt = got.dtype
    got = got.double().cpu()
    tol = size * ((K / 16 + 40) * 2.0 ** -23)
    if gelu:
        rel, low = (2.0 ** -12, 2.0 ** -18) if dt == B else (2.0 ** -15, 2.0 ** -21)
        tol = 1.13 * tol + want.abs() * rel + low
    tol = tol + want.abs() * (torch.finfo(dt).eps / 2) + TINY[dt]
    err = (got - want).abs()
    assert got.shape == want.shape and bool((err <= tol).all()), float((err / tol).nan_to_num(9e9).max())


def run(counts, N, K, dtype=B, out=None, gather=0, bias=False, gelu=False, behind=0, seed=0, idx=torch.int64):
    """A call on experts with these counts of rows, held to the definition; `gather`: tokens the rows are read of."""
    E, R = len(counts), sum(counts) + behind
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(gather or R, K, generator=gen).to(dtype)
    data, scales = ref.weights(E, N, K, seed)
    off = offsets_of(counts)
    rows = torch.randint(0, gather, (R,), generator=gen).to(idx) if gather else None
    b = torch.randn(E, N, generator=gen).to(dtype) if bias else None
    got = fm.fp4_linear(x.to(DEV), fm.Fp4Weights(data.to(DEV), scales.to(DEV), K), off.to(DEV),
                        rows=None if rows is None else rows.to(DEV), bias=None if b is None else b.to(DEV),
                        activation="gelu" if gelu else None, out_dtype=out)
    assert got.dtype == (out or dtype)
    want, size = ref.linear(x, ref.values(data, scales, K), off, rows, b, gelu, R)
    check(got, want, size, K, gelu)
    assert not got[sum(counts):].any()


COUNTS = [[1], [0, 1, 0, 2], [16, 0, 17, 5], [33, 64, 65, 31], [128, 1, 129, 0, 200], [300, 40]]


@pytest.mark.parametrize("dtype", [B, H], ids=str)
@pytest.mark.parametrize("N,K", [(1, 1), (16, 128), (17, 129), (100, 33), (256, 256), (257, 200), (64, 1000), (300, 1001)])
@pytest.mark.parametrize("counts", COUNTS, ids=str)
def test_products(counts, N, K, dtype):
    run(counts, N, K, dtype, seed=N + K)


@pytest.mark.parametrize("out", [F, B, H], ids=str)
@pytest.mark.parametrize("dtype", [B, H], ids=str)
@pytest.mark.parametrize("counts", COUNTS[2:], ids=str)
def test_bias_gelu_and_output_types(counts, dtype, out):
    run(counts, 130, 300, dtype, out, bias=True)
    run(counts, 130, 300, dtype, out, gelu=True)
    run(counts, 130, 256, dtype, out, bias=True, gelu=True, gather=50)


@pytest.mark.parametrize("idx", [torch.int64, torch.int32], ids=str)
@pytest.mark.parametrize("counts", COUNTS, ids=str)
def test_rows_through_an_index_and_rows_behind(counts, idx):
    run(counts, 70, 260, gather=9, behind=3, idx=idx)
    run(counts, 70, 256, behind=40, bias=True, gelu=True)
    run([0] * len(counts), 70, 256, behind=40, bias=True)


def test_many_experts():
    run([(7 * e) % 3 for e in range(600)], 40, 128, gather=30)
    run([(7 * e) % 5 for e in range(257)], 33, 130, behind=2, bias=True)


@pytest.mark.parametrize("T", [1, 15, 40, 200])
def test_one_expert_without_offsets(T):
    x = torch.randn(T, 192, generator=torch.Generator().manual_seed(1)).to(B)
    data, scales = ref.weights(1, 100, 192)
    want, size = ref.linear(x, ref.values(data, scales, 192), [0, T])
    for w in (fm.Fp4Weights(data.to(DEV), scales.to(DEV), 192), fm.Fp4Weights(data[0].to(DEV), scales[0].to(DEV), 192)):
        check(fm.fp4_linear(x.to(DEV), w), want, size, 192)
    bias = torch.randn(100).to(DEV)
    check(fm.fp4_linear(x.to(DEV), w, bias=bias), want + bias.double().cpu(), size + bias.abs().double().cpu(), 192)


@pytest.mark.parametrize("T", [5, 150])
@pytest.mark.parametrize("K", [256, 250])
def test_strides_alignment_and_gaps(T, K):
    gen = torch.Generator().manual_seed(3)
    data, scales = ref.weights(3, 90, K)
    w = fm.Fp4Weights(data.to(DEV), scales.to(DEV), K)
    flat = torch.randn(T * (K + 21) + 5, generator=gen).to(B)
    off = offsets_of([T // 3, 1, T - T // 3 - 1])
    for start, width in ((0, K + 16), (3, K + 21), (8, K + 8)):
        x = flat[start:start + T * width].view(T, width)[:, :K]
        on = flat.to(DEV)[start:start + T * width].view(T, width)[:, :K]
        want, size = ref.linear(x, ref.values(data, scales, K), off)
        check(fm.fp4_linear(on, w, off.to(DEV)), want, size, K)
    gaps = torch.zeros(8, dtype=torch.int64)
    gaps[::2] = off
    order = torch.arange(2 * T).flip(0) // 2  # every other entry
    check(fm.fp4_linear(on, w, gaps.to(DEV)[::2], rows=order.to(DEV)[::2]),
          *ref.linear(x, ref.values(data, scales, K), off, order[::2]), K)
    one = flat.to(DEV)[:K].view(1, K).expand(T, K)  # every row the same memory
    check(fm.fp4_linear(one, w, off.to(DEV)), *ref.linear(one.cpu(), ref.values(data, scales, K), off), K)


@pytest.mark.parametrize("counts", [[3, 2], [100, 60]], ids=str)
def test_indices_outside_are_zero_and_said(counts):
    R = sum(counts)
    x = torch.randn(20, 128, generator=torch.Generator().manual_seed(1)).to(B)
    data, scales = ref.weights(2, 48, 128)
    w = fm.Fp4Weights(data.to(DEV), scales.to(DEV), 128)
    rows = torch.randint(0, 20, (R,), generator=torch.Generator().manual_seed(2))
    rows[0], rows[2], rows[-1] = -1, 20, 1 << 40
    off, bias = offsets_of(counts), torch.randn(2, 48)
    got = fm.fp4_linear(x.to(DEV), w, off.to(DEV), rows=rows.to(DEV), bias=bias.to(DEV))
    check(got, *ref.linear(x, ref.values(data, scales, 128), off, rows, bias), 128)
    assert torch.equal(got[0].cpu(), bias[0].to(B))
    with pytest.raises(IndexError, match="3 entries"):
        fm.fp4_linear(x.to(DEV), w, off.to(DEV), rows=rows.to(DEV), validate=True)
    for bad in ([0, 5, R + 1], [0, R, R - 1], [1, 2, R]):
        with pytest.raises(IndexError):
            fm.fp4_linear(x.to(DEV), w, torch.tensor(bad, device=DEV), rows=rows.clamp(0, 19).to(DEV), validate=True)
    # offsets that are none: nothing outside the arrays, whatever comes out
    for bad in ([0, 5, R + 9], [0, R, 3], [-5, 2, 1 << 50], [0, -3, R]):
        out = fm.fp4_linear(x.to(DEV), w, torch.tensor(bad, device=DEV), rows=rows.clamp(0, 19).to(DEV))
        assert out.shape == (R, 48)


@pytest.mark.parametrize("counts", [[4], [140]], ids=str)
def test_what_is_not_finite_stays_in_its_row_or_column(counts):
    T, N, K = counts[0], 70, 200
    x = torch.randn(T, K, generator=torch.Generator().manual_seed(1)).to(B)
    data, scales = ref.weights(1, N, K)
    x[1, 5], x[2, 199] = float("nan"), float("inf")
    scales[0, 9, 2] = 255
    got = fm.fp4_linear(x.to(DEV), fm.Fp4Weights(data.to(DEV), scales.to(DEV), K)).cpu()
    want, size = ref.linear(x, ref.values(data, scales, K), [0, T])
    keep = torch.ones(T, dtype=torch.bool)
    keep[1:3] = False
    cols = torch.arange(N) != 9
    assert got[1].isnan().all() and not got[2].isfinite().any() and got[:, 9].isnan().all()
    check(got[keep][:, cols], want[keep][:, cols], size[keep][:, cols], K)
    # padding is not read as rows: what lies behind a row's end has no part in it
    wide = torch.full((T, K + 60), float("nan"), dtype=B)
    wide[:, :K] = torch.randn(T, K, generator=torch.Generator().manual_seed(4)).to(B)
    scales[0, 9, 2] = 120
    got = fm.fp4_linear(wide.to(DEV)[:, :K], fm.Fp4Weights(data.to(DEV), scales.to(DEV), K))
    check(got, *ref.linear(wide[:, :K], ref.values(data, scales, K), [0, T]), K)


def test_the_smallest_and_largest_scales():
    x = torch.ones(3, 128, dtype=B)
    for low in (0, 1, 60, 200, 240):
        data, scales = ref.weights(1, 40, 128, low=low, high=low + 3)
        got = fm.fp4_linear(x.to(DEV), fm.Fp4Weights(data.to(DEV), scales.to(DEV), 128), out_dtype=F)
        # matrix units may take the smallest numbers of all as zero
        want, size = ref.linear(x, ref.values(data, scales, 128), [0, 3])
        err = (got.double().cpu() - want).abs()
        assert bool((err <= size * 2.0 ** -16 + 128 * 2.0 ** -125).all())
    # fp16 holds every weight whose scale lies between 2^-23 and 2^13
    for low in (127 - 23, 127 + 11):
        data, scales = ref.weights(1, 40, 128, low=low, high=low + 3)
        got = fm.fp4_linear(x.to(H).to(DEV), fm.Fp4Weights(data.to(DEV), scales.to(DEV), 128), out_dtype=F)
        want, size = ref.linear(x, ref.values(data, scales, 128), [0, 3])
        check(got, want, size, 128)


@pytest.mark.parametrize("dtype", [F, B, H], ids=str)
@pytest.mark.parametrize("K", [1, 31, 32, 129, 1000])
def test_weights_to_four_bits_and_back(K, dtype):
    gen = torch.Generator().manual_seed(K)
    x = (torch.randn(3, 41, K, generator=gen) * torch.randn(3, 41, 1, generator=gen).exp()).to(dtype)
    x[0, 0] = 0
    x[1, 1, 0] = 6 * 2.0 ** -3                      # a block whose largest is just representable
    x[1, 2] = torch.randint(-12, 13, (K,), generator=gen).to(dtype) / 4  # ties
    if K > 30:
        x[2, 3, 7], x[2, 4, 30], x[2, 5, 0] = float("inf"), float("nan"), -float("inf")
    want, scales = ref.quantize(x)
    for given in (x.to(DEV), [p.to(DEV) for p in x]):
        w = fm.quantize_weights_fp4(given)
        assert w.features == K and torch.equal(w.scales.cpu(), scales) and torch.equal(w.data.cpu(), want)
    v = ref.values(want, scales, K)
    for dt in (F, B, H):
        assert torch.equal(w.dequantize(dt).cpu(), v.to(F).to(dt)) or K > 30
        back = w.dequantize(dt).cpu()
        assert torch.equal(back.isnan(), v.isnan()) and torch.equal(back.nan_to_num(0.0), v.nan_to_num(0.0).to(F).to(dt))
    one = fm.quantize_weights_fp4(x[1].to(DEV))
    assert one.data.shape[0] == 1 and torch.equal(one.data[0].cpu(), want[1])
    assert fm.Fp4Weights(one.data[0], one.scales[0], K).dequantize().shape == (41, K)


def test_weights_of_the_smallest_numbers():
    x = torch.tensor([[2.0 ** -126, 2.0 ** -130, 2.0 ** -149] + [0.0] * 29, [3e38, -3e38, 1e38] + [0.0] * 29])
    want, scales = ref.quantize(x)
    w = fm.quantize_weights_fp4(x.to(DEV))
    assert torch.equal(w.scales[0].cpu(), scales) and torch.equal(w.data[0].cpu(), want)


def test_graph_replays_and_two_streams():
    counts = [5, 0, 90, 33]
    data, scales = ref.weights(4, 200, 384)
    w = fm.Fp4Weights(data.to(DEV), scales.to(DEV), 384)
    x = torch.empty(40, 384, dtype=B, device=DEV)
    rows = torch.empty(128, dtype=torch.int64, device=DEV)
    off = torch.empty(5, dtype=torch.int64, device=DEV)

    def fill(seed):
        gen = torch.Generator().manual_seed(seed)
        x.copy_(torch.randn(40, 384, generator=gen).to(B))
        rows.copy_(torch.randint(0, 40, (128,), generator=gen))
        off.copy_(offsets_of([counts[(i + seed) % 4] for i in range(4)]))

    fill(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = fm.fp4_linear(x, w, off, rows=rows, activation="gelu")
    here = fm.fp4_linear(x, w, off, rows=rows, activation="gelu")
    torch.cuda.synchronize()
    assert torch.equal(other, here)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fm.fp4_linear(x, w, off, rows=rows, activation="gelu")
    for seed in range(4):
        fill(seed)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, fm.fp4_linear(x, w, off, rows=rows, activation="gelu"))


def test_refusals():
    data, scales = ref.weights(2, 16, 100)
    w = fm.Fp4Weights(data.to(DEV), scales.to(DEV), 100)
    x = torch.randn(8, 100, device=DEV).to(B)
    off = torch.tensor([0, 3, 8], device=DEV)
    fm.fp4_linear(x, w, off)
    with pytest.raises(TypeError, match="bfloat16 or float16"):
        fm.fp4_linear(x.float(), w, off)
    with pytest.raises(ValueError, match="features"):
        fm.fp4_linear(x[:, :99], w, off)
    with pytest.raises(ValueError, match="need expert_offsets"):
        fm.fp4_linear(x, w)
    with pytest.raises(ValueError, match="expert_offsets"):
        fm.fp4_linear(x, w, off[:2])
    with pytest.raises(ValueError, match="expert_offsets"):
        fm.fp4_linear(x, w, off.int())
    with pytest.raises(TypeError, match="rows"):
        fm.fp4_linear(x, w, off, rows=off.float())
    with pytest.raises(ValueError, match="bias"):
        fm.fp4_linear(x, w, off, bias=torch.zeros(16, device=DEV))
    with pytest.raises(ValueError, match="unknown activation"):
        fm.fp4_linear(x, w, off, activation="relu")
    with pytest.raises(TypeError, match="out_dtype"):
        fm.fp4_linear(x, w, off, out_dtype=torch.int8)
    with pytest.raises(ValueError, match="unit column stride"):
        fm.fp4_linear(torch.zeros(100, 8, device=DEV, dtype=B).t(), w, off)
    with pytest.raises(RuntimeError, match="no gradient"):
        fm.fp4_linear(x.clone().requires_grad_(True), w, off)
    with pytest.raises(TypeError, match="uint8"):
        fm.fp4_linear(x, fm.Fp4Weights(w.data.to(torch.int8), w.scales, 100), off)
    with pytest.raises(ValueError, match="stored"):
        fm.fp4_linear(x, fm.Fp4Weights(w.data[..., :50], w.scales, 100), off)
    with pytest.raises(ValueError, match="stored"):
        fm.fp4_linear(x, fm.Fp4Weights(w.data, w.scales[:1], 100), off)
    with pytest.raises(ValueError, match="contiguous"):
        fm.fp4_linear(x, fm.Fp4Weights(w.data.transpose(0, 1).contiguous().transpose(0, 1), w.scales, 100), off)
    moved = torch.zeros(w.data.numel() + 16, dtype=torch.uint8, device=DEV)[8:8 + w.data.numel()].view(w.data.shape)
    with pytest.raises(ValueError, match="multiples"):
        fm.fp4_linear(x, fm.Fp4Weights(moved, w.scales, 100), off)
    with pytest.raises(RuntimeError, match="only on the GPU"):
        fm.fp4_linear(x, fm.Fp4Weights(data, scales, 100), off)
    with pytest.raises(ValueError, match="must be"):
        fm.quantize_weights_fp4([x, x[:4]])
    with pytest.raises(ValueError, match="no weights"):
        fm.quantize_weights_fp4([])
    with pytest.raises(RuntimeError, match="only on the GPU"):
        fm.quantize_weights_fp4(x.cpu())
    assert fm.fp4_linear(x[:0], w, torch.zeros(3, dtype=torch.int64, device=DEV)).shape == (0, 16)


def _pick(rows, E, N, K):
    from fastmoe_amd import _abi

    return _abi.lib().fmoe_fp4_linear_tile(rows, E, N, K)


@pytest.mark.parametrize("tile,counts,N,K", [
    (16016, [1], 33, 700), (16016, [16], 250, 2304), (16016, [30], 130, 1100), (16016, [2], 17, 8192),
    (16032, [3], 5000, 1500), (16032, [16], 4200, 2600), (16032, [13, 1, 0], 2000, 1024),
    (16064, [4], 9000 + 5, 700), (16064, [40, 1, 2, 12], 2500, 520), (16064, [16, 16, 15, 1], 2300, 1792),
    (16128, [1] * 60, 900, 520), (16128, [5, 0, 16, 11] * 6, 1300, 1040), (16128, [100], 5000, 513),
    (96128, [30] * 40, 900, 512), (96128, [0, 97, 1, 64, 33, 200, 10, 70] * 3, 1050, 1001), (96128, [96, 95, 97, 31] * 8, 500, 832),
    (96256, [30] * 40, 2900, 320), (96256, [192, 1, 0, 130, 65, 96] * 8, 2300, 768), (96256, [400] * 10, 2049, 65),
], ids=str)
def test_every_variant(tile, counts, N, K):
    E, R = len(counts), sum(counts)
    assert _pick(R, E, N, K) == tile
    run(counts, N, K, bias=True, gelu=True)
    run(counts, N, K, H, F, gather=77, behind=0)


@pytest.mark.parametrize("K", [1, 5, 8, 9, 63, 66, 68, 71, 130, 189, 255])
@pytest.mark.parametrize("tile,counts,N", [
    (96128, [0, 97, 1, 64, 33, 200, 10, 70] * 3, 700), (96256, [30] * 40, 2900), (96256, [400, 90, 101, 0] * 10, 2049)], ids=str)
def test_rows_whose_last_piece_is_not_whole(tile, counts, N, K):
    assert _pick(sum(counts), len(counts), N, K) == tile
    run(counts, N, K, H if K % 2 else B, gather=50 if K % 3 else None)


@pytest.mark.parametrize("per", [79, 80, 81])
def test_rows_about_where_weights_stay_in_the_caches(per):
    assert _pick(per * 24, 24, 4096, 192) == 96256
    run([per] * 24, 4096, 192, bias=True)


def test_weights_and_rows_beyond_32_bits():
    """Codes of the last expert begin past 4 GiB, rows of x end past it: as a call on that expert, on those rows."""
    E, N, K = 5, 1 << 18, 8192
    gen = torch.Generator(device=DEV).manual_seed(0)
    data = torch.randint(0, 256, (E, N, K // 2), dtype=torch.uint8, generator=gen, device=DEV)
    scales = torch.randint(117, 122, (E, N, K // 32), dtype=torch.uint8, generator=gen, device=DEV)
    x = torch.zeros((1 << 18) + 200, K, dtype=B, device=DEV)
    x[-120:] = torch.randn(120, K, generator=gen, device=DEV).to(B)
    for per in (3, 120):
        off = torch.tensor([0, 0, 2, 2, 2, 2 + per], device=DEV)
        rows = torch.cat([torch.zeros(2, dtype=torch.int64), torch.arange(len(x) - per, len(x))]).to(DEV)
        out = fm.fp4_linear(x, fm.Fp4Weights(data, scales, K), off, rows=rows)
        assert not out[:2].any()
        pick = torch.arange(0, N, 1021)
        w = fm.Fp4Weights(data[4][pick], scales[4][pick], K)
        y = x[-per:]
        want, size = y.double() @ w.dequantize().double().T, y.double().abs() @ w.dequantize().double().abs().T
        check(out[2:][:, pick], want.cpu(), size.cpu(), K)
    del data, scales


@pytest.mark.parametrize("count", [4, 300])
def test_rows_outside_are_zero_whatever_x_holds(count):
    w = fm.Fp4Weights(*(t.to(DEV) for t in ref.weights(1, 300, 256)), 256)
    x = torch.full((3, 256), float("nan"), device=DEV, dtype=B)
    x[1] = 1
    rows = torch.full((count,), 1, device=DEV)
    rows[::3], rows[1::7] = -1, 99
    out = fm.fp4_linear(x, w, rows=rows)
    live = rows == 1
    assert not out[~live].any() and torch.equal(out[live], fm.fp4_linear(x[1:2], w).expand(int(live.sum()), -1))


@pytest.mark.parametrize("K", [3, 64, 100, 128, 192, 257, 400, 1000])
@pytest.mark.parametrize("counts", [[1], [3, 0, 12], [200, 97]], ids=str)
def test_what_lies_beside_the_rows_is_not_read(counts, K):
    """x is a slice of rows whose other columns hold NaN; padded codes are zero, their scales the largest."""
    data, scales = ref.weights(len(counts), 70, K)
    scales[..., (K + 31) // 32:] = 254
    w = fm.Fp4Weights(data.to(DEV), scales.to(DEV), K)
    x = torch.randn(sum(counts), K, generator=torch.Generator().manual_seed(K)).to(B)
    wide = torch.full((sum(counts), 16 + K + 24), float("nan"), dtype=B, device=DEV)
    off = offsets_of(counts)
    for at in (16, 11):
        wide.fill_(float("nan"))
        wide[:, at:at + K] = x.to(DEV)
        check(fm.fp4_linear(wide[:, at:at + K], w, off.to(DEV)), *ref.linear(x, ref.values(data, scales, K), off), K)
