"""int8_linear where scales, tiles and routing are at the ends of their ranges.

The sums are exact, so the roundings are the sum's conversion to fp32, three products and the bias'
addition, half a step u = 2^-24 each, and the output's own."""
from __future__ import annotations

import pytest
import torch

import fastmoe_amd as fm
from fastmoe_amd import _abi

from .test_int8_linear_gpu import TILES, U, check, make, ragged, reference, route

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("tile,E,mean,N", TILES + [(32128, 30, 5, 2000)])
def test_scales_of_every_size(tile, E, mean, N, dtype):
    """Scales from 2^-120 to 2^120: every result that the type holds is right, however large or small the
    factors on the way, and none is infinite that need not be."""
    K = 300
    counts = ragged(E, mean)
    R = sum(counts)
    assert _abi.lib().fmoe_int8_linear_tile(R, E, N, K) == tile
    x, w = make(R, K, E, N, seed=3)
    g = torch.Generator(device="cuda").manual_seed(4)
    spread = lambda *s: torch.exp2(torch.rand(s, generator=g, device="cuda") * 240 - 120)
    x = x._replace(scales=spread(R))
    w = w._replace(scales=spread(E, N))
    got = fm.int8_linear(x, w, route(counts), out_dtype=dtype).double()
    want, _ = reference(x, w, counts)
    normal = (want.abs() < 2.0 ** 127) & (want.abs() > 2.0 ** -100)
    assert normal.float().mean() > 0.3
    err = (got - want).abs()[normal]
    half = torch.finfo(dtype).eps / 2 if dtype is not torch.float32 else 0
    assert (err <= (half + 6 * U) * want.abs()[normal]).all()
    assert got[want.abs() > 2.0 ** 128].isinf().all()
    assert (got[want.abs() <= 2.0 ** -100].abs() <= 2.0 ** -99).all()


def test_rows_near_the_largest_numbers():
    """Rows of 1e38 by weights of 1e-3, quantised here: products of 1e35 times a few, far from the type's end."""
    for dtype in (torch.float32, torch.bfloat16):
        x = torch.full((3, 64), 1e38, dtype=dtype, device="cuda")
        w = torch.full((40, 64), 1e-3, device="cuda")
        got = fm.int8_linear(fm.quantize_rows(x), fm.quantize_weights(w), out_dtype=dtype)
        want = x.double() @ w.double().t()
        # both are their rows' largest: 127 steps of a scale, a few u off
        assert ((got.double() - want).abs() <= (torch.finfo(dtype).eps / 2 + 16 * U) * want).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("tile,E,mean,N", [(256256, 50, 130, 1024), (256256, 50, 130, 1025), (128256, 40, 40, 1024),
                                           (128256, 40, 40, 992)])
def test_rows_that_start_with_a_line_of_memory_and_inside_one(tile, E, mean, N, dtype):
    K = 300
    counts = ragged(E, mean)
    R = sum(counts)
    assert _abi.lib().fmoe_int8_linear_tile(R, E, N, K) == tile
    x, w = make(R, K, E, N, seed=3)
    got = fm.int8_linear(x, w, route(counts), out_dtype=dtype)
    check(got, *reference(x, w, counts), dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("tile,E,mean,N", [(256256, 50, 130, 1024), (256256, 50, 130, 1025), (128256, 40, 40, 1024),
                                           (128256, 40, 40, 992)])
def test_rows_that_start_with_a_line_of_memory_and_inside_one(tile, E, mean, N, dtype):
    K = 300
    counts = ragged(E, mean)
    R = sum(counts)
    assert _abi.lib().fmoe_int8_linear_tile(R, E, N, K) == tile
    x, w = make(R, K, E, N, seed=3)
    got = fm.int8_linear(x, w, route(counts), out_dtype=dtype)
    check(got, *reference(x, w, counts), dtype)


@pytest.mark.parametrize("tile,E,mean,N", TILES)
def test_scales_of_either_sign(tile, E, mean, N):
    """A scale may be negative; its size alone says which factor comes first."""
    counts = ragged(E, mean)
    R = sum(counts)
    x, w = make(R, 300, E, N, seed=3)
    g = torch.Generator(device="cuda").manual_seed(5)
    sign = lambda *s: torch.randint(0, 2, s, generator=g, device="cuda") * 2.0 - 1
    x = x._replace(scales=sign(R) * 1e36)
    w = w._replace(scales=sign(E, N) * 1e-36)
    want, _ = reference(x, w, counts)
    got = fm.int8_linear(x, w, route(counts), out_dtype=torch.float32).double()
    assert ((got - want).abs() <= 6 * U * want.abs()).all()
