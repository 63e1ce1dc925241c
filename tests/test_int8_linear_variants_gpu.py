"""Every kernel that int8_linear chooses from, on routing that is far from even too.

128 x 256 has two: up to 104 rows per expert its weights pass the caches, above they stay in them."""
from __future__ import annotations

import pytest
import torch

import fastmoe_amd as fm
from fastmoe_amd import _abi

from .test_int8_linear_gpu import KS, check, make, ragged, reference, route

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def one_and_many(tile, counts, N, K, dtype, seed=0):
    R, E = sum(counts), len(counts)
    assert _abi.lib().fmoe_int8_linear_tile(R, E, N, K) == tile
    x, w = make(R, K, E, N, seed=K)
    bias = torch.randn(E, N, device="cuda")
    check(fm.int8_linear(x, w, route(counts), bias=bias, out_dtype=dtype),
          *reference(x, w, counts, bias=bias), dtype)
    g = torch.Generator(device="cuda").manual_seed(K)
    rows = torch.randint(-2, R + 2, (R + 37,), generator=g, device="cuda", dtype=torch.int32)
    check(fm.int8_linear(x, w, route(counts), rows=rows, out_dtype=dtype),
          *reference(x, w, counts, rows), dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("K", KS + [1001])
def test_128_x_256_with_weights_kept_in_the_caches(K, dtype):
    counts = ragged(13, 346, seed=K)
    assert sum(counts) // 13 > 104
    one_and_many(128256, counts, 1003, K, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tile,counts,N,K", [
    (128256, [3000, 0, 1, 2, 1490, 0, 0, 0, 5, 0, 0, 0, 3], 1003, 500),
    (128256, [0] * 40 + [3800] + [0] * 22 + [70], 1000, 300),
    (256256, [6000, 0, 0, 255, 0, 1, 257, 2000], 4100, 300),
    (256256, [1] * 49 + [9000], 1000, 641),
    (128128, [0] * 15 + [1040], 1024, 500),
    (32064, [150] + [0] * 29, 300, 130),
    (32128, [0, 130] + [1] * 20 + [0] * 8, 2000, 300),
    (16016, [0, 0, 12], 130, 1100),
])
def test_a_few_experts_have_most_rows(tile, counts, N, K, dtype):
    one_and_many(tile, counts, N, K, dtype)
