"""The results of 16-bit types are the fp32 results rounded, whichever tile computes them."""
from __future__ import annotations

import pytest
import torch

import fastmoe_amd as fm
from fastmoe_amd import _abi

from .test_int8_linear_gpu import TILES, make, ragged, route

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tile,E,mean,N", TILES + [(32128, 30, 5, 2000)])
def test_a_result_is_the_fp32_one_rounded(tile, E, mean, N, dtype):
    counts = ragged(E, mean)
    R = sum(counts)
    assert _abi.lib().fmoe_int8_linear_tile(R, E, N, 300) == tile
    x, w = make(R, 300, E, N, seed=3)
    bias = torch.randn(E, N, device="cuda")
    for b in (None, bias):
        wide = fm.int8_linear(x, w, route(counts), bias=b, out_dtype=torch.float32)
        assert torch.equal(fm.int8_linear(x, w, route(counts), bias=b, out_dtype=dtype), wide.to(dtype))
