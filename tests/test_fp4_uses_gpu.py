"""Products with weights in 4 bits at the ends of their types and of K."""
from __future__ import annotations

import pytest
import torch

import fastmoe_amd as fm

from . import fp4_ref as ref
from .test_fp4_gpu import B, DEV, F, _pick, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tile,rows,N", [(16016, 1, 40), (16032, 3, 5000), (16064, 4, 9005), (16128, 100, 5000),
                                         (96128, 1000, 600), (96256, 9000, 1024)])
@pytest.mark.parametrize("K", [100, 128, 384, 1100, 2176])
def test_the_largest_weights_beside_others(tile, rows, N, K):
    """The first 32 weights have the largest scale, the last ones the largest codes: what fills up the last 256 of K for
    the matrix units meets zeros, and is finite with any of a row's scales."""
    assert _pick(rows, 1, N, K) == tile
    codes = torch.zeros(1, N, ref.pad(K), dtype=torch.uint8)
    codes[..., 0] = 2                     # 2^127
    codes[..., K - 32:K] = 7              # 6
    scales = torch.full((1, N, ref.pad(K) // 32), 127, dtype=torch.uint8)
    scales[..., 0] = 254
    data = ref.pack(codes)
    x = torch.ones(rows, K, dtype=B)
    x[:, 0] = 2.0 ** -120
    x[:, 32:] *= torch.randn(rows, K - 32, generator=torch.Generator().manual_seed(K)).to(B)
    got = fm.fp4_linear(x.to(DEV), fm.Fp4Weights(data.to(DEV), scales.to(DEV), K), out_dtype=F)
    some = torch.tensor([0, 1, N // 2, N - 1])
    want, size = ref.linear(x, ref.values(data[:, some], scales[:, some], K), [0, rows])
    check(got[:, some], want, size, K)
    assert got.isfinite().all()
