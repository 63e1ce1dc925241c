"""GELU before 8 bits: as near as fp16's own results, whatever the rows' type."""
from __future__ import annotations

import pytest
import torch

import fastmoe_amd as fm

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.mark.parametrize("C", [512, 20000])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_whole_numbers_of_negative_rows(dtype, C):
    """Rows of negative values, whose GELU lies within 0.17 of zero: a step is 0.0013, so the error shows.

    With a an absolute error of 4e-7 and 8 u of the value in GELU, the largest value t carries both too;
    the quotient 127 / t and its product add 2 u: q is within 127 (2 a / t + 24 u) of the ideal value,
    and then rounded."""
    g = torch.Generator(device="cuda").manual_seed(1)
    x = (torch.rand(1 << 20, generator=g, device="cuda") * -5).to(dtype)[:(1 << 20) // C * C].view(-1, C)
    q = fm.quantize_rows(x, activation="gelu")
    v = x.double() * 0.5 * torch.erfc(-x.double() * 0.5 ** 0.5)
    top = v.abs().amax(-1, keepdim=True)
    a = 4e-7
    assert ((q.scales.double().unsqueeze(1) - top / 127).abs() <= a / 127 + 12 * U * top / 127).all()
    off = (q.data[:, :C].double() - v * 127 / top).abs()
    bound = 0.5 + 127 * (2 * a / top + 24 * U)
    bad = off > bound
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()}, worst {float((off - bound)[bad].max())}"
