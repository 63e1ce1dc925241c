"""The norm's backward over more rows than it has in flight: every unit takes several in turn.

A row's gradient depends on that row alone, so it has the same bits in a call in which each unit has one
row at most; the weight's is compared with the formula in 64 bits."""
from __future__ import annotations

import pytest
import torch

import fastmoe_amd as fm

from .test_norm_quantize_gpu import TYPES, U, close, half, norm64, rand

pytestmark = pytest.mark.gpu

# (rows, columns, rows of a workgroup, most workgroups): every width class, with two full rounds of rows
# and a ragged third one, and rows beyond the registers
SIZES = [(4500, 129, 4, 512), (4500, 512, 4, 512), (6200, 1001, 4, 512), (1300, 2048, 1, 512), (1300, 4096, 1, 512),
         (700, 7168, 1, 256), (601, 8192, 1, 256), (600, 16384, 1, 256), (1100, 16391, 1, 512)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,D,per_group,groups", SIZES)
def test_gradients_of_many_rows(T, D, per_group, groups, dtype):
    assert T > 2 * per_group * groups
    x, r, w = rand(T, D, dtype=dtype, seed=1), rand(T, D, dtype=dtype, seed=2), rand(D, dtype=dtype, seed=3)
    gy, gh = rand(T, D, dtype=dtype, seed=4), rand(T, D, dtype=dtype, seed=5)

    def grads(rows, through_stream):
        leaves = [x[rows].clone().requires_grad_(True), r[rows].clone().requires_grad_(True),
                  w.clone().requires_grad_(True)]
        y, h = fm.add_rms_norm(leaves[0], leaves[2], leaves[1])
        if through_stream:
            return torch.autograd.grad([y, h], leaves, [gy[rows], gh[rows]])
        return torch.autograd.grad(y, leaves, gy[rows])

    for through_stream in (True, False):
        gx, gr, gw = grads(slice(0, T), through_stream)
        assert torch.equal(gx, gr)
        for first in range(0, T, groups):
            part = slice(first, min(first + groups, T))
            assert torch.equal(gx[part], grads(part, through_stream)[0]), f"rows from {first}"
        h64, c, _ = norm64(x, w, r, 1e-6)
        terms = gy.double() * h64 * c
        # a unit's rows, its workgroup's units, every sixteenth workgroup and the sixteen, one addition
        # each; a term carries 64 u (the norm's factor and two products)
        steps = -(-T // (per_group * groups)) + per_group + groups // 16 + 16 + 64
        close(gw, terms.sum(0), half(dtype), steps * U * terms.abs().sum(0) + 2.0 ** -25)
        again = grads(slice(0, T), through_stream)
        assert torch.equal(again[0], gx) and torch.equal(again[2], gw)


@pytest.mark.parametrize("dtype", TYPES)
def test_gradients_of_many_rows_without_a_residual(dtype):
    T, D = 2500, 1000
    x, w, gy = rand(T, D, dtype=dtype, seed=1), rand(D, seed=3), rand(T, D, dtype=dtype, seed=4)

    def grads(rows):
        leaves = [x[rows].clone().requires_grad_(True), w.clone().requires_grad_(True)]
        return torch.autograd.grad(fm.add_rms_norm(*leaves)[0], leaves, gy[rows])

    gx, gw = grads(slice(0, T))
    assert gw.dtype == torch.float32
    for first in range(0, T, 512):
        part = slice(first, min(first + 512, T))
        assert torch.equal(gx[part], grads(part)[0])
    h64, c, _ = norm64(x, w, None, 1e-6)
    terms = gy.double() * h64 * c
    close(gw, terms.sum(0), U, (2 + 4 + 32 + 16 + 64) * U * terms.abs().sum(0))
