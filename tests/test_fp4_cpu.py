"""Refusals of the 4-bit weights and their C entry points (CPU: nothing is launched)."""
from __future__ import annotations

import pytest
import torch

import fastmoe_amd as fm
from fastmoe_amd import _abi

DEV = 0x10000  # stands for a device address: every call here is refused before a launch
B = _abi.BF16


def test_cpu_tensors_raise():
    w = fm.Fp4Weights(torch.zeros(1, 4, 64, dtype=torch.uint8), torch.zeros(1, 4, 4, dtype=torch.uint8), 8)
    x = torch.zeros(2, 8, dtype=torch.bfloat16)
    for call in (lambda: fm.fp4_linear(x, w), lambda: w.dequantize(), lambda: fm.quantize_weights_fp4(x),
                 lambda: fm.quantize_weights_fp4([x.requires_grad_(True)])):
        with pytest.raises(RuntimeError, match="only on the GPU"):
            call()
    with pytest.raises(TypeError, match="tensor"):
        fm.quantize_weights_fp4([[1.0]])


def _linear(x=DEV, xs=8, xr=4, xd=B, idx=None, idt=_abi.I64, w=DEV, s=DEV, b=None, bd=B, act=0, off=DEV, E=2, N=8,
            K=8, rows=4, out=DEV, os=8, od=B):
    return _abi.lib().fmoe_fp4_linear(x, xs, xr, xd, idx, idt, w, s, b, bd, act, off, E, N, K, rows, out, os, od, None)


def test_linear_entry_point_refuses():
    for bad in (dict(rows=-1), dict(xr=-1), dict(N=0), dict(K=0), dict(E=0), dict(xd=_abi.F32), dict(od=_abi.I64),
                dict(idx=DEV, idt=B), dict(b=DEV, bd=_abi.I64), dict(act=2), dict(off=None), dict(os=7), dict(xs=-8),
                dict(w=DEV + 8), dict(s=DEV + 2), dict(xr=0), dict(x=None), dict(w=None), dict(s=None), dict(out=None)):
        assert _linear(**bad) == _abi.EINVAL, bad
    for bad in (dict(K=(1 << 17) + 1), dict(N=1 << 25, os=1 << 25), dict(E=1 << 17), dict(rows=1 << 31),
                dict(xr=1 << 31), dict(rows=(1 << 31) - 1, N=1 << 24, os=1 << 24)):
        assert _linear(**bad) == _abi.ERANGE, bad
    assert _linear(rows=0, x=None, xr=0) == _abi.OK


def test_weight_entry_points_refuse():
    lib = _abi.lib()

    def to(x=DEV, stride=8, rows=4, cols=8, dt=B, q=DEV, s=DEV):
        return lib.fmoe_quantize_fp4(x, stride, rows, cols, dt, q, s, None)

    def back(q=DEV, s=DEV, rows=4, cols=8, out=DEV, dt=B):
        return lib.fmoe_restore_fp4(q, s, rows, cols, out, dt, None)

    for bad in (dict(rows=-1), dict(cols=0), dict(dt=_abi.I64), dict(q=None), dict(s=None), dict(q=DEV + 8)):
        assert to(**bad) == _abi.EINVAL and back(**bad) == _abi.EINVAL, bad
    assert to(x=None) == _abi.EINVAL and to(stride=-1) == _abi.EINVAL and back(out=None) == _abi.EINVAL
    for bad in (dict(rows=1 << 31), dict(cols=1 << 25), dict(rows=1 << 30, cols=1 << 20)):
        assert to(**bad) == _abi.ERANGE and back(**bad) == _abi.ERANGE, bad
    assert to(rows=0, x=None) == _abi.OK and back(rows=0, out=None) == _abi.OK


def test_tile_introspection():
    tile = _abi.lib().fmoe_fp4_linear_tile
    for bad in ((0, 1, 1, 1), (1, 0, 1, 1), (1, 1, 0, 1), (1, 1, 1, 0)):
        assert tile(*bad) == -1
    assert tile(1, 1, 2048, 7168) == 16016 and tile(49152, 64, 2048, 4096) == 96256
    for rows in (1, 7, 64, 1000, (1 << 31) - 1):
        for E in (1, 3, 256, 1 << 16):
            for N in (1, 128, 129, 1 << 24):
                assert tile(rows, E, N, 128) in (16016, 16032, 16064, 16128, 96128, 96256)
