"""Refusals of the norms around a block and their C entry points (CPU: nothing is launched)."""
from __future__ import annotations

import pytest
import torch

import fastmoe_amd as fm
from fastmoe_amd import _abi

DEV = 0x10000  # stands for a device address: every call here is refused before a launch
B, F = _abi.BF16, _abi.F32


def test_cpu_tensors_raise():
    x, w = torch.zeros(2, 8), torch.ones(8)
    for t in (x, x.clone().requires_grad_(True)):
        with pytest.raises(RuntimeError, match="only on the GPU"):
            fm.sandwich_norm(t, w, x, w)


def _forward(x=DEV, xs=8, r=DEV, post=DEV, pre=DEV, wd=B, gate=None, gd=F, gr=0, rows=4, cols=8, dt=B, h=DEV, y=DEV):
    return _abi.lib().fmoe_sandwich_norm(x, xs, r, 8, post, pre, wd, gate, gd, gr, rows, cols, dt, 1.0, 1e-6, h, y,
                                         None, None)


def test_forward_entry_point_refuses():
    for bad in (dict(cols=0), dict(rows=-1), dict(dt=_abi.I64), dict(wd=_abi.F16), dict(post=None), dict(x=None),
                dict(r=None), dict(h=None), dict(y=None), dict(pre=None), dict(xs=-8), dict(gate=DEV),
                dict(gate=DEV, gr=3), dict(gate=DEV, gr=2, gd=_abi.F16), dict(gr=2), dict(gate=DEV, gr=-1)):
        assert _forward(**bad) == _abi.EINVAL, bad
    assert _forward(rows=1 << 40) == _abi.ERANGE
    assert _forward(cols=1 << 31) == _abi.ERANGE
    assert _forward(rows=0, x=None) == _abi.OK


def test_backward_entry_point_refuses():
    lib = _abi.lib()
    size = lib.fmoe_sandwich_norm_backward_workspace_bytes
    assert size(1000, 8, 0) == 250 * 8 * 8          # four rows in flight a workgroup
    assert size(100000, 2000, 0) == 512 * 2000 * 8
    assert size(100, 20000, 0) == 100 * 20000 * 8 + 400
    assert size(0, 8, 0) == 64
    assert size(-1, 8, 0) < 0 and size(4, 0, 0) < 0 and size(4, 8, 3) < 0 and size(4, 8, -1) < 0
    need = size(1000, 8, 2)

    def call(gy=DEV, gh=DEV, x=DEV, h=DEV, post=DEV, pre=DEV, wd=B, gate=DEV, gr=2, rstd=DEV, rows=1000, cols=8, gx=DEV,
             gpost=DEV, gpre=DEV, ggate=DEV, ws=DEV, nbytes=need):
        return lib.fmoe_sandwich_norm_backward(gy, 8, gh, 8, x, 8, h, post, pre, wd, gate, F, gr, rstd, rows, cols, B,
                                               1.0, gx, DEV, gpost, gpre, ggate, ws, nbytes, None)

    for bad in (dict(gy=None, gh=None), dict(x=None), dict(h=None), dict(rstd=None), dict(post=None), dict(pre=None),
                dict(wd=_abi.F16), dict(gate=None), dict(gate=None, gr=0), dict(gr=3), dict(ws=None),
                dict(ws=DEV + 4), dict(nbytes=need - 1), dict(rows=0),
                dict(cols=20000, gpost=None, gpre=None, ggate=None, ws=None)):
        assert call(**bad) == _abi.EINVAL, bad
    assert call(rows=1 << 40) == _abi.ERANGE


@pytest.mark.parametrize("scale,eps", [(float("inf"), 1e-6), (float("nan"), 1e-6), (1.0, float("inf")), (1.0, -1.0)])
def test_forward_entry_point_refuses_numbers(scale, eps):
    call = _abi.lib().fmoe_sandwich_norm
    assert call(DEV, 8, DEV, 8, DEV, DEV, B, None, F, 0, 4, 8, B, scale, eps, DEV, DEV, None, None) == _abi.EINVAL
