"""Refusals of the router and its C entry points (CPU: nothing is launched)."""
from __future__ import annotations

import pytest
import torch

import fastmoe_amd as fm
from fastmoe_amd import _abi

DEV = 0x10000  # stands for a device address: every call here is refused before a launch


def test_cpu_tensors_and_bad_options_raise():
    with pytest.raises(RuntimeError, match="only on the GPU"):
        fm.route_tokens(torch.zeros(2, 4), 2)
    with pytest.raises(RuntimeError, match="only on the GPU"):
        fm.route_tokens(torch.zeros(2, 4, requires_grad=True), 2)
    with pytest.raises(TypeError):
        fm.route_tokens([[1.0, 2.0]], 1)
    for bad in (dict(score="tanh"), dict(group_score="mean"), dict(groups=2, top_groups=3), dict(top_groups=0),
                dict(scale=float("inf")), dict(scale=float("nan"))):
        with pytest.raises(ValueError):
            fm.Routing(**bad)


def _route(x=DEV, stride=8, T=4, E=8, dt=_abi.F32, k=2, score=0, groups=1, top=1, gs=0, w=DEV, wd=_abi.F32, ids=DEV):
    return _abi.lib().fmoe_route(x, stride, T, E, dt, None, k, score, groups, top, gs, 1, 1.0, w, wd, ids, None,
                                 None, None, None)


def test_entry_point_refuses():
    assert _route(T=-1) == _abi.EINVAL
    assert _route(E=0) == _abi.EINVAL
    assert _route(k=0) == _abi.EINVAL
    assert _route(k=9) == _abi.EINVAL
    assert _route(dt=_abi.I64) == _abi.EINVAL
    assert _route(wd=_abi.I32) == _abi.EINVAL
    assert _route(score=2) == _abi.EINVAL
    assert _route(gs=2) == _abi.EINVAL
    assert _route(groups=3) == _abi.EINVAL
    assert _route(groups=4, top=5) == _abi.EINVAL
    assert _route(groups=4, top=0) == _abi.EINVAL
    assert _route(groups=4, top=1, k=3) == _abi.EINVAL
    assert _route(stride=-8) == _abi.EINVAL
    assert _route(x=None) == _abi.EINVAL
    assert _route(w=None) == _abi.EINVAL
    assert _route(ids=None) == _abi.EINVAL
    assert _route(E=4097) == _abi.ERANGE
    assert _route(E=100, k=65) == _abi.ERANGE
    assert _route(E=2048, groups=2) == _abi.ERANGE
    assert _route(E=1024, groups=128) == _abi.ERANGE
    assert _route(T=1 << 40) == _abi.ERANGE
    assert _route(T=0, x=None) == _abi.OK


def test_backward_entry_point_refuses():
    def call(g=DEV, gd=_abi.F32, ids=DEV, share=DEV, rest=None, norm=None, x=None, T=4, renorm=1, out=DEV):
        return _abi.lib().fmoe_route_backward(g, gd, ids, share, rest, norm, x, 8, T, 8, 2, _abi.F32, renorm, 1.0,
                                              out, None)

    assert call(g=None) == _abi.EINVAL
    assert call(ids=None) == _abi.EINVAL
    assert call(share=None) == _abi.EINVAL
    assert call(out=None) == _abi.EINVAL
    assert call(gd=_abi.I64) == _abi.EINVAL
    assert call(norm=DEV, renorm=0) == _abi.EINVAL             # reads the logits
    assert call(norm=DEV, x=DEV) == _abi.EINVAL                # renormalised
    assert call(norm=DEV, x=DEV, rest=DEV, renorm=0) == _abi.EINVAL
    assert call(T=1 << 40) == _abi.ERANGE
    assert call(T=0, g=None) == _abi.OK


@pytest.mark.parametrize("scale", [float("inf"), float("nan")])
def test_entry_point_refuses_a_scale_beyond_fp32(scale):
    call = _abi.lib().fmoe_route
    assert call(DEV, 8, 4, 8, _abi.F32, None, 2, 0, 1, 1, 0, 1, scale, DEV, _abi.F32, DEV, None, None, None,
                None) == _abi.EINVAL
