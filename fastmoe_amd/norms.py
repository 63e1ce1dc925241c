"""The norms around a block on gfx950 kernels: the one after it, its gate and residual scale, the addition to
the stream, and the norm before the next block, in one pass each way.

``quantize.add_rms_norm`` is the norm before a block alone.  The reference has no counterpart (its layer,
src/fastmoe/models/tiny_model.py:42-420, has no norm).  CPU tensors raise.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

from ._helper import call, check_matrix, need_gpu
from .ops import _refuse_autograd_capture
from .quantize import _not_taken, _refuse_transforms

__all__ = ["sandwich_norm"]


def sandwich_norm(x: torch.Tensor, post_weight: torch.Tensor, residual: torch.Tensor,
                  pre_weight: Optional[torch.Tensor] = None, *, gate: Optional[torch.Tensor] = None,
                  scale: float = 1.0, eps: float = 1e-6) -> Tuple[Optional[torch.Tensor], torch.Tensor]:
    """With ``rms(v) = v / sqrt(mean(v^2) + eps)``, of a block's output ``x`` and the stream ``residual``:

        h = residual + scale * gate * rms(x) * post_weight       the stream behind the block
        y = rms(h) * pre_weight                                  what the next block reads

    Returns ``(y, h)``, y None without ``pre_weight``.  ``x`` and ``residual`` [T, D] (unit column
    stride); the weights [D], both in x's type or both float32; ``gate`` [D], or [G, D] with a row for each
    of G equal runs of neighbouring rows (a sequence's, where T = G * its tokens), in x's type or float32; one that is
    not contiguous, as a slice or a broadcast one, is copied first.
    h is rounded to x's type and y computed from it in float32 and rounded once.  Differentiable in all five;
    sums over rows run in a fixed order.  A row of x whose sum of squares passes float32's range adds nothing.
    """
    _refuse_transforms("sandwich_norm")
    given = (x, post_weight, residual, pre_weight, gate)
    records = torch.is_grad_enabled() and any(getattr(t, "requires_grad", False) for t in given)
    if records:
        _refuse_autograd_capture("the autograd norms", next(t for t in given if getattr(t, "requires_grad", False)))
    out = call("sandwich", *given, scale, eps, records)
    if out is NotImplemented:
        _check_sandwich(*given, scale, eps)
        if gate is not None and not gate.is_contiguous():
            return sandwich_norm(x, post_weight, residual, pre_weight, gate=gate.contiguous(), scale=scale, eps=eps)
        _not_taken("sandwich_norm")
    return out


def _check_sandwich(x, post_weight, residual, pre_weight, gate, scale, eps) -> None:
    check_matrix(x, "x")
    check_matrix(residual, "residual")
    if residual.shape != x.shape or residual.dtype != x.dtype:
        raise ValueError(f"fastmoe_amd: residual must be {x.dtype} {tuple(x.shape)}, got {residual.dtype} "
                         f"{tuple(residual.shape)}")
    T, D = x.shape
    for name, t in (("post_weight", post_weight), ("pre_weight", pre_weight), ("gate", gate)):
        if t is None and name != "post_weight":
            continue
        need_gpu(t, name)
        if t.dim() not in ((1, 2) if name == "gate" else (1,)) or t.shape[-1] != D or \
                (name != "gate" and not t.is_contiguous()):
            raise ValueError(f"fastmoe_amd: {name} must be {'' if name == 'gate' else 'contiguous '}[{D}], got "
                             f"{tuple(t.shape)}")
        if t.dtype not in (x.dtype, torch.float32):
            raise TypeError(f"fastmoe_amd: {name} must be {x.dtype} or float32, got {t.dtype}")
        if t.device != x.device:
            raise ValueError(f"fastmoe_amd: {name} is on {t.device}, not on {x.device}")
    if residual.device != x.device:
        raise ValueError(f"fastmoe_amd: residual is on {residual.device}, not on {x.device}")
    if pre_weight is not None and pre_weight.dtype != post_weight.dtype:
        raise TypeError(f"fastmoe_amd: the weights must share a dtype, got {post_weight.dtype} and "
                        f"{pre_weight.dtype}")
    if gate is not None and gate.dim() == 2 and (T % gate.shape[0] if gate.shape[0] else T):
        raise ValueError(f"fastmoe_amd: {gate.shape[0]} rows of the gate do not share out {T} rows")
    if not math.isfinite(scale):
        raise ValueError(f"fastmoe_amd: the scale must be finite, got {scale}")
    if not 0.0 <= float(eps) < float("inf"):
        raise ValueError(f"fastmoe_amd: eps must be finite and not negative, got {eps}")
