"""Routing of tokens to experts on a gfx950 kernel: scores, a bias for balance, groups, top-k and weights.

The reference routes by ``torch.topk`` of the logits and a softmax of the chosen
(src/fastmoe/models/tiny_model.py:92-100), which ``moe.gate_and_sort`` does without a ``routing``;
:class:`Routing` has no counterpart there.  CPU tensors raise.
"""
from __future__ import annotations

import dataclasses
import math
from typing import NamedTuple, Optional

import torch

from . import _abi
from ._helper import call, check_matrix, need_gpu
from .ops import _FLOAT_CODES, _refuse_autograd_capture
from .quantize import _no_gradient, _not_taken, _refuse_transforms

__all__ = ["RoutedTokens", "Routing", "route_tokens"]

_SCORES = {"softmax": _abi.SCORE_SOFTMAX, "sigmoid": _abi.SCORE_SIGMOID}
_GROUP_SCORES = {"max": _abi.GROUP_MAX, "top2": _abi.GROUP_TOP2}


@dataclasses.dataclass(frozen=True)
class Routing:
    """How :func:`route_tokens` chooses experts and weighs them.

    ``score``: "softmax" (over all experts) or "sigmoid" of the logits.  ``groups``: neighbouring experts
    in this many groups of equal size, of which the ``top_groups`` best are kept, ranked by their highest
    choice (``group_score="max"``) or the sum of their two highest ("top2").  ``renormalize``: the chosen
    scores divided by their sum.  ``scale``: what the weights are multiplied by.
    """

    score: str = "softmax"
    groups: int = 1
    top_groups: int = 1
    group_score: str = "max"
    renormalize: bool = True
    scale: float = 1.0

    def __post_init__(self) -> None:
        if self.score not in _SCORES:
            raise ValueError(f"fastmoe_amd: unknown score {self.score!r} (expected 'softmax' or 'sigmoid')")
        if self.group_score not in _GROUP_SCORES:
            raise ValueError(f"fastmoe_amd: unknown group score {self.group_score!r} (expected 'max' or "
                             "'top2')")
        if not 1 <= self.top_groups <= self.groups:
            raise ValueError(f"fastmoe_amd: {self.top_groups} of {self.groups} groups")
        if not math.isfinite(self.scale):
            raise ValueError(f"fastmoe_amd: the scale must be finite, got {self.scale}")


class RoutedTokens(NamedTuple):
    """What :func:`route_tokens` returns, as ``permute_tokens`` takes it."""

    topk_weights: torch.Tensor  # [T, k]
    topk_indices: torch.Tensor  # int64 [T, k], highest choice first


_DEFAULT = Routing()


def route_tokens(logits: torch.Tensor, top_k: int, routing: Routing = _DEFAULT, *,
                 bias: Optional[torch.Tensor] = None,
                 out_dtype: Optional[torch.dtype] = None) -> RoutedTokens:
    """The ``top_k`` experts of each row of ``logits`` [T, E] (unit column stride), and their weights in
    ``out_dtype`` (None: the logits' type).

    With s the scores, experts are chosen by ``s + bias`` (``bias`` float32 [E]; s is computed to 2^-36 and rounded to
    float32, then the bias is added), or, without a bias and without groups ranked by a sum, by the logits, which
    rank alike.  Equal choices go to the lowest index.  The weights are of s alone, computed in 64 bits and
    rounded once; where the logits choose, the sum under a softmax over all experts is float32 (the weights then hold
    to 2^-17, and measured to 2^-20).  Differentiable in the logits; the bias only chooses, and one that
    requires a gradient is refused.

    A logit of -inf masks its expert: score and weight 0.  Where the logits choose, it is chosen only if nothing else is
    left; where ``s + bias`` does, its choice is its bias alone, and one above others' choices takes a place with weight
    0.  A bias of -inf leaves an expert out of every row.  Where nothing is left the ids are still different experts,
    with weights of 0.  A NaN ranks highest and makes the weights that depend on it NaN.  At most 64 of 4096
    experts; with groups at most 1024 experts in 64 groups.
    """
    _refuse_transforms("route_tokens")
    w_code = _FLOAT_CODES.get(out_dtype if out_dtype is not None else getattr(logits, "dtype", None), -1)
    args = (logits, bias, top_k, _SCORES[routing.score], routing.groups, routing.top_groups,
            _GROUP_SCORES[routing.group_score], bool(routing.renormalize), routing.scale, w_code)
    out = NotImplemented
    if w_code >= 0:
        records = torch.is_grad_enabled() and logits.requires_grad
        if records:
            _refuse_autograd_capture("the autograd router", logits)
        out = call("route", *args, records)
    if out is NotImplemented:
        _check_route(logits, top_k, routing, bias, out_dtype)
        _not_taken("route_tokens")
    return RoutedTokens(*out)


def _check_route(logits, top_k, routing, bias, out_dtype) -> None:
    check_matrix(logits, "logits")
    if out_dtype is not None and out_dtype not in _FLOAT_CODES:
        raise TypeError(f"fastmoe_amd: unsupported out_dtype {out_dtype}")
    E = logits.shape[1]
    if not 1 <= top_k <= E:
        raise ValueError(f"fastmoe_amd: top_k={top_k} of {E} experts")
    if bias is not None:
        need_gpu(bias, "bias")
        if bias.dtype != torch.float32 or tuple(bias.shape) != (E,) or not bias.is_contiguous():
            raise ValueError(f"fastmoe_amd: bias must be contiguous float32 [{E}], got {bias.dtype} "
                             f"{tuple(bias.shape)}")
        if bias.device != logits.device:
            raise ValueError(f"fastmoe_amd: bias is on {bias.device}, not on {logits.device}")
        _no_gradient("the router's bias", bias)
