"""Experts' weights in 4 bits with a scale for 32 of them, on gfx950 kernels, and every expert's product of 16-bit
rows with them (``moe.Fp4MoEFeedForward`` serves with these).

A weight is ``v * 2**(s - 127)``: v one of 0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives, a 4-bit code of sign, two bits of
exponent and one of mantissa, and s a byte for 32 neighbouring weights of an output (255: NaN).  The rows stay as
they are.

The reference has no counterpart (its experts, src/fastmoe/models/tiny_model.py:66-77, keep their weights in
the activations' type).  CPU tensors raise.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Sequence, Union

import torch

from ._helper import call, check_matrix, need_gpu
from .ops import _FLOAT_CODES, _INDEX_CODES, _validate_default
from .quantize import (_ACTIVATIONS, _float_code, _no_gradient, _not_taken, _same_device)

__all__ = ["Fp4Weights", "fp4_linear", "quantize_weights_fp4"]

PITCH = 128  # an output's weights are padded with zeros to a multiple of this many
BLOCK = 32   # weights that share a scale


def _pad(n: int) -> int:
    return -(-n // PITCH) * PITCH


class Fp4Weights(NamedTuple):
    """Weights in 4 bits: expert e's weight of output n and column c has its code in ``data[e, n, c // 2]`` (the
    low half for an even c) and its scale in ``scales[e, n, c // 32]``.  Two-dimensional weights are those of one
    expert."""

    data: torch.Tensor    # uint8 [E, N, features rounded up to 128, / 2], codes of zero from ``features`` on
    scales: torch.Tensor  # uint8 [E, N, features rounded up to 128, / 32], not 255 from ``features`` on
    features: int

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The weights in ``dtype``, [E, N, features]."""
        out = call("restore_fp4", self.data, self.scales, self.features, _float_code(dtype))
        if out is NotImplemented:
            _check_weights(self)
            _not_taken("dequantize")
        return out


def quantize_weights_fp4(weight: Union[torch.Tensor, Sequence[torch.Tensor]]) -> Fp4Weights:
    """Weights in 4 bits: from [E, N, K], from [N, K] (one expert), or from a list of E tensors [N, K]
    (``nn.Linear.weight``, whose gradients stay out of it).  Each 32 get the smallest power of two with which
    none of them passes 6 as their scale, and are rounded to the nearest (ties to even); an infinity or a NaN
    among them makes all 32 NaN."""
    parts = [weight] if isinstance(weight, torch.Tensor) and weight.dim() != 3 else list(weight)
    if not parts:
        raise ValueError("fastmoe_amd: no weights")
    need_gpu(parts[0], "weight 0")
    N, K = parts[0].shape if parts[0].dim() == 2 else (0, 0)
    for i, p in enumerate(parts):
        check_matrix(p, f"weight {i}")
        if tuple(p.shape) != (N, K) or N < 1:
            raise ValueError(f"fastmoe_amd: weight {i} must be [{N}, {K}], got {tuple(p.shape)}")
        _same_device(parts[0], **{f"weight {i}": p})
    dev = parts[0].device
    data = torch.empty((len(parts), N, _pad(K) // 2), dtype=torch.uint8, device=dev)
    scales = torch.empty((len(parts), N, _pad(K) // BLOCK), dtype=torch.uint8, device=dev)
    with torch.no_grad():
        for e, p in enumerate(parts):
            out = call("quantize_fp4", p.detach())
            if out is NotImplemented:
                _not_taken("quantize_weights_fp4")
            data[e], scales[e] = out
    return Fp4Weights(data, scales, K)


def fp4_linear(x: torch.Tensor, weights: Fp4Weights, expert_offsets: Optional[torch.Tensor] = None, *,
               rows: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               activation: Optional[str] = None, out_dtype: Optional[torch.dtype] = None,
               validate: Optional[bool] = None) -> torch.Tensor:
    """Every expert's product on its own rows: out [R, N] in ``out_dtype`` (None: x's type) with

        out[r] = act(x[i] @ W[e].T + bias[e])

    for r in [expert_offsets[e], expert_offsets[e + 1]), i = ``rows[r]`` (the reverse map of
    ``permute_tokens``), or i = r without ``rows``.  ``x`` [T, K], bfloat16 or float16 (unit column stride);
    W the weights in x's type (bfloat16 holds every one that float32 does, float16 those whose scale lies
    between 2^-23 and 2^13).  ``expert_offsets`` int64 [E + 1] on the device (``PermutedTokens.expert_offsets``), starting at 0
    and not falling; None for one expert's weights.  ``bias`` [E, N] (or [N]).  ``activation``: None or "gelu" (the
    exact form, as ``torch.nn.GELU()``).  Sums are float32; the result is rounded once.

    Nothing is read back by the host, so the call can be captured in a HIP graph.  Rows at or beyond
    ``expert_offsets[E]`` are zero, and so is the product of a row whose ``rows`` entry lies outside
    x; ``validate=True`` (or ``FASTMOE_VALIDATE=1``) raises IndexError for such entries and for
    offsets that fall or end outside the rows (one synchronisation).  It has no gradient.
    """
    if activation not in _ACTIVATIONS:
        raise ValueError(f"fastmoe_amd: unknown activation {activation!r} (expected None or 'gelu')")
    if _validate_default(validate):
        _check_linear(x, weights, expert_offsets, rows, bias, out_dtype)
        _validate_rows(x.shape[0], expert_offsets, rows, x.device)
    code = _FLOAT_CODES.get(out_dtype if out_dtype is not None else getattr(x, "dtype", None))
    args = (x, weights.data, weights.scales, weights.features)
    act = _ACTIVATIONS[activation]
    out = NotImplemented
    if code is not None:
        out = call("fp4_linear", *args, expert_offsets, rows, bias, act, code)
    if out is NotImplemented:
        _check_linear(x, weights, expert_offsets, rows, bias, out_dtype)
        # what is left: indices, offsets or a bias with gaps between their elements
        expert_offsets, rows, bias = (t if t is None else t.contiguous() for t in (expert_offsets, rows, bias))
        out = call("fp4_linear", *args, expert_offsets, rows, bias, act, code)
        if out is NotImplemented:
            _not_taken("fp4_linear")
    return out


def _check_weights(w: Fp4Weights) -> None:
    need_gpu(w.data, "weights' data")
    need_gpu(w.scales, "weights' scales")
    if w.data.dtype != torch.uint8 or w.scales.dtype != torch.uint8 or w.data.dim() not in (2, 3):
        raise TypeError(f"fastmoe_amd: weights' data and scales must be uint8 with 2 or 3 dimensions, got "
                        f"{w.data.dtype} {tuple(w.data.shape)} and {w.scales.dtype} {tuple(w.scales.shape)}")
    features = int(w.features)
    want = _pad(max(features, 1))
    if features < 1 or w.data.shape[-1] != want // 2 or \
            tuple(w.scales.shape) != (*w.data.shape[:-1], want // BLOCK):
        raise ValueError(f"fastmoe_amd: {features} features are stored in {want // 2} bytes of codes and "
                         f"{want // BLOCK} scales, got {tuple(w.data.shape)} and {tuple(w.scales.shape)}")
    if not w.data.is_contiguous() or not w.scales.is_contiguous() or \
            (w.data.numel() and (w.data.data_ptr() % 16 or w.scales.data_ptr() % 4)):
        raise ValueError("fastmoe_amd: weights' data and scales must be contiguous and start at multiples of "
                         "16 and 4 bytes")
    _same_device(w.data, **{"weights' scales": w.scales})


def _check_linear(x, weights, expert_offsets, rows, bias, out_dtype) -> None:
    """Says what is wrong with fp4_linear's arguments, if anything is."""
    check_matrix(x, "x")
    if x.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"fastmoe_amd: x must be bfloat16 or float16, got {x.dtype}")
    _check_weights(weights)
    E = weights.data.shape[0] if weights.data.dim() == 3 else 1
    N = weights.data.shape[-2]
    if weights.features != x.shape[1]:
        raise ValueError(f"fastmoe_amd: x has {x.shape[1]} features, the weights {weights.features}")
    if E < 1 or N < 1:
        raise ValueError("fastmoe_amd: no weights")
    _float_code(x.dtype if out_dtype is None else out_dtype, "out_dtype")
    if expert_offsets is None:
        if E != 1:
            raise ValueError(f"fastmoe_amd: {E} experts need expert_offsets")
    else:
        need_gpu(expert_offsets, "expert_offsets")
        if expert_offsets.dtype != torch.int64 or tuple(expert_offsets.shape) != (E + 1,):
            raise ValueError(f"fastmoe_amd: expert_offsets must be int64 [{E + 1}], got "
                             f"{expert_offsets.dtype} {tuple(expert_offsets.shape)}")
    if rows is not None:
        need_gpu(rows, "rows")
        if rows.dtype not in _INDEX_CODES or rows.dim() != 1:
            raise TypeError(f"fastmoe_amd: rows must be int64 or int32 with one dimension, got "
                            f"{rows.dtype} {tuple(rows.shape)}")
        if rows.shape[0] and not x.shape[0]:
            raise ValueError("fastmoe_amd: rows is not empty, and x is")
    if bias is not None:
        need_gpu(bias, "bias")
        if bias.dtype not in _FLOAT_CODES:
            raise TypeError(f"fastmoe_amd: unsupported bias dtype {bias.dtype}")
        if tuple(bias.shape) != (E, N) and not (E == 1 and tuple(bias.shape) == (N,)):
            raise ValueError(f"fastmoe_amd: bias must be [{E}, {N}], got {tuple(bias.shape)}")
    _no_gradient("fp4_linear", x, bias)
    _same_device(x, weights=weights.data, expert_offsets=expert_offsets, rows=rows, bias=bias)


def _validate_rows(x_rows: int, offsets, rows, device) -> None:
    R = x_rows if rows is None else rows.shape[0]
    bad = torch.zeros((), dtype=torch.int64, device=device)
    if rows is not None and R:
        bad = bad + ((rows < 0) | (rows >= x_rows)).sum()
    if offsets is not None:
        bad = bad + (offsets[0] != 0) + (offsets[1:] < offsets[:-1]).sum() + (offsets[-1] > R)
    if int(bad):
        raise IndexError(f"fastmoe_amd: {int(bad)} entries of rows or expert_offsets lie outside "
                         f"x's {x_rows} rows, or the {R} packed rows, or fall")
