"""The MoE layer's rows in 8 bits on gfx950 kernels: the norm at its entry, rows and weights as whole
numbers with scales, the experts' product of them, and activations held in 8 bits for the backward.

Serving (``moe.Int8MoEFeedForward`` runs them in this order):

    add_rms_norm_int8   h = x + residual; y = rms_norm(h) * weight, in its own type (the router reads
                        it) and in 8 bits (the experts read it)
    quantize_rows       any rows to 8 bits, optionally after GELU (between the experts' products)
    int8_linear         every expert's product on its own rows, which it reads through the
                        dispatch's reverse map: the tokens' rows are never copied for their experts

Training:

    add_rms_norm        the same norm with its gradients
    gelu_compress, gelu_compressed_backward
                        GELU whose input is held in 8 bits until the backward, which makes GELU's
                        output again from it (``moe.compute_experts(..., checkpoint="int8")``)
    compress_rows, restore_rows
                        any activation held in 8 bits

A value v is held as ``q = round(v * (127 / m))`` with the scale ``m / 127``, m the largest |v| of its row
(rows for products) or of its 128 columns of a row (held activations).  Values below 2^-118 only:
scale 0.  An infinity or a NaN among them: scale NaN, so that what is computed from them is NaN.

The reference has no counterpart (its layer, src/fastmoe/models/tiny_model.py:42-420, keeps every
row in the activations' type).  CPU tensors raise.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Sequence, Tuple, Union

import torch

from . import _abi
from .ops import (_FLOAT_CODES, _INDEX_CODES, _on_device, _refuse_autograd_capture, _runs_plain,
                  _span, _stream_handle, _validate_default)

__all__ = [
    "CompressedRows",
    "Int8NormedRows",
    "Int8Weights",
    "QuantizedRows",
    "add_rms_norm",
    "add_rms_norm_int8",
    "compress_rows",
    "gelu_compress",
    "gelu_compressed_backward",
    "int8_linear",
    "quantize_rows",
    "quantize_weights",
    "restore_rows",
]

PITCH = 128  # a row of whole numbers is padded with zeros to a multiple of this many
BLOCK = 128  # columns of a held activation that share a scale

_ACTIVATIONS = {None: _abi.ACT_NONE, "gelu": _abi.ACT_GELU}


def _pad(n: int) -> int:
    return -(-n // PITCH) * PITCH


def _need_gpu(t, what: str) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"fastmoe_amd: {what} must be a tensor, got {type(t).__name__}")
    if not t.is_cuda:
        raise RuntimeError(f"fastmoe_amd: {what} is on {t.device}; the 8-bit operators run only on "
                           "the GPU")


def _check_matrix(t, what: str) -> None:
    """``t`` is a 2-D float matrix on the GPU whose rows have unit stride."""
    _need_gpu(t, what)
    if t.dim() != 2:
        raise ValueError(f"fastmoe_amd: {what} must be [rows, columns], got {tuple(t.shape)}")
    if t.dtype not in _FLOAT_CODES:
        raise TypeError(f"fastmoe_amd: unsupported {what} dtype {t.dtype}")
    if t.shape[1] < 1:
        raise ValueError(f"fastmoe_amd: {what} has no columns")
    if t.shape[1] > 1 and t.stride(1) != 1 and t.shape[0] > 0:
        raise ValueError(f"fastmoe_amd: {what} must have unit column stride")


def _row_stride(t: torch.Tensor) -> int:
    """Elements from row to row (a single row's stride is free to be anything)."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _same_device(first: torch.Tensor, **others) -> None:
    for name, t in others.items():
        if t is not None and t.device != first.device:
            raise ValueError(f"fastmoe_amd: {name} is on {t.device}, not on {first.device}")


def _check_int8(data, scales, features, what: str, dims: int) -> None:
    _need_gpu(data, f"{what} data")
    _need_gpu(scales, f"{what} scales")
    _same_device(data, **{f"{what} scales": scales})
    if data.dtype != torch.int8 or data.dim() != dims:
        raise TypeError(f"fastmoe_amd: {what} data must be int8 with {dims} dimensions, got "
                        f"{data.dtype} {tuple(data.shape)}")
    if scales.dtype != torch.float32:
        raise TypeError(f"fastmoe_amd: {what} scales must be float32, got {scales.dtype}")
    features = int(features)
    if features < 1 or data.shape[-1] != _pad(features):
        raise ValueError(f"fastmoe_amd: {what} data has {data.shape[-1]} columns; {features} "
                         f"features are stored in {_pad(max(features, 1))} (padded with zeros)")
    if data.numel() and (data.stride(-1) != 1 or data.data_ptr() % 16):
        raise ValueError(f"fastmoe_amd: {what} data must have unit column stride and start at a "
                         "multiple of 16 bytes")


class QuantizedRows(NamedTuple):
    """Rows in 8 bits with one scale each: row r stands for ``data[r, :features] * scales[r]``."""

    data: torch.Tensor    # int8 [R, features rounded up to 128], zeros from ``features`` on
    scales: torch.Tensor  # float32 [R]
    features: int

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The values that the rows stand for, [R, features]."""
        _check_rows8(self, "rows")
        return _restore(self.data, self.scales, 1, self.features, dtype)


class Int8Weights(NamedTuple):
    """Weights in 8 bits with one scale for each output: expert e's weight of output n is
    ``data[e, n, :features] * scales[e, n]``.  Two-dimensional weights are those of one expert."""

    data: torch.Tensor    # int8 [E, N, features rounded up to 128], zeros from ``features`` on
    scales: torch.Tensor  # float32 [E, N]
    features: int


class CompressedRows(NamedTuple):
    """Held rows: ``data[r, c] * scales[r, c // 128]`` for c below ``features``."""

    data: torch.Tensor    # int8 [R, features rounded up to 128]
    scales: torch.Tensor  # float32 [R, ceil(features / 128)]
    features: int


class Int8NormedRows(NamedTuple):
    """What :func:`add_rms_norm_int8` returns."""

    rows: QuantizedRows                # the norm in 8 bits
    normed: Optional[torch.Tensor]     # the norm in its own type, if kept
    residual: torch.Tensor             # the stream: x + residual


def _check_rows8(x: QuantizedRows, what: str) -> None:
    _check_int8(x.data, x.scales, x.features, what, 2)
    if x.scales.shape != x.data.shape[:1] or not x.scales.is_contiguous():
        raise ValueError(f"fastmoe_amd: {what} scales must be contiguous [{x.data.shape[0]}], got "
                         f"{tuple(x.scales.shape)}")
    if x.data.shape[0] > 1 and (x.data.stride(0) < x.data.shape[1] or x.data.stride(0) % 16):
        raise ValueError(f"fastmoe_amd: {what} data's row stride must be a multiple of 16 and at "
                         "least its columns")


def _new_rows8(rows: int, cols: int, dev) -> QuantizedRows:
    return QuantizedRows(torch.empty((rows, _pad(cols)), dtype=torch.int8, device=dev),
                         torch.empty(rows, dtype=torch.float32, device=dev), cols)


# ---- the norm ---------------------------------------------------------------------------------

def _check_norm(x, weight, residual, eps) -> None:
    _check_matrix(x, "x")
    _need_gpu(weight, "weight")
    if weight.dim() != 1 or weight.shape[0] != x.shape[1] or not weight.is_contiguous():
        raise ValueError(f"fastmoe_amd: weight must be contiguous [{x.shape[1]}], got "
                         f"{tuple(weight.shape)}")
    if weight.dtype not in (x.dtype, torch.float32):
        raise TypeError(f"fastmoe_amd: weight must be {x.dtype} or float32, got {weight.dtype}")
    if residual is not None:
        _check_matrix(residual, "residual")
        if residual.shape != x.shape or residual.dtype != x.dtype:
            raise ValueError(f"fastmoe_amd: residual must be {x.dtype} {tuple(x.shape)}, got "
                             f"{residual.dtype} {tuple(residual.shape)}")
    _same_device(x, weight=weight, residual=residual)
    if not 0.0 <= float(eps) < float("inf"):
        raise ValueError(f"fastmoe_amd: eps must be finite and not negative, got {eps}")


def _norm(x, weight, residual, eps, *, y: bool, rstd: bool, rows8: bool):
    """(stream, y, rstd, 8-bit rows) of checked arguments; None where not asked for."""
    T, D = x.shape
    dev = x.device
    h = x if residual is None else torch.empty((T, D), dtype=x.dtype, device=dev)
    out = torch.empty((T, D), dtype=x.dtype, device=dev) if y else None
    factor = torch.empty(T, dtype=torch.float32, device=dev) if rstd else None
    q = _new_rows8(T, D, dev) if rows8 else None
    if T:
        with _on_device(dev), _span("add_rms_norm"):
            rc = _abi.lib().fmoe_add_rms_norm(
                x.data_ptr(), _row_stride(x),
                residual.data_ptr() if residual is not None else None,
                _row_stride(residual) if residual is not None else 0,
                weight.data_ptr(), _FLOAT_CODES[weight.dtype], T, D, _FLOAT_CODES[x.dtype],
                float(eps), h.data_ptr() if residual is not None else None,
                out.data_ptr() if y else None, factor.data_ptr() if rstd else None,
                q.data.data_ptr() if rows8 else None, q.data.shape[1] if rows8 else 0,
                q.scales.data_ptr() if rows8 else None, _stream_handle(dev))
        _abi.check(rc, "fmoe_add_rms_norm")
    return h, out, factor, q


class _AddRmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        h, y, rstd, _ = _norm(x, weight, residual, eps, y=True, rstd=True, rows8=False)
        ctx.save_for_backward(h, weight, rstd)
        ctx.has_residual = residual is not None
        ctx.set_materialize_grads(False)
        return (y, h) if residual is not None else y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gy, gh=None):
        h, weight, rstd = ctx.saved_tensors
        _refuse_autograd_capture("the norm's backward", h)
        need_x, need_w, need_r = ctx.needs_input_grad[:3]
        gw = None
        if gy is None:  # only the stream was used
            gw = torch.zeros_like(weight) if need_w else None
            return gh if need_x else None, gw, gh if need_r else None, None
        T, D = h.shape
        gy = gy if D == 1 or gy.stride(1) == 1 else gy.contiguous()
        if gh is not None and D > 1 and gh.stride(1) != 1:
            gh = gh.contiguous()
        lib = _abi.lib()
        gx = torch.empty((T, D), dtype=h.dtype, device=h.device)
        nbytes, ws = 0, None
        if need_w:
            gw = torch.empty_like(weight)
            nbytes = lib.fmoe_add_rms_norm_backward_workspace_bytes(T, D)
            ws = torch.empty(nbytes, dtype=torch.uint8, device=h.device)
        with _on_device(h.device), _span("add_rms_norm_backward"):
            rc = lib.fmoe_add_rms_norm_backward(
                gy.data_ptr(), _row_stride(gy), gh.data_ptr() if gh is not None else None,
                _row_stride(gh) if gh is not None else 0, h.data_ptr(), _row_stride(h),
                weight.data_ptr(), _FLOAT_CODES[weight.dtype], rstd.data_ptr(), T, D,
                _FLOAT_CODES[h.dtype], gx.data_ptr(), gw.data_ptr() if need_w else None,
                ws.data_ptr() if need_w else None, nbytes, _stream_handle(h.device))
        _abi.check(rc, "fmoe_add_rms_norm_backward")
        return gx if need_x else None, gw, gx if need_r else None, None


def add_rms_norm(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None, *,
                 eps: float = 1e-6) -> Tuple[torch.Tensor, torch.Tensor]:
    """``h = x + residual`` and ``y = h * weight / sqrt(mean(h^2) + eps)``; returns ``(y, h)``.

    ``x`` and ``residual`` [T, D] (unit column stride), ``weight`` [D] in x's type or float32.  h is
    rounded to x's type, as the tensors' sum is, and y is computed from it in float32 and rounded
    once.  Without a residual, h is ``x`` itself.  Differentiable in all three; the gradient of the
    weight sums the rows in a fixed order.
    """
    _check_norm(x, weight, residual, eps)
    inputs = [t for t in (x, weight, residual) if t is not None]
    if _runs_plain(inputs):
        h, y, _, _ = _norm(x, weight, residual, eps, y=True, rstd=False, rows8=False)
        return y, h
    records = torch.is_grad_enabled() and any(t.requires_grad for t in inputs)
    _refuse_autograd_capture("the autograd norm", x, records)
    out = _AddRmsNorm.apply(x, weight, residual, float(eps))
    return out if residual is not None else (out, x)


def _no_gradient(what: str, *tensors) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError(f"fastmoe_amd: {what} has no gradient; call it under torch.no_grad() or "
                           "on detached tensors")


def add_rms_norm_int8(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None,
                      *, eps: float = 1e-6, keep_normed: bool = True) -> Int8NormedRows:
    """:func:`add_rms_norm` whose y also comes in 8 bits, one scale a row, from the unrounded y.

    Without ``keep_normed`` only the 8-bit rows are written.  For serving: it records no backward,
    and refuses inputs that require one.
    """
    _check_norm(x, weight, residual, eps)
    _no_gradient("add_rms_norm_int8", x, weight, residual)
    h, y, _, q = _norm(x, weight, residual, eps, y=bool(keep_normed), rstd=False, rows8=True)
    return Int8NormedRows(q, y, h)


# ---- rows and weights in 8 bits ---------------------------------------------------------------

def quantize_rows(x: torch.Tensor, *, activation: Optional[str] = None) -> QuantizedRows:
    """Rows [R, C] (unit column stride) in 8 bits with one scale each, after ``activation``: None or
    "gelu" (the exact form, as ``torch.nn.GELU()``).  Records no backward, and refuses inputs that
    require one."""
    _check_matrix(x, "x")
    if activation not in _ACTIVATIONS:
        raise ValueError(f"fastmoe_amd: unknown activation {activation!r} (expected None or 'gelu')")
    _no_gradient("quantize_rows", x)
    R, C = x.shape
    q = _new_rows8(R, C, x.device)
    if R:
        with _on_device(x.device), _span("quantize_rows"):
            rc = _abi.lib().fmoe_quantize_rows(
                x.data_ptr(), _row_stride(x), R, C, _FLOAT_CODES[x.dtype], _ACTIVATIONS[activation],
                q.data.data_ptr(), q.data.shape[1], q.scales.data_ptr(), _stream_handle(x.device))
        _abi.check(rc, "fmoe_quantize_rows")
    return q


def quantize_weights(weight: Union[torch.Tensor, Sequence[torch.Tensor]]) -> Int8Weights:
    """Weights in 8 bits with one scale for each output: from [E, N, K], from [N, K] (one expert), or
    from a list of E tensors [N, K] (``nn.Linear.weight``, whose gradients stay out of it)."""
    parts = [weight] if isinstance(weight, torch.Tensor) else list(weight)
    if not parts:
        raise ValueError("fastmoe_amd: no weights")
    if isinstance(weight, torch.Tensor) and weight.dim() == 3:
        parts = list(weight)
        if not parts:
            raise ValueError("fastmoe_amd: no weights")
    N, K = parts[0].shape if parts[0].dim() == 2 else (0, 0)
    for i, p in enumerate(parts):
        _check_matrix(p, f"weight {i}")
        if tuple(p.shape) != (N, K) or p.shape[0] < 1:
            raise ValueError(f"fastmoe_amd: weight {i} must be [{N}, {K}], got {tuple(p.shape)}")
        _same_device(parts[0], **{f"weight {i}": p})
    data = torch.empty((len(parts), N, _pad(K)), dtype=torch.int8, device=parts[0].device)
    scales = torch.empty((len(parts), N), dtype=torch.float32, device=parts[0].device)
    with torch.no_grad():
        for e, p in enumerate(parts):
            q = quantize_rows(p.detach())
            data[e], scales[e] = q.data, q.scales
    return Int8Weights(data, scales, K)


def int8_linear(x: QuantizedRows, weights: Int8Weights,
                expert_offsets: Optional[torch.Tensor] = None, *,
                rows: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
                out_dtype: torch.dtype = torch.bfloat16,
                validate: Optional[bool] = None) -> torch.Tensor:
    """Every expert's product on its own rows: out [R, N] with

        out[r] = (x.data[i] @ weights.data[e].T) * x.scales[i] * weights.scales[e] + bias[e]

    for r in [expert_offsets[e], expert_offsets[e + 1]), i = ``rows[r]`` (the reverse map of
    ``permute_tokens``), or i = r without ``rows``.  ``expert_offsets`` int64 [E + 1] on the device
    (``PermutedTokens.expert_offsets``), starting at 0 and not falling; None for one expert's weights.
    ``bias`` [E, N] (or [N]).  The sums are exact; the result is rounded once, to ``out_dtype``.

    Nothing is read back by the host, so the call can be captured in a HIP graph.  Rows at or beyond
    ``expert_offsets[E]`` are zero, and so is the product of a row whose ``rows`` entry lies outside
    x; ``validate=True`` (or ``FASTMOE_VALIDATE=1``) raises IndexError for such entries and for
    offsets that fall or end outside the rows (one synchronisation).  It has no gradient.
    """
    _check_rows8(x, "x")
    data, scales = weights.data, weights.scales
    if data.dim() == 2:
        data, scales = data.unsqueeze(0), scales.unsqueeze(0)
    _check_int8(data, scales, weights.features, "weights", 3)
    E, N, Kp = data.shape
    if weights.features != x.features:
        raise ValueError(f"fastmoe_amd: x has {x.features} features, the weights {weights.features}")
    if E < 1 or N < 1 or tuple(scales.shape) != (E, N):
        raise ValueError(f"fastmoe_amd: weight scales must be [{E}, {N}], got {tuple(scales.shape)}")
    if not data.is_contiguous() or not scales.is_contiguous():
        raise ValueError("fastmoe_amd: weights and their scales must be contiguous")
    if out_dtype not in _FLOAT_CODES:
        raise TypeError(f"fastmoe_amd: unsupported out_dtype {out_dtype}")
    if expert_offsets is None:
        if E != 1:
            raise ValueError(f"fastmoe_amd: {E} experts need expert_offsets")
    else:
        _need_gpu(expert_offsets, "expert_offsets")
        if expert_offsets.dtype != torch.int64 or tuple(expert_offsets.shape) != (E + 1,):
            raise ValueError(f"fastmoe_amd: expert_offsets must be int64 [{E + 1}], got "
                             f"{expert_offsets.dtype} {tuple(expert_offsets.shape)}")
        expert_offsets = expert_offsets.contiguous()
    R = x.data.shape[0]
    if rows is not None:
        _need_gpu(rows, "rows")
        if rows.dtype not in _INDEX_CODES or rows.dim() != 1:
            raise TypeError(f"fastmoe_amd: rows must be int64 or int32 with one dimension, got "
                            f"{rows.dtype} {tuple(rows.shape)}")
        rows = rows.contiguous()
        R = rows.shape[0]
    if bias is not None:
        _need_gpu(bias, "bias")
        if bias.dtype not in _FLOAT_CODES:
            raise TypeError(f"fastmoe_amd: unsupported bias dtype {bias.dtype}")
        if tuple(bias.shape) != (E, N) and not (E == 1 and tuple(bias.shape) == (N,)):
            raise ValueError(f"fastmoe_amd: bias must be [{E}, {N}], got {tuple(bias.shape)}")
        _no_gradient("int8_linear", bias)
        bias = bias.contiguous()
    _same_device(x.data, weights=data, expert_offsets=expert_offsets, rows=rows, bias=bias)
    if R and not x.data.shape[0]:
        raise ValueError("fastmoe_amd: rows is not empty, and x is")
    dev = x.data.device
    if _validate_default(validate):
        _validate_linear(x, expert_offsets, rows, R)
    out = torch.empty((R, N), dtype=out_dtype, device=dev)
    if R:
        with _on_device(dev), _span("int8_linear"):
            rc = _abi.lib().fmoe_int8_linear(
                x.data.data_ptr(), x.data.stride(0) if x.data.shape[0] > 1 else Kp,
                x.data.shape[0], x.scales.data_ptr(),
                rows.data_ptr() if rows is not None else None,
                _INDEX_CODES[rows.dtype] if rows is not None else _abi.I64,
                data.data_ptr(), scales.data_ptr(), bias.data_ptr() if bias is not None else None,
                _FLOAT_CODES[bias.dtype] if bias is not None else _abi.F32,
                expert_offsets.data_ptr() if expert_offsets is not None else None, E, N, x.features,
                R, out.data_ptr(), N, _FLOAT_CODES[out_dtype], _stream_handle(dev))
        _abi.check(rc, "fmoe_int8_linear")
    return out


def _validate_linear(x: QuantizedRows, offsets, rows, R: int) -> None:
    bad = torch.zeros((), dtype=torch.int64, device=x.data.device)
    if rows is not None and R:
        bad = bad + ((rows < 0) | (rows >= x.data.shape[0])).sum()
    if offsets is not None:
        bad = bad + (offsets[0] != 0) + (offsets[1:] < offsets[:-1]).sum() + (offsets[-1] > R)
    if int(bad):
        raise IndexError(f"fastmoe_amd: {int(bad)} entries of rows or expert_offsets lie outside "
                         f"x's {x.data.shape[0]} rows, or the {R} packed rows, or fall")


# ---- activations held in 8 bits ---------------------------------------------------------------

def _restore(data, scales, per_row: int, features: int, dtype) -> torch.Tensor:
    if dtype not in _FLOAT_CODES:
        raise TypeError(f"fastmoe_amd: unsupported dtype {dtype}")
    R = data.shape[0]
    out = torch.empty((R, features), dtype=dtype, device=data.device)
    if R:
        with _on_device(data.device), _span("restore_rows"):
            rc = _abi.lib().fmoe_restore_rows(
                data.data_ptr(), data.stride(0) if R > 1 else data.shape[1], scales.data_ptr(),
                per_row, R, features, out.data_ptr(), _FLOAT_CODES[dtype],
                _stream_handle(data.device))
        _abi.check(rc, "fmoe_restore_rows")
    return out


def _check_held(held: CompressedRows) -> None:
    _check_int8(held.data, held.scales, held.features, "held", 2)
    want = (held.data.shape[0], -(-held.features // BLOCK))
    if tuple(held.scales.shape) != want or not held.scales.is_contiguous():
        raise ValueError(f"fastmoe_amd: held scales must be contiguous {list(want)}, got "
                         f"{tuple(held.scales.shape)}")
    if not held.data.is_contiguous():
        raise ValueError("fastmoe_amd: held data must be contiguous")


def _compress(x: torch.Tensor, gelu: bool):
    R, C = x.shape
    dev = x.device
    held = CompressedRows(torch.empty((R, _pad(C)), dtype=torch.int8, device=dev),
                          torch.empty((R, -(-C // BLOCK)), dtype=torch.float32, device=dev), C)
    a = torch.empty((R, C), dtype=x.dtype, device=dev) if gelu else None
    if R:
        with _on_device(dev), _span("compress_rows"):
            rc = _abi.lib().fmoe_compress_rows(
                x.data_ptr(), _row_stride(x), R, C, _FLOAT_CODES[x.dtype], held.data.data_ptr(),
                held.data.shape[1], held.scales.data_ptr(), a.data_ptr() if gelu else None,
                _stream_handle(dev))
        _abi.check(rc, "fmoe_compress_rows")
    return a, held


def compress_rows(x: torch.Tensor) -> CompressedRows:
    """Rows [R, C] (unit column stride) held in 8 bits, a scale for every 128 columns of a row: each
    value within 1/254 of the largest of its block.  Records no backward, and refuses inputs that
    require one (an autograd Function's forward, which records nothing, is where it is called)."""
    _check_matrix(x, "x")
    _no_gradient("compress_rows", x)
    return _compress(x, False)[1]


def restore_rows(held: CompressedRows, dtype: torch.dtype) -> torch.Tensor:
    """The values that held rows stand for, [R, C] in ``dtype``."""
    _check_held(held)
    return _restore(held.data, held.scales, held.scales.shape[1], held.features, dtype)


def gelu_compress(x: torch.Tensor) -> Tuple[torch.Tensor, CompressedRows]:
    """``(gelu(x), x held in 8 bits)`` in one pass: the forward of a GELU whose backward is
    :func:`gelu_compressed_backward`.  GELU is exact (``torch.nn.GELU()``) and taken of the exact x.
    Records no backward, and refuses inputs that require one."""
    _check_matrix(x, "x")
    _no_gradient("gelu_compress", x)
    return _compress(x, True)


def gelu_compressed_backward(held: CompressedRows, grad: torch.Tensor, *,
                             again: bool = True) -> Tuple[Optional[torch.Tensor], torch.Tensor]:
    """``(gelu(x'), grad * gelu'(x'))`` of the held rows x', in ``grad``'s type: GELU's output once
    more, which the gradient of the weights after it reads (None without ``again``), and the
    gradient of GELU's input."""
    _check_held(held)
    _check_matrix(grad, "grad")
    R, C = held.data.shape[0], held.features
    if tuple(grad.shape) != (R, C):
        raise ValueError(f"fastmoe_amd: grad must be [{R}, {C}], got {tuple(grad.shape)}")
    _same_device(held.data, grad=grad)
    _no_gradient("gelu_compressed_backward", grad)
    out = torch.empty((R, C), dtype=grad.dtype, device=grad.device)
    a = torch.empty_like(out) if again else None
    if R:
        with _on_device(grad.device), _span("gelu_compressed_backward"):
            rc = _abi.lib().fmoe_gelu_compressed_backward(
                held.data.data_ptr(), held.data.shape[1], held.scales.data_ptr(), grad.data_ptr(),
                _row_stride(grad), R, C, _FLOAT_CODES[grad.dtype], a.data_ptr() if again else None,
                out.data_ptr(), _stream_handle(grad.device))
        _abi.check(rc, "fmoe_gelu_compressed_backward")
    return a, out
