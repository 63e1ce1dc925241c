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

import ctypes
from typing import NamedTuple, Optional, Sequence, Tuple, Union

import torch
from torch.autograd import forward_ad

from . import _abi, ops
from .ops import _FLOAT_CODES, _INDEX_CODES, _refuse_autograd_capture, _validate_default

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

_ROWS: list = []


def _rows_module():
    """The host helper module ``fastmoe_amd._rows`` (built with the library), which allocates for and
    calls the entry points; raises if it or the library is missing."""
    if not _ROWS:
        lib = _abi.lib()
        try:
            from . import _rows as mod
        except ImportError as exc:
            raise _abi.FastMoEError(
                "fastmoe_amd: the host helper module fastmoe_amd._rows is not built "
                "(run python -m fastmoe_amd.build)") from exc
        names = [n for n in _abi.SIGNATURES if hasattr(lib, n)]
        mod.bind({n: ctypes.cast(getattr(lib, n), ctypes.c_void_p).value for n in names})
        _ROWS.append(mod)
    return _ROWS[0]


def _call(name: str, *args):
    """A function of the helper module, in a span of its name where calls are timed.  NotImplemented
    where it does not take its arguments: the caller then checks them one by one."""
    fn = getattr(_ROWS[0] if _ROWS else _rows_module(), name)
    if ops._TIMER is None:
        return fn(*args)
    with ops._TIMER.span(name):
        return fn(*args)


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


def _float_code(dtype, what: str = "dtype") -> int:
    code = _FLOAT_CODES.get(dtype)
    if code is None:
        raise TypeError(f"fastmoe_amd: unsupported {what} {dtype}")
    return code


def _refuse_transforms(what: str) -> None:
    """These calls are opaque to functorch's transforms, forward-mode gradients and tracing (which would
    record their results as constants)."""
    if torch.compiler.is_compiling():  # first: the compiler does not trace the others
        return
    if (torch._C._are_functorch_transforms_active() or forward_ad._current_level >= 0
            or torch._C._get_tracing_state() is not None
            or torch._C._get_dispatch_mode(torch._C._TorchDispatchModeKey.PROXY) is not None):
        raise RuntimeError(f"fastmoe_amd: {what} does not run under functorch transforms, "
                           "forward-mode gradients or tracing")


def _not_taken(what: str) -> None:
    _refuse_transforms(what)
    raise ValueError(f"fastmoe_amd: {what} does not take these tensors (forward-mode gradients, views that "
                     "stand for negated memory, and tensors without memory of their own are not read)")


class QuantizedRows(NamedTuple):
    """Rows in 8 bits with one scale each: row r stands for ``data[r, :features] * scales[r]``."""

    data: torch.Tensor    # int8 [R, features rounded up to 128], zeros from ``features`` on
    scales: torch.Tensor  # float32 [R]
    features: int

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The values that the rows stand for, [R, features]."""
        out = _call("restore", self.data, self.scales, False, self.features, _float_code(dtype))
        if out is NotImplemented:
            _check_rows8(self, "rows")
            _no_gradient("dequantize", self.scales)
            _not_taken("dequantize")
        return out


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


def add_rms_norm(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None, *,
                 eps: float = 1e-6) -> Tuple[torch.Tensor, torch.Tensor]:
    """``h = x + residual`` and ``y = h * weight / sqrt(mean(h^2) + eps)``; returns ``(y, h)``.

    ``x`` and ``residual`` [T, D] (unit column stride), ``weight`` [D] in x's type or float32.  h is
    rounded to x's type, as the tensors' sum is, and y is computed from it in float32 and rounded
    once.  Without a residual, h is ``x`` itself.  Differentiable in all three; the gradient of the
    weight sums the rows in a fixed order.  A row whose sum of squares passes float32's range gives zeros.
    """
    _refuse_transforms("add_rms_norm")
    out = _call("norm", x, weight, residual, eps, True, False)
    if out is not NotImplemented:  # nothing to record
        return out[1], x if residual is None else out[0]
    _check_norm(x, weight, residual, eps)
    _refuse_autograd_capture("the autograd norm", x)
    out = _call("norm_recorded", x, weight, residual, eps)
    if out is NotImplemented:
        _not_taken("add_rms_norm")
    return out


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
    out = _call("norm", x, weight, residual, eps, bool(keep_normed), True)
    if out is NotImplemented:
        _check_norm(x, weight, residual, eps)
        _no_gradient("add_rms_norm_int8", x, weight, residual)
        _not_taken("add_rms_norm_int8")
    h, y, q, scales = out
    return Int8NormedRows(QuantizedRows(q, scales, x.shape[1]), y, x if residual is None else h)


# ---- rows and weights in 8 bits ---------------------------------------------------------------

def quantize_rows(x: torch.Tensor, *, activation: Optional[str] = None) -> QuantizedRows:
    """Rows [R, C] (unit column stride) in 8 bits with one scale each, after ``activation``: None or
    "gelu" (the exact form, as ``torch.nn.GELU()``).  Records no backward, and refuses inputs that
    require one."""
    if activation not in _ACTIVATIONS:
        raise ValueError(f"fastmoe_amd: unknown activation {activation!r} (expected None or 'gelu')")
    out = _call("quantize", x, _ACTIVATIONS[activation])
    if out is NotImplemented:
        _check_matrix(x, "x")
        _no_gradient("quantize_rows", x)
        _not_taken("quantize_rows")
    return QuantizedRows(*out, x.shape[1])


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
    _need_gpu(parts[0], "weight 0")
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
    if _validate_default(validate):
        _check_linear(x, weights, expert_offsets, rows, bias, out_dtype)
        _validate_linear(x, expert_offsets, rows)
    args = (x.data, x.scales, x.features, weights.data, weights.scales)
    code = _FLOAT_CODES.get(out_dtype)
    out = NotImplemented
    if code is not None and weights.features == x.features:
        out = _call("linear", *args, expert_offsets, rows, bias, code)
    if out is NotImplemented:
        _check_linear(x, weights, expert_offsets, rows, bias, out_dtype)
        # what is left: indices, offsets or a bias with gaps between their elements
        expert_offsets, rows, bias = (t if t is None else t.contiguous()
                                      for t in (expert_offsets, rows, bias))
        out = _call("linear", *args, expert_offsets, rows, bias, code)
        if out is NotImplemented:
            _not_taken("int8_linear")
    return out


def _check_linear(x, weights, expert_offsets, rows, bias, out_dtype) -> None:
    """Says what is wrong with int8_linear's arguments, if anything is."""
    _check_rows8(x, "x")
    data, scales = weights.data, weights.scales
    if isinstance(data, torch.Tensor) and data.dim() == 2:
        data, scales = data.unsqueeze(0), scales.unsqueeze(0)
    _check_int8(data, scales, weights.features, "weights", 3)
    E, N, _ = data.shape
    if weights.features != x.features:
        raise ValueError(f"fastmoe_amd: x has {x.features} features, the weights {weights.features}")
    if E < 1 or N < 1 or tuple(scales.shape) != (E, N):
        raise ValueError(f"fastmoe_amd: weight scales must be [{E}, {N}], got {tuple(scales.shape)}")
    if not data.is_contiguous() or not scales.is_contiguous():
        raise ValueError("fastmoe_amd: weights and their scales must be contiguous")
    _float_code(out_dtype, "out_dtype")
    if expert_offsets is None:
        if E != 1:
            raise ValueError(f"fastmoe_amd: {E} experts need expert_offsets")
    else:
        _need_gpu(expert_offsets, "expert_offsets")
        if expert_offsets.dtype != torch.int64 or tuple(expert_offsets.shape) != (E + 1,):
            raise ValueError(f"fastmoe_amd: expert_offsets must be int64 [{E + 1}], got "
                             f"{expert_offsets.dtype} {tuple(expert_offsets.shape)}")
    if rows is not None:
        _need_gpu(rows, "rows")
        if rows.dtype not in _INDEX_CODES or rows.dim() != 1:
            raise TypeError(f"fastmoe_amd: rows must be int64 or int32 with one dimension, got "
                            f"{rows.dtype} {tuple(rows.shape)}")
        if rows.shape[0] and not x.data.shape[0]:
            raise ValueError("fastmoe_amd: rows is not empty, and x is")
    if bias is not None:
        _need_gpu(bias, "bias")
        if bias.dtype not in _FLOAT_CODES:
            raise TypeError(f"fastmoe_amd: unsupported bias dtype {bias.dtype}")
        if tuple(bias.shape) != (E, N) and not (E == 1 and tuple(bias.shape) == (N,)):
            raise ValueError(f"fastmoe_amd: bias must be [{E}, {N}], got {tuple(bias.shape)}")
    _no_gradient("int8_linear", x.scales, weights.scales, bias)
    _same_device(x.data, weights=data, expert_offsets=expert_offsets, rows=rows, bias=bias)


def _validate_linear(x: QuantizedRows, offsets, rows) -> None:
    R = x.data.shape[0] if rows is None else rows.shape[0]
    bad = torch.zeros((), dtype=torch.int64, device=x.data.device)
    if rows is not None and R:
        bad = bad + ((rows < 0) | (rows >= x.data.shape[0])).sum()
    if offsets is not None:
        bad = bad + (offsets[0] != 0) + (offsets[1:] < offsets[:-1]).sum() + (offsets[-1] > R)
    if int(bad):
        raise IndexError(f"fastmoe_amd: {int(bad)} entries of rows or expert_offsets lie outside "
                         f"x's {x.data.shape[0]} rows, or the {R} packed rows, or fall")


# ---- activations held in 8 bits ---------------------------------------------------------------

def _check_held(held: CompressedRows) -> None:
    _check_int8(held.data, held.scales, held.features, "held", 2)
    want = (held.data.shape[0], -(-held.features // BLOCK))
    if tuple(held.scales.shape) != want or not held.scales.is_contiguous():
        raise ValueError(f"fastmoe_amd: held scales must be contiguous {list(want)}, got "
                         f"{tuple(held.scales.shape)}")
    if not held.data.is_contiguous():
        raise ValueError("fastmoe_amd: held data must be contiguous")


def _compress(x: torch.Tensor, gelu: bool, what: str = "compress_rows", hold: bool = True):
    """(gelu(x) or None, x held in 8 bits, or nothing in it without ``hold``)."""
    out = _call("compress", x, gelu, hold)
    if out is NotImplemented:
        _check_matrix(x, "x")
        _no_gradient(what, x)
        _not_taken(what)
    a, q, scales = out
    return a, CompressedRows(q, scales, x.shape[1])


def compress_rows(x: torch.Tensor) -> CompressedRows:
    """Rows [R, C] (unit column stride) held in 8 bits, a scale for every 128 columns of a row: each
    value within 1/254 of the largest of its block.  Records no backward, and refuses inputs that
    require one (an autograd Function's forward, which records nothing, is where it is called)."""
    return _compress(x, False)[1]


def restore_rows(held: CompressedRows, dtype: torch.dtype) -> torch.Tensor:
    """The values that held rows stand for, [R, C] in ``dtype``."""
    out = _call("restore", held.data, held.scales, True, held.features, _float_code(dtype))
    if out is NotImplemented:
        _check_held(held)
        _no_gradient("restore_rows", held.scales)
        _not_taken("restore_rows")
    return out


def gelu_compress(x: torch.Tensor) -> Tuple[torch.Tensor, CompressedRows]:
    """``(gelu(x), x held in 8 bits)`` in one pass: the forward of a GELU whose backward is
    :func:`gelu_compressed_backward`.  GELU is exact (``torch.nn.GELU()``) and taken of the exact x.
    Records no backward, and refuses inputs that require one."""
    return _compress(x, True, "gelu_compress")


def gelu_compressed_backward(held: CompressedRows, grad: torch.Tensor, *,
                             again: bool = True) -> Tuple[Optional[torch.Tensor], torch.Tensor]:
    """``(gelu(x'), grad * gelu'(x'))`` of the held rows x', in ``grad``'s type: GELU's output once
    more, which the gradient of the weights after it reads (None without ``again``), and the
    gradient of GELU's input."""
    out = _call("gelu_backward", held.data, held.scales, held.features, grad, bool(again))
    if out is NotImplemented:
        _check_held(held)
        _check_matrix(grad, "grad")
        R, C = held.data.shape[0], held.features
        if tuple(grad.shape) != (R, C):
            raise ValueError(f"fastmoe_amd: grad must be [{R}, {C}], got {tuple(grad.shape)}")
        _same_device(held.data, grad=grad)
        _no_gradient("gelu_compressed_backward", held.scales, grad)
        _not_taken("gelu_compressed_backward")
    return out
