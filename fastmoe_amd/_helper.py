"""Loader of the host helper module ``fastmoe_amd._block`` and the checks that its callers share."""
from __future__ import annotations

import ctypes

import torch

from . import _abi, ops
from .ops import _FLOAT_CODES

_BLOCK: list = []


def _block_module():
    """The helper module (built with the library); raises if it or the library is missing."""
    if not _BLOCK:
        lib = _abi.lib()
        try:
            from . import _block as mod
        except ImportError as exc:
            raise _abi.FastMoEError(
                "fastmoe_amd: the host helper module fastmoe_amd._block is not built "
                "(run python -m fastmoe_amd.build)") from exc
        mod.bind({n: ctypes.cast(getattr(lib, n), ctypes.c_void_p).value for n in _abi.SIGNATURES})
        _BLOCK.append(mod)
    return _BLOCK[0]


def call(name: str, *args):
    """A function of the helper module, in a span of its name where calls are timed.  NotImplemented
    where it does not take its arguments: the caller then checks them one by one."""
    fn = getattr(_BLOCK[0] if _BLOCK else _block_module(), name)
    if ops._TIMER is None:
        return fn(*args)
    with ops._TIMER.span(name):
        return fn(*args)


def need_gpu(t, what: str) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"fastmoe_amd: {what} must be a tensor, got {type(t).__name__}")
    if not t.is_cuda:
        raise RuntimeError(f"fastmoe_amd: {what} is on {t.device}; this operator runs only on the GPU")


def check_matrix(t, what: str) -> None:
    """``t`` is a 2-D float matrix on the GPU whose rows have unit stride."""
    need_gpu(t, what)
    if t.dim() != 2:
        raise ValueError(f"fastmoe_amd: {what} must be [rows, columns], got {tuple(t.shape)}")
    if t.dtype not in _FLOAT_CODES:
        raise TypeError(f"fastmoe_amd: unsupported {what} dtype {t.dtype}")
    if t.shape[1] < 1:
        raise ValueError(f"fastmoe_amd: {what} has no columns")
    if t.shape[1] > 1 and t.stride(1) != 1 and t.shape[0] > 0:
        raise ValueError(f"fastmoe_amd: {what} must have unit column stride")
