"""Tensor subclasses without memory of their own are refused, wherever they are passed."""
from __future__ import annotations

import pytest
import torch

import fastmoe_amd as fm

pytestmark = pytest.mark.gpu


class Wrapper(torch.Tensor):
    """A subclass that says it is a tensor on the GPU; its address is null."""

    @staticmethod
    def __new__(cls, t):
        return torch.Tensor._make_wrapper_subclass(cls, t.shape, strides=t.stride(), dtype=t.dtype,
                                                   device=t.device, requires_grad=t.requires_grad)

    def __init__(self, t):
        pass

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        raise NotImplementedError(f"{func}")


class Named(torch.Tensor):
    """A subclass with memory of its own."""


def test_wrappers_are_refused():
    x, w, bias = (torch.randn(*s, device="cuda") for s in ((4, 256), (256,), (2, 8)))
    rows = torch.tensor([0, 1, 2, 3], device="cuda")
    off = torch.tensor([0, 2, 4], device="cuda")
    q, weights = fm.quantize_rows(x), fm.quantize_weights(torch.randn(2, 8, 256, device="cuda"))
    one = fm.Int8Weights(weights.data[:1], weights.scales[:1], 256)
    held = fm.compress_rows(x)
    W = Wrapper
    for call in (lambda: fm.add_rms_norm(W(x), w, x), lambda: fm.add_rms_norm(x, w, W(x)),
                 lambda: fm.add_rms_norm(x, W(w)), lambda: fm.add_rms_norm_int8(x, w, W(x)),
                 lambda: fm.quantize_rows(W(x)), lambda: fm.gelu_compress(W(x)),
                 lambda: q._replace(scales=W(q.scales)).dequantize(),
                 lambda: fm.restore_rows(held._replace(data=W(held.data)), torch.float32),
                 lambda: fm.gelu_compressed_backward(held, W(x)),
                 lambda: fm.int8_linear(q, weights, off, rows=W(rows)),
                 lambda: fm.int8_linear(q, weights, off, bias=W(bias)),
                 lambda: fm.int8_linear(q, one, W(off[:2]))):
        with pytest.raises((ValueError, RuntimeError, NotImplementedError, TypeError)):
            call()


def test_subclasses_with_memory_are_taken():
    x, w = torch.randn(4, 64, device="cuda"), torch.randn(64, device="cuda")
    y, _ = fm.add_rms_norm(x.as_subclass(Named), torch.nn.Parameter(w), x)
    assert torch.equal(y.as_subclass(torch.Tensor), fm.add_rms_norm(x, w, x)[0])


def test_zeros_without_memory_are_refused():
    """What forward-mode and complex views make for zeros: no memory, a null address."""
    x, w = torch.randn(4, 256, device="cuda"), torch.randn(256, device="cuda")
    zero = torch._efficientzerotensor((4, 256), device="cuda")
    assert zero.is_cuda and not zero.any()
    q, weights = fm.quantize_rows(x), fm.quantize_weights(torch.randn(8, 256, device="cuda"))
    for call in (lambda: fm.add_rms_norm(x, w, zero), lambda: fm.add_rms_norm_int8(x, w, zero),
                 lambda: fm.quantize_rows(zero), lambda: fm.gelu_compressed_backward(fm.compress_rows(x), zero),
                 lambda: fm.int8_linear(q, weights, bias=torch._efficientzerotensor((8,), device="cuda"))):
        with pytest.raises((ValueError, RuntimeError)):
            call()


def test_gradients_of_every_kind():
    """Zeros without memory count as zeros; wrappers and batched gradients raise."""
    x, w, r = (torch.randn(*s, device="cuda").requires_grad_(True) for s in ((4, 32), (32,), (4, 32)))
    g, gh = torch.randn(4, 32, device="cuda"), torch.randn(4, 32, device="cuda")

    def grads(of_y, of_h, **kw):
        y, h = fm.add_rms_norm(x, w, r)
        return torch.autograd.grad([y, h], [x, w, r], [of_y, of_h], **kw)

    zero = torch._efficientzerotensor((4, 32), device="cuda")
    for a, b in ((g, zero), (zero, gh)):
        plain = [torch.zeros_like(g) if t is zero else t for t in (a, b)]
        assert all(torch.equal(u, v) for u, v in zip(grads(a, b), grads(*plain)))
    for which in range(2):
        y, h = fm.add_rms_norm(x, w, r)
        (y, h)[which].register_hook(Wrapper)
        with pytest.raises((ValueError, RuntimeError, NotImplementedError, TypeError)):
            torch.autograd.grad([y, h], [x, w, r], [g, gh])
    with pytest.raises(RuntimeError):
        grads(torch.stack([g, g]), torch.stack([gh, gh]), is_grads_batched=True)
    assert all(t.isfinite().all() for t in grads(g, gh))  # and leaves nothing behind
