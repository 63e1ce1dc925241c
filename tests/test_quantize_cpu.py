"""Refusals of the 8-bit operators and their C entry points (CPU: nothing is launched)."""
from __future__ import annotations

import pytest
import torch

import fastmoe_amd as fm
from fastmoe_amd import _abi

DEV = 0x10000  # stands for a device address: every call here is refused before a launch


def test_cpu_tensors_raise():
    x, w = torch.zeros(2, 8), torch.ones(8)
    q = fm.QuantizedRows(torch.zeros(2, 128, dtype=torch.int8), torch.ones(2), 8)
    held = fm.CompressedRows(torch.zeros(2, 128, dtype=torch.int8), torch.ones(2, 1), 8)
    for call in (lambda: fm.add_rms_norm(x, w), lambda: fm.add_rms_norm_int8(x, w, x),
                 lambda: fm.quantize_rows(x), lambda: fm.quantize_weights([x]),
                 lambda: fm.compress_rows(x), lambda: fm.gelu_compress(x),
                 lambda: q.dequantize(), lambda: fm.restore_rows(held, torch.float32),
                 lambda: fm.gelu_compressed_backward(held, x),
                 lambda: fm.int8_linear(q, fm.Int8Weights(q.data, q.scales, 8))):
        with pytest.raises(RuntimeError, match="only on the GPU"):
            call()


def _norm(x=DEV, xs=8, r=None, w=DEV, wd=_abi.BF16, rows=4, cols=8, dt=_abi.BF16, h=None, y=DEV,
          q=None, qs=0, sc=None):
    return _abi.lib().fmoe_add_rms_norm(x, xs, r, xs, w, wd, rows, cols, dt, 1e-6, h, y, None, q, qs,
                                        sc, None)


def test_norm_entry_point_refuses():
    assert _norm(cols=0) == _abi.EINVAL
    assert _norm(rows=-1) == _abi.EINVAL
    assert _norm(dt=_abi.I64) == _abi.EINVAL
    assert _norm(wd=_abi.F16) == _abi.EINVAL          # neither the rows' type nor fp32
    assert _norm(w=None) == _abi.EINVAL
    assert _norm(x=None) == _abi.EINVAL
    assert _norm(xs=-8) == _abi.EINVAL
    assert _norm(r=DEV) == _abi.EINVAL                # a residual without the stream's output
    assert _norm(q=DEV, qs=112, sc=DEV) == _abi.EINVAL   # 8 columns are stored in 128
    assert _norm(q=DEV + 8, qs=128, sc=DEV) == _abi.EINVAL
    assert _norm(q=DEV, qs=128) == _abi.EINVAL        # no scales
    assert _norm(rows=1 << 40) == _abi.ERANGE
    assert _norm(cols=1 << 31) == _abi.ERANGE
    assert _norm(rows=0, x=None) == _abi.OK           # nothing to do


def test_norm_backward_entry_point_refuses():
    lib = _abi.lib()
    need = lib.fmoe_add_rms_norm_backward_workspace_bytes(1000, 8)
    assert need == 512 * 8 * 4
    assert lib.fmoe_add_rms_norm_backward_workspace_bytes(3, 8) == 3 * 8 * 4
    assert lib.fmoe_add_rms_norm_backward_workspace_bytes(-1, 8) < 0

    def call(ws=DEV, nbytes=need, gy=DEV, gw=DEV, wd=_abi.BF16, rows=1000):
        return lib.fmoe_add_rms_norm_backward(gy, 8, None, 0, DEV, 8, DEV, wd, DEV, rows, 8,
                                              _abi.BF16, DEV, gw, ws, nbytes, None)

    assert call(nbytes=need - 1) == _abi.EINVAL
    assert call(ws=None) == _abi.EINVAL
    assert call(ws=DEV + 4) == _abi.EINVAL
    assert call(gy=None) == _abi.EINVAL
    assert call(wd=_abi.F16) == _abi.EINVAL
    assert call(rows=1 << 40) == _abi.ERANGE


def test_row_entry_points_refuse():
    lib = _abi.lib()

    def rows(act=0, q=DEV, qs=128, sc=DEV, x=DEV, cols=8, n=4, dt=_abi.F16):
        return lib.fmoe_quantize_rows(x, 8, n, cols, dt, act, q, qs, sc, None)

    assert rows(act=2) == _abi.EINVAL
    assert rows(q=DEV + 4) == _abi.EINVAL
    assert rows(qs=136) == _abi.EINVAL
    assert rows(cols=129) == _abi.EINVAL              # needs a pitch of 256
    assert rows(sc=None) == _abi.EINVAL
    assert rows(x=None) == _abi.EINVAL
    assert rows(dt=_abi.I32) == _abi.EINVAL
    assert rows(n=1 << 40) == _abi.ERANGE
    assert lib.fmoe_compress_rows(DEV, 8, 4, 8, _abi.F16, DEV, 64, DEV, None, None) == _abi.EINVAL
    assert lib.fmoe_compress_rows(None, 8, 4, 8, _abi.F16, DEV, 128, DEV, None, None) == _abi.EINVAL
    assert lib.fmoe_compress_rows(DEV, 8, 1 << 40, 8, _abi.F16, DEV, 128, DEV, None,
                                  None) == _abi.ERANGE
    # three scales per row are neither one nor the two blocks of 200 columns
    assert lib.fmoe_restore_rows(DEV, 256, DEV, 3, 4, 200, DEV, _abi.F32, None) == _abi.EINVAL
    assert lib.fmoe_restore_rows(DEV, 256, DEV, 2, 4, 200, None, _abi.F32, None) == _abi.EINVAL
    assert lib.fmoe_gelu_compressed_backward(DEV, 256, DEV, None, 8, 4, 200, _abi.F32, None, DEV,
                                             None) == _abi.EINVAL


def test_int8_linear_entry_point_refuses():
    def call(x=DEV, xs=128, xr=4, w=DEV, off=DEV, E=2, N=16, K=100, rows=4, out=DEV, os_=16,
             od=_abi.BF16, idx=None, it=_abi.I64, bias=None, bt=_abi.F32):
        return _abi.lib().fmoe_int8_linear(x, xs, xr, DEV, idx, it, w, DEV, bias, bt, off, E, N, K,
                                           rows, out, os_, od, None)

    assert call(off=None) == _abi.EINVAL              # two experts without offsets
    assert call(xs=112) == _abi.EINVAL
    assert call(xs=136) == _abi.EINVAL
    assert call(x=DEV + 8) == _abi.EINVAL
    assert call(w=DEV + 8) == _abi.EINVAL
    assert call(os_=15) == _abi.EINVAL
    assert call(od=_abi.I64) == _abi.EINVAL
    assert call(idx=DEV, it=_abi.F32) == _abi.EINVAL
    assert call(bias=DEV, bt=_abi.I32) == _abi.EINVAL
    assert call(xr=0) == _abi.EINVAL
    assert call(E=0) == _abi.EINVAL
    assert call(K=131072, xs=131072) == _abi.ERANGE   # (-128)^2 * K would pass int32
    assert call(rows=1 << 31) == _abi.ERANGE
    assert call(N=1 << 25, os_=1 << 25) == _abi.ERANGE
    assert call(rows=0, x=None) == _abi.OK


def test_modules_that_compute_something_else_are_refused():
    """The experts' parameters are read without calling the modules."""
    nn = torch.nn

    class Scaled(nn.Linear):
        def forward(self, x):
            return super().forward(x) * 2

    class Named(nn.Linear):  # a subclass that computes the same
        pass

    class Residual(nn.Sequential):
        def forward(self, x):
            return x + super().forward(x)

    def experts(first=nn.Linear, outer=nn.Sequential, act=nn.GELU):
        return [outer(first(8, 16), act(), nn.Linear(16, 8)) for _ in range(2)]

    x = torch.zeros(4, 8)
    run = lambda e: fm.compute_experts(e, x, [2, 2], checkpoint="int8")
    for wrong in (experts(Scaled), experts(outer=Residual), experts(act=nn.SiLU)):
        with pytest.raises(TypeError, match="Sequential"):
            run(wrong)
    for right in (experts(), experts(Named)):
        with pytest.raises(RuntimeError, match="only on the GPU"):
            run(right)
    patched = experts()
    patched[1][0].forward = lambda x: x
    with pytest.raises(TypeError, match="Sequential"):
        run(patched)
    shared = nn.Linear(8, 8)  # the same module twice: its weight has two gradients
    with pytest.raises(RuntimeError, match="only on the GPU"):
        run([nn.Sequential(shared, nn.GELU(), shared) for _ in range(2)])
    hooked = experts()
    hooked[0][2].register_full_backward_hook(lambda *a: None)
    with pytest.raises(ValueError, match="hooks"):
        run(hooked)
    layer = fm.MoEFeedForward(8, 16, 2, 1)
    layer.router = Scaled(8, 2, bias=False)
    with pytest.raises(TypeError, match="router"):
        layer.int8()


def test_recording_is_refused():
    """make_fx and torch.jit.trace would keep the example's results as constants."""
    from torch.fx.experimental.proxy_tensor import make_fx

    w = torch.ones(8)
    norm = lambda x: fm.add_rms_norm(x, w)[0]
    for record in (lambda: make_fx(norm)(torch.zeros(2, 8)),
                   lambda: torch.jit.trace(norm, (torch.zeros(2, 8),))):
        with pytest.raises(RuntimeError, match="tracing"):
            record()


def test_layers_that_compute_something_else_are_refused():
    """The 8-bit layer reads a layer's parts without calling the layer."""
    class Shared(fm.MoEFeedForward):
        def __init__(self, *args):
            super().__init__(*args)
            self.shared = torch.nn.Linear(args[0], args[0])

        def forward(self, x):
            return super().forward(x) + self.shared(x)

    class Scaled(fm.NormedMoEFeedForward):
        def forward(self, x, residual=None):
            out, stream = super().forward(x, residual)
            return out * 0.5, stream

    class Called(fm.MoEFeedForward):
        def __call__(self, x):
            return super().__call__(x) * 2

    class Named(fm.MoEFeedForward):  # a subclass that computes the same
        pass

    sizes = (8, 16, 2, 1)
    for wrong in (Shared(*sizes), Called(*sizes), fm.NormedMoEFeedForward(Shared(*sizes)),
                  Scaled(fm.MoEFeedForward(*sizes))):
        with pytest.raises(TypeError, match="forward"):
            wrong.int8()
    with pytest.raises(TypeError, match="forward"):
        fm.Int8MoEFeedForward(Shared(*sizes))
    patched = fm.MoEFeedForward(*sizes)
    patched.forward = lambda x: x
    with pytest.raises(TypeError, match="forward"):
        patched.int8()
    for hook in ("register_forward_hook", "register_forward_pre_hook", "register_full_backward_hook"):
        plain, normed = fm.MoEFeedForward(*sizes), fm.NormedMoEFeedForward(fm.MoEFeedForward(*sizes))
        inner = fm.NormedMoEFeedForward(fm.MoEFeedForward(*sizes))
        for module, layer in ((plain, plain), (normed, normed), (inner.moe, inner)):
            getattr(module, hook)(lambda *a: None)
            with pytest.raises(ValueError, match="hooks"):
                layer.int8()
    for right in (Named(*sizes), fm.NormedMoEFeedForward(Named(*sizes))):
        with pytest.raises(RuntimeError, match="only on the GPU"):  # the weights are next
            right.int8()


def test_gelu_without_held_rows_at_the_entry_point():
    lib = _abi.lib()

    def call(q=None, qs=0, sc=None, gelu=DEV, x=DEV, rows=4):
        return lib.fmoe_compress_rows(x, 8, rows, 8, _abi.F16, q, qs, sc, gelu, None)

    assert call(gelu=None) == _abi.EINVAL             # nothing to write
    assert call(q=DEV, qs=128) == _abi.EINVAL         # rows without scales
    assert call(sc=DEV, qs=128) == _abi.EINVAL        # scales without rows
    assert call(x=None) == _abi.EINVAL
    assert call(rows=1 << 40) == _abi.ERANGE
    assert call(rows=0, x=None) == _abi.OK


def test_the_tile_does_not_alternate_with_the_rows():
    """One row more per expert does not change the tile there and back: at these sizes (none of which is a
    tie of two tiles' rounds) a choice between two equal ones lasts three row counts at least."""
    tile = _abi.lib().fmoe_int8_linear_tile
    for E in (1, 4, 8, 13, 16, 20, 32, 50, 64, 128, 160, 256):
        for N in (16, 100, 256, 640, 1003, 2048, 3000, 4096, 8192):
            for K in (128, 2048, 7168):
                runs = []  # (tile, row counts that it lasts)
                for per in range(1, 420):
                    t = tile(per * E, E, N, K)
                    if runs and runs[-1][0] == t:
                        runs[-1][1] += 1
                    else:
                        runs.append([t, 1])
                for a, b, c in zip(runs, runs[1:], runs[2:]):
                    assert a[0] != c[0] or b[1] >= 3, (E, N, K, runs)


def test_a_residual_of_another_shape_is_refused():
    """Of as many rows, but in another order: batch and tokens exchanged."""
    layer = fm.NormedMoEFeedForward(fm.MoEFeedForward(8, 16, 2, 1))
    x = torch.zeros(2, 3, 8)
    for wrong in (torch.zeros(3, 2, 8), torch.zeros(6, 8), torch.zeros(1, 3, 8)):
        with pytest.raises(ValueError, match="residual must be"):
            layer(x, wrong)
    with pytest.raises(RuntimeError, match="only on the GPU"):
        layer(x, torch.zeros(2, 3, 8))


def test_weights_that_are_no_tensors_are_refused():
    for wrong in ([1.0, 2.0], [[1.0]], [None]):
        with pytest.raises(TypeError, match="weight 0 must be a tensor"):
            fm.quantize_weights(wrong)
    with pytest.raises(ValueError, match="no weights"):
        fm.quantize_weights([])


def test_tensors_that_only_stand_for_memory_are_refused():
    """Fake tensors say that they are on the GPU, and have no memory anywhere."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        x, w = torch.empty(2, 8, device="cuda"), torch.empty(8, device="cuda")
        q = fm.QuantizedRows(torch.empty(2, 128, dtype=torch.int8, device="cuda"),
                             torch.empty(2, device="cuda"), 8)
        held = fm.CompressedRows(q.data, torch.empty(2, 1, device="cuda"), 8)
    for call in (lambda: fm.add_rms_norm_int8(x, w), lambda: fm.quantize_rows(x),
                 lambda: fm.compress_rows(x), lambda: fm.gelu_compress(x), lambda: q.dequantize(), lambda: fm.restore_rows(held, torch.float32),
                 lambda: fm.gelu_compressed_backward(held, x)):
        with pytest.raises(ValueError, match="memory of their own"):
            call()
