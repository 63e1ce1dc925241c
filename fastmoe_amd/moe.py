"""The MoE layer's stages around the combine, single GPU (the callers on either side of the path).

Mirrors ``MoEFeedForward`` (src/fastmoe/models/tiny_model.py:42-420) at world size 1 -- where
every exchange of the reference short-circuits (:168-175, :314-315) -- with the combine fed the
ragged per-expert list instead of a ``torch.cat`` of it:

  gate_and_sort    (:79-164)  router -> top-k -> fp32 softmax -> ``permute_tokens`` (HIP sort +
                              gather); returns the reference's 6-tuple
  compute_experts  (:282-294) each expert on its own rows; returns the list of per-expert outputs
                              (the reference concatenates them, :294 -- the copy the grouped
                              combine exists to avoid)
  unpermute        (:396-409) FAST: ``grouped_weighted_scatter_add`` over the per-expert list;
                              STANDARD: the reference's torch formulation (mul + index_add_),
                              kept as the comparison implementation the selector names -- FAST
                              never falls back to it
  MoEFeedForward   the layer wiring these stages (router + experts as in :66-77)

The router GEMM, top-k, softmax and the expert MLPs are torch library calls, as in the reference.

Beyond the reference, on the 8-bit operators of ``quantize``:

  compute_experts(..., checkpoint="int8")  holds the experts' inputs and hidden rows in 8 bits until
                              the backward (``MoEFeedForward(..., checkpoint="int8")``)
  NormedMoEFeedForward        the layer behind a root-mean-square norm with the residual's addition
  Int8MoEFeedForward          either layer for serving, with rows and experts' weights in 8 bits

and on those of ``routing``, ``fp4`` and ``norms``:

  gate_and_sort(..., routing=Routing(...)), MoEFeedForward(..., routing=...)  scores, groups, a bias for
                              balance and weights by ``route_tokens`` instead of the reference's rule
  Fp4MoEFeedForward           the layer for serving, with the experts' weights in 4 bits
  SandwichMoEFeedForward      the layer between two norms, with a gate and a scale for what it adds
"""
from __future__ import annotations

from typing import List, Optional, Sequence, Union

import torch
import torch.nn as nn
import torch.nn.functional as F

from .consts import MoEImplementation
from .dispatch import PermutedTokens, permute_tokens
from .fp4 import Fp4Weights, fp4_linear, quantize_weights_fp4
from .norms import sandwich_norm
from .ops import (_apply, _combine_forward, _GroupedCombinePermuted, _refuse_autograd_capture,
                  _runs_plain, grouped_weighted_scatter_add)
from .quantize import (CompressedRows, Int8Weights, _check_matrix, _compress, _no_gradient, add_rms_norm,
                       add_rms_norm_int8, gelu_compressed_backward, int8_linear, quantize_rows,
                       quantize_weights, restore_rows)
from .routing import Routing, route_tokens

__all__ = ["Fp4MoEFeedForward", "Int8MoEFeedForward", "MoEFeedForward", "NormedMoEFeedForward",
           "SandwichMoEFeedForward", "compute_experts", "gate_and_sort", "unpermute"]


def _route(x_flat: torch.Tensor, router: nn.Module, top_k: int, routing: Optional[Routing] = None,
           bias: Optional[torch.Tensor] = None):
    """(gates in x's type, expert ids), each [T, k] (tiny_model.py:92-100; ``routing``: by route_tokens)."""
    logits = router(x_flat)
    if routing is not None:
        return route_tokens(logits, top_k, routing, bias=bias, out_dtype=x_flat.dtype)
    topk_weights, topk_indices = torch.topk(logits, top_k, dim=-1)
    return F.softmax(topk_weights, dim=-1, dtype=torch.float32).type_as(x_flat), topk_indices


def gate_and_sort(x: torch.Tensor, router: nn.Module, top_k: int, num_experts: int, *,
                  routing: Optional[Routing] = None, bias: Optional[torch.Tensor] = None):
    """Routing and permutation of tiny_model.py:79-164 at world size 1; with a ``routing``, experts and
    weights are those of ``route_tokens`` (``bias`` float32 [E], for the choice alone).

    Returns ``(permuted_data, rank_counts, expert_counts_by_rank, reverse_map_indices,
    sorted_weights, (B, T))`` like the reference (:160-166): ``rank_counts`` = [T*k] (:158),
    ``expert_counts_by_rank`` = counts viewed [1, E] (:157).
    """
    B, T, D = x.shape
    x_flat = x.reshape(-1, D)
    if routing is None and bias is not None:
        raise ValueError("fastmoe_amd: a bias needs a routing")
    topk_weights, topk_indices = _route(x_flat, router, top_k, routing, bias)
    p = permute_tokens(x_flat, topk_indices, topk_weights, num_experts)
    rank_counts = torch.tensor([p.permuted_data.shape[0]], device=x.device, dtype=torch.long)
    return _Routed((p.permuted_data, rank_counts, p.expert_counts.view(1, num_experts),
                    p.reverse_map_indices, p.sorted_weights, (B, T)), p)


class _Routed(tuple):
    """gate_and_sort's 6-tuple (tiny_model.py:160-166) that also carries the permutation."""

    def __new__(cls, items, permutation):
        self = super().__new__(cls, items)
        self.permutation = permutation
        return self


def compute_experts(experts: Sequence[nn.Module], recv_data: torch.Tensor,
                    tokens_per_expert: Sequence[int], *,
                    checkpoint: Optional[str] = None) -> List[torch.Tensor]:
    """Each expert on its own rows (tiny_model.py:282-291); the per-expert outputs stay separate
    allocations (no :294 cat).  An expert with no rows yields an empty [0, D] tensor.

    ``checkpoint="int8"`` (experts ``Sequential(Linear, GELU(), Linear)``) keeps for the backward the
    rows and the first product in 8 bits, a scale for every 128 columns, instead of the rows, the
    first product and GELU's output in their own type: about D + F bytes a row instead of 2 D + 4 F at 16
    bits.  The forward computes with the rows as they are (GELU within the results' rounding); the
    gradients are those of the held values (each within 1/254 of its block's largest).  Without a
    backward to record nothing is held.  Rows and weights share one dtype (autocast's, where it is on).
    """
    if checkpoint is not None:
        if checkpoint != "int8":
            raise ValueError(f"fastmoe_amd: unknown checkpoint {checkpoint!r} (expected None or "
                             "'int8')")
        return _compute_experts_held(experts, recv_data, [int(n) for n in tokens_per_expert])
    chunks = recv_data.split(list(tokens_per_expert), dim=0)
    out = []
    for chunk, expert in zip(chunks, experts):
        if chunk.shape[0] > 0:
            out.append(expert(chunk))
        else:
            out.append(torch.empty(0, recv_data.shape[1], device=recv_data.device,
                                   dtype=recv_data.dtype))
    return out


_HOOKS = ("_forward_hooks", "_forward_pre_hooks", "_backward_hooks", "_backward_pre_hooks")


def _computes_as(module: nn.Module, kind: type) -> bool:
    """``module`` is a ``kind`` whose forward is that class's own."""
    return (isinstance(module, kind) and type(module).forward is kind.forward
            and type(module).__call__ is kind.__call__ and "forward" not in vars(module))


def _hooked(*modules: nn.Module) -> bool:
    return any(getattr(m, hooks, None) for m in modules for hooks in _HOOKS)


def _check_layer(layer: nn.Module, kind: type, form: str) -> None:
    """What ``form`` ("int8" or "fp4") reads of a layer is all that its call computes."""
    if not _computes_as(layer, kind):
        raise TypeError(f"fastmoe_amd: {type(layer).__name__} is not a {kind.__name__} with that class's "
                        f"forward; {form}() would lose what it adds")
    if _hooked(layer):
        raise ValueError(f"fastmoe_amd: the {kind.__name__} has hooks, which the layer that {form}() makes would "
                         "not call")


def _mlp_parameters(experts: Sequence[nn.Module], bits: int = 8):
    """[(w1, b1, w2, b2), ...] of experts Sequential(Linear, GELU(), Linear); biases may be None.  ``bits``: of the
    operators that are to compute them."""
    out = []
    for e, expert in enumerate(experts):
        parts = list(expert) if _computes_as(expert, nn.Sequential) else []
        if len(parts) != 3 or not all(
                _computes_as(p, k) for p, k in zip(parts, (nn.Linear, nn.GELU, nn.Linear))):
            raise TypeError(f"fastmoe_amd: expert {e} is not Sequential(Linear, GELU, Linear)")
        if parts[1].approximate != "none":
            raise ValueError(f"fastmoe_amd: expert {e} has a GELU approximation "
                             f"({parts[1].approximate!r}); the {bits}-bit operators compute the exact form")
        out.append((parts[0].weight, parts[0].bias, parts[2].weight, parts[2].bias))
        if _hooked(expert, *parts):
            raise ValueError(f"fastmoe_amd: expert {e} has hooks, which the {bits}-bit operators would "
                             "not call")
    if not out:
        raise ValueError("fastmoe_amd: no experts")
    return out


def _compute_experts_held(experts, recv_data, counts) -> List[torch.Tensor]:
    params = _mlp_parameters(experts)
    if torch.is_autocast_enabled("cuda"):
        dtype = torch.get_autocast_dtype("cuda")
        recv_data = recv_data.to(dtype)
        params = [tuple(None if t is None else t.to(dtype) for t in p) for p in params]
    _check_matrix(recv_data, "recv_data")
    N, D = recv_data.shape
    hidden = params[0][0].shape[0]
    if len(counts) != len(params) or sum(counts) != N or min(counts) < 0:
        raise ValueError(f"fastmoe_amd: tokens_per_expert {counts} does not split {N} rows over "
                         f"{len(params)} experts")
    for e, (w1, b1, w2, b2) in enumerate(params):
        if tuple(w1.shape) != (hidden, D) or w2.shape[1] != hidden or w2.shape[0] != params[0][2].shape[0]:
            raise ValueError(f"fastmoe_amd: expert {e} has weights {tuple(w1.shape)} and "
                             f"{tuple(w2.shape)}; expert 0 has ({hidden}, {D}) and "
                             f"{tuple(params[0][2].shape)}")
        for t in (w1, b1, w2, b2):
            if t is not None and (t.dtype != recv_data.dtype or t.device != recv_data.device):
                raise TypeError(f"fastmoe_amd: expert {e} has {t.dtype} parameters on {t.device}, "
                                f"the rows are {recv_data.dtype} on {recv_data.device}")
    flat = [t for p in params for t in p]
    records = torch.is_grad_enabled() and any(
        t is not None and t.requires_grad for t in (recv_data, *flat))
    _refuse_autograd_capture("the experts with held activations", recv_data, records)
    # autocast has done its casts: the products below run in the rows' type
    with torch.autocast("cuda", enabled=False):
        return list(_HeldExperts.apply((counts, records), recv_data, *flat))


def _mm(x, w, bias, out):
    """out = x @ w + bias"""
    if bias is None:
        torch.mm(x, w, out=out)
    else:
        torch.addmm(bias, x, w, out=out)


class _HeldExperts(torch.autograd.Function):
    """Every expert's Linear, GELU, Linear over the packed rows; what the backward needs of the
    activations is held in 8 bits.  One launch each way holds or restores all experts' rows.  The first
    argument is the experts' rows and whether a backward is recorded: ctx.needs_input_grad does not
    say so (under no_grad it is still true of parameters)."""

    @staticmethod
    def forward(ctx, plan, x, *flat):
        counts, records = plan
        params = [flat[i:i + 4] for i in range(0, len(flat), 4)]
        h = x.new_empty((x.shape[0], params[0][0].shape[0]))
        for xe, he, (w1, b1, _, _) in zip(x.split(counts), h.split(counts), params):
            if xe.shape[0]:
                _mm(xe, w1.t(), b1, he)
        a, held_h = _compress(h, True, hold=records)
        del h, he  # he: the last expert's part of it
        outs = []
        for ae, (_, _, w2, b2) in zip(a.split(counts), params):
            y = a.new_empty((ae.shape[0], w2.shape[0]))
            if ae.shape[0]:
                _mm(ae, w2.t(), b2, y)
            outs.append(y)
        if not records:
            return tuple(outs)
        held_x = _compress(x, False)[1] if any(ctx.needs_input_grad[2::4]) else None
        ctx.counts, ctx.dtype = counts, x.dtype
        ctx.features = (x.shape[1], a.shape[1])
        ctx.save_for_backward(held_h.data, held_h.scales, *(held_x[:2] if held_x else (None, None)),
                              *flat)
        ctx.set_materialize_grads(False)
        return tuple(outs)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, *grads):
        hd, hs, xd, xs, *flat = ctx.saved_tensors
        _refuse_autograd_capture("the held experts' backward", hd)
        counts, (D, hidden) = ctx.counts, ctx.features
        params = [flat[i:i + 4] for i in range(0, len(flat), 4)]
        needs = ctx.needs_input_grad[2:]
        N = hd.shape[0]
        da = torch.empty((N, hidden), dtype=ctx.dtype, device=hd.device)
        for g, de, (_, _, w2, _) in zip(grads, da.split(counts), params):
            if g is None:
                de.zero_()  # this expert's output had no part in the loss
            elif de.shape[0]:
                torch.mm(g, w2, out=de)
        a, dh = gelu_compressed_backward(CompressedRows(hd, hs, hidden), da, again=any(needs[2::4]))
        del da, de
        x = None
        if any(needs[0::4]):
            x = restore_rows(CompressedRows(xd, xs, D), ctx.dtype).split(counts)
        dx = torch.empty((N, D), dtype=ctx.dtype, device=hd.device) if ctx.needs_input_grad[1] else None
        dxs = dx.split(counts) if dx is not None else None
        a = a.split(counts) if a is not None else None
        out = []
        for e, (g, he, (w1, _, w2, _)) in enumerate(zip(grads, dh.split(counts), params)):
            n1, nb1, n2, nb2 = needs[4 * e:4 * e + 4]
            live = counts[e] > 0 and g is not None
            if dx is not None and counts[e]:
                if live:
                    torch.mm(he, w1, out=dxs[e])
                else:  # zeros, whatever its rows held
                    dxs[e].zero_()
            out += [torch.mm(he.t(), x[e]) if n1 and live else None,
                    he.sum(0) if nb1 and live else None,
                    torch.mm(g.t(), a[e]) if n2 and live else None,
                    g.sum(0) if nb2 and live else None]
        return (None, dx, *out)


def unpermute(x_out: Union[torch.Tensor, Sequence[torch.Tensor]], reverse_map_indices: torch.Tensor,
              sorted_weights: torch.Tensor, original_shape, implementation=MoEImplementation.FAST,
              permutation: Optional[PermutedTokens] = None):
    """Combine of tiny_model.py:396-409.  ``x_out`` is the packed [T*k, D] tensor (as the
    reference passes it) or the list of per-expert outputs (no concatenation).  Given the
    ``permutation`` that produced ``reverse_map_indices``, the FAST combine builds its plan from
    the permutation's slot map (one kernel) instead of inverting the scatter index."""
    B, T = original_shape
    parts = list(x_out) if isinstance(x_out, (list, tuple)) else [x_out]
    D = parts[0].shape[1]
    impl = MoEImplementation(implementation)
    if impl == MoEImplementation.FAST:
        if permutation is not None:
            k = permutation.slot_pos.numel() // (B * T) if B * T else 0
            slots = (permutation.slot_pos, k)
            if _runs_plain((reverse_map_indices, sorted_weights, *parts)):
                out = _combine_forward(None, None, None, reverse_map_indices, sorted_weights,
                                       (B * T, D), parts, False, slots)
            else:
                out = _apply(_GroupedCombinePermuted, slots, reverse_map_indices, sorted_weights,
                             (B * T, D), *parts)
        else:
            out = grouped_weighted_scatter_add(parts, reverse_map_indices, sorted_weights,
                                               (B * T, D))
        return out.view(B, T, D)
    if impl == MoEImplementation.STANDARD:
        packed = parts[0] if len(parts) == 1 else torch.cat(parts, dim=0)
        weighted = packed * sorted_weights.unsqueeze(-1)
        out = torch.zeros(B * T, D, device=packed.device, dtype=weighted.dtype)
        out.index_add_(0, reverse_map_indices, weighted)
        return out.view(B, T, D)
    raise NotImplementedError(impl)


class _Balanced(nn.Module):
    """A layer whose ``balance_bias`` (float32 [E], or None) stays float32 when the layer is cast: steps of
    1e-3 and less would be lost in 16 bits.  ``expert_load`` (int64 [E], or None) moves with the layer, but is no
    buffer: data-parallel wrappers copy the first process's buffers over the others' before a forward."""

    expert_load: Optional[torch.Tensor] = None

    def _apply(self, fn, recurse=True):
        bias = self._buffers.get("balance_bias")
        super()._apply(fn, recurse)
        if bias is not None:
            moved = self._buffers["balance_bias"]
            if moved.dtype != torch.float32:
                self._buffers["balance_bias"] = bias.to(moved.device)
        load = self.expert_load
        if load is not None:
            moved = fn(load)
            if load.is_meta and not moved.is_meta:  # memory without values
                moved = torch.zeros_like(moved)
            self.expert_load = moved if moved.dtype == load.dtype else load.to(moved.device)
        return self

    def __setstate__(self, state):
        super().__setstate__(state)
        if "routing" not in self.__dict__:  # pickled before layers had one
            self.routing = None
            self._buffers.update(balance_bias=None)
        if "expert_load" in self._buffers:  # pickled when it was one
            self._non_persistent_buffers_set.discard("expert_load")
            self.expert_load = self._buffers.pop("expert_load")


class MoEFeedForward(_Balanced):
    """MoE feed-forward layer of tiny_model.py:42-77 on one GPU: router, E experts
    (Linear -> GELU -> Linear), HIP permutation, per-expert compute, grouped combine.

    ``checkpoint="int8"`` holds the experts' activations in 8 bits until the backward (see
    ``compute_experts``); :meth:`int8` makes the layer that serves with 8-bit rows and weights, :meth:`fp4`
    the one with 4-bit weights.

    ``routing``: how experts are chosen and weighed (``route_tokens``) instead of the reference's rule.
    ``balance=True`` (with a routing) adds ``balance_bias`` to the scores that choose; in training mode the
    layer counts the rows that each expert gets in ``expert_load``, and :meth:`update_balance`, called
    after the optimiser's step, moves the bias against it.  ``expert_load`` is what this process counted (a forward that
    activation checkpointing runs again counts again), neither a buffer nor part of the layer's state.  Where several
    processes train copies of the layer, sum it over them first, so that their biases stay alike."""

    def __init__(self, dim: int, ff_dim: int, num_experts: int, top_k: int,
                 implementation=MoEImplementation.FAST, checkpoint: Optional[str] = None,
                 routing: Optional[Routing] = None, balance: bool = False) -> None:
        super().__init__()
        if balance and routing is None:
            raise ValueError("fastmoe_amd: balance needs a routing")
        self.routing = routing
        if checkpoint not in (None, "int8"):
            raise ValueError(f"fastmoe_amd: unknown checkpoint {checkpoint!r} (expected None or "
                             "'int8')")
        self.checkpoint = checkpoint
        self.dim = dim
        self.num_experts = num_experts
        self.top_k = top_k
        self.implementation = MoEImplementation(implementation)
        self.router = nn.Linear(dim, num_experts, bias=False)
        self.experts = nn.ModuleList(
            [nn.Sequential(nn.Linear(dim, ff_dim, bias=False), nn.GELU(),
                           nn.Linear(ff_dim, dim, bias=False)) for _ in range(num_experts)])
        self.register_buffer("balance_bias", torch.zeros(num_experts) if balance else None)
        self.expert_load = torch.zeros(num_experts, dtype=torch.int64) if balance else None

    @torch.no_grad()
    def update_balance(self, rate: float = 1e-3) -> None:
        """``balance_bias += rate * sign(mean load - load)`` of the rows counted since the last call, which
        are forgotten.  A bias of -inf stays: an expert that the router masks in every row is to have it, else its bias
        rises until it takes places with weight 0."""
        if self.balance_bias is None:
            raise ValueError("fastmoe_amd: the layer was made without balance")
        load = self.expert_load.double()
        self.balance_bias.add_((rate * torch.sign(load.mean() - load)).float())
        self.expert_load.zero_()

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        routed = gate_and_sort(x, self.router, self.top_k, self.num_experts, routing=self.routing,
                               bias=self.balance_bias)
        permuted, _, counts_by_rank, rev, weights, shape = routed
        if self.training and self.balance_bias is not None:
            self.expert_load.add_(counts_by_rank.view(-1))
        # the split sizes go to the host, as in the reference (recv_splits .tolist(), :197-207)
        tokens_per_expert = counts_by_rank.view(-1).tolist()
        outs = compute_experts(self.experts, permuted, tokens_per_expert,
                               checkpoint=self.checkpoint)
        if self.implementation == MoEImplementation.FAST:
            return unpermute(outs, rev, weights, shape, self.implementation,
                             permutation=routed.permutation)
        return unpermute(torch.cat(outs, 0), rev, weights, shape, self.implementation)

    def int8(self) -> "Int8MoEFeedForward":
        """This layer for serving, its experts' weights in 8 bits (a copy: later changes of this layer
        do not reach it).  A layer with hooks, or a subclass with a forward of its own, is refused: what
        they add would be lost."""
        return Int8MoEFeedForward(self)

    def fp4(self) -> "Fp4MoEFeedForward":
        """As :meth:`int8`, with the experts' weights in 4 bits and the rows as they are."""
        return Fp4MoEFeedForward(self)


def _check_residual(x: torch.Tensor, residual: Optional[torch.Tensor]) -> None:
    """Before both become rows: [T, B, D] would pass for [B, T, D] there."""
    if residual is not None and residual.shape != x.shape:
        raise ValueError(f"fastmoe_amd: residual must be {tuple(x.shape)}, got "
                         f"{tuple(residual.shape)}")


def _copy_parameters(of: nn.Module, to: nn.Module, *names: str) -> None:
    """``to`` gets copies of these parameters of ``of`` in their own type: a norm may be float32 around a layer in
    16 bits."""
    for name in names:
        p = getattr(of, name)
        setattr(to, name, None if p is None else nn.Parameter(p.detach().clone()))


class NormedMoEFeedForward(nn.Module):
    """A :class:`MoEFeedForward` behind the root-mean-square norm of a pre-norm block: the residual's
    addition and the norm are one kernel (``add_rms_norm``).  ``forward(x, residual=None)`` returns
    ``(moe(norm(x + residual)), x + residual)``: the layer's output and the stream it is added to."""

    def __init__(self, moe: MoEFeedForward, eps: float = 1e-6) -> None:
        super().__init__()
        self.moe = moe
        self.eps = eps
        self.norm_weight = nn.Parameter(torch.ones(moe.dim, dtype=moe.router.weight.dtype,
                                                   device=moe.router.weight.device))

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None):
        _check_residual(x, residual)
        flat = None if residual is None else residual.reshape(-1, x.shape[-1])
        y, stream = add_rms_norm(x.reshape(-1, x.shape[-1]), self.norm_weight, flat, eps=self.eps)
        return self.moe(y.view(x.shape)), stream.view(x.shape)

    def int8(self) -> "Int8MoEFeedForward":
        """As :meth:`MoEFeedForward.int8`, the norm included."""
        _check_layer(self, NormedMoEFeedForward, "int8")
        return Int8MoEFeedForward(self.moe, self.norm_weight, self.eps)

    def fp4(self) -> "NormedMoEFeedForward":
        """As :meth:`MoEFeedForward.fp4`, behind a copy of the norm."""
        _check_layer(self, NormedMoEFeedForward, "fp4")
        block = NormedMoEFeedForward(self.moe.fp4(), self.eps)
        _copy_parameters(self, block, "norm_weight")
        return block.requires_grad_(False)


class SandwichMoEFeedForward(nn.Module):
    """A layer between two norms: ``h = stream + scale * gate * rms(moe(rms(stream) * norm_weight)) *
    post_weight``, where ``rms(v) = v / sqrt(mean(v^2) + eps)`` (``sandwich_norm``).

    ``forward(stream, normed=None, gate=None, next_weight=None)`` returns ``(h, y)``: ``y = rms(h) *
    next_weight`` is what the next block's layer reads, made in the same pass, and the next call's
    ``normed`` (None without ``next_weight``).  ``gate``: [dim], or [batch, dim] with one for each sequence;
    ``gated=True`` adds a parameter ``gate`` [dim], ones at first, for calls that give none.  ``moe``: a
    :class:`MoEFeedForward`, or one of its serving forms without a norm."""

    def __init__(self, moe: nn.Module, eps: float = 1e-6, scale: float = 1.0, gated: bool = False) -> None:
        super().__init__()
        self.moe, self.eps, self.scale = moe, eps, scale
        like = dict(dtype=moe.router.weight.dtype, device=moe.router.weight.device)
        self.norm_weight = nn.Parameter(torch.ones(moe.dim, **like))
        self.post_weight = nn.Parameter(torch.ones(moe.dim, **like))
        self.gate = nn.Parameter(torch.ones(moe.dim, **like)) if gated else None

    def forward(self, stream: torch.Tensor, normed: Optional[torch.Tensor] = None,
                gate: Optional[torch.Tensor] = None, next_weight: Optional[torch.Tensor] = None):
        D = stream.shape[-1]
        flat = stream.reshape(-1, D)
        if normed is None:
            normed = add_rms_norm(flat, self.norm_weight, eps=self.eps)[0]
        else:
            _check_residual(stream, normed)
        gate = self.gate if gate is None else gate
        if gate is not None and gate.dim() > 1 and gate.shape[0] != stream.shape[0]:
            raise ValueError(f"fastmoe_amd: gate must be [{D}] or [{stream.shape[0]}, {D}], got "
                             f"{tuple(gate.shape)}")
        out = self.moe(normed.reshape(stream.shape)).reshape(-1, D)
        if len(flat) and torch.is_grad_enabled() and normed.requires_grad and not out.requires_grad:
            raise RuntimeError("fastmoe_amd: the layer between the norms has no gradients; call the block under "
                               "torch.no_grad()")
        y, h = sandwich_norm(out, self.post_weight, flat, next_weight, gate=gate, scale=self.scale, eps=self.eps)
        return h.view(stream.shape), None if y is None else y.view(stream.shape)

    def fp4(self) -> "SandwichMoEFeedForward":
        """This block for serving: a copy with the experts' weights in 4 bits."""
        _check_layer(self, SandwichMoEFeedForward, "fp4")
        block = SandwichMoEFeedForward(self.moe.fp4(), self.eps, self.scale, self.gate is not None)
        _copy_parameters(self, block, "norm_weight", "post_weight", "gate")
        return block.requires_grad_(False)


class Fp4MoEFeedForward(_Balanced):
    """An MoE layer for serving with the experts' weights in 4 bits, a scale for 32 of them (Linear -> GELU ->
    Linear, biases in their own type), and 16-bit rows.  Made by :meth:`MoEFeedForward.fp4` (or those of
    the layers around it).

    ``forward(x)`` returns the layer's output.  The experts' first product reads each token's row
    through the reverse map and applies GELU: no [T*k, D] copy of the rows is made.  The host reads
    nothing back, so a call can be captured in a HIP graph.  It has no gradients, and refuses an x that requires one.
    """

    def __init__(self, moe: MoEFeedForward) -> None:
        super().__init__()
        _check_layer(moe, MoEFeedForward, "fp4")
        params = _mlp_parameters(moe.experts, 4)
        if not _computes_as(moe.router, nn.Linear) or _hooked(moe.router):
            raise TypeError("fastmoe_amd: the router is not a Linear without hooks")
        if moe.router.weight.dtype not in (torch.bfloat16, torch.float16):
            raise TypeError(f"fastmoe_amd: the 4-bit layer's rows are bfloat16 or float16; this one is "
                            f"{moe.router.weight.dtype}")
        self.dim, self.num_experts, self.top_k = moe.dim, moe.num_experts, moe.top_k
        self.routing = moe.routing
        self.hidden = params[0][0].shape[0]
        self.router = nn.Linear(moe.dim, moe.num_experts, bias=moe.router.bias is not None,
                                dtype=moe.router.weight.dtype, device=moe.router.weight.device)
        self.router.load_state_dict(moe.router.state_dict())
        self.router.requires_grad_(False)

        def keep(name, t):
            self.register_buffer(name, None if t is None else t.detach().clone())

        keep("balance_bias", moe.balance_bias)
        for i, name in ((0, "1"), (2, "2")):
            w = quantize_weights_fp4([p[i] for p in params])
            self.register_buffer("w" + name, w.data)
            self.register_buffer("s" + name, w.scales)
            biases = [p[i + 1] for p in params]
            if any((b is None) != (biases[0] is None) for b in biases):
                raise ValueError("fastmoe_amd: some experts have biases and some have none")
            keep("b" + name, None if biases[0] is None else torch.stack([b.detach() for b in biases]))

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if x.dim() != 3 or x.shape[2] != self.dim:
            raise ValueError(f"fastmoe_amd: x must be [batch, tokens, {self.dim}], got "
                             f"{tuple(x.shape)}")
        _no_gradient("the layer in 4 bits", x)
        with torch.no_grad():
            return self._serve(x)

    def _serve(self, x: torch.Tensor) -> torch.Tensor:
        B, T, D = x.shape
        flat = x.reshape(-1, D)
        if flat.shape[0] == 0:
            return x.new_empty(x.shape)
        gates, ids = _route(flat, self.router, self.top_k, self.routing, self.balance_bias)
        # the sort alone: what it gathers is one column
        p = permute_tokens(flat[:, :1], ids, gates, self.num_experts)
        h = fp4_linear(flat, Fp4Weights(self.w1, self.s1, D), p.expert_offsets, rows=p.reverse_map_indices,
                       bias=self.b1, activation="gelu")
        h = fp4_linear(h, Fp4Weights(self.w2, self.s2, self.hidden), p.expert_offsets, bias=self.b2)
        return unpermute(h, p.reverse_map_indices, p.sorted_weights, (B, T), permutation=p)


class Int8MoEFeedForward(_Balanced):
    """An MoE layer for serving in 8 bits: rows with one scale each, experts' weights with one scale for
    each output (Linear -> GELU -> Linear, biases in their own type).  Made by
    :meth:`MoEFeedForward.int8` or :meth:`NormedMoEFeedForward.int8`.

    ``forward(x)`` without a norm returns the layer's output; with one, ``forward(x, residual=None)``
    returns ``(output, x + residual)``.  The router stays in its own type and reads the unquantised
    rows.  The experts' first product reads each token's 8-bit row through the reverse map: no
    [T*k, D] copy of the rows is made.  The host reads nothing back, so a call can be captured in a
    HIP graph.  No gradients; convert the layer to its type before making this one (casting it
    later would cast the scales, which the products refuse).
    """

    def __init__(self, moe: MoEFeedForward, norm_weight: Optional[torch.Tensor] = None,
                 eps: float = 1e-6) -> None:
        super().__init__()
        _check_layer(moe, MoEFeedForward, "int8")
        params = _mlp_parameters(moe.experts)
        if not _computes_as(moe.router, nn.Linear) or _hooked(moe.router):
            raise TypeError("fastmoe_amd: the router is not a Linear without hooks")
        self.dim, self.num_experts, self.top_k, self.eps = moe.dim, moe.num_experts, moe.top_k, eps
        self.routing = moe.routing
        self.hidden = params[0][0].shape[0]
        self.router = nn.Linear(moe.dim, moe.num_experts, bias=moe.router.bias is not None,
                                dtype=moe.router.weight.dtype, device=moe.router.weight.device)
        self.router.load_state_dict(moe.router.state_dict())
        self.router.requires_grad_(False)

        def keep(name, t):
            self.register_buffer(name, None if t is None else t.detach().clone())

        keep("norm_weight", norm_weight)
        keep("balance_bias", moe.balance_bias)
        for i, name in ((0, "1"), (2, "2")):
            w = quantize_weights([p[i] for p in params])
            self.register_buffer("w" + name, w.data)
            self.register_buffer("s" + name, w.scales)
            biases = [p[i + 1] for p in params]
            if any((b is None) != (biases[0] is None) for b in biases):
                raise ValueError("fastmoe_amd: some experts have biases and some have none")
            keep("b" + name, None if biases[0] is None else torch.stack([b.detach() for b in biases]))

    @torch.no_grad()
    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None):
        if x.dim() != 3 or x.shape[2] != self.dim:
            raise ValueError(f"fastmoe_amd: x must be [batch, tokens, {self.dim}], got "
                             f"{tuple(x.shape)}")
        B, T, D = x.shape
        flat = x.reshape(-1, D)
        if self.norm_weight is None:
            if residual is not None:
                raise ValueError("fastmoe_amd: a residual needs the norm (NormedMoEFeedForward.int8)")
            rows, y = quantize_rows(flat), flat
        else:
            _check_residual(x, residual)
            rows, y, stream = add_rms_norm_int8(
                flat, self.norm_weight, None if residual is None else residual.reshape(-1, D),
                eps=self.eps)
        if flat.shape[0] == 0:
            out = x.new_empty(x.shape)
        else:
            gates, ids = _route(y, self.router, self.top_k, self.routing, self.balance_bias)
            # the sort alone: what it gathers are the rows' scales, four bytes each
            p = permute_tokens(rows.scales.view(-1, 1), ids, gates, self.num_experts)
            h = int8_linear(rows, Int8Weights(self.w1, self.s1, D), p.expert_offsets,
                            rows=p.reverse_map_indices, bias=self.b1, out_dtype=x.dtype)
            h = int8_linear(quantize_rows(h, activation="gelu"),
                            Int8Weights(self.w2, self.s2, self.hidden), p.expert_offsets,
                            bias=self.b2, out_dtype=x.dtype)
            out = unpermute(h, p.reverse_map_indices, p.sorted_weights, (B, T), permutation=p)
        return out if self.norm_weight is None else (out, stream.view(x.shape))
