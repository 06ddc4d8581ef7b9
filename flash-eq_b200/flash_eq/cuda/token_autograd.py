"""Layer norm and mixture-of-experts operators with autograd: native forward, native backward.

``layer_norm`` normalises the last dimension.  ``expert_route`` turns router logits into a plan
(``ExpertRoute``): the chosen experts, their weights and every pair's place in the order by
expert.  ``expert_dispatch`` brings token rows into that order, ``expert_linear`` applies each
expert's linear map to its rows (equivariant rows (rows, dim, channels) with one weight per irrep,
or plain rows), and ``expert_combine`` sums the weighted rows back onto their tokens.  The row
counts of the experts stay on the device: no call synchronises the host.  All sums have a fixed
order, so results and gradients are reproducible bit for bit.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch
from torch.autograd.function import once_differentiable

from . import token_ops


def _tracks(*tensors) -> bool:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, stats = token_ops.layer_norm_fwd(x, weight, bias, eps, keep_stats=True)
        ctx.save_for_backward(x, weight, stats)
        ctx.param_dtype = next((p.dtype for p in (weight, bias) if p is not None), None)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out):
        x, weight, stats = ctx.saved_tensors
        need = ctx.needs_input_grad
        return (*token_ops.layer_norm_bwd(grad_out, x, weight, stats, need[0], need[1], need[2], ctx.param_dtype),
                None)


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               eps: float = 1e-5) -> torch.Tensor:
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dimension, in float32, rounded once
    to x's type (float32, bfloat16, float16).  weight and bias: x's type or float32, or None."""
    if _tracks(x, weight, bias):
        return _LayerNorm.apply(x, weight, bias, eps)
    return token_ops.layer_norm_fwd(x, weight, bias, eps, keep_stats=False)[0]


@dataclass
class ExpertRoute:
    """Where the (token, choice) pairs go.

    experts (tokens, top_k) int32: the chosen experts, best first; -1 where a choice is missing
    weights (tokens, top_k) float32: their weights (differentiable with respect to the logits)
    slots   (tokens, top_k) int32: each pair's place in the order by expert; pairs without an expert last
    offsets (num_experts + 1,) int32: the first place of each expert; the last entry counts the pairs
            that have one
    """
    experts: torch.Tensor
    weights: torch.Tensor
    slots: torch.Tensor
    offsets: torch.Tensor

    @property
    def num_experts(self) -> int:
        return self.offsets.shape[0] - 1

    @property
    def top_k(self) -> int:
        return self.slots.shape[1]

    @property
    def num_tokens(self) -> int:
        return self.slots.shape[0]


class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, top_k, normalize):
        ids, weights, slots, offsets = token_ops.expert_route(logits, top_k, normalize)
        ctx.mark_non_differentiable(ids, slots, offsets)
        ctx.save_for_backward(logits, ids, weights)
        ctx.normalize = normalize
        return ids, weights, slots, offsets

    @staticmethod
    @once_differentiable
    def backward(ctx, _ids, grad_weights, _slots, _offsets):
        logits, ids, weights = ctx.saved_tensors
        return token_ops.expert_route_bwd(logits, ids, weights, grad_weights, ctx.normalize), None, None


def expert_route(logits: torch.Tensor, top_k: int, normalize: bool = True) -> ExpertRoute:
    """The ``top_k`` best experts of every token and the order by expert, from logits (tokens,
    num_experts).  Equal logits: the lower expert first; a logit of -inf is never chosen, so masking
    a token's whole row leaves it without an expert (weight 0, zero rows).  ``normalize``: weights are
    the softmax over the chosen logits, else the chosen entries of the softmax over all of them."""
    if _tracks(logits):
        return ExpertRoute(*_Route.apply(logits, int(top_k), bool(normalize)))
    return ExpertRoute(*token_ops.expert_route(logits, top_k, normalize))


class _Dispatch(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, slots, offsets):
        ctx.save_for_backward(slots, offsets)
        return token_ops.expert_dispatch(x, slots, offsets)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_sorted):
        slots, offsets = ctx.saved_tensors
        return token_ops.expert_combine(grad_sorted, slots, offsets), None, None


def _flat(t: torch.Tensor, name: str):
    if t.dim() < 2:
        raise ValueError(f"{name} must be (rows, ...); got {tuple(t.shape)}")
    return t if t.dim() == 2 else t.flatten(1)


def expert_dispatch(x: torch.Tensor, route: ExpertRoute) -> torch.Tensor:
    """Token rows x (tokens, ...) -> (tokens * top_k, ...) in the order by expert; zeros where a pair
    has no expert.  The gradient sums the copies of a token."""
    rows = _flat(x, "x")
    if _tracks(x):
        out = _Dispatch.apply(rows, route.slots, route.offsets)
    else:
        out = token_ops.expert_dispatch(rows, route.slots, route.offsets)
    return out if x.dim() == 2 else out.view(out.shape[0], *x.shape[1:])


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, weights, slots, offsets):
        ctx.save_for_backward(y, weights, slots, offsets)
        return token_ops.expert_combine(y, slots, offsets, weights)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out):
        y, weights, slots, offsets = ctx.saved_tensors
        gy, gw = token_ops.expert_combine_bwd(grad_out, y, slots, offsets, weights)
        return gy, gw, None, None


def expert_combine(y: torch.Tensor, route: ExpertRoute) -> torch.Tensor:
    """Rows y (tokens * top_k, ...) in the order by expert -> (tokens, ...): the sum over a token's
    choices of weight * row.  Differentiable in y and, through route.weights, in the logits."""
    rows = _flat(y, "y")
    if _tracks(y, route.weights):
        out = _Combine.apply(rows, route.weights, route.slots, route.offsets)
    else:
        out = token_ops.expert_combine(rows, route.slots, route.offsets, route.weights)
    return out if y.dim() == 2 else out.view(out.shape[0], *y.shape[1:])


class _ExpertLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, offsets, lvals):
        ctx.save_for_backward(x, weight, offsets)
        ctx.lvals = lvals
        return token_ops.expert_linear_fwd(x, weight, bias, offsets, lvals)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out):
        x, weight, offsets = ctx.saved_tensors
        need = ctx.needs_input_grad
        return (*token_ops.expert_linear_bwd(grad_out, x, weight, offsets, ctx.lvals, need[0], need[1], need[2]),
                None, None)


def expert_linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None, offsets: torch.Tensor,
                  lvals=(0,)) -> torch.Tensor:
    """Each expert's linear map on its rows offsets[e] .. offsets[e + 1) (rows past offsets[-1]: zeros).

    Plain rows: x (rows, c_in), weight (num_experts, c_out, c_in), bias (num_experts, c_out) or None.
    Equivariant rows: x (rows, dim, c_in) with dim = sum(2 l + 1) over ``lvals``, weight (num_experts,
    len(lvals), c_out, c_in), bias (num_experts, number of l = 0 irreps, c_out) on the l = 0
    components.  float32, bfloat16 or float16, one type for all; sums in float32."""
    if type(lvals) is not tuple:
        lvals = tuple(int(v) for v in lvals)
    if _tracks(x, weight, bias):
        return _ExpertLinear.apply(x, weight, bias, offsets, lvals)
    return token_ops.expert_linear_fwd(x, weight, bias, offsets, lvals)
