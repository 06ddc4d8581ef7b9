"""Mixture-of-experts feed-forward on equivariant node features (no counterpart in the reference).

Each node is routed by its invariants to ``top_k`` of ``num_experts`` experts and gets the weighted
sum of their outputs: layer norm of the irrep norms -> router logits -> choice; the rows (N, dim, C)
sorted by expert -> per-irrep linear maps to a wider multiplicity -> gate by the l = 0 channels ->
linear maps back -> weighted sum per node.  The router sees invariants only and every
step after it acts on channels, so the layer is equivariant.  The experts' row counts stay on the
device: no step synchronises the host, forward or backward.
"""
from __future__ import annotations

import torch
import torch.nn as nn

from ..cuda.token_autograd import expert_combine, expert_dispatch, expert_linear, expert_route
from ..representations import Repr
from .norm import InvariantLayerNorm, RepNorm


class EquivariantExperts(nn.Module):
    """(N, C, dim) -> (N, C, dim): ``top_k`` of ``num_experts`` gated equivariant MLPs per node."""

    def __init__(self, repr: Repr, num_experts: int, top_k: int = 2, mlp_ratio: int = 2, normalize: bool = True) -> None:
        super().__init__()
        nscalar, locs = repr.find_scalar()
        if nscalar == 0:
            raise ValueError("EquivariantExperts gates by the l = 0 channels; "
                             f"lvals {repr.lvals.tolist()} have no l = 0")
        if not 1 <= top_k <= num_experts:
            raise ValueError(f"top_k must be in [1, num_experts = {num_experts}]; got {top_k}")
        self.repr, self.num_experts, self.top_k, self.normalize = repr, num_experts, top_k, normalize
        self.lvals = tuple(repr.lvals.tolist())
        self.hidden = repr.mult * mlp_ratio
        self._gate_at = int(locs[0])
        reps, c, h = repr.nreps(), repr.mult, self.hidden
        self.invariants = RepNorm(repr)
        self.router_norm = InvariantLayerNorm(reps * c)
        self.router = nn.Linear(reps * c, num_experts, bias=False)
        self.weight_up = nn.Parameter(torch.empty(num_experts, reps, h, c))
        self.bias_up = nn.Parameter(torch.zeros(num_experts, nscalar, h))
        self.weight_down = nn.Parameter(torch.empty(num_experts, reps, c, h))
        self.bias_down = nn.Parameter(torch.zeros(num_experts, nscalar, c))
        nn.init.xavier_uniform_(self.router.weight)
        for w in (self.weight_up, self.weight_down):        # as EquivariantLinear, expert by expert
            for expert in w.detach():
                nn.init.xavier_uniform_(expert.view(-1, expert.shape[-1]))

    def route(self, x: torch.Tensor, mask: torch.Tensor | None = None):
        """The plan for nodes x (N, C, dim); nodes where ``mask`` (N,) is False get no expert."""
        logits = self.router(self.router_norm(self.invariants(x).flatten(-2, -1)))
        if mask is not None:
            logits = logits.masked_fill(~mask.unsqueeze(-1), float("-inf"))
        return expert_route(logits, self.top_k, self.normalize)

    def forward(self, x: torch.Tensor, mask: torch.Tensor | None = None) -> torch.Tensor:
        if x.dim() != 3 or x.shape[1] != self.repr.mult or x.shape[2] != self.repr.dim():
            raise ValueError(f"expected (N, {self.repr.mult}, {self.repr.dim()}) features; got {tuple(x.shape)}")
        plan = self.route(x, mask)
        rows = expert_dispatch(x.transpose(1, 2).contiguous(), plan)                 # (N k, dim, C)
        h = expert_linear(rows, self.weight_up, self.bias_up, plan.offsets, self.lvals)
        h = h * torch.sigmoid(h[:, self._gate_at:self._gate_at + 1])
        y = expert_linear(h, self.weight_down, self.bias_down, plan.offsets, self.lvals)
        return expert_combine(y, plan).transpose(1, 2).contiguous()

    def extra_repr(self) -> str:
        return f"repr={self.repr}, num_experts={self.num_experts}, top_k={self.top_k}, hidden={self.hidden}"
