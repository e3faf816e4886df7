"""Layers of a residual block over typed rows: one Linear per node type, tissue or donor, and the norms, gate and residual around a block.

The reference applies one Linear to every node and leaves the ``norm`` of a layer to the caller (dance/models/nn/gnn.py:41-60,84-96;
scdeepsort.py:39-46).  ``TypedLinear`` stands beside ``autograd.HipLinear``; ``RowNorm`` fits the ``norm`` argument of scDeepSort's ``GNN`` and
the ``norm_layer`` of ``AdaptiveSAGE``.
"""
import math
from typing import Optional

import torch
import torch.nn as nn

from ..autograd import grouped_linear, residual_norm


def group_rows(types: torch.Tensor, n_types: int):
    """(order, group_ptr) of integer row types: ``order`` sorts rows by type (rows of one type keep their order), ``group_ptr`` int32
    [n_types + 1] are the types' bounds among the sorted rows.  Types below 0 or from ``n_types`` on belong to no group (they sort in front
    and behind).  Stays on the types' device."""
    if types.dim() != 1 or types.dtype.is_floating_point or types.dtype.is_complex or types.dtype == torch.bool:
        raise ValueError(f"types must be a 1-d integer tensor, got {tuple(types.shape)} of {types.dtype}")
    if n_types < 0:
        raise ValueError(f"n_types must not be negative, got {n_types}")
    ordered, order = torch.sort(types.to(torch.int64), stable=True)
    bounds = torch.arange(n_types + 1, device=types.device)
    return order, torch.searchsorted(ordered, bounds).to(torch.int32)


class TypedLinear(nn.Module):
    """``nn.Linear`` with one weight and bias per row type: rows group_ptr[t] <= i < group_ptr[t + 1] of the input take weight[t], bias[t]."""

    def __init__(self, in_features: int, out_features: int, n_types: int, bias: bool = True):
        super().__init__()
        self.in_features, self.out_features, self.n_types = in_features, out_features, n_types
        self.weight = nn.Parameter(torch.empty(n_types, out_features, in_features))
        self.bias = nn.Parameter(torch.empty(n_types, out_features)) if bias else None
        self.reset_parameters()

    def reset_parameters(self):  # torch.nn.Linear's, for every type
        bound = 1.0 / math.sqrt(self.in_features) if self.in_features > 0 else 0.0
        nn.init.uniform_(self.weight, -bound, bound)
        if self.bias is not None:
            nn.init.uniform_(self.bias, -bound, bound)

    def forward(self, input, group_ptr, fuse_relu: bool = False):
        return grouped_linear(input, self.weight, group_ptr, self.bias, relu=fuse_relu)

    def extra_repr(self):
        return f"in_features={self.in_features}, out_features={self.out_features}, n_types={self.n_types}, bias={self.bias is not None}"


class RowNorm(nn.Module):
    """Layer norm (``kind="layer"``) or RMS norm (``"rms"``) over the columns of a [N, dim] matrix, fp32 or bf16 rows, fp32 parameters."""

    def __init__(self, dim: int, kind: str = "layer", eps: float = 1e-5, affine: bool = True):
        super().__init__()
        self.dim, self.kind, self.eps = dim, kind, eps
        self.weight = nn.Parameter(torch.ones(dim)) if affine else None
        self.bias = nn.Parameter(torch.zeros(dim)) if affine and kind == "layer" else None

    def forward(self, input):
        return residual_norm(input, None, post=(self.weight, self.bias), kind=self.kind, eps=self.eps)[0]

    def extra_repr(self):
        return f"{self.dim}, kind={self.kind!r}, eps={self.eps}"


class GatedResidualNorm(nn.Module):
    """(r, h) = (x + scale * act(gate) * norm(f), norm(r)) between two blocks; see ``autograd.residual_norm``.

    ``post`` / ``pre`` switch the two norms, each with its own parameters.  ``gate``: "channel" or "scalar" (a parameter that starts at one,
    or at zero behind a sigmoid), or None: then ``forward`` may be given one, [N, 1] or [N, dim]."""

    def __init__(self, dim: int, *, post: bool = True, pre: bool = True, gate: Optional[str] = "channel", gate_act: str = "none",
                 scale: float = 1.0, kind: str = "layer", eps: float = 1e-5):
        super().__init__()
        if gate not in (None, "scalar", "channel"):
            raise ValueError(f"gate must be None, 'scalar' or 'channel', got {gate!r}")
        self.dim, self.gate_act, self.scale, self.kind, self.eps = dim, gate_act, scale, kind, eps
        self.has_post, self.has_pre = post, pre
        bias = kind == "layer"
        self.post_weight = nn.Parameter(torch.ones(dim)) if post else None
        self.post_bias = nn.Parameter(torch.zeros(dim)) if post and bias else None
        self.pre_weight = nn.Parameter(torch.ones(dim)) if pre else None
        self.pre_bias = nn.Parameter(torch.zeros(dim)) if pre and bias else None
        start = torch.zeros if gate_act == "sigmoid" else torch.ones
        self.gate = None if gate is None else nn.Parameter(start(1 if gate == "scalar" else dim))

    def forward(self, f, x=None, gate=None):
        if gate is not None and self.gate is not None:
            raise ValueError("GatedResidualNorm: a gate was given to a module that has its own")
        return residual_norm(f, x, post=(self.post_weight, self.post_bias) if self.has_post else None, gate=self.gate if gate is None else gate,
                             gate_act=self.gate_act, scale=self.scale, pre=(self.pre_weight, self.pre_bias) if self.has_pre else None,
                             kind=self.kind, eps=self.eps)

    def extra_repr(self):
        return f"{self.dim}, kind={self.kind!r}, gate_act={self.gate_act!r}, scale={self.scale}, eps={self.eps}"
