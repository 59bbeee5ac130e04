"""Linears chosen per row by an expert id (an atom's element), for any widths, in FP32, bfloat16 or FP16.

  y[n] = W[id n] x[n] + b[id n]      W [experts, outputs, inputs], b [experts, outputs]

The rows' order by expert is made once per batch (``expert_order``) and shared by every layer and both passes.  The
adjoints are the same two products with their roles exchanged, so the operator is differentiable to any order (a loss
on forces differentiates it twice).  Checks, allocations and autograd nodes are in csrc/torch_ops.cpp.
"""
from __future__ import annotations

import torch

from ictc_o3 import _native as nat


class ExpertOrder:
    """Rows in the order of their expert: perm [rows] int32 row numbers sorted by expert (stable), offsets
    [experts + 2] int32 with expert e at sorted rows offsets[e] .. offsets[e + 1] and the rows whose id is outside
    [0, experts) last."""

    __slots__ = ("perm", "offsets", "rows", "experts")

    def __init__(self, ids: torch.Tensor, experts: int):
        self.perm, self.offsets = nat.ops().expert_order(ids, experts)
        self.rows, self.experts = ids.shape[0], experts
