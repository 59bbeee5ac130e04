"""Layer norm on HIP kernels, with first and second derivatives.

y = (x - mean) / sqrt(var + eps) * weight + bias over the last axis, as the scalar
node features and the radial layers of a potential take it.  A loss on forces
differentiates the row gradient once more: that gradient has a kernel of its own
(ictc_layer_norm_bwd2), so both backward passes read every row once.  Checks,
allocations and autograd nodes are in csrc/torch_ops.cpp.
"""
from __future__ import annotations

import torch

from ictc_o3 import _native as nat


def layer_norm(x: torch.Tensor, weight=None, bias=None, eps: float = 1e-5) -> torch.Tensor:
    return nat.ops().layer_norm(x, weight, bias, eps)
