"""Linears chosen per row by an expert id (an atom's element), for any widths, in FP32, bfloat16 or FP16.

  y[n] = W[id n] x[n] + b[id n]      W [experts, outputs, inputs], b [experts, outputs]

The rows' order by expert is made once per batch (``expert_order``) and shared by every layer and both passes.  The
adjoints are the same two products with their roles exchanged, so the operator is differentiable to any order (a loss
on forces differentiates it twice).
"""
from __future__ import annotations

import torch

from ictc_o3 import _native as nat
from ictc_o3.ops.layer_norm import DTYPES
from ictc_o3.ops.tensor_product import Csr


class ExpertOrder:
    """Rows in the order of their expert: perm [rows] int32 row numbers sorted by expert (stable), offsets
    [experts + 2] int32 with expert e at sorted rows offsets[e] .. offsets[e + 1] and the rows whose id is outside
    [0, experts) last."""

    def __init__(self, ids: torch.Tensor, experts: int):
        csr = Csr(ids if ids.is_contiguous() else ids.contiguous(), experts)
        self.perm, self.offsets, self.rows, self.experts = csr.order, csr.ptr, ids.shape[0], experts
        self.device = ids.device


def _rows(t):
    """t [N, C] itself, or a copy, with unit column stride and a row pitch of at least C."""
    if t.is_contiguous() or ((t.stride(1) == 1 or t.shape[1] == 1) and (t.stride(0) >= t.shape[1] or t.shape[0] <= 1)):
        return t
    return t.contiguous()


def _pitch(t):
    return max(t.stride(0), t.shape[1])


def _c(t):
    return t if t is None or t.is_contiguous() else t.contiguous()


def _linear(x, W, b, order, trans):
    x, W, b = _rows(x), _c(W), _c(b)
    outputs = W.shape[2] if trans else W.shape[1]
    out = torch.empty((x.shape[0], outputs), dtype=x.dtype, device=x.device)
    nat.call("ictc_expert_linear", DTYPES[x.dtype], x.data_ptr(), _pitch(x), x.shape[0], x.shape[1], W.data_ptr(),
             nat.ptr(b), outputs, order.experts, order.perm.data_ptr(), order.offsets.data_ptr(), 1 if trans else 0,
             out.data_ptr(), nat.stream_of(x))
    return out


def _outer(g, x, order, need_b):
    g, x = _rows(g), _rows(x)
    N, M, K, E, dtype = x.shape[0], g.shape[1], x.shape[1], order.experts, DTYPES[x.dtype]
    gW = torch.empty((E, M, K), dtype=x.dtype, device=x.device)
    gb = torch.empty((E, M), dtype=x.dtype, device=x.device) if need_b else None
    nbytes = nat.lib().ictc_expert_outer_workspace_bytes(dtype, N, K, M, E)
    ws = torch.empty(nbytes // 4, dtype=torch.float32, device=x.device) if nbytes else None
    nat.call("ictc_expert_outer", dtype, g.data_ptr(), _pitch(g), x.data_ptr(), _pitch(x), N, K, M, E,
             order.perm.data_ptr(), order.offsets.data_ptr(), gW.data_ptr(), nat.ptr(gb), nat.ptr(ws), nbytes,
             nat.stream_of(x))
    return gW, gb


class _ExpertLinear(torch.autograd.Function):
    """y[n] = W[e] x[n] + b[e], or with trans W[e]^T x[n]."""

    @staticmethod
    def forward(ctx, x, W, b, order, trans):
        ctx.order, ctx.trans = order, trans
        ctx.save_for_backward(x, W)
        return _linear(x, W, b, order, trans)

    @staticmethod
    def backward(ctx, g):
        x, W = ctx.saved_tensors
        order, trans = ctx.order, ctx.trans
        need_x, need_W, need_b = ctx.needs_input_grad[:3]
        again = torch.is_grad_enabled()   # the gradient will be differentiated
        dx = dW = db = None
        if need_x:
            dx = _ExpertLinear.apply(g, W, None, order, not trans) if again else _linear(g, W, None, order, not trans)
        if need_W or need_b:
            a, b = (x, g) if trans else (g, x)
            dW, db = _ExpertOuter.apply(a, b, order, need_b) if again else _outer(a, b, order, need_b)
        return dx, dW if need_W else None, db, None, None


class _ExpertOuter(torch.autograd.Function):
    """(sum over an expert's rows of g[n] x[n]^T, sum of g[n]) per expert."""

    @staticmethod
    def forward(ctx, g, x, order, need_b):
        ctx.set_materialize_grads(False)
        ctx.order = order
        ctx.save_for_backward(g, x)
        return _outer(g, x, order, need_b)

    @staticmethod
    def backward(ctx, H, h):
        g, x = ctx.saved_tensors
        order = ctx.order
        if H is None and h is None:
            return None, None, None, None
        if H is None:   # (the bias gradient alone was used)
            H = torch.zeros((order.experts, g.shape[1], x.shape[1]), dtype=x.dtype, device=x.device)
        dg = _ExpertLinear.apply(x, H, h, order, False) if ctx.needs_input_grad[0] else None
        dx = _ExpertLinear.apply(g, H, None, order, True) if ctx.needs_input_grad[1] else None
        return dg, dx, None, None


def expert_linear(x: torch.Tensor, weight: torch.Tensor, order: ExpertOrder, bias=None) -> torch.Tensor:
    return _ExpertLinear.apply(x, weight, bias, order, False)
