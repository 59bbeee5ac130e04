"""Layer norm on HIP kernels, with first and second derivatives.

y = (x - mean) / sqrt(var + eps) * weight + bias over the last axis, as the scalar
node features and the radial layers of a potential take it.  A loss on forces
differentiates the row gradient once more: that gradient has a kernel of its own
(ictc_layer_norm_bwd2), so both backward passes read every row once.
"""
from __future__ import annotations

import torch

from ictc_o3 import _native as nat

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _rows(t):
    """t [N, C] itself, or a copy, with unit column stride and a row pitch of at least C."""
    if t.is_contiguous():
        return t
    if (t.stride(1) == 1 or t.shape[1] == 1) and (t.stride(0) >= t.shape[1] or t.shape[0] <= 1):
        return t
    return t.contiguous()


def _param(t):
    return t if t is None or t.is_contiguous() else t.contiguous()


def _pitch(t):
    return max(t.stride(0), t.shape[1])   # (a single row's stride may be anything)


def _forward(x, weight, bias, eps):
    x, weight, bias = _rows(x), _param(weight), _param(bias)
    N, C = x.shape
    y = torch.empty((N, C), dtype=x.dtype, device=x.device)
    stats = torch.empty((2, N), dtype=torch.float32, device=x.device)   # the rows' mean and 1 / deviation
    at = stats.data_ptr()
    nat.call("ictc_layer_norm_fwd", DTYPES[x.dtype], x.data_ptr(), _pitch(x), N, C, nat.ptr(weight), nat.ptr(bias), eps,
             y.data_ptr(), at, at + 4 * N, nat.stream_of(x))
    return y, stats


def _workspace(x):
    nbytes = nat.lib().ictc_layer_norm_workspace_bytes(DTYPES[x.dtype], x.shape[0], x.shape[1])
    return torch.empty(nbytes // 4, dtype=torch.float32, device=x.device), nbytes


def _backward(x, weight, g, stats, need_x, need_w, need_b):
    x, weight, g = _rows(x), _param(weight), _rows(g)
    N, C = x.shape
    dx = torch.empty((N, C), dtype=x.dtype, device=x.device) if need_x else None
    dw = torch.empty(C, dtype=x.dtype, device=x.device) if need_w else None
    db = torch.empty(C, dtype=x.dtype, device=x.device) if need_b else None
    ws, nbytes = _workspace(x) if need_w or need_b else (None, 0)
    at = stats.data_ptr()
    nat.call("ictc_layer_norm_bwd", DTYPES[x.dtype], x.data_ptr(), _pitch(x), g.data_ptr(), _pitch(g), N, C,
             nat.ptr(weight), at, at + 4 * N, nat.ptr(dx), nat.ptr(dw), nat.ptr(db), nat.ptr(ws), nbytes,
             nat.stream_of(x))
    return dx, dw, db


def _backward2(x, weight, g, vx, vw, vb, stats, need_x, need_w, need_g):
    v = _rows(torch.zeros_like(x) if vx is None else vx)
    x, weight, g, vw, vb = _rows(x), _param(weight), _rows(g), _param(vw), _param(vb)
    N, C = x.shape
    dx = x.new_empty(N, C) if need_x else None
    dg = x.new_empty(N, C) if need_g else None
    dw = x.new_empty(C) if need_w else None
    ws, nbytes = _workspace(x) if need_w else (None, 0)
    at = stats.data_ptr()
    nat.call("ictc_layer_norm_bwd2", DTYPES[x.dtype], nat.ptr(x), _pitch(x), nat.ptr(g), _pitch(g), nat.ptr(v),
             _pitch(v), nat.ptr(vw), nat.ptr(vb), N, C, nat.ptr(weight), at, at + 4 * N, nat.ptr(dx),
             nat.ptr(dg), nat.ptr(dw), nat.ptr(ws), nbytes, nat.stream_of(x))
    return dx, dw, dg


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, stats = _forward(x, weight, bias, eps)
        ctx.save_for_backward(x, weight, stats)
        return y

    @staticmethod
    def backward(ctx, g):
        x, weight, stats = ctx.saved_tensors
        needs = ctx.needs_input_grad
        if torch.is_grad_enabled():   # the gradient will be differentiated
            return (*_LayerNormGrad.apply(x, weight, g, stats, *needs[:3]), None)
        return (*_backward(x, weight, g, stats, *needs[:3]), None)


class _LayerNormGrad(torch.autograd.Function):
    """(dx, dweight, dbias) as functions of x, weight and the output gradient g."""

    @staticmethod
    def forward(ctx, x, weight, g, stats, need_x, need_w, need_b):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, weight, g, stats)
        return _backward(x, weight, g, stats, need_x, need_w, need_b)

    @staticmethod
    def backward(ctx, vx, vw, vb):
        x, weight, g, stats = ctx.saved_tensors
        needs = ctx.needs_input_grad[:3]
        if vx is None and vw is None and vb is None:
            return (None,) * 7
        if torch.is_grad_enabled():
            return (*_LayerNormGrad2.apply(x, weight, g, vx, vw, vb, stats, *needs), *(None,) * 4)
        return (*_backward2(x, weight, g, vx, vw, vb, stats, *needs), *(None,) * 4)


class _LayerNormGrad2(torch.autograd.Function):
    """The second derivative as a node of the graph, so that a third one raises wherever it would pass here."""

    @staticmethod
    def forward(ctx, x, weight, g, vx, vw, vb, stats, need_x, need_w, need_g):
        return _backward2(x, weight, g, vx, vw, vb, stats, need_x, need_w, need_g)

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError("layer_norm: third derivatives are not supported")


def layer_norm(x: torch.Tensor, weight=None, bias=None, eps: float = 1e-5) -> torch.Tensor:
    if x.dim() == 2:
        return _LayerNorm.apply(x, weight, bias, eps)
    return _LayerNorm.apply(x.reshape(-1, x.shape[-1]), weight, bias, eps).view(x.shape)
