"""LayerNorm without an activation, for rows in fp32, bf16 or fp16 (``nn.LayerNorm(E)``; the world model's blocks use the form fused
with SiLU, lib/world_model.py:153-160).

``layer_norm`` is one kernel forward and two backward (the row pass, which also forms the column sums of the weight's and the
bias's gradient, and their sum over workgroups).  Statistics and sums are fp32 whatever the rows' type; results are rounded once.
Host tensors take the formula in tensor operations.
"""
from __future__ import annotations

from typing import Optional

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from . import _native as N


def _layer_norm_grads(ctx, dy):
    rows, weight, stats = ctx.saved_tensors
    need = ctx.needs_input_grad
    dx, dw, db = N.layer_norm_backward(rows, N.as_rows(dy), weight, stats, need[0], need[1], need[2], ctx.bias_dtype)
    return dx if dx is None or dy.dim() == 2 else dx.view(dy.shape), dw, db, None


_layer_norm_grads_once = once_differentiable(_layer_norm_grads)


class _LayerNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        rows = N.as_rows(x)
        y, stats = N.layer_norm_forward(rows, weight, bias, eps, True)
        ctx.save_for_backward(rows, weight, stats)
        ctx.bias_dtype = None if bias is None else bias.dtype
        return y if x.dim() == 2 else y.view(x.shape)

    @staticmethod
    def backward(ctx, dy):
        # (the wrapper that refuses a second differentiation is only needed where one could follow)
        return _layer_norm_grads_once(ctx, dy) if torch.is_grad_enabled() else _layer_norm_grads(ctx, dy)


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5) -> torch.Tensor:
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dimension of x (any leading shape; rows may be strided).

    x in fp32, bf16 or fp16; weight and bias (E,), or None, both in fp32 or both in x's type.  The result is dense, in x's type, and
    differentiable with respect to x, weight and bias (once)."""
    if x.dim() < 1 or x.shape[-1] < 1:
        raise N.NativeError(f"layer_norm: rows of at least one element, got shape {tuple(x.shape)}")
    if x.is_cuda:
        if weight is not None and not weight.is_contiguous():
            weight = weight.contiguous()
        if bias is not None and not bias.is_contiguous():
            bias = bias.contiguous()
        if N.wants_grad(x, weight, bias):
            return _LayerNormFn.apply(x, weight, bias, float(eps))
        y, _ = N.layer_norm_forward(N.as_rows(x), weight, bias, float(eps), False)
        return y if x.dim() == 2 else y.view(x.shape)
    N.dtype_id(x, "x")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None and (t.shape != x.shape[-1:] or t.dtype not in (torch.float32, x.dtype) or t.device != x.device):
            raise N.NativeError(f"layer_norm: {name} {tuple(t.shape)} {t.dtype} on {t.device} does not fit rows {tuple(x.shape)} {x.dtype}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise N.NativeError(f"layer_norm: weight is {weight.dtype}, bias {bias.dtype}")
    v = x.float()
    c = v - v.mean(-1, keepdim=True)
    y = c * torch.rsqrt(c.square().mean(-1, keepdim=True) + eps)
    y = y if weight is None else y * weight.float()
    return (y if bias is None else y + bias.float()).to(x.dtype)


class LayerNorm(nn.LayerNorm):
    """``nn.LayerNorm`` over the last dimension (same parameters and state-dict keys) on ``layer_norm``; parameters may stay in
    fp32 while the rows are bf16 or fp16."""

    def __init__(self, normalized_shape, eps: float = 1e-5, elementwise_affine: bool = True, bias: bool = True, device=None, dtype=None):
        super().__init__(normalized_shape, eps, elementwise_affine, bias, device, dtype)
        if len(self.normalized_shape) != 1:
            raise ValueError(f"LayerNorm normalises the last dimension only, got normalized_shape={tuple(self.normalized_shape)}")

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if x.shape[-1:] != tuple(self.normalized_shape):
            raise ValueError(f"LayerNorm over {self.normalized_shape[0]} elements got rows of {x.shape[-1] if x.dim() else 0}")
        return layer_norm(x, self.weight, self.bias, self.eps)
