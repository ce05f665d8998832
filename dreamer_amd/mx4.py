"""Microscaled 4-bit matrices: blocks of 32 elements along a row, each a 4-bit float (1 sign, 2 exponent, 1 mantissa bit) times
the block's power of two.  ``quantize`` makes them, ``linear`` multiplies with them: the Linear layers of lib/world_model.py:153-160
with weights of 4.25 bits, for acting (few rows: the weight is streamed once) and for training what lies in front of a frozen
layer (input and bias gradients).
"""
from __future__ import annotations

from typing import Optional, Union

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from . import _native as N

BLOCK = 32


class MX4Tensor:
    """A matrix (rows, columns) in 4 bits on the device.

    codes: uint8 (rows, nb * 16), nb = ceil(columns / 32): element 2i of a block in the low half of its byte i, element 2i + 1 in the
    high half; bit 3 is the sign, bits 0-2 number 0, 0.5, 1, 1.5, 2, 3, 4, 6; codes behind the last column are 0.
    scales: uint8 (rows, nb): byte s stands for 2**(s - 127), 255 for a block of NaN.
    """

    __slots__ = ("codes", "scales", "columns")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, columns: int):
        N._mx4_operand(codes, scales, int(columns), "MX4Tensor")
        self.codes, self.scales, self.columns = codes, scales, int(columns)

    @classmethod
    def _of(cls, codes: torch.Tensor, scales: torch.Tensor, columns: int) -> "MX4Tensor":
        """From tensors that are known to fit (the quantisation's own)."""
        t = cls.__new__(cls)
        t.codes, t.scales, t.columns = codes, scales, columns
        return t

    @property
    def shape(self) -> torch.Size:
        return torch.Size((self.codes.shape[0], self.columns))

    @property
    def device(self) -> torch.device:
        return self.codes.device

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The values as a float matrix (fp32 and bf16 hold them exactly, fp16 inside its range)."""
        return N.mx4_dequantize(self.codes, self.scales, self.columns, dtype)

    def __repr__(self) -> str:
        return f"MX4Tensor({self.codes.shape[0]} x {self.columns}, device={self.device})"


def quantize(x: torch.Tensor) -> MX4Tensor:
    """A float matrix (fp32, bf16 or fp16; leading dimensions are flattened to rows) in 4 bits: the block's scale is
    2**(floor(log2(max |x|)) - 2), elements go to the nearest value (ties to the even code), at most 6 scales.  Blocks that hold an
    infinity or NaN become NaN.  Not differentiable."""
    if x.dim() < 1 or x.shape[-1] < 1:
        raise N.NativeError(f"quantize: rows of at least one element, got shape {tuple(x.shape)}")
    rows = N.as_rows(x.detach())
    return MX4Tensor._of(*N.mx4_quantize(rows), rows.shape[1])


def _versions(codes: torch.Tensor, scales: torch.Tensor):
    """Counts of in-place writes (tensors made under inference_mode have none)."""
    return None if codes.is_inference() or scales.is_inference() else (codes._version, scales._version)


def _mx4_linear_grads(ctx, dy):
    rows = N.as_rows(dy)
    if ctx.versions != _versions(ctx.codes, ctx.scales):
        raise N.NativeError("linear: the 4-bit weight was written to between the product and its gradient")
    dx = db = None
    if ctx.needs_input_grad[0]:
        dx = N.mx4_linear_dgrad(rows, ctx.codes, ctx.scales, ctx.columns)
        dx = dx if dy.dim() == 2 else dx.view(*dy.shape[:-1], ctx.columns)
    if ctx.needs_input_grad[1]:
        db = N.mx4_bias_grad(rows, ctx.bias_dtype)
    return dx, db, None


_mx4_linear_grads_once = once_differentiable(_mx4_linear_grads)


class _MX4LinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, bias, weight):
        # the tensors of this product: the caller may put others into the MX4Tensor afterwards (kept as attributes, since tensors
        # made under inference_mode cannot be saved for backward)
        ctx.codes, ctx.scales, ctx.columns = weight.codes, weight.scales, weight.columns
        ctx.versions = _versions(ctx.codes, ctx.scales)
        ctx.bias_dtype = None if bias is None else bias.dtype
        y = N.mx4_linear(N.as_rows(x), weight.codes, weight.scales, bias)
        return y if x.dim() == 2 else y.view(*x.shape[:-1], weight.codes.shape[0])

    @staticmethod
    def backward(ctx, dy):
        # (the wrapper that refuses a second differentiation is only needed where one could follow)
        return _mx4_linear_grads_once(ctx, dy) if torch.is_grad_enabled() else _mx4_linear_grads(ctx, dy)


def _mx4_product_grad(ctx, dy):
    return N.mx4_bias_grad(N.as_rows(dy), ctx.bias_dtype), None, None, None


_mx4_product_grad_once = once_differentiable(_mx4_product_grad)


class _MX4ProductFn(torch.autograd.Function):
    """The product of rows and weight that are both in 4 bits, for the gradient of its bias."""

    @staticmethod
    def forward(ctx, bias, x, weight, out_dtype):
        ctx.bias_dtype = bias.dtype
        return N.mx4_product(x.codes, x.scales, weight.codes, weight.scales, weight.columns, bias, out_dtype)

    @staticmethod
    def backward(ctx, dy):
        return _mx4_product_grad_once(ctx, dy) if torch.is_grad_enabled() else _mx4_product_grad(ctx, dy)


def linear(x: Union[torch.Tensor, MX4Tensor], weight: MX4Tensor, bias: Optional[torch.Tensor] = None,
           out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """x @ weight.T + bias for a weight (N, K) in 4 bits.

    x a float tensor (..., K), fp32 / bf16 / fp16: the result has x's type (``out_dtype`` may only repeat it); each product is exact,
    sums are fp32.  Differentiable with respect to x and bias (once); the weight is frozen.
    x an MX4Tensor (M, K): the result is (M, N) in ``out_dtype`` (default fp32); differentiable with respect to bias only (once).
    bias (N,) in any of the three types."""
    if not isinstance(weight, MX4Tensor):
        raise N.NativeError(f"linear: the weight must be an MX4Tensor, got {type(weight).__name__}")
    if isinstance(x, MX4Tensor):
        if x.columns != weight.columns:
            raise N.NativeError(f"linear: rows of {x.columns} elements, weight {tuple(weight.shape)}")
        if bias is not None:
            bias = bias if bias.is_contiguous() else bias.contiguous()
            if N.wants_grad(bias):
                return _MX4ProductFn.apply(bias, x, weight, out_dtype or torch.float32)
        return N.mx4_product(x.codes, x.scales, weight.codes, weight.scales, weight.columns, bias, out_dtype or torch.float32)
    if x.dim() < 1 or x.shape[-1] != weight.columns:
        raise N.NativeError(f"linear: rows {tuple(x.shape)}, weight {tuple(weight.shape)}")
    if out_dtype is not None and out_dtype != x.dtype:
        raise N.NativeError(f"linear: a product with {x.dtype} rows has {x.dtype} results, not {out_dtype}")
    if bias is not None and not bias.is_contiguous():
        bias = bias.contiguous()
    if N.wants_grad(x, bias):
        return _MX4LinearFn.apply(x, bias, weight)
    y = N.mx4_linear(N.as_rows(x), weight.codes, weight.scales, bias)
    return y if x.dim() == 2 else y.view(*x.shape[:-1], weight.codes.shape[0])


class MX4Linear(nn.Module):
    """A Linear layer whose frozen weight is held in 4 bits (``from_linear`` quantises one).  ``activations="mx4"`` also quantises
    the rows, without gradients; ``"float"`` (default) multiplies them as they are.  A layer of this kind works in models that are
    evaluated module by module; the rollout and the recurrence kernels (``imagine``, ``observe``) read float weights and refuse a
    model in which it stands for one of their Linears."""

    def __init__(self, weight: MX4Tensor, bias: Optional[torch.Tensor] = None, activations: str = "float"):
        super().__init__()
        if activations not in ("float", "mx4"):
            raise ValueError(f"MX4Linear: activations must be 'float' or 'mx4', got {activations!r}")
        self.in_features, self.out_features, self.activations = weight.columns, weight.codes.shape[0], activations
        self.register_buffer("codes", weight.codes)
        self.register_buffer("scales", weight.scales)
        self.bias = None if bias is None else nn.Parameter(bias.detach().clone())

    @classmethod
    def from_linear(cls, layer: nn.Linear, activations: str = "float") -> "MX4Linear":
        return cls(quantize(layer.weight), layer.bias, activations)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        w = MX4Tensor(self.codes, self.scales, self.in_features)
        if self.activations == "float":
            return linear(x, w, self.bias)
        if N.wants_grad(x, self.bias):
            raise N.NativeError("MX4Linear: products of quantised rows have no gradient; call under torch.no_grad()")
        return linear(quantize(x), w, self.bias, x.dtype).view(*x.shape[:-1], self.out_features)
