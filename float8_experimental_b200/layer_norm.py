"""Layer norm over the last dimension, forward and backward on the sm_100a kernels.

`layer_norm(x, weight, bias, eps)` computes what `torch.nn.functional.layer_norm` does over the last dimension:
the moments, the normalised values and every sum in fp32, the results rounded once.  `LayerNorm` is the module.
Like RMSNorm (`fused_norm.py`) it is what stands in front of a `Float8Linear`
(float8_experimental/benchmarks/profile_linear_float8.py:129-149 has the reference's form of that).
"""
from __future__ import annotations

from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import _native as N
from ._ops import _layer_norm_bwd_cuda, _layer_norm_cuda, eager_cuda, layer_norm_into, ops

__all__ = ["layer_norm", "LayerNorm"]


class _LayerNormFunc(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        forward = _layer_norm_cuda if eager_cuda(x) else ops.layer_norm
        y, mean, rstd = forward(x, weight, bias, eps, True)
        ctx.save_for_backward(x, weight, mean, rstd)
        ctx.affine_dtype = next((t.dtype for t in (weight, bias) if t is not None), x.dtype)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        x, weight, mean, rstd = ctx.saved_tensors
        need = ctx.needs_input_grad[:3]
        backward = _layer_norm_bwd_cuda if eager_cuda(x) else ops.layer_norm_bwd
        grads = backward(x, g, weight, mean, rstd, ctx.affine_dtype, *need)
        return (*[t if n else None for t, n in zip(grads, need)], None)


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5) -> torch.Tensor:
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dimension of `x` [..., D].

    `x` is bf16, fp16 or fp32; `weight` and `bias` [D] are optional and share x's dtype or are both float32.
    The result has x's dtype.  Differentiable once in x, weight and bias."""
    N.hp_code(x.dtype)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias)):
        return _LayerNormFunc.apply(x, weight, bias, float(eps))
    if eager_cuda(x):
        return layer_norm_into(x, weight, bias, float(eps), None, None)
    return ops.layer_norm(x, weight, bias, float(eps), False)[0]


class LayerNorm(torch.nn.LayerNorm):
    """`torch.nn.LayerNorm` over one dimension, on the kernels of this package: same arguments, same state."""

    def __init__(self, *args, **kwargs):
        super().__init__(*args, **kwargs)
        if len(self.normalized_shape) != 1:
            raise ValueError(f"LayerNorm: normalises the last dimension only, got {tuple(self.normalized_shape)}")

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if x.shape[-1] != self.normalized_shape[0]:
            raise RuntimeError(f"LayerNorm: the last dimension must be {self.normalized_shape[0]}, got {x.shape[-1]}")
        return layer_norm(x, self.weight, self.bias, self.eps)
