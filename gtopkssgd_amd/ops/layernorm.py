"""Layer norm with its backward pass (csrc/layernorm.hip).

    y  = (x - mean) rstd weight + bias,  rstd = 1 / sqrt(var + eps)
    dx = rstd (g - mean(g) - xh mean(g xh)),  g = dy weight, xh = (x - mean) rstd
    dweight = sum of dy xh over the rows,  dbias = sum of dy

On the GPU each direction reads its inputs once; the weight's and bias's
gradients are summed in the same pass, in a fixed order.  With ``act8=True``
the input is kept in 8 bits for the backward pass (``act8`` module).
"""
from __future__ import annotations

from typing import Optional

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from . import _ext
from .act8 import _wide, act8_pack, act8_unpack


class _NormCPU(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, act8):
        v = _wide(x)
        mean = v.mean(-1, keepdim=True)
        rstd = torch.rsqrt((v - mean).square().mean(-1, keepdim=True) + eps)
        y = (v - mean) * rstd
        if weight is not None:
            y = y * weight
        if bias is not None:
            y = y + bias
        kept = act8_pack(x) if act8 else (x,)
        ctx.save_for_backward(weight, bias, mean, rstd, *kept)
        return y.to(x.dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        weight, bias, mean, rstd, *kept = ctx.saved_tensors
        x = act8_unpack(*kept) if len(kept) == 2 else _wide(kept[0])
        xh = (x - mean) * rstd
        d = _wide(dy)
        g = d if weight is None else d * weight
        dx = rstd * (g - g.mean(-1, keepdim=True) -
                     xh * (g * xh).mean(-1, keepdim=True))
        rows = tuple(range(dy.dim() - 1))
        dw = None if weight is None else \
            (d * xh).sum(rows).to(weight.dtype) if rows else d * xh
        db = None if bias is None else \
            d.sum(rows).to(bias.dtype) if rows else d
        return dx.to(dy.dtype), dw, db, None, None


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None,
               bias: Optional[torch.Tensor] = None, eps: float = 1e-5,
               act8: bool = False) -> torch.Tensor:
    """Layer norm over the last dimension, any length from 1 on.

    x: bf16, fp16 or fp32, any leading dimensions and strides.
    weight, bias: [x.size(-1)], both of x's type or both fp32; either may be
    None.  The result has x's type; statistics and sums are fp32.  No second
    derivative; on the GPU forward mode, torch.func's transforms and tracing
    are refused."""
    if x.is_cuda:
        return _ext().layer_norm(x, weight, bias, float(eps), bool(act8))
    if x.dim() < 1 or x.size(-1) == 0:
        raise RuntimeError("layer_norm needs a last dimension, got "
                           f"{tuple(x.shape)}")
    for name, p in (("weight", weight), ("bias", bias)):
        if p is not None and tuple(p.shape) != (x.size(-1),):
            raise RuntimeError(f"{name} must have shape [{x.size(-1)}], got "
                               f"{list(p.shape)}")
    return _NormCPU.apply(x, weight, bias, float(eps), bool(act8))


class FusedLayerNorm(nn.LayerNorm):
    """``nn.LayerNorm`` over one dimension (same state_dict) through
    ``layer_norm``."""

    def __init__(self, dim: int, eps: float = 1e-5, act8: bool = False,
                 **kwargs):
        super().__init__(dim, eps=eps, **kwargs)
        if len(self.normalized_shape) != 1:
            raise ValueError("FusedLayerNorm takes one dimension, got "
                             f"{self.normalized_shape}")
        self.act8 = act8

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return layer_norm(x, self.weight, self.bias, self.eps, self.act8)
