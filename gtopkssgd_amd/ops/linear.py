"""Linear layer with bias, activation and residual in its product's epilogue,
and its backward pass (csrc/linear.hip).

    y = act(x W^T + b) + residual
    p = dy act'(u),  u = x W^T + b
    dx = p W,  dW = p^T x,  db = sum of p over the rows,  dresidual = dy

For the backward pass the layer keeps x, W and, for gelu and silu, u (on the GPU
with more bits than the result: in fp16 beside bf16, in fp32 beside fp16); relu
keeps one bit a value.  ``act8=True`` keeps x and u in 8 bits (``act8``
module): half the memory, and gradients from what those stand for.  On the GPU
long 16-bit operands of wide products are copied to rows that start on lines of
128 bytes, and the backward pass uses the copy.
"""
from __future__ import annotations

from typing import Optional

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from . import _ext
from ._autocast import check_cast_leaves
from .act8 import _wide, act8_pack, act8_unpack

ACTS = {"none": 0, "relu": 1, "gelu": 2, "silu": 3}


def _act_code(act: str) -> int:
    if act not in ACTS:
        raise ValueError(f"unknown activation '{act}' (have {sorted(ACTS)})")
    return ACTS[act]


def _value(u: torch.Tensor, act: str) -> torch.Tensor:
    if act == "relu":
        return torch.relu(u)
    if act == "gelu":
        return u * 0.5 * (1.0 + torch.erf(u * 0.5 ** 0.5))
    if act == "silu":
        return u * torch.sigmoid(u)
    return u


def _slope(u: torch.Tensor, act: str) -> torch.Tensor:
    if act == "gelu":
        return 0.5 * (1.0 + torch.erf(u * 0.5 ** 0.5)) + \
            u * torch.exp(-0.5 * u * u) * 0.3989422804014327
    s = torch.sigmoid(u)
    return s * (1.0 + u * (1.0 - s))


class _LinearCPU(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act, act8):
        u = _wide(x) @ _wide(weight).t()
        if bias is not None:
            u = u + bias
        y = _value(u, act)
        if residual is not None:
            y = y + residual
        kept_x = act8_pack(x) if act8 else (x,)
        if act == "none":
            kept_u = ()
        elif act == "relu":
            kept_u = (~(u <= 0),)
        else:
            kept_u = act8_pack(u) if act8 else (u.to(x.dtype),)
        ctx.save_for_backward(weight, *kept_x, *kept_u)
        ctx.act, ctx.act8 = act, act8
        ctx.bias_type = None if bias is None else bias.dtype
        ctx.has_residual = residual is not None
        return y.to(x.dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        weight, *kept = ctx.saved_tensors
        n = 2 if ctx.act8 else 1
        x = act8_unpack(*kept[:2]) if ctx.act8 else _wide(kept[0])
        p = _wide(dy)
        if ctx.act == "relu":
            p = torch.where(kept[n], p, torch.zeros_like(p))
        elif ctx.act != "none":
            u = act8_unpack(*kept[n:]) if ctx.act8 else _wide(kept[n])
            p = p * _slope(u, ctx.act)
        flat = p.reshape(-1, p.size(-1))
        dx = (p @ _wide(weight)).to(dy.dtype)
        dw = (flat.t() @ x.reshape(-1, x.size(-1))).to(dy.dtype)
        db = None if ctx.bias_type is None else flat.sum(0).to(ctx.bias_type)
        return dx, dw, db, dy if ctx.has_residual else None, None, None


def linear_act(x: torch.Tensor, weight: torch.Tensor,
               bias: Optional[torch.Tensor] = None,
               residual: Optional[torch.Tensor] = None, act: str = "none",
               act8: bool = False) -> torch.Tensor:
    """``act(x weight^T + bias) + residual``.

    x: [..., in], weight: [out, in], residual: [..., out], of one type (bf16,
    fp16 or fp32); bias: [out] of that type or fp32.  act: "none", "relu",
    "gelu" (the exact one) or "silu".  Sums are fp32, the result is rounded
    once.  Under autocast x, weight and residual are cast to its type.  No
    second derivative; on the GPU forward mode, torch.func's transforms and
    tracing are refused."""
    code = _act_code(act)
    if x.is_cuda:
        if torch.is_autocast_enabled("cuda"):
            check_cast_leaves(x, weight, bias, residual)
            t = torch.get_autocast_dtype("cuda")
            x, weight = x.to(t), weight.to(t)
            residual = None if residual is None else residual.to(t)
            if bias is not None and bias.dtype != torch.float32:
                bias = bias.to(t)
        return _ext().linear_act(x, weight, bias, residual, code, bool(act8))
    if weight.dim() != 2 or x.dim() < 1 or weight.size(1) != x.size(-1) or \
            weight.numel() == 0:
        raise RuntimeError(f"weight must have shape [out, {x.shape[-1:]}], "
                           f"got {list(weight.shape)}")
    if bias is not None and tuple(bias.shape) != (weight.size(0),):
        raise RuntimeError(f"bias must have shape [{weight.size(0)}], got "
                           f"{list(bias.shape)}")
    want = (*x.shape[:-1], weight.size(0))
    if residual is not None and tuple(residual.shape) != want:
        raise RuntimeError(f"residual must have the output's shape {want}, "
                           f"got {tuple(residual.shape)}")
    return _LinearCPU.apply(x, weight, bias, residual, act, bool(act8))


class FusedLinearAct(nn.Linear):
    """``nn.Linear`` (same state_dict) with activation and residual."""

    def __init__(self, in_features: int, out_features: int, bias: bool = True,
                 act: str = "none", act8: bool = False, **kwargs):
        super().__init__(in_features, out_features, bias=bias, **kwargs)
        _act_code(act)
        self.act = act
        self.act8 = act8

    def forward(self, x: torch.Tensor,
                residual: Optional[torch.Tensor] = None) -> torch.Tensor:
        return linear_act(x, self.weight, self.bias, residual, self.act,
                          self.act8)
