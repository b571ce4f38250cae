"""The pre-norm feed-forward block, one autograd function over the layer norm,
the two products and the 8-bit form:

    y = x + W2 act(W1 norm(x) + b1) + b2

What goes from one operator to the next, in both directions, has x's type.  The
backward pass takes the gradient through the activation in the epilogue of the
product that makes it, and adds dy onto the norm's gradient in the norm's own
pass.  With ``act8=True`` the inputs of the norm and of both products and the
value before the activation are kept in 8 bits.
"""
from __future__ import annotations

from typing import Optional

import torch
import torch.nn as nn
import torch.nn.functional as F
from torch.nn.modules import module as _module

from . import _ext
from ._autocast import check_cast_leaves
from .layernorm import FusedLayerNorm, layer_norm
from .linear import FusedLinearAct, _act_code, linear_act


def ffn_block(x: torch.Tensor, norm_weight: Optional[torch.Tensor],
              norm_bias: Optional[torch.Tensor], w1: torch.Tensor,
              b1: Optional[torch.Tensor], w2: torch.Tensor,
              b2: Optional[torch.Tensor], act: str = "gelu",
              eps: float = 1e-5, act8: bool = False) -> torch.Tensor:
    """``x + w2 act(w1 norm(x) + b1) + b2``.

    x: [..., dim], w1: [hidden, dim], w2: [dim, hidden], of one type (bf16,
    fp16 or fp32); norm_weight, norm_bias: [dim], b1: [hidden], b2: [dim], of
    that type or fp32, or None.  Under autocast x, w1 and w2 are cast to its
    type, and with x the residual: y has that type, too, as a linear layer's
    result; a residual of fp32 needs the block in fp32, outside autocast.  No
    second derivative; on the GPU forward mode, torch.func's transforms and
    tracing are refused."""
    code = _act_code(act)
    if x.is_cuda:
        if torch.is_autocast_enabled("cuda"):
            check_cast_leaves(x, norm_weight, norm_bias, w1, b1, w2, b2)
            t = torch.get_autocast_dtype("cuda")
            x, w1, w2 = x.to(t), w1.to(t), w2.to(t)
            norm_weight, norm_bias, b1, b2 = (
                p if p is None or p.dtype == torch.float32 else p.to(t)
                for p in (norm_weight, norm_bias, b1, b2))
        return _ext().ffn_block(x, norm_weight, norm_bias, w1, b1, w2, b2,
                                code, float(eps), bool(act8))
    if w1.dim() != 2 or w2.dim() != 2 or w2.size(0) != x.size(-1):
        raise RuntimeError(f"w2 must have shape [{x.size(-1)}, hidden], got "
                           f"{list(w2.shape)}")
    h = layer_norm(x, norm_weight, norm_bias, eps, act8)
    a = linear_act(h, w1, b1, act=act, act8=act8)
    return linear_act(a, w2, b2, residual=x, act8=act8)


def _nothing_hangs_on(m: nn.Module) -> bool:
    """Calling ``m`` does what its parameters say, and nothing else."""
    return not (m._forward_pre_hooks or m._forward_hooks or
                m._backward_pre_hooks or m._backward_hooks or
                "forward" in vars(m))


class FFNBlock(nn.Module):
    """``ffn_block`` with its parameters.

    Its children ``norm``, ``fc1`` and ``fc2`` are the layer norm and the two
    linear layers without activation or residual, and keep the parameters.  They
    are called, with the activation and the addition of x between and after
    them, where something hangs on that: hooks of theirs or of all modules
    (pruning and the like work by such), or another module in a child's place.
    Otherwise the block is one call, with fewer roundings on its way."""

    def __init__(self, dim: int, hidden: int, act: str = "gelu",
                 act8: bool = False, eps: float = 1e-5):
        super().__init__()
        _act_code(act)
        self.norm = FusedLayerNorm(dim, eps=eps, act8=act8)
        self.fc1 = FusedLinearAct(dim, hidden, act8=act8)
        self.fc2 = FusedLinearAct(hidden, dim, act8=act8)
        self.act = act
        self.act8 = act8

    def _as_one_call(self) -> bool:
        fc = (self.fc1, self.fc2)
        return type(self.norm) is FusedLayerNorm and \
            all(type(m) is FusedLinearAct and m.act == "none" for m in fc) and \
            all(map(_nothing_hangs_on, (self.norm, *fc))) and \
            not _module._has_any_global_hook()

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if not self._as_one_call():
            if x.is_cuda and torch.is_autocast_enabled("cuda"):
                check_cast_leaves(x)
                x = x.to(torch.get_autocast_dtype("cuda"))
            u = self.fc1(self.norm(x))
            a = u if self.act == "none" else getattr(F, self.act)(u)
            return x + self.fc2(a)
        return ffn_block(x, self.norm.weight, self.norm.bias, self.fc1.weight,
                         self.fc1.bias, self.fc2.weight, self.fc2.bias,
                         self.act, self.norm.eps, self.act8)
