"""Activations kept in 8 bits for the backward pass.

A row's values go in groups of 128 (the last one may be shorter); each group
keeps one fp32 scale::

    a     = max |x|                    over the group
    codes = rint(x * fl(127 / a))      int8, ties to even
    scale = fl(a * fl(1 / 127))
    x'    = codes * scale

``fl`` is rounding to fp32, so the codes are the same on every device.  A group
whose ``a`` is under 2^-119 is kept as zeros, and one that holds an infinity or
a NaN gets the scale NaN: all of it reads as NaN, so that a broken activation
shows in the gradients.

``layer_norm``, ``linear_act`` and ``ffn_block`` use this form with
``act8=True``; ``act8_pack`` and ``act8_unpack`` are for functions of one's own.
"""
from __future__ import annotations

from typing import NamedTuple

import torch
import torch.nn.functional as F

from . import _ext

GROUP = 128
_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


class Act8(NamedTuple):
    """``codes``: int8, shaped as the activation; ``scales``: fp32, with one
    value for each 128 of the last dimension."""
    codes: torch.Tensor
    scales: torch.Tensor


def _groups(x: torch.Tensor) -> torch.Tensor:
    dim = x.size(-1)
    n = -(-dim // GROUP)
    return F.pad(x, (0, n * GROUP - dim)).reshape(*x.shape[:-1], n, GROUP)


def act8_pack(x: torch.Tensor) -> Act8:
    """The 8-bit form of ``x`` (bf16, fp16 or fp32), by groups of its last
    dimension.  Not differentiable; on the GPU forward mode, torch.func's
    transforms and tracing are refused."""
    if x.is_cuda:
        return Act8(*_ext().act8_pack(x))
    if x.dim() < 1 or x.size(-1) == 0 or not x.is_floating_point():
        raise RuntimeError("act8_pack needs floating values with a last "
                           f"dimension, got {x.dtype} {tuple(x.shape)}")
    g = _groups(x.detach().float())
    a = g.abs().amax(-1, keepdim=True)
    fine = torch.isfinite(a)
    some = fine & (a >= 2.0 ** -119)
    by = torch.where(some, torch.full_like(a, 127.0) / a,
                     torch.zeros_like(a))
    codes = torch.where(some, torch.round(g * by), torch.zeros_like(g))
    codes = codes.to(torch.int8).flatten(-2)[..., :x.size(-1)].contiguous()
    scales = torch.where(some, a * torch.full_like(a, 1.0 / 127.0),
                         torch.zeros_like(a))
    scales = torch.where(fine, scales, torch.full_like(a, float("nan")))
    return Act8(codes, scales.squeeze(-1))


def act8_unpack(codes: torch.Tensor, scales: torch.Tensor,
                dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values that an 8-bit form stands for, rounded once to ``dtype``.  On
    the GPU scales that require a gradient are refused, and what ``act8_pack``
    refuses."""
    if codes.is_cuda:
        if dtype not in _TYPES:
            raise RuntimeError(f"act8_unpack gives {list(_TYPES)}, "
                               f"not {dtype}")
        return _ext().act8_unpack(codes, scales, _TYPES[dtype])
    if codes.dtype != torch.int8 or scales.dtype != torch.float32:
        raise RuntimeError("codes must be int8 and scales float32, got "
                           f"{codes.dtype} and {scales.dtype}")
    want = (*codes.shape[:-1], -(-codes.size(-1) // GROUP))
    if tuple(scales.shape) != want:
        raise RuntimeError(f"scales must have shape {want}, got "
                           f"{tuple(scales.shape)}")
    x = _groups(codes.float()) * scales.unsqueeze(-1)
    return x.flatten(-2)[..., :codes.size(-1)].to(dtype)


def _wide(x: torch.Tensor) -> torch.Tensor:
    """CPU: what arithmetic is done in."""
    return x if x.dtype == torch.float64 else x.float()
