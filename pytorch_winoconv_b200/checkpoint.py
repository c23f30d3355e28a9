"""Activations kept in eight bits between the forward and the backward pass (``csrc/wino_e4m3.cu``).

32 neighbours of the last dimension share a power of two, the smallest (from 2^-127 on) that brings the largest finite magnitude
among them within e4m3's 448, and are rounded to e4m3 (half to even): 1 + 1/32 bytes a value instead of two, a relative error of at
most 2^-4 for all but the values that are 2^-13 or less of their block's largest.  A power of two costs none of the four significant
bits, so what comes back is held by float16 and bfloat16 without another rounding.  Infinities and NaN come back as NaN; a value that
rounds up beyond the type's largest (65504 in float16) comes back as that largest.

``linear.Linear``, ``conv.Conv2d`` and ``conv.Conv3d`` use it with ``checkpoint="e4m3"`` (a convolution packs the channels of each
pixel: fewer than 32 save less); :func:`pack` and :func:`unpack` are the operators themselves, for a program's own autograd functions
(calls that a tracer would record or that carry a forward-mode gradient are errors).
"""
from __future__ import annotations

from typing import Tuple

import torch

from . import _backend

__all__ = ["BLOCK", "pack", "unpack"]

BLOCK = 32
_native = None


def _module():
    global _native
    _native = _backend.load()
    return _native


def pack(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(q, scale)`` of a float16 or bfloat16 tensor: ``q`` of x's shape in ``torch.float8_e4m3fn``, ``scale``
    ``[..., ceil(C / 32)]`` in ``torch.float8_e8m0fnu``, both contiguous.  Not differentiable."""
    return (_native or _module()).e4m3_pack(x)


def unpack(q: torch.Tensor, scale: torch.Tensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values that :func:`pack` kept, in ``dtype`` (float16 or bfloat16)."""
    return (_native or _module()).e4m3_unpack(q, scale, dtype)
