"""Fully connected layers on the engine: ``y = act(x W^T + bias) + residual``, with gradients.

The layers that stand between and behind convolutions -- 1x1 heads on pooled features, classifiers, feed-forward blocks -- run on
the tensor cores like them (``csrc/wino_linear.cu``): 16-bit operands, products and sums in fp32, bias, activation and residual
applied to the fp32 sums, one rounding at the end.  One or two rows are served by a kernel that reads the weights once, a few by
clusters that share the reduction, thousands by one that keeps the tensor cores busy; all take any size and any row stride, and
give the same bits every time.

* :func:`linear` -- the operator on tensors; :class:`Linear` -- the ``torch.nn.Linear`` subclass, as ``conv.Conv2d`` is one of
  ``torch.nn.Conv2d``.
* Backward: the gradient through the activation with the bias gradient beside it (``csrc/wino_e4m3.cu``), the data and weight
  gradients as two more products of the same kernels, which read W, x and the gradient as they lie.
* What the backward pass needs is x (for the weight gradient) and, with an activation, the pre-activation, in x's type.
  ``checkpoint="e4m3"`` keeps both in eight bits instead (:mod:`.checkpoint`): half the memory, gradients as if x and the
  pre-activation had been rounded to four significant bits; the forward result is the same.

The gradients are not differentiable again.  There is no CPU path and no library product.  Calls keep nothing but what autograd
saves: they may run on several threads and streams and in captured graphs.  (As with every operator of torch, a backward pass can only
be captured when no eager graph of the same parameters, built on another stream, is still alive: torch raises there.)  A call that a
tracer would record (``torch.jit.trace``, ``make_fx``, ``torch.export``) or that carries a forward-mode gradient is an error.
"""
from __future__ import annotations

from typing import Optional

import torch
import torch.nn as nn

from . import _backend

__all__ = ["ACTIVATIONS", "Linear", "linear"]

#: activation name -> code of the C ABI (``winoconv_act_t``)
ACTIVATIONS = {None: 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}


def _activation(name) -> int:
    try:
        return ACTIVATIONS[name]
    except (KeyError, TypeError):
        raise ValueError(f"activation must be one of {list(ACTIVATIONS)}, got {name!r}") from None


def _packs(checkpoint) -> bool:
    if checkpoint not in (None, "e4m3"):
        raise ValueError(f"checkpoint must be None or 'e4m3', got {checkpoint!r}")
    return checkpoint is not None


_call = None


def _native():
    global _call
    _call = _backend.load().linear_call
    return _call


def linear(input: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,      # noqa: A002  (torch's argument name)
           residual: Optional[torch.Tensor] = None, *, activation: Optional[str] = None,
           checkpoint: Optional[str] = None) -> torch.Tensor:
    """``act(input @ weight.T + bias) + residual`` in the type of ``input`` (float16 or bfloat16).

    ``input`` [..., in_features], ``weight`` [out_features, in_features] of the same type or float32 (then rounded once),
    ``bias`` [out_features] of the same type or float32, ``residual`` of the result's shape and type.  ``activation``: ``None``,
    ``"relu"``, ``"gelu"`` (erf), ``"gelu_tanh"`` or ``"silu"``.  ``checkpoint="e4m3"`` keeps what the backward pass needs in
    eight bits.  Weights that are float32, transposed or have rows that do not start on 16 bytes are copied on every call.
    """
    return (_call or _native())(input, weight, bias, residual, _activation(activation), _packs(checkpoint))


class Linear(nn.Linear):
    """``torch.nn.Linear`` on the engine: same arguments, parameters and ``state_dict``.

    Extra keyword arguments, as for ``conv.Conv2d``: ``compute_dtype`` (default ``torch.float16``; ``None`` keeps the input's
    type, which must then be a 16-bit one) is the type of the operands and the result; ``activation``; ``checkpoint``
    (``None`` / ``"e4m3"``).  ``forward`` takes the residual as a second argument.

    Parameters of the compute type are read as they lie; float32 ones, a training loop's master copies, are rounded on every
    call and get float32 gradients.  For serving, keep them in the compute type: ``layer.to(layer.compute_dtype)``.
    """

    def __init__(self, in_features, out_features, bias=True, device=None, dtype=None, *,
                 compute_dtype: Optional[torch.dtype] = torch.float16, activation: Optional[str] = None,
                 checkpoint: Optional[str] = None):
        super().__init__(in_features, out_features, bias, device=device, dtype=dtype)
        if compute_dtype not in (None, torch.float16, torch.bfloat16):
            raise ValueError(f"compute_dtype must be None, torch.float16 or torch.bfloat16, got {compute_dtype}")
        _activation(activation)
        _packs(checkpoint)
        self.compute_dtype = compute_dtype
        self.activation = activation
        self.checkpoint = checkpoint

    def forward(self, input: torch.Tensor, residual: Optional[torch.Tensor] = None) -> torch.Tensor:      # noqa: A002
        dtype = self.compute_dtype if self.compute_dtype is not None else input.dtype
        weight, bias = self.weight, self.bias
        # (differentiable: a gradient comes back in the type of what was given)
        x = input if input.dtype == dtype else input.to(dtype)
        if residual is not None and residual.dtype != dtype:
            residual = residual.to(dtype)
        if weight.dtype not in (dtype, torch.float32):
            weight = weight.to(dtype)
        if bias is not None and bias.dtype not in (dtype, torch.float32):
            bias = bias.to(dtype)
        return linear(x, weight, bias, residual, activation=self.activation, checkpoint=self.checkpoint)

    def extra_repr(self) -> str:
        s = super().extra_repr() + f", compute_dtype={self.compute_dtype}"
        if self.activation:
            s += f", activation={self.activation}"
        if self.checkpoint:
            s += f", checkpoint={self.checkpoint}"
        return s
