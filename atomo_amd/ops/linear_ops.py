"""Fully connected layer with its epilogue in the product's kernel (kernels:
ops/csrc/linear_kernels.hip).

    y = act(x W^T + b) + residual        act: none, relu, gelu (erf), silu

and its gradients.  ``models.fuse_linears`` puts it in the place of the model
zoo's Linear (+ ReLU) layers (``--fused-linear``).  CUDA (= ROCm) tensors take
the HIP kernels, CPU tensors the torch oracle (64-bit inside).
"""

from __future__ import annotations

import math
from typing import Optional

import torch
import torch.nn as nn
import torch.nn.functional as F

from . import ext

_FLOATS = (torch.float32, torch.bfloat16, torch.float16)
ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "silu": 3}
_APPLY = {"none": lambda h: h, "relu": F.relu, "gelu": F.gelu, "silu": F.silu}


def _same(t: torch.Tensor, x: torch.Tensor, shape, name: str) -> torch.Tensor:
    if t.dtype != x.dtype:
        raise TypeError(f"{name} is {t.dtype}, x is {x.dtype}")
    if t.device != x.device:
        raise ValueError(f"{name} is on {t.device}, x on {x.device}")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must be {tuple(shape)}, not {tuple(t.shape)}")
    return t


def _matrix(t: torch.Tensor) -> torch.Tensor:
    """(..., columns) as (rows, columns) with contiguous rows."""
    if t.dim() != 2:
        t = t.reshape(math.prod(t.shape[:-1]), t.shape[-1])
    if t.shape[1] > 1 and t.stride(1) != 1:
        t = t.contiguous()
    return t


def linear_act(
    x: torch.Tensor,
    weight: torch.Tensor,
    bias: Optional[torch.Tensor] = None,
    activation: str = "none",
    residual: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """``act(x @ weight.T + bias) + residual`` for x (..., in), weight
    (out, in), bias (out), residual (..., out), all of one type: fp32, bf16 or
    fp16.

    Sums are fp32, the result is rounded once.  fp32 operands of more than
    four rows are multiplied as three bf16 parts each, six products of nine:
    to 2^-25 of a product, but what a part holds below 2^-126 may count as 0,
    so that operands below 2^-101 have fewer digits.  The slope of gelu and
    silu is kept for the backward pass in fp32; dy times the slope is rounded to
    the operands' type before it is multiplied.  A result of relu that is above
    0 and too small for the type is -0, which keeps its slope of 1.  Rows may be
    strided; other layouts are copied first.  The gradients cannot be
    differentiated again on a GPU.
    """
    if activation not in ACTIVATIONS:
        raise ValueError(
            f"activation must be one of {sorted(ACTIVATIONS)}, not {activation!r}")
    if x.dtype not in _FLOATS:
        raise TypeError(f"x must be fp32, bf16 or fp16, not {x.dtype}")
    if weight.dim() != 2 or 0 in weight.shape:
        raise ValueError("weight must be (out, in), neither of them 0")
    n, k = weight.shape
    if x.dim() < 1 or x.shape[-1] != k:
        raise ValueError(f"x must be (..., {k}), not {tuple(x.shape)}")
    lead = x.shape[:-1]
    _same(weight, x, (n, k), "weight")
    if bias is not None:
        _same(bias, x, (n,), "bias")
    if residual is not None:
        _same(residual, x, (*lead, n), "residual")
    if x.is_cuda:
        y = ext().linear_act(
            _matrix(x), _matrix(weight),
            None if bias is None else bias.contiguous(),
            None if residual is None else _matrix(residual),
            ACTIVATIONS[activation])
        return y if len(lead) == 1 else y.view(*lead, n)
    wide = None if bias is None else bias.double()
    h = F.linear(x.double(), weight.double(), wide)
    if activation == "relu":
        h = h.relu()
    elif activation != "none":
        # at both ends their limits, with the slopes 0 and 1
        far = h.detach().abs() > 1e4
        near = _APPLY[activation](h.masked_fill(far, 0.0))
        h = torch.where(far, h.masked_fill(h.detach() < 0.0, 0.0), near)
    if residual is not None:
        h = h + residual.double()
    return h.to(x.dtype)


def linear_relu(layer: nn.Module, x: torch.Tensor) -> torch.Tensor:
    """ReLU of a layer's output, unless the layer has it in its kernel."""
    y = layer(x)
    return y if getattr(layer, "activation", None) == "relu" else F.relu(y)


class FusedLinear(nn.Linear):
    """``nn.Linear`` with its activation in the same kernel; same parameters,
    same names.  Types that the kernel does not take (fp64) go the way of
    ``nn.Linear``."""

    def __init__(self, in_features: int, out_features: int, bias: bool = True,
                 activation: str = "none"):
        super().__init__(in_features, out_features, bias)
        if activation not in ACTIVATIONS:
            raise ValueError(
                f"activation must be one of {sorted(ACTIVATIONS)}, not {activation!r}")
        self.activation = activation

    @classmethod
    def of(cls, linear: nn.Linear, activation: str = "none") -> "FusedLinear":
        """Takes over a layer's parameters (the same objects)."""
        fused = cls.__new__(cls)
        nn.Module.__init__(fused)
        fused.in_features = linear.in_features
        fused.out_features = linear.out_features
        fused.weight, fused.bias = linear.weight, linear.bias
        fused.activation = activation
        return fused.train(linear.training)

    def forward(self, x: torch.Tensor,
                residual: Optional[torch.Tensor] = None) -> torch.Tensor:
        weight, bias = self.weight, self.bias
        if torch.is_autocast_enabled(x.device.type):
            kind = torch.get_autocast_dtype(x.device.type)
            # as torch's own layers: fp64 stays
            x, weight, bias, residual = (
                t if t is None or t.dtype == torch.float64 else t.to(kind)
                for t in (x, weight, bias, residual))
        if x.dtype not in _FLOATS:
            y = _APPLY[self.activation](F.linear(x, weight, bias))
            return y if residual is None else y + residual
        return linear_act(x, weight, bias, self.activation, residual)

    def extra_repr(self) -> str:
        return f"{super().extra_repr()}, activation={self.activation}"
