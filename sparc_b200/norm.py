"""Layer norm over the last dimension, y = (x - mean) (var + eps)^(-1/2) weight + bias, forward and
backward with the weight's and bias's gradients, on the kernels of csrc/layer_norm.cu: the norm
the reference's networks put before each layer (sparc-impl/sparc/networks/sequence_classifier.py),
next to the RMSNorm of `stack.py`, whose stack takes either (``norm="layer"``).

x is float32 or bfloat16 with any leading dimensions (rows whose columns are adjacent are read in
place, others copied first); the statistics, the sums and the parameters are float32. There is no
forward-mode derivative: an input with a tangent is refused (NotImplementedError).
"""
from __future__ import annotations

import torch
from torch import nn

from . import torch_ops


def layer_norm(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None,
               eps: float = 1e-5) -> torch.Tensor:
    """Layer norm over x's last dimension, in x's dtype; differentiable (once) with respect to x,
    the weight and the bias."""
    return torch_ops.call("layer_norm", x, weight, bias, eps)


class LayerNorm(nn.Module):
    """Layer norm over the last dimension (parameters: weight, ones, and bias, zeros, unless bias
    is False), as torch.nn.LayerNorm's state dict has them."""

    def __init__(self, width: int, eps: float = 1e-5, bias: bool = True):
        super().__init__()
        self.eps = eps
        self.weight = nn.Parameter(torch.ones(width))
        self.bias = nn.Parameter(torch.zeros(width)) if bias else None

    def forward(self, x):
        return layer_norm(x, self.weight, self.bias, self.eps)
