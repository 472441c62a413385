"""Layer norm with an optional residual add, forward and backward.

``layer_norm`` normalises the last dimension through ``gdn2_layer_norm_fwd`` /
``gdn2_layer_norm_bwd``; ``LayerNorm`` is the module around it.  Statistics,
and the sums of the weight's and the bias's gradients, are fp32.
"""

from __future__ import annotations

import torch
import torch.nn as nn

from . import _lib


def layer_norm(
    x: torch.Tensor,
    weight: torch.Tensor | None = None,
    bias: torch.Tensor | None = None,
    eps: float = 1e-5,
    residual: torch.Tensor | None = None,
):
    r"""Layer norm over the last dimension D (at most 32768).

    ``y = (s - mean) / sqrt(var + eps) * weight + bias`` with ``s = x``, or
    ``s = x + residual``.  x: bf16 or fp32; weight, bias: ``[D]``, bf16 or
    fp32 (one type), either may be None; residual: the shape of x, x's type or
    fp32.  Returns ``y`` in x's type, or ``(y, s)`` with a residual, ``s`` in
    the residual's type (s is rounded to it before the statistics).
    Differentiable in every tensor (once, in reverse mode; forward-mode tangents are refused).
    """
    y, s = _lib.ops().layer_norm(x, weight, bias, eps, residual)
    return y if residual is None else (y, s)


class LayerNorm(nn.Module):
    """``layer_norm`` with its parameters (ones and zeros; names and shapes of ``torch.nn.LayerNorm``)."""

    def __init__(self, size: int, eps: float = 1e-5, elementwise_affine: bool = True, bias: bool = True):
        super().__init__()
        self.size, self.eps = size, eps
        self.weight = nn.Parameter(torch.ones(size)) if elementwise_affine else None
        self.bias = nn.Parameter(torch.zeros(size)) if elementwise_affine and bias else None

    def forward(self, x: torch.Tensor, residual: torch.Tensor | None = None):
        return layer_norm(x, self.weight, self.bias, self.eps, residual)
