"""Layers on the HIP kernels: ComplexLinear on the complex GEMM (trnfft/nn.py:18-49) and GroupNorm.

Same parameters, initialisation and state_dict keys as the reference (``W_re.weight``,
``W_im.weight``, ``bias_re``, ``bias_im``), so checkpoints move between the two unchanged.  The
forward pass is one fused kernel: the four real products share their A/B tiles and the bias is
added in the epilogue.
"""

from __future__ import annotations

import math

import torch
import torch.nn as nn

from .complex import ComplexTensor
from .dispatch import complex_linear
from .norm import ACTIVATIONS, group_norm


class ComplexLinear(nn.Module):
    """Complex-valued linear layer: y = W x + b (complex arithmetic)."""

    def __init__(self, in_features: int, out_features: int, bias: bool = True):
        super().__init__()
        self.W_re = nn.Linear(in_features, out_features, bias=False)
        self.W_im = nn.Linear(in_features, out_features, bias=False)
        self.bias_re = nn.Parameter(torch.zeros(out_features)) if bias else None
        self.bias_im = nn.Parameter(torch.zeros(out_features)) if bias else None
        self._reset_parameters()

    def _reset_parameters(self):
        # trnfft/nn.py:29-31
        nn.init.kaiming_uniform_(self.W_re.weight, a=math.sqrt(5))
        nn.init.kaiming_uniform_(self.W_im.weight, a=math.sqrt(5))

    def forward(self, x: ComplexTensor) -> ComplexTensor:
        # differentiable in x, both weights and the bias (adjoint GEMMs on the same kernel)
        return complex_linear(x, self.W_re.weight, self.W_im.weight, self.bias_re, self.bias_im)


class GroupNorm(nn.Module):
    """Group norm with an activation on channels-last data (batch, ..., channels); parameters as torch.nn.GroupNorm's.

    The reference has no counterpart."""

    def __init__(self, num_groups: int, num_channels: int, eps: float = 1e-5, affine: bool = True,
                 activation: str | None = None):
        super().__init__()
        if num_groups < 1 or num_channels < 1 or num_channels % num_groups:
            raise ValueError(f"GroupNorm: {num_channels} channels cannot be divided into {num_groups} groups")
        if activation not in ACTIVATIONS:
            raise ValueError(f"GroupNorm: activation must be one of {tuple(ACTIVATIONS)}, got {activation!r}")
        self.num_groups, self.num_channels, self.eps, self.activation = num_groups, num_channels, eps, activation
        self.weight = nn.Parameter(torch.ones(num_channels)) if affine else None
        self.bias = nn.Parameter(torch.zeros(num_channels)) if affine else None

    def forward(self, x: torch.Tensor, lengths: torch.Tensor | None = None) -> torch.Tensor:
        return group_norm(x, self.num_groups, self.weight, self.bias, self.eps, self.activation, lengths)

    def extra_repr(self) -> str:
        return f"{self.num_groups}, {self.num_channels}, eps={self.eps}, activation={self.activation!r}"
