"""Layers on the HIP kernels: ComplexLinear on the complex GEMM (trnfft/nn.py:18-49), GroupNorm and StateSpace.

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
from .state_space import causal_conv, causal_conv_step, selective_scan, selective_scan_step


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


class StateSpace(nn.Module):
    """A selective state space layer on (batch, frames, features): a projection to a signal and its gate, a short causal
    convolution, the selective scan with steps, inputs and outputs that the signal itself gives, and a projection back.

    Each frame sees those up to it.  ``step`` takes the next frame of every stream; what a stream keeps is ``state``: the last
    width - 1 inputs of the convolution and ``states`` values a channel.  The reference has no counterpart."""

    def __init__(self, features: int, states: int = 16, width: int = 4, expand: int = 2, rank: int | None = None):
        super().__init__()
        if features < 1 or states < 1 or width < 1 or expand < 1 or (rank is not None and rank < 1):
            raise ValueError("StateSpace: features, states, width, expand and rank must be at least 1")
        self.features, self.inner, self.states, self.width = features, expand * features, states, width
        self.rank = -(-features // 16) if rank is None else rank
        self.enter = nn.Linear(features, 2 * self.inner, bias=False)
        self.conv_weight = nn.Parameter(torch.empty(self.inner, width))
        self.conv_bias = nn.Parameter(torch.zeros(self.inner))
        self.select = nn.Linear(self.inner, self.rank + 2 * states, bias=False)
        self.steps = nn.Linear(self.rank, self.inner, bias=False)
        self.dt_bias = nn.Parameter(torch.empty(self.inner))
        self.a_log = nn.Parameter(torch.empty(self.inner, states))
        self.skip = nn.Parameter(torch.ones(self.inner))
        self.leave = nn.Linear(self.inner, features, bias=False)
        self._reset_parameters()

    @torch.no_grad()
    def _reset_parameters(self):
        nn.init.uniform_(self.conv_weight, -self.width**-0.5, self.width**-0.5)
        # steps of 1e-3 to 1e-1 to begin with (softplus of the bias), decays of 1 to `states` for a step of 1
        step = torch.exp(torch.rand(self.inner) * math.log(100.0) + math.log(1e-3))
        self.dt_bias.copy_(step + torch.log(-torch.expm1(-step)))
        self.a_log.copy_(torch.log(torch.arange(1, self.states + 1, dtype=torch.float32)).expand(self.inner, -1))

    def state(self, batch: int, device=None, dtype: torch.dtype | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """What a stream begins with: zeros for the convolution (in the layer's dtype) and the scan (float32)."""
        device, dtype = device or self.enter.weight.device, dtype or self.enter.weight.dtype
        return (torch.zeros(batch, self.width - 1, self.inner, dtype=dtype, device=device),
                torch.zeros(batch, self.inner, self.states, dtype=torch.float32, device=device))

    def _operands(self, x: torch.Tensor):
        """dt, a, b and c of the convolved signal."""
        step, b, c = self.select(x).split([self.rank, self.states, self.states], dim=-1)
        return self.steps(step), -torch.exp(self.a_log.float()), b.unsqueeze(-2), c.unsqueeze(-2)

    def forward(self, x: torch.Tensor, lengths: torch.Tensor | None = None,
                state: tuple[torch.Tensor, torch.Tensor] | None = None, return_state: bool = False):
        """Frames at and past a row's length are padding.  state: where the sequences go on from; return_state: where they end."""
        signal, gate = self.enter(x).chunk(2, dim=-1)
        before, start = (None, None) if state is None else state
        signal = causal_conv(signal, self.conv_weight, self.conv_bias, activation="silu", initial_state=before, lengths=lengths,
                             return_state=return_state)
        signal, last = signal if return_state else (signal, None)
        dt, a, b, c = self._operands(signal)
        y = selective_scan(signal, dt, a, b, c, d=self.skip, z=gate, dt_bias=self.dt_bias, initial_state=start, lengths=lengths,
                           return_state=return_state)
        y, end = y if return_state else (y, None)
        return (self.leave(y), (last, end)) if return_state else self.leave(y)

    def step(self, x: torch.Tensor, state: tuple[torch.Tensor, torch.Tensor]) -> torch.Tensor:
        """The next frame (batch, features) of every stream; both parts of the state are updated in place.  No gradients."""
        with torch.no_grad():
            signal, gate = self.enter(x).chunk(2, dim=-1)
            signal = causal_conv_step(signal, state[0], self.conv_weight, self.conv_bias, activation="silu")
            dt, a, b, c = self._operands(signal)
            y = selective_scan_step(signal, dt, a, b, c, state[1], d=self.skip, z=gate, dt_bias=self.dt_bias)
            return self.leave(y)

    def extra_repr(self) -> str:
        return f"{self.features}, states={self.states}, width={self.width}, inner={self.inner}, rank={self.rank}"
