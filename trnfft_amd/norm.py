"""Group norm with an activation on channels-last data (csrc/kernels_norm.hip).

Features of STFT frames are channels last (batch, frames, channels) or (batch, frames, bins, channels), as frames-major
spectra are; normalisation, affine map and activation are one operator, forward and backward.  The reference has no
counterpart.
"""

from __future__ import annotations

import ctypes
import math

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .attention import DTYPES, _on
from .dispatch import _require_hip, addr, launch, refuse_tangents, target_device

ACTIVATIONS = {None: _lib.ACT_NONE, "silu": _lib.ACT_SILU, "gelu": _lib.ACT_GELU, "relu": _lib.ACT_RELU}


def _whole(x: torch.Tensor) -> torch.Tensor:
    return x if x.data_ptr() % 16 == 0 else x.clone()


def _channels(w: torch.Tensor | None, dev: torch.device) -> torch.Tensor | None:
    return None if w is None else _on(w if w.dtype == torch.float32 else w.float(), dev).contiguous()


def _workspace(desc: _lib.NormDesc, backward: int, dev: torch.device, what: str) -> torch.Tensor | None:
    nbytes = ctypes.c_size_t()
    _lib.check(_lib.lib().tfa_group_norm_workspace_size(desc, backward, nbytes), what)
    return torch.empty(nbytes.value, dtype=torch.uint8, device=dev) if nbytes.value else None


def _forward(x, weight, bias, lengths, desc):
    y = torch.empty_like(x)
    stats = torch.empty(2, desc.batch, desc.groups, dtype=torch.float32, device=x.device)
    ws = _workspace(desc, 0, x.device, "group_norm")
    launch("group_norm", x.device, _lib.lib().tfa_group_norm, desc, addr(x), addr(weight), addr(bias), addr(lengths),
           addr(y), *_mean_rstd(stats), addr(ws))
    return y, stats


def _mean_rstd(stats: torch.Tensor) -> tuple[int, int]:
    at = stats.data_ptr()
    return at, at + 2 * stats.numel()  # (two halves of 4-byte values)


class _GroupNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, lengths, desc):
        y, stats = _forward(x, weight, bias, lengths, desc)
        ctx.desc = desc
        ctx.save_for_backward(x, weight, bias, lengths, stats)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        x, weight, bias, lengths, stats = ctx.saved_tensors
        what, dev, desc, need = "group_norm backward", x.device, ctx.desc, ctx.needs_input_grad
        g = _whole(_on(g, dev).contiguous())
        dx = torch.empty_like(x)
        fresh = torch.empty_like if x.numel() else torch.zeros_like  # (of no data there is no launch)
        dw = fresh(weight) if weight is not None and need[1] else None
        db = fresh(bias) if bias is not None and need[2] else None
        ws = _workspace(desc, 1, dev, what)
        launch(what, dev, _lib.lib().tfa_group_norm_backward, desc, addr(x), addr(g), addr(weight), addr(bias),
               addr(lengths), *_mean_rstd(stats), addr(dx), addr(dw), addr(db), addr(ws))
        return dx if need[0] else None, dw, db, None, None


def group_norm(x: torch.Tensor, num_groups: int, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               eps: float = 1e-5, activation: str | None = None, lengths: torch.Tensor | None = None) -> torch.Tensor:
    """act(group_norm(x) * weight + bias) of channels-last x (batch, ..., channels), differentiable.

    Statistics are those of a sample's group of channels / num_groups channels over all positions.  x: float32, bfloat16 or
    float16; weight and bias (channels,) in float32 or x's dtype; activation: None, "silu", "gelu" (by the error function)
    or "relu".  lengths: (batch,) whole numbers, the positions along axis 1 that are no padding: padding is not read, takes
    no part in the statistics and is zero in the result.  Gradients cannot be differentiated again, and there is no forward mode.
    """
    what = "group_norm"
    if x.dtype not in DTYPES:
        raise TypeError(f"{what}: float32, bfloat16 or float16 expected, got {x.dtype}")
    if x.dim() < 2:
        raise ValueError(f"{what}: expects (batch, ..., channels), got {x.dim()} dimensions")
    channels, batch = x.shape[-1], x.shape[0]
    if num_groups < 1 or channels < 1 or channels % num_groups:
        raise ValueError(f"{what}: {channels} channels cannot be divided into {num_groups} groups")
    if activation not in ACTIVATIONS:
        raise ValueError(f"{what}: activation must be one of {tuple(ACTIVATIONS)}, got {activation!r}")
    if not (math.isfinite(eps) and eps >= 0):
        raise ValueError(f"{what}: eps must be finite and not negative")
    for name, w in (("weight", weight), ("bias", bias)):
        if w is None:
            continue
        if w.shape != (channels,):
            raise ValueError(f"{what}: {name} must be ({channels},), got {tuple(w.shape)}")
        if w.dtype not in (torch.float32, x.dtype):
            raise TypeError(f"{what}: {name} must be float32 or {x.dtype}, got {w.dtype}")
    if lengths is not None:
        if x.dim() < 3 or lengths.shape != (batch,):
            raise ValueError(f"{what}: lengths must be ({batch},) for (batch, positions, ..., channels) data")
        if lengths.dtype not in (torch.int64, torch.int32, torch.int16, torch.uint8, torch.int8):
            raise TypeError(f"{what}: lengths must be whole numbers, got {lengths.dtype}")
    refuse_tangents(what, x, weight, bias)
    _require_hip(what)
    dev, out_dev = target_device(x), x.device
    x = _whole(_on(x, dev).contiguous())
    weight, bias = _channels(weight, dev), _channels(bias, dev)
    lengths = None if lengths is None else lengths.to(dev, torch.int64).contiguous()
    positions = math.prod(x.shape[1:-1])
    inner = max(1, math.prod(x.shape[2:-1])) if x.dim() > 2 else 1
    desc = _lib.NormDesc(DTYPES[x.dtype], channels, num_groups, ACTIVATIONS[activation], batch, positions, inner, eps, 0)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias)):
        y = _GroupNormFn.apply(x, weight, bias, lengths, desc)
    else:
        y, _ = _forward(x, weight, bias, lengths, desc)
    return y if out_dev == dev else y.to(out_dev)
