"""The operators of a selective state space layer over frames (csrc/kernels_conv.hip, csrc/scan_blocks.h).

    causal_conv:     y_t = act(bias + sum_j weight[:, j] x_{t - width + 1 + j})
    selective_scan:  s_t = softplus(dt_t + dt_bias),  h_t = exp(s_t a) h_{t-1} + s_t x_t b_t,  y_t = (c_t . h_t + d x_t) silu(z_t)

A sequence model for STFT frames whose memory each frame sets for itself: what a stream keeps is the last inputs of a short
filter and a few states a channel, however long it runs.  ``causal_conv`` and ``selective_scan`` take whole sequences
(training, prompts, blocks of a stream), their ``_step`` one frame.  The reference has no counterpart.
"""

from __future__ import annotations

import torch
from torch.autograd import forward_ad

from . import _lib
from .attention import DTYPES, _features, _on
from .dispatch import _current_device, _require_hip, _use_hip, addr, launch, refuse_tangents, target_device
from .norm import ACTIVATIONS, _channels

_WHOLE = (torch.int64, torch.int32, torch.int16, torch.uint8, torch.int8)


def _check_lengths(what: str, lengths: torch.Tensor | None, b: int) -> None:
    if lengths is None:
        return
    if lengths.shape != (b,):
        raise ValueError(f"{what}: lengths must be ({b},), got {tuple(lengths.shape)}")
    if lengths.dtype not in _WHOLE:
        raise TypeError(f"{what}: lengths must be whole numbers, got {lengths.dtype}")


def _check_channels(what: str, c: int, dtype: torch.dtype, **vectors: torch.Tensor | None) -> None:
    for name, v in vectors.items():
        if v is None:
            continue
        if v.shape != (c,):
            raise ValueError(f"{what}: {name} must be ({c},), got {tuple(v.shape)}")
        if v.dtype not in (torch.float32, dtype):
            raise TypeError(f"{what}: {name} must be float32 or {dtype}, got {v.dtype}")


def _whole_numbers(lengths: torch.Tensor | None, dev: torch.device) -> torch.Tensor | None:
    return None if lengths is None else lengths.to(dev, torch.int64).contiguous()


def _wants(*tensors: torch.Tensor | None) -> bool:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


def _dense(g: torch.Tensor | None, dev: torch.device) -> torch.Tensor | None:
    return None if g is None else _on(g, dev).contiguous()


def _tokens(x: torch.Tensor, dev: torch.device) -> torch.Tensor:
    """x on dev with contiguous channels and frames less than 2^24 values apart (x itself where it is so)."""
    x = _features(x, dev)
    return x if x.stride(1) < 1 << 24 or x.shape[1] == 1 else x.contiguous()


def _check_state(what: str, state: torch.Tensor) -> torch.device:
    """The device of a state that is updated in place."""
    if not state.is_cuda or not state.is_contiguous() or state.is_neg():
        raise ValueError(f"{what}: the state is updated in place and must be contiguous on the GPU")
    return state.device


def _results(what: str, out, dev: torch.device):
    """A native call's results on dev; raises for a status."""
    if type(out) is int:
        _lib.check(out, what)
    if type(out) is tuple:
        return tuple(v if v.device == dev else v.to(dev) for v in out)
    return out if out.device == dev else out.to(dev)


def _direct(what: str, name: str, *args):
    """A sequence's call made natively: its results, or None where an operand has to be converted or refused first."""
    if not _use_hip() or getattr(forward_ad, "_current_level", 0) >= 0:
        return None
    out = getattr(_lib.state_space(), name)(*args, False)
    if type(out) is int:
        _lib.check(out, what)
    return out


def _step(what: str, step: str, state: torch.Tensor, *args) -> torch.Tensor | None:
    """A stream's step called natively: its result, or None where an operand has to be converted or refused first, or the state is
    on another device than the current one."""
    if not _use_hip():
        return None
    index = state.get_device()
    if index < 0 or _current_device() != index or getattr(forward_ad, "_current_level", 0) >= 0:
        return None
    y = getattr(_lib.state_space(), step)(index, *args)
    if type(y) is int:
        _lib.check(y, what)
    return y


# ---------------------------------------------------------------------------------------------
# causal convolution
# ---------------------------------------------------------------------------------------------


def _check_conv(what: str, x, weight, bias, activation, dims: int) -> None:
    if x.dim() != dims:
        raise ValueError(f"{what}: x must have {dims} dimensions, got {x.dim()}")
    if x.dtype not in DTYPES:
        raise TypeError(f"{what}: float32, bfloat16 or float16 expected, got {x.dtype}")
    c = x.shape[-1]
    if c < 1 or weight.dim() != 2 or weight.shape[0] != c or weight.shape[1] < 1:
        raise ValueError(f"{what}: weight must be (channels, width) for {c} channels, got {tuple(weight.shape)}")
    if weight.dtype not in (torch.float32, x.dtype):
        raise TypeError(f"{what}: weight must be float32 or {x.dtype}, got {weight.dtype}")
    if bias is not None:
        _check_channels(what, c, x.dtype, bias=bias)
    if activation not in ACTIVATIONS:
        raise ValueError(f"{what}: activation must be one of {tuple(ACTIVATIONS)}, got {activation!r}")


def causal_conv(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *, activation: str | None = None,
                initial_state: torch.Tensor | None = None, lengths: torch.Tensor | None = None, return_state: bool = False):
    """Causal convolution over frames with a filter for each channel and an activation, differentiable in every tensor but
    `lengths`.

    x (batch, frames, channels): float32, bfloat16 or float16; views of a larger projection are taken as they are.  weight
    (channels, width), widths 1 to 8, the last tap on the frame itself; bias (channels,); both float32 or x's dtype.
    activation: None, "silu", "gelu" or "relu".  initial_state: (batch, width - 1, channels) of x's dtype, the inputs before
    the first frame (zeros without).  lengths: (batch,) whole numbers; frames at and past a sequence's length are padding,
    whatever they hold: outputs and gradients are zero there.

    Returns y (batch, frames, channels) in x's dtype, and with return_state the last width - 1 inputs up to each sequence's
    length.  Sums are fp32.  Gradients cannot be differentiated again, and there is no forward mode.
    """
    what = "causal_conv"
    if activation in ACTIVATIONS:
        out = _direct(what, what, x, weight, bias, initial_state, lengths, ACTIVATIONS[activation], return_state)
        if out is not None:  # (as it mostly is: nothing to convert, nothing to refuse)
            return out
    _check_conv(what, x, weight, bias, activation, 3)
    (b, _, c), width = x.shape, weight.shape[1]
    if initial_state is not None:
        if initial_state.shape != (b, width - 1, c):
            raise ValueError(f"{what}: initial_state must be (batch, width - 1, channels), got {tuple(initial_state.shape)}")
        if initial_state.dtype != x.dtype:
            raise TypeError(f"{what}: initial_state must be {x.dtype}, got {initial_state.dtype}")
    _check_lengths(what, lengths, b)
    refuse_tangents(what, x, weight, bias, initial_state)
    _require_hip(what)
    dev, out_dev = target_device(x), x.device
    x, weight, bias = _features(x, dev), _channels(weight, dev), _channels(bias, dev)
    state, lengths = _dense(initial_state, dev), _whole_numbers(lengths, dev)
    return _results(what, _lib.state_space().causal_conv(x, weight, bias, state, lengths, ACTIVATIONS[activation], return_state, True), out_dev)


def causal_conv_step(x: torch.Tensor, state: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *,
                     activation: str | None = None) -> torch.Tensor:
    """The next frame of every stream: `state` (batch, width - 1, channels), the last inputs, is shifted in place.

    x (batch, channels); weight, bias and activation as in causal_conv; returns y (batch, channels) in x's dtype.  state: contiguous
    in x's dtype on the GPU.  No gradients.
    """
    what = "causal_conv_step"
    if activation in ACTIVATIONS:
        y = _step(what, "conv_step", state, x, state, weight, bias, ACTIVATIONS[activation])
        if y is not None:  # (as it mostly is: nothing to convert, nothing to refuse)
            return y
    _check_conv(what, x, weight, bias, activation, 2)
    (b, c), width = x.shape, weight.shape[1]
    if state.shape != (b, width - 1, c):
        raise ValueError(f"{what}: state must be (batch, width - 1, channels), got {tuple(state.shape)}")
    if state.dtype != x.dtype:
        raise TypeError(f"{what}: state must be {x.dtype}, got {state.dtype}")
    if _wants(x, state, weight, bias):
        raise RuntimeError(f"{what}: no gradients; use causal_conv, or torch.no_grad()")
    refuse_tangents(what, x, state, weight, bias)
    _require_hip(what)
    dev, out_dev = _check_state(what, state), x.device
    x, weight, bias = _features(x, dev), _channels(weight, dev), _channels(bias, dev)
    desc = _lib.ConvDesc(DTYPES[x.dtype], c, width, ACTIVATIONS[activation], b, 1, x.stride(0), 0)
    y = x.new_empty(b, c)
    launch(what, dev, _lib.lib().tfa_causal_conv_step, desc, addr(x), addr(weight), addr(bias), addr(state), addr(y))
    torch.autograd.graph.increment_version(state)
    return y if out_dev == dev else y.to(out_dev)


# ---------------------------------------------------------------------------------------------
# selective scan
# ---------------------------------------------------------------------------------------------


def _check_scan(what: str, x, dt, a, b, c, d, z, dt_bias, dims: int) -> None:
    if x.dim() != dims:
        raise ValueError(f"{what}: x must have {dims} dimensions, got {x.dim()}")
    dtype, shape = x.dtype, x.shape
    lead, channels = shape[:-1], shape[-1]
    if dtype not in DTYPES:
        raise TypeError(f"{what}: float32, bfloat16 or float16 expected, got {dtype}")
    if a.dim() != 2 or a.shape[0] != channels or a.shape[1] < 1 or channels < 1:
        raise ValueError(f"{what}: a must be (channels, states) for {channels} channels, got {tuple(a.shape)}")
    if a.dtype != torch.float32:
        raise TypeError(f"{what}: a must be float32, got {a.dtype}")
    if dt.shape != shape or (z is not None and z.shape != shape):
        raise ValueError(f"{what}: dt and z must be {tuple(shape)} as x, got {tuple(dt.shape)} and {None if z is None else tuple(z.shape)}")
    bs = b.shape
    if len(bs) != dims + 1 or bs[:-2] != lead or bs[-1] != a.shape[1] or bs[-2] < 1 or channels % bs[-2]:
        raise ValueError(f"{what}: b must be (*{tuple(lead)}, groups, {a.shape[1]}) with groups that divide {channels} channels, "
                         f"got {tuple(bs)}")
    if c.shape != bs:
        raise ValueError(f"{what}: c must be {tuple(bs)} as b, got {tuple(c.shape)}")
    if dt.dtype != dtype or b.dtype != dtype or c.dtype != dtype or (z is not None and z.dtype != dtype):
        raise TypeError(f"{what}: dt, b, c and z must be {dtype} as x")
    if d is not None or dt_bias is not None:
        _check_channels(what, channels, dtype, d=d, dt_bias=dt_bias)


def selective_scan(x: torch.Tensor, dt: torch.Tensor, a: torch.Tensor, b: torch.Tensor, c: torch.Tensor, *,
                   d: torch.Tensor | None = None, z: torch.Tensor | None = None, dt_bias: torch.Tensor | None = None,
                   softplus: bool = True, initial_state: torch.Tensor | None = None, lengths: torch.Tensor | None = None,
                   return_state: bool = False):
    """The selective scan of a state space layer over whole sequences, differentiable in every tensor but `lengths`.

    x, dt, z (batch, frames, channels), b, c (batch, frames, groups, states): one dtype of float32, bfloat16, float16; views of
    larger projections are taken as they are.  Neighbouring channels share a group of b and c.  a (channels, states) float32, at
    most 0 where steps are positive (above it states grow; -inf: no memory); d (skip) and dt_bias (channels,), float32 or x's dtype.  Steps are
    softplus(dt + dt_bias), or dt + dt_bias without softplus; z gates the output by silu(z).  Up to 64 states.
    initial_state: (batch, channels, states) float32.  lengths: (batch,) whole numbers; frames at and past a sequence's length
    are padding, whatever they hold: outputs and gradients are zero there.

    Returns y (batch, frames, channels) in x's dtype, and with return_state the state after each sequence's last frame (float32).
    States and sums are fp32.  A decay is rounded once a frame: where steps are the same from frame to frame, a state with a memory
    of m frames can be off by m 2^-25 of itself.  Gradients cannot be differentiated again, and there is no forward mode.  In a captured pass
    leaves are refused whose graph of an eager pass still lives: autograd would leave the capture for them.  A pass with gradients
    keeps n / 4 bytes a value of x, n being the states filled up to 4, 8, 16, 32 or 64, and takes n / 8 more (32 at 64) while the
    gradients of b and c are summed up.
    A value that is not finite makes NaN or infinities of its channel from its frame on (of b and c: of its group's channels), but for
    dt + dt_bias of -inf under softplus, a step of 0: such a frame leaves the state.
    """
    what = "selective_scan"
    out = _direct(what, what, x, dt, a, b, c, d, z, dt_bias, initial_state, lengths, softplus, return_state)
    if out is not None:  # (as it mostly is: nothing to convert, nothing to refuse)
        return out
    _check_scan(what, x, dt, a, b, c, d, z, dt_bias, 3)
    rows = x.shape[0]
    if initial_state is not None:
        if initial_state.shape != (rows, *a.shape):
            raise ValueError(f"{what}: initial_state must be (batch, channels, states), got {tuple(initial_state.shape)}")
        if initial_state.dtype != torch.float32:
            raise TypeError(f"{what}: states are float32, got {initial_state.dtype}")
    _check_lengths(what, lengths, rows)
    refuse_tangents(what, x, dt, a, b, c, d, z, dt_bias, initial_state)
    _require_hip(what)
    dev, out_dev = target_device(x, dt, b, c), x.device
    x, dt, b, c = _tokens(x, dev), _tokens(dt, dev), _tokens(b, dev), _tokens(c, dev)
    z = None if z is None else _tokens(z, dev)
    a, d, dt_bias = _dense(a, dev), _channels(d, dev), _channels(dt_bias, dev)
    state, lengths = _dense(initial_state, dev), _whole_numbers(lengths, dev)
    return _results(what, _lib.state_space().selective_scan(x, dt, a, b, c, d, z, dt_bias, state, lengths, softplus, return_state, True), out_dev)


def selective_scan_step(x: torch.Tensor, dt: torch.Tensor, a: torch.Tensor, b: torch.Tensor, c: torch.Tensor,
                        state: torch.Tensor, *, d: torch.Tensor | None = None, z: torch.Tensor | None = None,
                        dt_bias: torch.Tensor | None = None, softplus: bool = True) -> torch.Tensor:
    """The next frame of every stream: `state` (batch, channels, states) is updated in place.

    x, dt, z (batch, channels), b, c (batch, groups, states); the rest as in selective_scan; returns y (batch, channels) in x's
    dtype.  state: contiguous float32 on the GPU.  No gradients.
    """
    what = "selective_scan_step"
    y = _step(what, "scan_step", state, x, dt, a, b, c, state, d, z, dt_bias, softplus)
    if y is not None:  # (as it mostly is: nothing to convert, nothing to refuse)
        return y
    _check_scan(what, x, dt, a, b, c, d, z, dt_bias, 2)
    rows, channels = x.shape
    if state.shape != (rows, *a.shape):
        raise ValueError(f"{what}: state must be (batch, channels, states), got {tuple(state.shape)}")
    if state.dtype != torch.float32:
        raise TypeError(f"{what}: states are float32, got {state.dtype}")
    if _wants(x, dt, a, b, c, state, d, z, dt_bias):
        raise RuntimeError(f"{what}: no gradients; use selective_scan, or torch.no_grad()")
    refuse_tangents(what, x, dt, a, b, c, state, d, z, dt_bias)
    _require_hip(what)
    dev, out_dev = _check_state(what, state), x.device
    x, dt, b, c = _features(x, dev), _features(dt, dev), _features(b, dev), _features(c, dev)
    z = None if z is None else _features(z, dev)
    a, d, dt_bias = _dense(a, dev), _channels(d, dev), _channels(dt_bias, dev)
    (bs, bg, _), (cs, cg, _) = b.stride(), c.stride()
    desc = _lib.ScanDesc(DTYPES[x.dtype], channels, b.shape[1], a.shape[1], int(bool(softplus)), 0, rows, 1, x.stride(0), 0,
                         dt.stride(0), 0, 0 if z is None else z.stride(0), 0, bs, 0, bg, cs, 0, cg)
    y = x.new_empty(rows, channels)
    launch(what, dev, _lib.lib().tfa_selective_scan_step, desc, addr(x), addr(dt), addr(a), addr(b), addr(c), addr(d), addr(z),
           addr(dt_bias), addr(state), addr(y))
    torch.autograd.graph.increment_version(state)
    return y if out_dev == dev else y.to(out_dev)
