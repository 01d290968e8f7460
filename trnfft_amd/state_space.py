"""The operators of a selective state space layer over frames (csrc/kernels_conv.hip, csrc/scan_blocks.h).

    causal_conv:     y_t = act(bias + sum_j weight[:, j] x_{t - width + 1 + j})
    selective_scan:  s_t = softplus(dt_t + dt_bias),  h_t = exp(s_t a) h_{t-1} + s_t x_t b_t,  y_t = (c_t . h_t + d x_t) silu(z_t)

A sequence model for STFT frames whose memory each frame sets for itself: what a stream keeps is the last inputs of a short
filter and a few states a channel, however long it runs.  ``causal_conv`` and ``selective_scan`` take whole sequences
(training, prompts, blocks of a stream), their ``_step`` one frame.  The reference has no counterpart.
"""

from __future__ import annotations

import ctypes

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .attention import DTYPES, _features, _on
from .dispatch import _require_hip, _use_hip, addr, launch, refuse_tangents, step_here, target_device
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


def _conv_forward(x, weight, bias, state, lengths, activation, want_state: bool):
    b, t, c = x.shape
    width, dev, what = weight.shape[1], x.device, "causal_conv"
    desc = _lib.ConvDesc(DTYPES[x.dtype], c, width, activation, b, t, *x.stride()[:2])
    y = x.new_empty(b, t, c)
    last = x.new_empty(b, width - 1, c) if want_state else None
    launch(what, dev, _lib.lib().tfa_causal_conv, desc, addr(x), addr(weight), addr(bias), addr(lengths), addr(state), addr(y),
           addr(last))
    return y, last


class _CausalConvFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, state, lengths, activation):
        ctx.set_materialize_grads(False)
        ctx.activation = activation
        ctx.save_for_backward(x, weight, bias, state, lengths)
        return _conv_forward(x, weight, bias, state, lengths, activation, True)

    @staticmethod
    @once_differentiable
    def backward(ctx, g_y, g_last):
        x, weight, bias, state, lengths = ctx.saved_tensors
        (b, t, c), width, dev, what, need = x.shape, weight.shape[1], x.device, "causal_conv backward", ctx.needs_input_grad
        desc = _lib.ConvDesc(DTYPES[x.dtype], c, width, ctx.activation, b, t, *x.stride()[:2])
        g_y = x.new_zeros(b, t, c) if g_y is None else _dense(g_y, dev)
        g_last = _dense(g_last, dev)
        d_x = x.new_empty(b, t, c) if need[0] else None
        d_w = torch.empty_like(weight) if need[1] else None
        d_b = torch.empty_like(bias) if bias is not None and need[2] else None
        d_s = torch.empty_like(state) if state is not None and need[3] else None
        ws = None
        if need[1] or need[2]:
            nbytes = ctypes.c_size_t()
            _lib.check(_lib.lib().tfa_causal_conv_workspace_size(desc, nbytes), what)
            ws = torch.empty(nbytes.value, dtype=torch.uint8, device=dev) if nbytes.value else None
        launch(what, dev, _lib.lib().tfa_causal_conv_backward, desc, addr(x), addr(weight), addr(bias), addr(lengths), addr(state),
               addr(g_y), addr(g_last), addr(d_x), addr(d_w), addr(d_b), addr(d_s), addr(ws))
        return d_x, d_w, d_b, d_s, None, None


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
    if _wants(x, weight, bias, state):
        y, last = _CausalConvFn.apply(x, weight, bias, state, lengths, ACTIVATIONS[activation])
    else:
        y, last = _conv_forward(x, weight, bias, state, lengths, ACTIVATIONS[activation], return_state)
    if out_dev != dev:
        y, last = y.to(out_dev), None if last is None else last.to(out_dev)
    return (y, last) if return_state else y


def causal_conv_step(x: torch.Tensor, state: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *,
                     activation: str | None = None) -> torch.Tensor:
    """The next frame of every stream: `state` (batch, width - 1, channels), the last inputs, is shifted in place.

    x (batch, channels); weight, bias and activation as in causal_conv; returns y (batch, channels) in x's dtype.  state: contiguous
    in x's dtype on the GPU.  No gradients.
    """
    what = "causal_conv_step"
    if activation in ACTIVATIONS and _use_hip():  # (as it mostly is: nothing to convert, nothing to refuse)
        y = step_here(what, "conv_step", state, x, state, weight, bias, ACTIVATIONS[activation])
        if y is not None:
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


def _scan_desc(x, dt, b, c, z, softplus: bool) -> _lib.ScanDesc:
    (rows, t, channels), (groups, n) = x.shape, b.shape[2:]
    return _lib.ScanDesc(DTYPES[x.dtype], channels, groups, n, int(softplus), 0, rows, t, *x.stride()[:2], *dt.stride()[:2],
                         *((0, 0) if z is None else z.stride()[:2]), *b.stride()[:3], *c.stride()[:3])


def _scan_forward(x, dt, a, b, c, d, z, dt_bias, state, lengths, softplus: bool, want_state: bool, want_kept: bool):
    (rows, t, channels), n, dev, what = x.shape, a.shape[1], x.device, "selective_scan"
    desc = _scan_desc(x, dt, b, c, z, softplus)
    sizes = [ctypes.c_size_t() for _ in range(3)]
    _lib.check(_lib.lib().tfa_selective_scan_sizes(desc, *sizes), what)
    kept, ws = (torch.empty(s.value, dtype=torch.uint8, device=dev) if s.value and want else None
                for s, want in zip(sizes, (want_kept, True)))
    y = x.new_empty(rows, t, channels)
    last = torch.empty(rows, channels, n, dtype=torch.float32, device=dev) if want_state else None
    launch(what, dev, _lib.lib().tfa_selective_scan, desc, addr(x), addr(dt), addr(a), addr(b), addr(c), addr(d), addr(z),
           addr(dt_bias), addr(lengths), addr(state), addr(y), addr(last), addr(kept), addr(ws))
    return y, last, kept


class _SelectiveScanFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, dt, a, b, c, d, z, dt_bias, state, lengths, softplus):
        ctx.set_materialize_grads(False)
        ctx.softplus = softplus
        y, last, kept = _scan_forward(x, dt, a, b, c, d, z, dt_bias, state, lengths, softplus, True, True)
        ctx.save_for_backward(x, dt, a, b, c, d, z, dt_bias, state, lengths, kept)
        return y, last

    @staticmethod
    @once_differentiable
    def backward(ctx, g_y, g_last):
        x, dt, a, b, c, d, z, dt_bias, state, lengths, kept = ctx.saved_tensors
        dev, what = x.device, "selective_scan backward"
        desc = _scan_desc(x, dt, b, c, z, ctx.softplus)
        sizes = [ctypes.c_size_t() for _ in range(3)]
        _lib.check(_lib.lib().tfa_selective_scan_sizes(desc, *sizes), what)
        ws = torch.empty(sizes[2].value, dtype=torch.uint8, device=dev) if sizes[2].value else None
        g_y = torch.zeros(x.shape, dtype=x.dtype, device=dev) if g_y is None else _dense(g_y, dev)
        g_last = _dense(g_last, dev)
        grads = [torch.empty(v.shape, dtype=v.dtype, device=dev) if v is not None and need else None
                 for v, need in zip((x, dt, a, b, c, d, z, dt_bias, state), ctx.needs_input_grad)]
        d_x, d_dt, d_a, d_b, d_c, d_d, d_z, d_bias, d_state = map(addr, grads)
        table = _lib.ScanGrads(addr(g_y), addr(g_last), d_x, d_dt, d_b, d_c, d_z, d_a, d_d, d_bias, d_state)
        launch(what, dev, _lib.lib().tfa_selective_scan_backward, desc, addr(x), addr(dt), addr(a), addr(b), addr(c), addr(d),
               addr(z), addr(dt_bias), addr(lengths), addr(state), addr(kept), table, addr(ws))
        return *grads, None, None


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
    States and sums are fp32.  Gradients cannot be differentiated again, and there is no forward mode.
    A value that is not finite makes NaN or infinities of its channel from its frame on (of b and c: of its group's channels).
    """
    what = "selective_scan"
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
    if _wants(x, dt, a, b, c, d, z, dt_bias, state):
        y, last = _SelectiveScanFn.apply(x, dt, a, b, c, d, z, dt_bias, state, lengths, bool(softplus))
    else:
        y, last, _ = _scan_forward(x, dt, a, b, c, d, z, dt_bias, state, lengths, bool(softplus), return_state, False)
    if out_dev != dev:
        y, last = y.to(out_dev), None if last is None else last.to(out_dev)
    return (y, last) if return_state else y


def selective_scan_step(x: torch.Tensor, dt: torch.Tensor, a: torch.Tensor, b: torch.Tensor, c: torch.Tensor,
                        state: torch.Tensor, *, d: torch.Tensor | None = None, z: torch.Tensor | None = None,
                        dt_bias: torch.Tensor | None = None, softplus: bool = True) -> torch.Tensor:
    """The next frame of every stream: `state` (batch, channels, states) is updated in place.

    x, dt, z (batch, channels), b, c (batch, groups, states); the rest as in selective_scan; returns y (batch, channels) in x's
    dtype.  state: contiguous float32 on the GPU.  No gradients.
    """
    what = "selective_scan_step"
    if _use_hip():  # (as it mostly is: nothing to convert, nothing to refuse)
        y = step_here(what, "scan_step", state, x, dt, a, b, c, state, d, z, dt_bias, softplus)
        if y is not None:
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
