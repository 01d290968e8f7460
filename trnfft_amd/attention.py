"""Linear attention with a decay for each head, over frames (csrc/kernels_attention.hip).

    S_t = exp(log_decay[h]) S_{t-1} + k_t v_t^T,    o_t = scale * S_t^T q_t

A sequence model for STFT frames: frame t sees the frames up to it, older ones by exp(log_decay[h]) less for every
frame, and what a stream has to keep is one (key_dim, value_dim) state a head, however long it runs.
``linear_attention`` takes whole sequences (training, prompts, blocks of a stream), ``linear_attention_step`` one frame.
The reference has no counterpart.
"""

from __future__ import annotations

import ctypes
import math

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .dispatch import _require_hip, addr, launch, refuse_tangents, target_device

DTYPES = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16}


def _check_operands(what: str, q, k, v, log_decay, dims: int) -> int:
    """Shapes and types of a call; returns the number of heads."""
    qs, ks, vs = q.shape, k.shape, v.shape
    if not len(qs) == len(ks) == len(vs) == dims:
        raise ValueError(f"{what}: q, k and v must have {dims} dimensions, got {len(qs)}, {len(ks)} and {len(vs)}")
    dtype = q.dtype
    if dtype not in DTYPES:
        raise TypeError(f"{what}: float32, bfloat16 or float16 expected, got {dtype}")
    if k.dtype != dtype or v.dtype != dtype:
        raise TypeError(f"{what}: q, k and v must have one dtype, got {dtype}, {k.dtype} and {v.dtype}")
    if log_decay.dim() != 1 or log_decay.dtype != torch.float32:
        raise TypeError(f"{what}: log_decay must be a float32 vector, one value for each head")
    if not qs[:-2] == ks[:-2] == vs[:-2]:
        raise ValueError(f"{what}: q, k and v must agree up to their heads")
    if qs[-1] != ks[-1]:
        raise ValueError(f"{what}: q and k must have the same features, got {qs[-1]} and {ks[-1]}")
    if qs[-1] < 1 or vs[-1] < 1:
        raise ValueError(f"{what}: heads must have features")
    heads = log_decay.shape[0]
    for n in (qs[-2], ks[-2], vs[-2]):
        if n < 1 or heads < 1 or heads % n:
            raise ValueError(f"{what}: the {heads} heads of log_decay must be a multiple of q's, k's and v's ({n})")
    return heads


def _scale(scale, key_dim: int, what: str) -> float:
    scale = key_dim**-0.5 if scale is None else float(scale)
    if not math.isfinite(scale) or scale == 0.0:
        raise ValueError(f"{what}: scale must be finite and not zero")
    return scale


def _on(x: torch.Tensor, dev: torch.device) -> torch.Tensor:
    """x on dev, as its memory says it (the imaginary part of a conjugated tensor is a view that negates what it reads)."""
    x = x.resolve_neg() if x.is_neg() else x
    return x if x.device == dev else x.to(dev)


def _features(x: torch.Tensor, dev: torch.device) -> torch.Tensor:
    """x on dev with contiguous features (x itself where it is so)."""
    x = _on(x, dev)
    return x if x.stride(-1) == 1 or x.shape[-1] == 1 else x.contiguous()


def _rows(x: torch.Tensor, dev: torch.device) -> torch.Tensor:
    """The same at a 16-byte boundary."""
    x = _features(x, dev)
    return x if x.data_ptr() % 16 == 0 else x.clone(memory_format=torch.contiguous_format)


def _desc(q, k, v, heads: int, scale: float) -> _lib.AttnDesc:
    (b, t, qh, dk), kh, (vh, dv) = q.shape, k.shape[2], v.shape[2:]
    return _lib.AttnDesc(DTYPES[q.dtype], heads, qh, kh, vh, dk, dv, scale, b, t, *q.stride()[:3], *k.stride()[:3],
                         *v.stride()[:3])


def _workspace(desc: _lib.AttnDesc, backward: int, dev: torch.device, what: str) -> torch.Tensor | None:
    nbytes = ctypes.c_size_t()
    _lib.check(_lib.lib().tfa_linear_attention_workspace_size(desc, backward, nbytes), what)
    return torch.empty(nbytes.value, dtype=torch.uint8, device=dev) if nbytes.value else None


def _forward(q, k, v, log_decay, lengths, state, scale: float, want_state: bool):
    b, t, _, _ = q.shape
    heads, dev, what = log_decay.numel(), q.device, "linear_attention"
    desc = _desc(q, k, v, heads, scale)
    out = q.new_empty(b, t, heads, v.shape[3])
    last = torch.empty(b, heads, q.shape[3], v.shape[3], dtype=torch.float32, device=dev) if want_state else None
    ws = _workspace(desc, 0, dev, what)
    launch(what, dev, _lib.lib().tfa_linear_attention, desc, addr(q), addr(k), addr(v), addr(log_decay), addr(lengths),
           addr(state), addr(out), addr(last), addr(ws))
    return out, last


class _LinearAttentionFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, log_decay, state, lengths, scale):
        ctx.set_materialize_grads(False)
        ctx.scale = scale
        ctx.save_for_backward(q, k, v, log_decay, state, lengths)
        return _forward(q, k, v, log_decay, lengths, state, scale, True)

    @staticmethod
    @once_differentiable
    def backward(ctx, g_out, g_last):
        q, k, v, log_decay, state, lengths = ctx.saved_tensors
        need = ctx.needs_input_grad
        heads, dev, what = log_decay.numel(), q.device, "linear_attention backward"
        desc = _desc(q, k, v, heads, ctx.scale)
        if g_out is None:
            g_out = q.new_zeros(*q.shape[:2], heads, v.shape[3])
        g_out = _rows(_on(g_out, dev).contiguous(), dev)
        g_last = None if g_last is None else _on(g_last, dev).contiguous()
        # (the decays' gradient comes with the queries' and keys', the state's with the values')
        d_q = torch.empty(q.shape, dtype=q.dtype, device=dev) if need[0] or need[3] else None
        d_k = torch.empty(k.shape, dtype=q.dtype, device=dev) if need[1] or need[3] else None
        d_state = torch.empty_like(state) if state is not None and need[4] else None
        d_v = torch.empty(v.shape, dtype=q.dtype, device=dev) if need[2] or d_state is not None else None
        d_g = torch.empty_like(log_decay) if need[3] else None
        ws = _workspace(desc, 2 if need[3] else 1, dev, what)
        launch(what, dev, _lib.lib().tfa_linear_attention_backward, desc, addr(q), addr(k), addr(v), addr(log_decay),
               addr(lengths), addr(state), addr(g_out), addr(g_last), addr(d_q), addr(d_k), addr(d_v), addr(d_g),
               addr(d_state), addr(ws))
        return d_q if need[0] else None, d_k if need[1] else None, d_v if need[2] else None, d_g, d_state, None, None


def linear_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor, *,
                     scale: float | None = None, initial_state: torch.Tensor | None = None,
                     lengths: torch.Tensor | None = None, return_state: bool = False):
    """Causal linear attention with decays over whole sequences, differentiable in every tensor but `lengths`.

    q (batch, frames, q_heads, key_dim), k (batch, frames, k_heads, key_dim), v (batch, frames, v_heads, value_dim): one
    dtype of float32, bfloat16, float16; views of a larger projection are taken as they are.  log_decay: (heads,) float32, at
    most 0 (-inf: no memory); heads is a multiple of each operand's heads, whose neighbouring heads then share it.
    scale: key_dim ** -0.5 unless given.  initial_state: (batch, heads, key_dim, value_dim) float32.  lengths: (batch,) whole
    numbers; frames at and past a sequence's length are padding, whatever they hold: outputs and gradients are zero there.

    Returns o (batch, frames, heads, value_dim) in q's dtype, and with return_state the state after each
    sequence's last frame (float32).  States and sums are fp32.  Gradients cannot be differentiated again, and there is no
    forward mode.
    A value that is not finite makes NaN (or infinities) of what depends on it by the recurrence: its frame and those after it.
    """
    what = "linear_attention"
    heads = _check_operands(what, q, k, v, log_decay, 4)
    scale = _scale(scale, q.shape[-1], what)
    b = q.shape[0]
    if initial_state is not None:
        if initial_state.shape != (b, heads, q.shape[-1], v.shape[-1]):
            raise ValueError(f"{what}: initial_state must be (batch, heads, key_dim, value_dim), got "
                             f"{tuple(initial_state.shape)}")
        if initial_state.dtype != torch.float32:
            raise TypeError(f"{what}: states are float32, got {initial_state.dtype}")
    if lengths is not None:
        if lengths.shape != (b,):
            raise ValueError(f"{what}: lengths must be ({b},), got {tuple(lengths.shape)}")
        if lengths.dtype not in (torch.int64, torch.int32, torch.int16, torch.uint8, torch.int8):
            raise TypeError(f"{what}: lengths must be whole numbers, got {lengths.dtype}")
    refuse_tangents(what, q, k, v, log_decay, initial_state)
    _require_hip(what)
    dev, out_dev = target_device(q, k, v), q.device
    q, k, v = _rows(q, dev), _rows(k, dev), _rows(v, dev)
    log_decay = _on(log_decay, dev).contiguous()
    state = None if initial_state is None else _on(initial_state, dev).contiguous()
    lengths = None if lengths is None else lengths.to(dev, torch.int64).contiguous()
    if torch.is_grad_enabled() and any(x is not None and x.requires_grad for x in (q, k, v, log_decay, state)):
        out, last = _LinearAttentionFn.apply(q, k, v, log_decay, state, lengths, scale)
    else:
        out, last = _forward(q, k, v, log_decay, lengths, state, scale, return_state)
    if out_dev != dev:
        out, last = out.to(out_dev), None if last is None else last.to(out_dev)
    return (out, last) if return_state else out


def linear_attention_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor,
                          state: torch.Tensor, *, scale: float | None = None) -> torch.Tensor:
    """The next frame of every stream: `state` (batch, heads, key_dim, value_dim) is updated in place.

    q (batch, q_heads, key_dim), k (batch, k_heads, key_dim), v (batch, v_heads, value_dim) and log_decay as in
    linear_attention; returns o (batch, heads, value_dim) in q's dtype.  state: contiguous float32 on the GPU.  No gradients.
    """
    what = "linear_attention_step"
    heads = _check_operands(what, q, k, v, log_decay, 3)
    (b, qh, dk), kh, (vh, dv) = q.shape, k.shape[1], v.shape[1:]
    scale = _scale(scale, dk, what)
    if state.shape != (b, heads, dk, dv):
        raise ValueError(f"{what}: state must be (batch, heads, key_dim, value_dim), got {tuple(state.shape)}")
    if state.dtype != torch.float32:
        raise TypeError(f"{what}: states are float32, got {state.dtype}")
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or log_decay.requires_grad
                                    or state.requires_grad):
        raise RuntimeError(f"{what}: no gradients; use linear_attention, or torch.no_grad()")
    refuse_tangents(what, q, k, v, log_decay, state)
    _require_hip(what)
    if not state.is_cuda or not state.is_contiguous() or state.is_neg():
        raise ValueError(f"{what}: the state is updated in place and must be contiguous on the GPU")
    dev, out_dev = state.device, q.device
    q, k, v, log_decay = _features(q, dev), _features(k, dev), _features(v, dev), _on(log_decay, dev).contiguous()
    (qb, qs, _), (kb, ks, _), (vb, vs, _) = q.stride(), k.stride(), v.stride()
    desc = _lib.AttnDesc(DTYPES[q.dtype], heads, qh, kh, vh, dk, dv, scale, b, 1, qb, 0, qs, kb, 0, ks, vb, 0, vs)
    out = q.new_empty(b, heads, dv)
    launch(what, dev, _lib.lib().tfa_linear_attention_step, desc, addr(q), addr(k), addr(v), addr(log_decay), addr(state),
           addr(out))
    torch.autograd.graph.increment_version(state)
    return out if out_dev == dev else out.to(out_dev)
