"""AdamW over all tensors of a model in few launches, states in 32 or 8 bits (csrc/kernels_adamw.hip).

``adamw_step`` is the step itself on lists of tensors, ``AdamW`` the torch optimizer on it.  8-bit states keep one fp32
scale s for every 256 values of a tensor: first moments s sgn(c) (c / 127)^2 of int8 codes c, second moments
s (c / 255)^4 of uint8 codes (at least 1 where there is any).  The reference has no counterpart.
"""

from __future__ import annotations

import torch

from . import _lib
from .attention import DTYPES, _on
from .dispatch import _require_hip, launch

BLOCK = 256  # values that share a scale


def _blocks(n: int) -> int:
    return -(-n // BLOCK)


def _listed(tensors):
    return tensors if tensors is None or type(tensors) is list else list(tensors)


_ADAM_LISTS = ("params", "grads", "exp_avgs", "exp_avg_sqs", "exp_avg_scales", "exp_avg_sq_scales", "masters")


@torch.no_grad()
def adamw_step(params, grads, exp_avgs, exp_avg_sqs, *, step: int, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8,
               weight_decay: float = 1e-2, exp_avg_scales=None, exp_avg_sq_scales=None, masters=None) -> None:
    """One AdamW step (decoupled weight decay) over lists of contiguous GPU tensors, in place.

    params: one dtype of float32, bfloat16, float16; grads: one dtype, the parameters' or float32.  exp_avgs and exp_avg_sqs:
    float32, or int8 and uint8 codes with their exp_avg_scales and exp_avg_sq_scales (float32, one for every 256 values).
    masters: float32 copies that the step is taken on; params then receive them rounded.  step counts from 1; it, lr and the other
    numbers are those of the call, so a captured call replays the same step, bias correction included.
    A gradient that is not finite makes its 8-bit block NaN, as it makes a float32 state.
    """
    what = "adamw_step"
    params, grads, masters = list(params), list(grads), _listed(masters)
    if not params:
        return
    eight = exp_avg_scales is not None
    if eight != (exp_avg_sq_scales is not None):
        raise ValueError(f"{what}: 8-bit states need both lists of scales")
    p_dtype, g_dtype, dev = params[0].dtype, grads[0].dtype if grads else None, params[0].device
    if p_dtype not in DTYPES:
        raise TypeError(f"{what}: float32, bfloat16 or float16 parameters expected, got {p_dtype}")
    if g_dtype not in (p_dtype, torch.float32):
        raise TypeError(f"{what}: gradients must be {p_dtype} or float32, got {g_dtype}")
    if step < 1 or int(step) != step:
        raise ValueError(f"{what}: steps count from 1, got {step}")
    _require_hip(what)
    if dev.type != "cuda":
        raise ValueError(f"{what}: the parameters are updated in place and must be on the GPU")
    moments = (torch.int8, torch.uint8) if eight else (torch.float32, torch.float32)
    table = _lib.tensor_table()(what, _ADAM_LISTS,
                                (params, grads, *map(_listed, (exp_avgs, exp_avg_sqs, exp_avg_scales, exp_avg_sq_scales)), masters),
                                (p_dtype, g_dtype, *moments, torch.float32, torch.float32, torch.float32), dev.index)
    desc = _lib.AdamDesc(DTYPES[p_dtype], DTYPES[g_dtype], 8 if eight else 32, 0, int(step), lr, betas[0], betas[1], eps,
                         weight_decay)
    launch(what, dev, _lib.lib().tfa_adamw_step, len(params), table, desc)
    # (autograd sees the update as it sees any in-place operation)
    torch.autograd.graph.increment_version(params)
    if masters is not None:
        torch.autograd.graph.increment_version(masters)


@torch.no_grad()
def adamw_state_values(codes, scales, out=None) -> list[torch.Tensor]:
    """The float32 values that 8-bit states stand for: first moments of int8 codes, second moments of uint8 codes."""
    what = "adamw_state_values"
    codes = list(codes)
    if not codes:
        return []
    dtype, dev = codes[0].dtype, codes[0].device
    if dtype not in (torch.int8, torch.uint8):
        raise TypeError(f"{what}: codes are int8 (first moments) or uint8 (second moments), got {dtype}")
    _require_hip(what)
    if dev.type != "cuda":
        raise ValueError(f"{what}: the states must be on the GPU")
    out = [torch.empty(c.shape, dtype=torch.float32, device=dev) for c in codes] if out is None else _listed(out)
    table = _lib.tensor_table()(what, ("codes", "scales", "out"), (codes, _listed(scales), out),
                                (dtype, torch.float32, torch.float32), dev.index)
    launch(what, dev, _lib.lib().tfa_adamw_state_values, len(codes), table, int(dtype == torch.uint8))
    torch.autograd.graph.increment_version(out)
    return out


class AdamW(torch.optim.Optimizer):
    """torch.optim.AdamW's update through ``adamw_step``, all tensors of a group and dtype in one call.

    state_bits: 32, or 8 for states of a quarter of the size (tensors below 4096 values keep 32 bits: they cost nothing, and
    norms and biases are the most sensitive).  Values whose gradients are 1e3 to 1e5 times smaller than others of their 256 may
    update several times faster with 8 bits (up to 13 lr for 1), still smaller ones slower.
    master_weights: float32 copies of 16-bit parameters, on which the step is taken (without them updates below half a unit in
    the last place of a 16-bit parameter are lost).  A parameter that was written between two steps (weights loaded, clamped)
    takes its master along; writes through ``.data`` are not seen.
    Parameters must be contiguous.  The step count and lr live on the host: ``step`` is refused while a graph is captured,
    whose replays would repeat one step's.
    """

    def __init__(self, params, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2,
                 state_bits: int = 32, master_weights: bool = True):
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits,
                                      master_weights=master_weights))

    def add_param_group(self, param_group):
        own = {**self.defaults, **param_group}
        betas = own["betas"]
        if own["state_bits"] not in (32, 8):
            raise ValueError(f"AdamW: state_bits must be 32 or 8, got {own['state_bits']}")
        if not (0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0):
            raise ValueError(f"AdamW: betas must be in [0, 1), got {betas}")
        if own["lr"] < 0.0 or own["eps"] < 0.0 or own["weight_decay"] < 0.0:
            raise ValueError("AdamW: lr, eps and weight_decay must not be negative")
        super().add_param_group(param_group)

    def _state_of(self, p: torch.Tensor, group: dict) -> dict:
        state = self.state[p]
        if not state:
            eight = group["state_bits"] == 8 and p.numel() >= 4096
            flat = {"dtype": torch.float32, "device": p.device}
            state["step"] = 0
            state["exp_avg"] = torch.zeros(p.shape, dtype=torch.int8 if eight else torch.float32, device=p.device)
            state["exp_avg_sq"] = torch.zeros(p.shape, dtype=torch.uint8 if eight else torch.float32, device=p.device)
            if eight:
                state["exp_avg_scale"] = torch.zeros(_blocks(p.numel()), **flat)
                state["exp_avg_sq_scale"] = torch.zeros(_blocks(p.numel()), **flat)
            if p.dtype != torch.float32 and group["master_weights"]:
                state["master"] = p.detach().float().contiguous()
        elif "master" in state and state.get("seen") != p._version:
            # written since the last step (weights that were loaded, clamped, averaged): those values hold, others keep their master
            master = state["master"]
            master.copy_(torch.where(master.to(p.dtype) == p, master, p.float()))
        return state

    @torch.no_grad()
    def step(self, closure=None):
        if torch.cuda.is_initialized() and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AdamW: step cannot be captured in a graph: its replays would repeat this step's bias correction")
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            calls: dict = {}
            for p in group["params"]:
                if p.grad is None:
                    continue
                if p.grad.is_sparse:
                    raise RuntimeError("AdamW: sparse gradients are not supported")
                state = self._state_of(p, group)
                key = (p.dtype, p.grad.dtype, p.device, state["step"] + 1, "exp_avg_scale" in state, "master" in state)
                calls.setdefault(key, []).append((p, _on(p.grad, p.device).contiguous(), state))
            for (_, _, _, step, eight, master), items in calls.items():
                states = [s for _, _, s in items]
                adamw_step([p for p, _, _ in items], [g for _, g, _ in items], [s["exp_avg"] for s in states],
                           [s["exp_avg_sq"] for s in states], step=step, lr=group["lr"], betas=group["betas"],
                           eps=group["eps"], weight_decay=group["weight_decay"],
                           exp_avg_scales=[s["exp_avg_scale"] for s in states] if eight else None,
                           exp_avg_sq_scales=[s["exp_avg_sq_scale"] for s in states] if eight else None,
                           masters=[s["master"] for s in states] if master else None)
                for p, _, s in items:
                    s["step"] = step
                    if master:
                        s["seen"] = p._version
        return loss

    def load_state_dict(self, state_dict):
        super().load_state_dict(state_dict)
        # torch casts floating states to their parameter's dtype: states are fp32 whatever it is
        for group, saved in zip(self.param_groups, state_dict["param_groups"]):
            for p, index in zip(group["params"], saved["params"]):
                for name, value in state_dict["state"].get(index, {}).items():
                    if torch.is_tensor(value):
                        self.state[p][name] = value.to(p.device).clone()
                if p in self.state:
                    self.state[p].pop("seen", None)
