"""A selective state space layer on STFT frames: its operators, their training passes, their forms for streams that get
one frame at a time, and the clipping of a model's gradients, as cases that can be timed and checked.

* the short causal convolution over frames with an activation, and its step;
* the selective scan h_t = exp(dt_t a) h_{t-1} + dt_t b_t x_t, y_t = c_t . h_t + d x_t, gated by silu(z_t), and its step;
* the global norm of all gradients of a model, and their clipping.

Sizes: the benchmark's 64 signals of 10 s (626 frames of hop 256, 1001 frames of hop 160), the complex linear layer's
1024 features, and generic ones.  Every operator has a plain form of elementary torch operations in fp32 here (norms in
fp64), rounded once at the end; with ``own`` set, ``run`` calls the package instead.
"""

from __future__ import annotations

import math
import random

import torch

own = False

_DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_ALIGN = 256  # values: where tensors start in a flat bucket


def listed():
    return [
        # one stream's next frame: nothing but latency
        {"name": "conv_step_1x1024_fp32", "op": "conv_step", "b": 1, "c": 1024, "width": 4, "act": "silu", "bias": True,
         "dtype": "fp32"},
        # the next frame of 256 streams served together
        {"name": "conv_step_256x2048_bf16", "op": "conv_step", "b": 256, "c": 2048, "width": 4, "act": "silu", "bias": True,
         "dtype": "bf16"},
        # the benchmark's 64 signals, ragged, one half of a layer's input projection; the streams go on from the state
        {"name": "conv_64x626x1024_bf16", "op": "conv", "b": 64, "t": 626, "c": 1024, "width": 4, "act": "silu",
         "bias": True, "dtype": "bf16", "lengths": True, "state": True, "packed": True, "grad": False},
        # a training pass of a wide layer
        {"name": "conv_train_8x4096x2048_bf16", "op": "conv", "b": 8, "t": 4096, "c": 2048, "width": 4, "act": "silu",
         "bias": True, "dtype": "bf16", "lengths": False, "state": False, "packed": False, "grad": True},
        # one stream's next frame
        {"name": "scan_step_1x512x16_fp32", "op": "scan_step", "b": 1, "c": 512, "n": 16, "groups": 1, "gate": True,
         "softplus": True, "dtype": "fp32"},
        # the next frame of 256 streams: the states are most of what is moved
        {"name": "scan_step_256x2048x16_bf16", "op": "scan_step", "b": 256, "c": 2048, "n": 16, "groups": 1, "gate": True,
         "softplus": True, "dtype": "bf16"},
        # the benchmark's 64 signals, ragged; b and c are columns of one projection, z is half of another; state kept
        {"name": "scan_64x626x512_bf16", "op": "scan", "b": 64, "t": 626, "c": 512, "n": 16, "groups": 1, "gate": True,
         "softplus": True, "dtype": "bf16", "lengths": True, "state": True, "packed": True, "grad": False},
        # one long recording: few channels, the long axis has to be shared out
        {"name": "scan_1x65536x1024_bf16", "op": "scan", "b": 1, "t": 65536, "c": 1024, "n": 16, "groups": 1, "gate": True,
         "softplus": True, "dtype": "bf16", "lengths": False, "state": False, "packed": True, "grad": False},
        # training on short utterances in fp32: an odd state size, two groups, ragged, from a state
        {"name": "scan_train_4x1001x384_fp32", "op": "scan", "b": 4, "t": 1001, "c": 384, "n": 12, "groups": 2,
         "gate": True, "softplus": True, "dtype": "fp32", "lengths": True, "state": True, "packed": False, "grad": True},
        # a training pass of a wide layer: every gradient
        {"name": "scan_train_8x4096x2048_bf16", "op": "scan", "b": 8, "t": 4096, "c": 2048, "n": 16, "groups": 1,
         "gate": True, "softplus": True, "dtype": "bf16", "lengths": False, "state": False, "packed": False, "grad": True},
        # the gradients of a small denoiser, over the bound
        {"name": "clip_24x0.5M_fp32", "op": "clip", "tensors": 24, "numel": 500_000, "dtype": "fp32", "clips": True},
        # those of a large model as they come out of a reduced bucket, over the bound
        {"name": "clip_320x120M_bf16", "op": "clip", "tensors": 320, "numel": 120_000_000, "dtype": "bf16", "clips": True},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["conv", "conv", "conv_step", "scan", "scan", "scan", "scan_step", "clip"])
    dtype = rng.choice(["fp32", "bf16", "bf16", "fp16"])
    if op == "clip":
        tensors = _log_int(rng, 1, 400)
        return {"op": op, "tensors": tensors, "numel": _log_int(rng, max(1000, 4 * tensors), 60_000_000), "dtype": dtype,
                "clips": rng.random() < 0.7}
    if op in ("conv", "conv_step"):
        base = {"op": op, "width": rng.choice([2, 3, 4, 4, 4, 5, 8]), "act": rng.choice(["silu", "silu", "none"]),
                "bias": rng.random() < 0.8, "dtype": dtype}
        c = 8 * _log_int(rng, 2, 384) if rng.random() < 0.7 else _log_int(rng, 5, 4000)
        if op == "conv_step":
            return {**base, "b": _log_int(rng, 1, 256), "c": c}
        grad = rng.random() < 0.5
        most = (1 << 24 if dtype == "fp32" else 1 << 25) // c
        t = _log_int(rng, 1, min(65536, most))
        return {**base, "b": _log_int(rng, 1, max(1, min(64, most // t))), "t": t, "c": c, "lengths": rng.random() < 0.5,
                "state": rng.random() < 0.5, "packed": not grad and rng.random() < 0.5, "grad": grad}
    n = rng.choice([4, 8, 12, 16, 16, 16, 32, 64]) if rng.random() < 0.8 else rng.randint(1, 64)
    groups = rng.choice([1, 1, 1, 2, 4])
    c = groups * (16 * _log_int(rng, 1, 128 // groups) if rng.random() < 0.7 else _log_int(rng, 3, 2000 // groups))
    base = {"op": op, "c": c, "n": n, "groups": groups, "gate": rng.random() < 0.8, "softplus": rng.random() < 0.8,
            "dtype": dtype}
    if op == "scan_step":
        return {**base, "b": _log_int(rng, 1, 256)}
    grad = rng.random() < 0.5
    most = min(1 << 29, (1 << 24 if dtype == "fp32" else 1 << 25) * n) // (c * n)
    t = _log_int(rng, 1, min(65536, most))
    return {**base, "b": _log_int(rng, 1, max(1, min(64, most // t))), "t": t, "lengths": rng.random() < 0.5,
            "state": rng.random() < 0.5, "packed": not grad and rng.random() < 0.5, "grad": grad}


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------


def _lengths(case, g):
    """Utterances of a batch end early: whole ones, half ones and very short ones."""
    if not case["lengths"]:
        return None
    lengths = (torch.rand(case["b"], generator=g, device="cuda") * (case["t"] + 1)).to(torch.int64).clamp_(max=case["t"])
    lengths[0] = case["t"]
    return lengths


def _sizes(case):
    """Sizes of a model's tensors: matrices over three decades of size, vectors between them, ordinary and odd."""
    r = random.Random(case["tensors"] * 7919 + case["numel"])
    weight = [math.exp(r.uniform(0.0, 6.9)) if i % 3 != 2 else 0.05 for i in range(case["tensors"])]
    total = sum(weight)
    return [max(1, int(case["numel"] * w / total)) for w in weight]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype = _DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, to=dtype):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(to)

    st = {"case": case}
    if case["op"] == "clip":
        sizes = _sizes(case)
        starts, end = [], 0
        for s in sizes:
            starts.append(end)
            end += -(-s // _ALIGN) * _ALIGN
        inside = torch.zeros(end, dtype=torch.bool, device="cuda")
        for s, at in zip(sizes, starts):
            inside[at:at + s] = True
        st["bucket"] = (torch.randn(end, generator=g, device="cuda") * 1e-2 * inside).to(dtype)
        st["grads"] = st["bucket"].clone()
        st["list"] = [st["grads"][at:at + s] for s, at in zip(sizes, starts)]
        # (the norm is about 1e-2 sqrt(numel))
        st["max_norm"] = 1e-2 * math.sqrt(sum(sizes)) * (0.3 if case["clips"] else 3.0)
        return st
    b, c = case["b"], case["c"]
    if case["op"] in ("conv", "conv_step"):
        width = case["width"]
        st["weight"] = normal(c, width, scale=width**-0.5, to=torch.float32)
        st["bias"] = normal(c, scale=0.1, to=torch.float32) if case["bias"] else None
        if case["op"] == "conv_step":
            st["x"], st["state"] = normal(b, c), normal(b, width - 1, c)
            return st
        if case["packed"]:
            st["xz"] = normal(b, case["t"], 2 * c)
        else:
            st["x"] = normal(b, case["t"], c)
        st["state"] = normal(b, width - 1, c) if case["state"] else None
        st["lengths"] = _lengths(case, g)
        if case["grad"]:
            st["dy"] = normal(b, case["t"], c)
            st["dstate"] = normal(b, width - 1, c, scale=0.1) if case["state"] else None
            for name in _wanted(case):
                st[name].requires_grad_()
        return st
    n, groups = case["n"], case["groups"]
    # decays as such layers start with: rates 1 to n a channel, steps of 1e-3 to 1e-1
    st["a"] = -torch.arange(1, n + 1, device="cuda") * torch.exp(normal(c, 1, scale=0.1, to=torch.float32))
    step = torch.exp(torch.rand(c, generator=g, device="cuda") * math.log(100.0) + math.log(1e-3))
    st["dt_bias"] = step + torch.log(-torch.expm1(-step)) if case["softplus"] else None
    st["d"] = 1.0 + normal(c, scale=0.1, to=torch.float32)
    lead = (b,) if case["op"] == "scan_step" else (b, case["t"])

    def steps():
        v = torch.randn(*lead, c, generator=g, device="cuda")
        return (v * 0.5 if case["softplus"] else step * torch.exp(0.5 * v)).to(dtype)

    st["dt"] = steps()
    st["x"] = torch.nn.functional.silu(normal(*lead, c, to=torch.float32)).to(dtype)
    if case["op"] == "scan" and case["packed"]:
        st["rank"] = -(-c // 16)
        st["proj"] = normal(*lead, st["rank"] + 2 * groups * n)
        st["xz"] = normal(*lead, 2 * c) if case["gate"] else None
    else:
        st["b"], st["c"] = normal(*lead, groups, n), normal(*lead, groups, n)
        st["z"] = normal(*lead, c) if case["gate"] else None
    if case["op"] == "scan_step":
        st["state"] = normal(b, c, n, to=torch.float32)
        return st
    st["state"] = normal(b, c, n, to=torch.float32) if case["state"] else None
    st["lengths"] = _lengths(case, g)
    if case["grad"]:
        st["dy"] = normal(*lead, c)
        st["dstate"] = normal(b, c, n, scale=0.1, to=torch.float32) if case["state"] else None
        for name in _wanted(case):
            st[name].requires_grad_()
    return st


def _wanted(case):
    """The inputs that gradients are asked of."""
    if case["op"] == "conv":
        return ("x", "weight") + (("bias",) if case["bias"] else ()) + (("state",) if case["state"] else ())
    return (("x", "dt", "a", "b", "c", "d") + (("z",) if case["gate"] else ()) + (("dt_bias",) if case["softplus"] else ())
            + (("state",) if case["state"] else ()))


def _scan_operands(st):
    """x, dt, b, c and z, views of their projections where they come so."""
    case = st["case"]
    if "proj" not in st:
        return st["x"], st["dt"], st["b"], st["c"], st["z"]
    groups, n, rank = case["groups"], case["n"], st["rank"]
    b, c = (st["proj"][..., at:at + groups * n].unflatten(-1, (groups, n)) for at in (rank, rank + groups * n))
    return st["x"], st["dt"], b, c, st["xz"][..., case["c"]:] if case["gate"] else None


def _conv_input(st):
    return st["xz"][..., :st["case"]["c"]] if "xz" in st else st["x"]


# ---------------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------------


def _silu(x):
    return x / (1.0 + torch.exp(-x))


def _plain_conv(x, weight, bias, act, state, lengths):
    dtype, (b, t, c), width = x.dtype, x.shape, weight.shape[1]
    ends = torch.full((b,), t, device=x.device) if lengths is None else lengths
    inside = (torch.arange(t, device=x.device) < ends[:, None])[..., None]
    before = x.new_zeros(b, width - 1, c) if state is None else state
    whole = torch.cat([before, torch.where(inside, x, 0.0)], dim=1)
    y = (whole.float().unfold(1, width, 1) * weight).sum(-1)
    y = y if bias is None else y + bias
    y = torch.where(inside, _silu(y) if act == "silu" else y, 0.0)
    at = ends[:, None] + torch.arange(width - 1, device=x.device)
    return y.to(dtype), torch.gather(whole, 1, at[..., None].expand(-1, -1, c))


def _plain_conv_step(st):
    case, state, x = st["case"], st["state"], st["x"]
    whole = torch.cat([state, x[:, None]], dim=1)
    y = (whole.float() * st["weight"].t()).sum(1)
    y = y if st["bias"] is None else y + st["bias"]
    state.copy_(whole[:, 1:])
    return (_silu(y) if case["act"] == "silu" else y).to(x.dtype)


def _plain_dt(dt, dt_bias, softplus):
    dt = dt.float() if dt_bias is None else dt.float() + dt_bias
    return dt.clamp(min=0.0) + torch.log1p(torch.exp(-dt.abs())) if softplus else dt


def _plain_scan(x, dt, a, b, c, d, z, dt_bias, softplus, state, lengths):
    """Stretches of frames side by side, frame after frame: from zero for the states between the stretches, then again from
    those for the outputs."""
    dtype, (rows, t, channels), (groups, n) = x.dtype, x.shape, b.shape[2:]
    each = channels // groups
    ends = torch.full((rows,), t, device=x.device) if lengths is None else lengths
    inside = (torch.arange(t, device=x.device) < ends[:, None])[..., None]
    x, dt = torch.where(inside, x.float(), 0.0), torch.where(inside, _plain_dt(dt, dt_bias, softplus), 0.0)
    b, c = (torch.where(inside[..., None], v.float(), 0.0) for v in (b, c))
    size = max(1, math.isqrt(t))
    count = -(-t // size)

    def stretches(v, *last):  # (rows, stretches, size, groups, ...)
        v = torch.cat([v, v.new_zeros(rows, count * size - t, *v.shape[2:])], dim=1)
        return v.reshape(rows, count, size, groups, *last)

    steps, inputs = stretches(dt, each, 1), stretches(dt * x, each, 1)
    b, c, rates = stretches(b, 1, n), stretches(c, 1, n), a.view(groups, each, n)

    def frame(h, i):
        return h * torch.exp(steps[:, :, i] * rates) + inputs[:, :, i] * b[:, :, i]

    h = x.new_zeros(rows, count, groups, each, n)
    for i in range(size if count > 1 else 0):
        h = frame(h, i)
    keeps = torch.exp(steps.sum(2) * rates)
    s = x.new_zeros(rows, groups, each, n) if state is None else state.view(rows, groups, each, n)
    starts = [s]
    for j in range(count - 1):
        s = s * keeps[:, j] + h[:, j]
        starts.append(s)
    h, y = torch.stack(starts, 1), []
    for i in range(size):
        h = frame(h, i)
        y.append((h * c[:, :, i]).sum(-1))
    y = torch.stack(y, 2).reshape(rows, count * size, channels)[:, :t] + d * x
    y = y if z is None else y * _silu(torch.where(inside, z.float(), 0.0))
    return torch.where(inside, y, 0.0).to(dtype), h[:, -1].reshape(rows, channels, n)


def _plain_scan_step(st):
    case, state = st["case"], st["state"]
    x, dt, b, c, z = (None if v is None else v.float() for v in _scan_operands(st))
    each = case["c"] // case["groups"]
    dt = _plain_dt(dt, st["dt_bias"], case["softplus"])[..., None]
    b, c = (v.repeat_interleave(each, dim=1) for v in (b, c))
    state.mul_(torch.exp(dt * st["a"])).add_(dt * x[..., None] * b)
    y = (state * c).sum(-1) + st["d"] * x
    return (y if z is None else y * _silu(z)).to(st["x"].dtype)


def _plain_clip(st):
    g = st["grads"]
    norm = torch.sqrt(g.double().square().sum())
    g.copy_(g.float() * (st["max_norm"] / (norm + 1e-6)).clamp(max=1.0).float())
    return norm.float()


# ---------------------------------------------------------------------------------------------
# a pass
# ---------------------------------------------------------------------------------------------


def run(st):
    if own:
        import trnfft_amd
    case = st["case"]
    act = "silu" if case.get("act") == "silu" else None
    if case["op"] == "clip":
        if case["clips"]:  # the step's gradients come out of their bucket
            st["grads"].copy_(st["bucket"])
        norm = trnfft_amd.clip_grads(st["list"], st["max_norm"]) if own else _plain_clip(st)
        return {"norm": norm, "grads": st["grads"]}
    if case["op"] == "conv_step":
        if own:
            y = trnfft_amd.causal_conv_step(st["x"], st["state"], st["weight"], st["bias"], activation=act)
        else:
            y = _plain_conv_step(st)
        return {"y": y, "state": st["state"]}
    if case["op"] == "scan_step":
        if own:
            y = trnfft_amd.selective_scan_step(st["x"], st["dt"], st["a"], st["b"], st["c"], st["state"], d=st["d"], z=st["z"],
                                               dt_bias=st["dt_bias"], softplus=case["softplus"])
        else:
            y = _plain_scan_step(st)
        return {"y": y, "state": st["state"]}
    if case["op"] == "conv":
        x = _conv_input(st)
        if own:
            y, last = trnfft_amd.causal_conv(x, st["weight"], st["bias"], activation=act, initial_state=st["state"],
                                             lengths=st["lengths"], return_state=True)
        else:
            y, last = _plain_conv(x, st["weight"], st["bias"], act, st["state"], st["lengths"])
    else:
        x, dt, b, c, z = _scan_operands(st)
        if own:
            y, last = trnfft_amd.selective_scan(x, dt, st["a"], b, c, d=st["d"], z=z, dt_bias=st["dt_bias"],
                                                softplus=case["softplus"], initial_state=st["state"],
                                                lengths=st["lengths"], return_state=True)
        else:
            y, last = _plain_scan(x, dt, st["a"], b, c, st["d"], z, st["dt_bias"], case["softplus"], st["state"],
                                  st["lengths"])
    if not case["grad"]:
        return {"y": y, "last": last}
    outputs, seeds = ([y, last], [st["dy"], st["dstate"]]) if case["state"] else ([y], [st["dy"]])
    grads = torch.autograd.grad(outputs, [st[name] for name in _wanted(case)], seeds)
    return {"y": y.detach(), "last": last.detach(), **{"d_" + name: v for name, v in zip(_wanted(case), grads)}}


def work(case):
    size = {"fp32": 4, "bf16": 2, "fp16": 2}[case["dtype"]]
    if case["op"] == "clip":
        n = sum(_sizes(case))
        # the norm reads every gradient; those that are scaled are written, and were taken out of their bucket
        return {"bytes": size * n * (4 if case["clips"] else 1), "flops": n * (3 if case["clips"] else 2)}
    b, t, c = case["b"], case.get("t", 1), case["c"]
    values = b * t * c
    if case["op"] in ("conv", "conv_step"):
        w = case["width"]
        weights = 4 * c * (w + (1 if case["bias"] else 0))
        state = size * b * (w - 1) * c
        each = 2 * w + 5
        if case["op"] == "conv_step":
            return {"bytes": 2 * size * values + 2 * state + weights, "flops": values * each}
        bytes_ = 2 * size * values + state * (2 if case["state"] else 1) + weights
        if case["grad"]:
            bytes_ += 2 * size * values + weights + (2 * state if case["state"] else 0)
            each *= 3
        return {"bytes": bytes_, "flops": values * each}
    n, groups = case["n"], case["groups"]
    weights = 4 * c * (n + 1 + (1 if case["softplus"] else 0))
    planes, shared, state = (4 if case["gate"] else 3) * values, 2 * b * t * groups * n, 4 * b * c * n
    if case["op"] == "scan_step":
        return {"bytes": size * (planes + shared) + 2 * state + weights, "flops": values * (7 * n + 12)}
    bytes_ = size * (planes + shared) + state * (2 if case["state"] else 1) + weights
    flops = values * (7 * n + 12)
    if case["grad"]:
        bytes_ += size * (planes + shared) + weights + (2 * state if case["state"] else 0)
        flops = values * (24 * n + 40)
    return {"bytes": bytes_, "flops": flops}


# ---------------------------------------------------------------------------------------------
# definitions in 64 bits
# ---------------------------------------------------------------------------------------------


def _slope(v):
    """The derivative of silu."""
    s = torch.sigmoid(v)
    return s * (1.0 + v * (1.0 - s))


def _exact_conv(case, st):
    """Tap by tap; row by row where sequences end."""
    x, w = _conv_input(st).detach().double(), st["weight"].detach().double()
    b, t, c, width = case["b"], case["t"], case["c"], case["width"]
    ends = [t] * b if st["lengths"] is None else st["lengths"].tolist()
    y, last = torch.zeros_like(x), torch.zeros(b, width - 1, c, dtype=torch.float64, device="cuda")
    grad = case["grad"]
    dx, dw, db, ds = torch.zeros_like(x), torch.zeros_like(w), torch.zeros_like(w[:, 0]), torch.zeros_like(last)
    for i, end in enumerate(ends):
        before = last[i] if st["state"] is None else st["state"][i].detach().double()
        seq = torch.cat([before, x[i, :end]])
        pre = torch.zeros(end, c, dtype=torch.float64, device="cuda")
        for j in range(width):
            pre += w[:, j] * seq[j:j + end]
        if case["bias"]:
            pre += st["bias"].detach().double()
        y[i, :end] = pre * torch.sigmoid(pre) if case["act"] == "silu" else pre
        if grad:
            dpre = st["dy"][i, :end].double() * (_slope(pre) if case["act"] == "silu" else 1.0)
            dseq = torch.zeros_like(seq)
            if st["dstate"] is not None:
                dseq[end:] += st["dstate"][i].double()
            for j in range(width):
                dseq[j:j + end] += w[:, j] * dpre
                dw[:, j] += (dpre * seq[j:j + end]).sum(0)
            db += dpre.sum(0)
            dx[i, :end], ds[i] = dseq[width - 1:], dseq[:width - 1]
        last[i] = seq[end:]
    out = {"y": y, "last": last}
    if grad:
        out |= {"d_x": dx, "d_weight": dw}
        out |= {"d_bias": db} if case["bias"] else {}
        out |= {"d_state": ds} if case["state"] else {}
    return out


def _exact_scan(case, st):
    """The recurrence itself, frame by frame; its gradients by the same recurrence backwards."""
    rows, t, ch, n, groups = case["b"], case["t"], case["c"], case["n"], case["groups"]
    x, dt, b, c, z = (None if v is None else v.detach().double() for v in _scan_operands(st))
    a, d = st["a"].detach().double(), st["d"].detach().double()
    v = dt if st["dt_bias"] is None else dt + st["dt_bias"].detach().double()
    dt = torch.logaddexp(v, torch.zeros_like(v)) if case["softplus"] else v
    if st["lengths"] is None:
        live = torch.ones(rows, t, 1, dtype=torch.float64, device="cuda")
    else:
        live = (torch.arange(t, device="cuda") < st["lengths"][:, None]).double()[..., None]
    dt = dt * live  # (a frame past the end: the state stays)

    def share(v):  # (rows, groups, n) for every channel
        return v.repeat_interleave(ch // groups, dim=1)

    h = torch.zeros(rows, ch, n, dtype=torch.float64, device="cuda") if st["state"] is None else st["state"].detach().double()
    inner = torch.empty(rows, t, ch, dtype=torch.float64, device="cuda")
    kept = torch.empty(t + 1, rows, ch, n, dtype=torch.float64, device="cuda") if case["grad"] else None
    u = dt * x
    for i in range(t):
        if case["grad"]:
            kept[i] = h
        h = torch.addcmul(h * torch.exp(dt[:, i, :, None] * a), u[:, i, :, None], share(b[:, i]))
        inner[:, i] = (h * share(c[:, i])).sum(-1)
    inner += d * x
    gate = torch.ones_like(x) if z is None else z * torch.sigmoid(z)
    out = {"y": inner * gate * live, "last": h}
    if not case["grad"]:
        return out
    kept[t] = h
    dy = st["dy"].double() * live
    out_z = dy * inner * _slope(z) if z is not None else None
    dy = dy * gate
    dx, ddt, db, dc, da = dy * d, torch.empty_like(x), torch.empty_like(b), torch.empty_like(c), torch.zeros_like(a)
    carry = torch.zeros_like(h) if st["dstate"] is None else st["dstate"].double()
    for i in range(t - 1, -1, -1):
        g = torch.addcmul(carry, dy[:, i, :, None], share(c[:, i]))
        dc[:, i] = (dy[:, i, :, None] * kept[i + 1]).unflatten(1, (groups, -1)).sum(2)
        db[:, i] = (g * u[:, i, :, None]).unflatten(1, (groups, -1)).sum(2)
        du = (g * share(b[:, i])).sum(-1)
        carry = g * torch.exp(dt[:, i, :, None] * a)
        flow = carry * kept[i]
        ddt[:, i] = (flow * a).sum(-1) + du * x[:, i]
        da += (flow * dt[:, i, :, None]).sum(0)
        dx[:, i] += du * dt[:, i]
    ddt, dx = ddt * live, dx * live
    ddt = ddt * torch.sigmoid(v) if case["softplus"] else ddt
    db, dc = db * live[..., None], dc * live[..., None]
    out |= {"d_x": dx, "d_dt": ddt, "d_a": da, "d_b": db, "d_c": dc, "d_d": (dy * x).sum((0, 1))}
    out |= {"d_z": out_z} if z is not None else {}
    out |= {"d_dt_bias": ddt.sum((0, 1))} if case["softplus"] else {}
    out |= {"d_state": carry} if case["state"] else {}
    return out


def exact(case, seed):
    st = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "conv":
            return _exact_conv(case, st)
        if case["op"] == "scan":
            return _exact_scan(case, st)
        if case["op"] == "clip":
            g = st["bucket"].double()
            norm = torch.linalg.vector_norm(g)
            return {"norm": norm, "grads": g * min(1.0, st["max_norm"] / (float(norm) + 1e-6))}
        if case["op"] == "conv_step":
            w = st["weight"].double()
            seq = torch.cat([st["state"].double(), st["x"].double()[:, None]], dim=1)
            y = torch.einsum("bjc,cj->bc", seq, w) + (0.0 if st["bias"] is None else st["bias"].double())
            return {"y": y * torch.sigmoid(y) if case["act"] == "silu" else y, "state": seq[:, 1:]}
        x, dt, b, c, z = (None if v is None else v.double() for v in _scan_operands(st))
        each = case["c"] // case["groups"]
        v = dt if st["dt_bias"] is None else dt + st["dt_bias"].double()
        dt = torch.logaddexp(v, torch.zeros_like(v)) if case["softplus"] else v
        h = st["state"].double() * torch.exp(dt[..., None] * st["a"].double())
        h = h + (dt * x)[..., None] * b.repeat_interleave(each, dim=1)
        y = (h * c.repeat_interleave(each, dim=1)).sum(-1) + st["d"].double() * x
        return {"y": y if z is None else y * z * torch.sigmoid(z), "state": h}
