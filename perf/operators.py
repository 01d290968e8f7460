"""The operators that a model on STFT frames is trained and served with, as cases that can be timed and checked.

* linear attention with a decay for each head: whole sequences of frames, their training pass, and the step of a
  stream that gets one frame at a time;
* group norm with an activation on channels-last frames, forward and training pass;
* the AdamW step over all tensors of a model, with states in 32 or 8 bits.

Sizes: the benchmark's 64 signals of 10 s (626 frames of 257 bins at n_fft 512, 1001 frames at n_fft 400, hop 160),
the complex linear layer's 8192 rows of 1024 features and its 1024 x 1024 weights, and generic ones.  Every
operator has a plain form of elementary torch operations in fp32 here, rounded once at the end; with ``own`` set, ``run``
calls the package instead.
"""

from __future__ import annotations

import math
import random

import torch

own = False

_DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_CHUNK = 64  # frames a block of the plain attention
_QBLOCK = 256  # values that share a scale of the 8-bit states
_LR, _BETAS, _EPS, _DECAY, _STEP = 1e-3, (0.9, 0.99), 1e-8, 0.01, 10


def listed():
    return [
        # one stream's next frame: nothing but latency
        {"name": "step_1x8x64_fp32", "op": "step", "b": 1, "h": 8, "hq": 8, "hk": 8, "hv": 8, "dk": 64, "dv": 64,
         "dtype": "fp32"},
        # the next frame of 256 streams served together; keys and queries shared by four heads
        {"name": "step_256x16x128_bf16", "op": "step", "b": 256, "h": 16, "hq": 4, "hk": 4, "hv": 16, "dk": 128,
         "dv": 128, "dtype": "bf16"},
        # the benchmark's 64 signals, ragged: projections come as one tensor and are split by views; state kept for the stream
        {"name": "attend_64x626_bf16", "op": "attend", "b": 64, "t": 626, "h": 8, "hq": 8, "hk": 8, "hv": 8, "dk": 64,
         "dv": 64, "dtype": "bf16", "lengths": True, "state": True, "packed": True, "grad": False},
        # one long recording: few rows, the long axis has to be shared out
        {"name": "attend_1x65536_bf16", "op": "attend", "b": 1, "t": 65536, "h": 16, "hq": 16, "hk": 16, "hv": 16,
         "dk": 128, "dv": 128, "dtype": "bf16", "lengths": False, "state": False, "packed": False, "grad": False},
        # training on short utterances in fp32: odd head sizes, shared keys, ragged, from a state
        {"name": "train_4x1001_fp32", "op": "attend", "b": 4, "t": 1001, "h": 6, "hq": 6, "hk": 2, "hv": 6, "dk": 48,
         "dv": 80, "dtype": "fp32", "lengths": True, "state": True, "packed": False, "grad": True},
        # a training pass of a wide model: every gradient, the decays' too
        {"name": "train_8x4096_bf16", "op": "attend", "b": 8, "t": 4096, "h": 16, "hq": 16, "hk": 16, "hv": 16,
         "dk": 128, "dv": 128, "dtype": "bf16", "lengths": False, "state": False, "packed": False, "grad": True},
        # a stream's block of 10 frames: latency
        {"name": "norm_1x10x64_fp32", "op": "norm", "n": 1, "t": 10, "f": 1, "c": 64, "groups": 8, "act": "silu",
         "dtype": "fp32", "lengths": False, "grad": False},
        # feature maps over (frames, bins), the largest activations of such a model
        {"name": "norm_32x626x257x32_bf16", "op": "norm", "n": 32, "t": 626, "f": 257, "c": 32, "groups": 8,
         "act": "silu", "dtype": "bf16", "lengths": False, "grad": False},
        # the training pass between two layers of 512 features, ragged utterances
        {"name": "norm_train_64x626x512_bf16", "op": "norm", "n": 64, "t": 626, "f": 1, "c": 512, "groups": 32,
         "act": "gelu", "dtype": "bf16", "lengths": True, "grad": True},
        # the weights of a small denoiser: a few complex layers, biases and norms
        {"name": "adamw_24x0.5M_fp32", "op": "adamw", "tensors": 24, "numel": 500_000, "dtype": "fp32", "bits": 32,
         "masters": False},
        # bf16 weights with fp32 masters
        {"name": "adamw_160x40M_bf16", "op": "adamw", "tensors": 160, "numel": 40_000_000, "dtype": "bf16",
         "bits": 32, "masters": True},
        # a large model whose states are held in 8 bits
        {"name": "adamw8_320x120M_fp32", "op": "adamw", "tensors": 320, "numel": 120_000_000, "dtype": "fp32",
         "bits": 8, "masters": False},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_heads(rng, most):
    h = rng.choice([x for x in (1, 2, 3, 4, 6, 8, 12, 16, 32) if x <= most])
    share = [x for x in range(1, h + 1) if h % x == 0]
    hv = h if rng.random() < 0.7 else rng.choice(share)
    hk = h if rng.random() < 0.5 else rng.choice(share)
    hq = h if rng.random() < 0.7 else hk
    sizes = (16, 24, 32, 48, 64, 64, 80, 96, 128, 128)
    dk = rng.choice(sizes) if rng.random() < 0.8 else rng.randint(8, 128)
    dv = dk if rng.random() < 0.5 else rng.choice(sizes) if rng.random() < 0.8 else rng.randint(8, 128)
    return {"h": h, "hq": hq, "hk": hk, "hv": hv, "dk": dk, "dv": dv}


def draw(rng):
    op = rng.choice(["step", "attend", "attend", "norm", "norm", "adamw"])
    dtype = rng.choice(["fp32", "bf16", "bf16", "fp16"])
    if op == "step":
        return {"op": op, "b": _log_int(rng, 1, 256), **_draw_heads(rng, 16), "dtype": dtype}
    if op == "attend":
        grad = rng.random() < 0.5
        heads = _draw_heads(rng, 32)
        t = _log_int(rng, 1, 16384)
        rows = (1 << 19 if grad else 1 << 20) * 256 // (t * heads["h"] * (heads["dk"] + heads["dv"]))
        return {"op": op, "b": _log_int(rng, 1, min(64, max(1, rows // (2 if dtype == "fp32" else 1)))), "t": t, **heads, "dtype": dtype,
                "lengths": rng.random() < 0.5, "state": rng.random() < 0.5,
                "packed": not grad and rng.random() < 0.5, "grad": grad}
    if op == "norm":
        grad = rng.random() < 0.5
        groups = rng.choice([1, 2, 4, 8, 16, 32])
        each = rng.choice([1, 2, 3, 4, 6, 8, 16, 24, 32, 64])
        c = groups * each
        n = _log_int(rng, 1, 64)
        most = min(160_882, (64 << 20 if grad else 128 << 20) // (n * c))
        f = rng.choice([1, 1, 9, 257])
        t = _log_int(rng, 1, max(1, most // f))
        if t * f * each < 16:
            t = -(-16 // (f * each))
        return {"op": op, "n": n, "t": t, "f": f, "c": c, "groups": groups,
                "act": rng.choice(["none", "silu", "gelu", "relu"]), "dtype": dtype,
                "lengths": t >= 32 and rng.random() < 0.4, "grad": grad}
    masters = dtype != "fp32" and rng.random() < 0.7
    tensors = _log_int(rng, 1, 400)
    return {"op": op, "tensors": tensors, "numel": _log_int(rng, max(1000, 4 * tensors), 60_000_000), "dtype": dtype,
            "bits": rng.choice([32, 8]), "masters": masters}


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------


def _lengths(case, rows, t, g, least):
    """Utterances of a batch end early: whole ones, half ones and very short ones."""
    if not case["lengths"]:
        return None
    u = torch.rand(rows, generator=g, device="cuda")
    lengths = (least + u * (t - least)).to(torch.int64).clamp_(max=t)
    lengths[0] = t
    return lengths


def _decays(h):
    # memories from 4 to 256 frames, one per head
    return torch.tensor([math.log1p(-(2.0 ** -(2.0 + 6.0 * i / max(1, h - 1)))) for i in range(h)],
                        dtype=torch.float32, device="cuda")


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
    if case["op"] in ("step", "attend"):
        b, h, dk, dv = case["b"], case["h"], case["dk"], case["dv"]
        st["scale"] = dk**-0.5
        st["log_decay"] = _decays(h)
        if case["op"] == "step":
            st["q"], st["k"], st["v"] = (normal(b, case[n], d) for n, d in (("hq", dk), ("hk", dk), ("hv", dv)))
            st["state"] = normal(b, h, dk, dv, to=torch.float32)
            return st
        t = case["t"]
        if case["packed"]:
            st["qkv"] = normal(b, t, case["hq"] * dk + case["hk"] * dk + case["hv"] * dv)
        else:
            for name, heads, d in (("q", "hq", dk), ("k", "hk", dk), ("v", "hv", dv)):
                st[name] = normal(b, t, case[heads], d)
        st["lengths"] = _lengths(case, b, t, g, 0)
        st["state"] = normal(b, h, dk, dv, to=torch.float32) if case["state"] else None
        if case["grad"]:
            st["do"] = normal(b, t, h, dv)
            st["dstate"] = normal(b, h, dk, dv, scale=0.1, to=torch.float32) if case["state"] else None
            for name in ("q", "k", "v", "log_decay") + (("state",) if case["state"] else ()):
                st[name].requires_grad_()
        return st
    if case["op"] == "norm":
        n, t, f, c = case["n"], case["t"], case["f"], case["c"]
        offset = torch.randn(c, generator=g, device="cuda")
        x = torch.randn(n, t, f, c, generator=g, device="cuda").mul_(1.5).add_(offset)
        st["x"] = x.to(dtype).view(n, t, c) if f == 1 else x.to(dtype)
        del x
        st["weight"] = 1.0 + normal(c, scale=0.2, to=torch.float32)
        st["bias"] = normal(c, scale=0.2, to=torch.float32)
        st["lengths"] = _lengths(case, n, t, g, 16)
        if case["grad"]:
            st["dy"] = normal(*st["x"].shape)
            for name in ("x", "weight", "bias"):
                st[name].requires_grad_()
        return st
    sizes = _sizes(case)
    starts, end = [], 0
    for s in sizes:  # every tensor starts at a whole block of the flat buffers that hold them
        starts.append(end)
        end += -(-s // _QBLOCK) * _QBLOCK
    inside = torch.zeros(end, dtype=torch.bool, device="cuda")
    for s, at in zip(sizes, starts):
        inside[at:at + s] = True

    def flat(scale, to=torch.float32):
        return (torch.randn(end, generator=g, device="cuda") * scale * inside).to(to)

    def views(buffer, parts=sizes, at=starts):
        return [buffer[i:i + s] for s, i in zip(parts, at)]

    st["masters"] = flat(0.05) if case["masters"] else None
    st["params"] = st["masters"].to(dtype) if case["masters"] else flat(0.05, dtype)
    st["grads"] = flat(1e-2, dtype)
    blocks, block_starts = [-(-s // _QBLOCK) for s in sizes], [i // _QBLOCK for i in starts]
    m, v = flat(3e-3), flat(1e-2).square_()
    if case["bits"] == 8:
        st["m"], st["m_scales"] = _encode(m, 1, 127, torch.int8)
        st["v"], st["v_scales"] = _encode(v, 2, 255, torch.uint8)
        st["m_values"], st["v_values"] = torch.zeros_like(m), torch.zeros_like(v)
    else:
        st["m"], st["v"] = m, v
    for name in ("params", "grads", "masters", "m", "v", "m_values", "v_values"):
        if st.get(name) is not None:
            st[name + "_list"] = views(st[name])
    for name in ("m_scales", "v_scales"):
        if name in st:
            st[name + "_list"] = views(st[name], blocks, block_starts)
    return st


# ---------------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------------


def _split(st):
    case = st["case"]
    if "qkv" not in st:
        return st["q"], st["k"], st["v"]
    b, t = st["qkv"].shape[:2]
    wide = [case["hq"] * case["dk"], case["hk"] * case["dk"], case["hv"] * case["dv"]]
    parts = st["qkv"].split(wide, dim=-1)
    return tuple(x.unflatten(-1, (-1, d)) for x, d in zip(parts, (case["dk"], case["dk"], case["dv"])))


def _plain_attention(q, k, v, log_decay, scale, state, lengths):
    """Blocks of frames: inside a block the masked, decayed products, between blocks the states."""
    dtype, (b, t), h = q.dtype, q.shape[:2], log_decay.numel()
    q, k, v = (x.float().repeat_interleave(h // x.shape[2], dim=2).transpose(1, 2) for x in (q, k, v))
    at = torch.arange(t, device=q.device)
    ends = torch.full((b,), t, device=q.device) if lengths is None else lengths
    inside = (at < ends[:, None])[:, None, :, None]
    q, k, v = (torch.where(inside, x, 0.0) for x in (q, k, v))
    g = log_decay[:, None]
    left = (ends[:, None, None] - 1 - at).clamp(min=0)
    last = (k * torch.exp(g * left)[..., None]).transpose(-1, -2) @ v
    if state is not None:
        last = last + torch.exp(log_decay * ends[:, None])[..., None, None] * state
    blocks = -(-t // _CHUNK)
    q, k, v = (torch.nn.functional.pad(x, (0, 0, 0, blocks * _CHUNK - t)).unflatten(2, (blocks, _CHUNK)) for x in (q, k, v))
    row = torch.arange(_CHUNK, device=q.device)
    lag = row[:, None] - row
    weights = torch.where(lag >= 0, torch.exp(g[..., None] * lag.clamp(min=0)), 0.0)
    o = ((q @ k.transpose(-1, -2)) * weights[:, None]) @ v
    gains = (k * torch.exp(g * (_CHUNK - 1 - row))[:, None, :, None]).transpose(-1, -2) @ v
    block = torch.arange(blocks, device=q.device)
    gap = block[:, None] - 1 - block
    carry = torch.where(gap >= 0, torch.exp(g[..., None] * (_CHUNK * gap.clamp(min=0))), 0.0)
    states = (carry @ gains.flatten(3)).view_as(gains)
    if state is not None:
        states = states + torch.exp(g * (_CHUNK * block))[..., None, None] * state[:, :, None]
    o = o + (q * torch.exp(g * (row + 1))[:, None, :, None]) @ states
    o = o.flatten(2, 3)[:, :, :t].transpose(1, 2) * scale
    return o.to(dtype), last


def _plain_step(st):
    h = st["log_decay"].numel()
    q, k, v = (st[n].float().repeat_interleave(h // st[n].shape[1], dim=1) for n in ("q", "k", "v"))
    state = st["state"]
    state.mul_(torch.exp(st["log_decay"])[:, None, None]).add_(k[..., None] * v[..., None, :])
    return ((q[..., None, :] @ state)[..., 0, :] * st["scale"]).to(st["q"].dtype)


def _activate(z, act):
    if act == "silu":
        return z / (1.0 + torch.exp(-z))
    if act == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    return z.clamp(min=0.0) if act == "relu" else z


def _plain_norm(x, weight, bias, groups, act, lengths, eps=1e-5):
    dtype, shape = x.dtype, x.shape
    x = x.float().reshape(shape[0], shape[1], -1, groups, shape[-1] // groups)
    count, inside = x[0, :, :, 0].numel(), None
    if lengths is not None:
        inside = (torch.arange(shape[1], device=x.device) < lengths[:, None])[:, :, None, None, None]
        x = torch.where(inside, x, 0.0)
        count = (lengths * x[0, 0, :, 0].numel()).clamp(min=1)[:, None, None, None, None]
    mean = x.sum((1, 2, 4), keepdim=True) / count
    x = x - mean
    if inside is not None:
        x = torch.where(inside, x, 0.0)
    x = x / torch.sqrt((x * x).sum((1, 2, 4), keepdim=True) / count + eps)
    y = _activate(x.flatten(3) * weight + bias, act)
    if inside is not None:
        y = torch.where(inside[..., 0], y, 0.0)
    return y.reshape(shape).to(dtype)


def _encode(x, roots, top, to):
    """8-bit codes of blocks: the value over the block's largest, its square root taken `roots` times."""
    x = x.view(-1, _QBLOCK)
    scales = x.abs().amax(1)
    r = torch.where(scales[:, None] > 0, x.abs() / scales[:, None], 0.0)
    for _ in range(roots):
        r = r.sqrt()
    return (torch.round(r * top) * torch.sign(x)).to(to).view(-1), scales


def _decode(codes, scales, roots, top, to=torch.float32):
    t = codes.to(to).view(-1, _QBLOCK) / top
    t = t * t.abs()
    for _ in range(roots - 1):
        t = t * t
    return (t * scales.to(to)[:, None]).view(-1)


def _plain_adamw(st):
    case, (b1, b2) = st["case"], _BETAS
    small = case["bits"] == 8
    g = st["grads"].float()
    m = _decode(st["m"], st["m_scales"], 1, 127) if small else st["m"]
    v = _decode(st["v"], st["v_scales"], 2, 255) if small else st["v"]
    m = m * b1 + g * (1 - b1)
    v = v * b2 + (g * g) * (1 - b2)
    p = st["masters"] if case["masters"] else st["params"].float()
    p = p * (1 - _LR * _DECAY) - (_LR / (1 - b1**_STEP)) * (m / (torch.sqrt(v) / math.sqrt(1 - b2**_STEP) + _EPS))
    if case["masters"]:
        st["masters"].copy_(p)
    st["params"].copy_(p)
    if not small:
        st["m"].copy_(m)
        st["v"].copy_(v)
        return
    for name, x, roots, top in (("m", m, 1, 127), ("v", v, 2, 255)):
        codes, scales = _encode(x, roots, top, st[name].dtype)
        st[name].copy_(codes)
        st[name + "_scales"].copy_(scales)
        st[name + "_values"].copy_(_decode(codes, scales, roots, top))


# ---------------------------------------------------------------------------------------------
# a pass
# ---------------------------------------------------------------------------------------------


def run(st):
    if own:
        import trnfft_amd
    case = st["case"]
    if case["op"] == "step":
        if own:
            o = trnfft_amd.linear_attention_step(st["q"], st["k"], st["v"], st["log_decay"], st["state"],
                                                 scale=st["scale"])
        else:
            o = _plain_step(st)
        return {"o": o, "state": st["state"]}
    if case["op"] == "attend":
        q, k, v = _split(st)
        if own:
            o, last = trnfft_amd.linear_attention(q, k, v, st["log_decay"], scale=st["scale"],
                                                  initial_state=st["state"], lengths=st["lengths"], return_state=True)
        else:
            o, last = _plain_attention(q, k, v, st["log_decay"], st["scale"], st["state"], st["lengths"])
        if not case["grad"]:
            return {"o": o, "state": last}
        wrt = ("q", "k", "v", "log_decay") + (("state",) if case["state"] else ())
        outputs, seeds = ([o, last], [st["do"], st["dstate"]]) if case["state"] else ([o], [st["do"]])
        grads = torch.autograd.grad(outputs, [st[n] for n in wrt], seeds)
        return {"o": o.detach(), "state": last.detach(), **{"d" + n: d for n, d in zip(wrt, grads)}}
    if case["op"] == "norm":
        if own:
            y = trnfft_amd.group_norm(st["x"], case["groups"], st["weight"], st["bias"],
                                      activation=None if case["act"] == "none" else case["act"],
                                      lengths=st["lengths"])
        else:
            y = _plain_norm(st["x"], st["weight"], st["bias"], case["groups"], case["act"], st["lengths"])
        if not case["grad"]:
            return y
        dx, dw, db = torch.autograd.grad(y, [st["x"], st["weight"], st["bias"]], st["dy"])
        return {"y": y.detach(), "dx": dx, "dweight": dw, "dbias": db}
    if own:
        eight = case["bits"] == 8
        trnfft_amd.adamw_step(st["params_list"], st["grads_list"], st["m_list"], st["v_list"], step=_STEP, lr=_LR,
                              betas=_BETAS, eps=_EPS, weight_decay=_DECAY, masters=st.get("masters_list"),
                              exp_avg_scales=st["m_scales_list"] if eight else None,
                              exp_avg_sq_scales=st["v_scales_list"] if eight else None)
        if eight:
            trnfft_amd.adamw_state_values(st["m_list"], st["m_scales_list"], out=st["m_values_list"])
            trnfft_amd.adamw_state_values(st["v_list"], st["v_scales_list"], out=st["v_values_list"])
    else:
        _plain_adamw(st)
    values = ("m_values", "v_values") if case["bits"] == 8 else ("m", "v")
    out = {"params": st["params"], "m": st[values[0]], "v": st[values[1]]}
    if case["masters"]:
        out["masters"] = st["masters"]
    return out


def work(case):
    size = {"fp32": 4, "bf16": 2, "fp16": 2}[case["dtype"]]
    if case["op"] in ("step", "attend"):
        b, t, h, dk, dv = case["b"], case.get("t", 1), case["h"], case["dk"], case["dv"]
        qk, vs, os = (case["hq"] + case["hk"]) * dk, case["hv"] * dv, h * dv
        state = 4 * b * h * dk * dv
        if case["op"] == "step":
            return {"bytes": size * b * (qk + vs + os) + 2 * state, "flops": 4 * b * h * dk * dv}
        bytes_ = size * b * t * (qk + vs + os) + state * (2 if case["state"] else 1)
        flops = 4 * b * t * h * dk * dv
        if case["grad"]:
            bytes_ += size * b * t * (2 * (qk + vs) + os) + (3 * state if case["state"] else 0)
            flops *= 3
        return {"bytes": bytes_, "flops": flops}
    if case["op"] == "norm":
        values = case["n"] * case["t"] * case["f"] * case["c"]
        return {"bytes": size * values * (5 if case["grad"] else 2), "flops": values * (30 if case["grad"] else 12)}
    n = sum(_sizes(case))
    each = size + (8 if case["masters"] else size) + size  # parameter (written, and read where there is no master), gradient
    each += 16 if case["bits"] == 32 else 4 + 8  # states; 8-bit codes are also returned as the values they stand for
    return {"bytes": n * each, "flops": 16 * n}


# ---------------------------------------------------------------------------------------------
# definitions in 64 bits
# ---------------------------------------------------------------------------------------------


def _exact_attend(case, st):
    """The recurrence itself, frame by frame; its gradients by the same recurrence backwards."""
    h, t, b = case["h"], case["t"], case["b"]
    q, k, v = (x.detach().double().repeat_interleave(h // x.shape[2], dim=2) for x in _split(st))
    decay = torch.exp(st["log_decay"].detach().double())[:, None, None]
    ends = torch.full((b,), t, device="cuda") if st["lengths"] is None else st["lengths"]
    inside = (torch.arange(t, device="cuda") < ends[:, None])
    live = inside[..., None, None].double()
    q, k, v = q * live, k * live, v * live
    keep = torch.where(inside[..., None, None, None], decay, 1.0) if case["lengths"] else None
    zero = torch.zeros(b, h, case["dk"], case["dv"], dtype=torch.float64, device="cuda")
    s0 = zero if st["state"] is None else st["state"].detach().double()
    o = torch.empty(b, t, h, case["dv"], dtype=torch.float64, device="cuda")
    dq = torch.empty_like(q) if case["grad"] else None
    do = st["do"].double() * live * st["scale"] if case["grad"] else None
    s, tangent, dg = s0, zero, 0.0  # tangent: the derivative of s by the log decay
    for i in range(t):
        w = decay if keep is None else keep[:, i]
        if case["grad"]:
            tangent = w * (tangent + s)
            if keep is not None:
                tangent = torch.where(inside[:, i, None, None, None], tangent, old_tangent) if i else tangent * live[:, i, :, :, None]
            old_tangent = tangent
        s = torch.baddbmm((w * s).flatten(0, 1), k[:, i].flatten(0, 1)[:, :, None], v[:, i].flatten(0, 1)[:, None]).view_as(s)
        o[:, i] = (q[:, i, :, None] @ s)[:, :, 0]
        if case["grad"]:
            dq[:, i] = (s @ do[:, i, :, :, None])[..., 0]
            dg = dg + (q[:, i, :, None] @ tangent @ do[:, i, :, :, None]).sum((0, 2, 3))
    out = {"o": o * st["scale"], "state": s}
    if not case["grad"]:
        return out
    ds = zero if st["dstate"] is None else st["dstate"].double()
    dg = dg + (ds * tangent).sum((0, 2, 3))
    dk, dv = torch.empty_like(k), torch.empty_like(v)
    for i in range(t - 1, -1, -1):
        ds = torch.baddbmm(ds.flatten(0, 1), q[:, i].flatten(0, 1)[:, :, None], do[:, i].flatten(0, 1)[:, None]).view_as(ds)
        dk[:, i] = (ds @ v[:, i, :, :, None])[..., 0] * live[:, i]
        dv[:, i] = (k[:, i, :, None] @ ds)[:, :, 0]
        ds = ds * (decay if keep is None else keep[:, i])
    for name, d, heads in (("dq", dq, "hq"), ("dk", dk, "hk"), ("dv", dv, "hv")):
        out[name] = d.unflatten(2, (case[heads], -1)).sum(3)
    out["dlog_decay"] = dg
    if case["state"]:
        out["dstate"] = ds
    return out


def _exact_norm(case, st):
    x, w, b = (st[n].detach().double() for n in ("x", "weight", "bias"))
    n, c, groups = case["n"], case["c"], case["groups"]
    ends = [case["t"]] * n if st["lengths"] is None else st["lengths"].tolist()
    y = torch.zeros_like(x)
    dx, dw, db = torch.zeros_like(x) if case["grad"] else None, 0.0, 0.0
    for i, end in enumerate(ends):
        r = x[i, :end].reshape(-1, groups, c // groups)
        var, mean = torch.var_mean(r, (0, 2), correction=0, keepdim=True)
        rstd = (var + 1e-5) ** -0.5
        xhat = ((r - mean) * rstd).flatten(1)
        z = xhat * w + b
        sig, cdf = torch.sigmoid(z), 0.5 * torch.erfc(-z / math.sqrt(2.0))
        y[i, :end] = {"silu": z * sig, "gelu": z * cdf, "relu": torch.relu(z), "none": z}[case["act"]].view_as(x[i, :end])
        if case["grad"]:
            slope = {"silu": sig * (1 + z * (1 - sig)), "relu": (z > 0).double(), "none": torch.ones_like(z),
                     "gelu": cdf + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)}[case["act"]]
            dz = st["dy"][i, :end].double().reshape_as(z) * slope
            dw, db = dw + (dz * xhat).sum(0), db + dz.sum(0)
            u, xh = (dz * w).unflatten(1, (groups, -1)), xhat.unflatten(1, (groups, -1))
            d = rstd * (u - u.mean((0, 2), keepdim=True) - xh * (u * xh).mean((0, 2), keepdim=True))
            dx[i, :end] = d.reshape(x[i, :end].shape)
    return {"y": y, "dx": dx, "dweight": dw, "dbias": db} if case["grad"] else y


def _exact_adamw(case, st):
    b1, b2 = _BETAS
    g = st["grads"].double()
    eight = case["bits"] == 8
    m = _decode(st["m"], st["m_scales"], 1, 127, torch.float64) if eight else st["m"].double()
    v = _decode(st["v"], st["v_scales"], 2, 255, torch.float64) if eight else st["v"].double()
    m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g.square()
    p = (st["masters"] if case["masters"] else st["params"]).double()
    mhat, vhat = m / (1 - b1**_STEP), v / (1 - b2**_STEP)
    p = p - _LR * (mhat / (vhat.sqrt() + _EPS) + _DECAY * p)
    out = {"params": p, "m": m, "v": v}
    if eight:  # the nearest of the 127 and 255 steps
        for name, power, top in (("m", 2, 127), ("v", 4, 255)):
            x = out[name].view(-1, _QBLOCK)
            s = x.abs().amax(1, keepdim=True)
            step = torch.round((x.abs() / s.clamp(min=1e-300)) ** (1 / power) * top)
            out[name] = (torch.sign(x) * (step / top) ** power * s).view(-1)
    if case["masters"]:
        out["masters"] = p
    return out


def exact(case, seed):
    st = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "step":
            h = case["h"]
            q, k, v = (st[n].double().repeat_interleave(h // st[n].shape[1], dim=1) for n in ("q", "k", "v"))
            s = torch.exp(st["log_decay"].double())[:, None, None] * st["state"].double()
            s = s + k[..., None] * v[..., None, :]
            return {"o": (q[..., None] * s).sum(2) * st["scale"], "state": s}
        if case["op"] == "attend":
            return _exact_attend(case, st)
        return _exact_norm(case, st) if case["op"] == "norm" else _exact_adamw(case, st)
