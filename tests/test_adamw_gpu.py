"""The AdamW step over many tensors against its definition in 64 bits; 8-bit states against their format.

Tolerances: a step is some ten fp32 operations, each within 2^-24 of its result, on terms of one sign but for the last
difference: 1e-6 relative (2-norm).  16-bit parameters are rounded once.  8-bit codes are the nearest: a state's value lies
within half a step (plus fp32 rounding, 1e-5 of a step) of what was encoded."""

from __future__ import annotations

import math

import pytest
import torch

import trnfft_amd
from trnfft_amd.optim import AdamW

pytestmark = pytest.mark.gpu

SIZES = [1, 3, 255, 256, 257, 4095, 4096, 4097, 12345, 0, 70000, 5]
HYPER = dict(lr=2e-3, betas=(0.9, 0.98), eps=1e-8, weight_decay=0.1)


def rel(got, ref):
    d, n = float((got.double().cpu() - ref).norm()), float(ref.norm())
    return d / n if n else d


def definition(p, g, m, v, step, lr, betas, eps, weight_decay):
    m = betas[0] * m + (1 - betas[0]) * g
    v = betas[1] * v + (1 - betas[1]) * g * g
    p = p - lr * weight_decay * p
    return p - lr * (m / (1 - betas[0]**step)) / ((v / (1 - betas[1]**step)).sqrt() + eps), m, v


def make(sizes, dtype, seed=0, offset=0):
    """Lists of tensors; with an offset every one starts that many elements past a 16-byte boundary."""
    r = torch.Generator().manual_seed(seed)

    def tensors(scale, to, square=False):
        out = []
        for n in sizes:
            x = torch.randn(n, generator=r) * scale
            buf = torch.zeros(n + offset, dtype=to, device="cuda")
            view = buf[offset:]
            view.copy_(x * x if square else x)
            out.append(view)
        return out

    return tensors(0.1, dtype), tensors(0.01, dtype), tensors(0.003, torch.float32), tensors(0.01, torch.float32, True)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("masters", [False, True])
@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("step", [1, 1000])
def test_step_with_fp32_states(dtype, masters, offset, step):
    params, grads, ms, vs = make(SIZES, dtype, offset=offset)
    copies = [p.float() * 1.0001 for p in params] if masters else None
    before = [[t.double().cpu() for t in x] for x in (copies or params, grads, ms, vs)]
    versions = [p._version for p in params]
    trnfft_amd.adamw_step(params, grads, ms, vs, step=step, masters=copies, **HYPER)
    for i, n in enumerate(SIZES):
        p, m, v = definition(*(x[i] for x in before), step, **HYPER)
        assert rel(ms[i], m) <= 1e-6 and rel(vs[i], v) <= 1e-6
        full = copies[i] if masters else params[i]
        if full.dtype == torch.float32:
            assert rel(full, p) <= 1e-6
        if dtype != torch.float32:
            # one rounding to nearest: half a unit in the last place (2^-9, 2^-12 of the next power of two), or denormal
            ulp = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}[dtype]
            assert ((params[i].double().cpu() - p).abs() <= 0.51 * ulp * 2 * p.abs() + 2.0**-25).all()
            if masters:
                assert torch.equal(params[i], copies[i].to(dtype))
    assert all(p._version > v for p, v in zip(params, versions))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("offset", [0, 3])
def test_steps_with_8_bit_states(dtype, offset):
    params, grads, ms, vs = make(SIZES, dtype, seed=1, offset=offset)
    blocks = [-(-n // 256) for n in SIZES]

    def odd(n, to):  # at odd addresses where the parameters are
        return torch.zeros(n + offset, dtype=to, device="cuda")[offset:]

    mc, vc = [odd(n, torch.int8) for n in SIZES], [odd(n, torch.uint8) for n in SIZES]
    msc, vsc = [odd(n, torch.float32) for n in blocks], [odd(n, torch.float32) for n in blocks]
    for step in (1, 2, 3):
        held = [trnfft_amd.adamw_state_values(mc, msc), trnfft_amd.adamw_state_values(vc, vsc)]
        before = [[t.double().cpu() for t in x] for x in (params, grads, *held)]
        trnfft_amd.adamw_step(params, grads, mc, vc, step=step, exp_avg_scales=msc, exp_avg_sq_scales=vsc, **HYPER)
        values = [trnfft_amd.adamw_state_values(mc, msc), trnfft_amd.adamw_state_values(vc, vsc)]
        for i, n in enumerate(SIZES):
            p, m, v = definition(*(x[i] for x in before), step, **HYPER)
            if dtype == torch.float32:
                assert rel(params[i], p) <= 1e-6
            else:
                assert ((params[i].double().cpu() - p).abs() <= 0.51 * 2.0**-7 * p.abs() + 2.0**-25).all()
            for x, codes, scales, got, power, top in ((m, mc[i], msc[i], values[0][i], 2, 127), (v, vc[i], vsc[i], values[1][i], 4, 255)):
                s = torch.stack([b.abs().max() for b in x.split(256)]) if n else x
                assert rel(scales, s) <= 1e-6
                s = s.repeat_interleave(256)[:n]
                # the code's place on the root scale is within half a step of the value's
                at = (x.abs() / s.clamp(min=1e-300)) ** (1 / power) * top
                assert ((codes.double().cpu().abs() - at).abs() <= 0.5 + 1e-4).all()
                decoded = torch.sign(x) * (codes.double().cpu().abs() / top) ** power * s
                assert (got.double().cpu() - decoded).abs().max() <= 2e-6 * s.max() if n else True
        grads = [g * 0.5 + 0.001 for g in grads]


def test_8_bit_blocks_of_zeros_and_of_what_is_not_finite():
    n = 600
    p, g = torch.ones(n, device="cuda"), torch.zeros(n, device="cuda")
    g[300], g[520] = float("nan"), float("inf")
    mc, vc = torch.zeros(n, dtype=torch.int8, device="cuda"), torch.zeros(n, dtype=torch.uint8, device="cuda")
    ms, vs = torch.zeros(3, device="cuda"), torch.zeros(3, device="cuda")
    trnfft_amd.adamw_step([p], [g], [mc], [vc], step=1, exp_avg_scales=[ms], exp_avg_sq_scales=[vs], weight_decay=0.0)
    assert (p[:256] == 1).all() and not mc[:256].any() and ms[0] == 0
    m, v = trnfft_amd.adamw_state_values([mc], [ms])[0], trnfft_amd.adamw_state_values([vc], [vs])[0]
    assert not m[:256].any() and not v[:256].any()
    assert m[256:].isnan().all() and v[256:].isnan().all()  # loud, not lost
    assert p[300].isnan() and torch.isfinite(p[:256]).all()


def test_more_tensors_than_one_launch_takes():
    sizes = [1 + (7 * i) % 700 for i in range(333)]
    params, grads, ms, vs = make(sizes, torch.float32, seed=3)
    before = [[t.double().cpu() for t in x] for x in (params, grads, ms, vs)]
    trnfft_amd.adamw_step(params, grads, ms, vs, step=5, **HYPER)
    for i in range(len(sizes)):
        p, m, v = definition(*(x[i] for x in before), 5, **HYPER)
        assert rel(params[i], p) <= 1e-6 and rel(ms[i], m) <= 1e-6 and rel(vs[i], v) <= 1e-6


def test_neighbours_are_left_alone():
    # tensors inside one buffer, with guards between them, for every state kind
    for bits in (32, 8):
        n = 1000
        p = torch.full((n + 8,), 3.0, device="cuda")
        g = torch.full((n,), 0.1, device="cuda")
        if bits == 32:
            m, v = torch.full((n + 8,), 3.0, device="cuda"), torch.full((n + 8,), 3.0, device="cuda")
            trnfft_amd.adamw_step([p[4:-4]], [g], [m[4:-4]], [v[4:-4]], step=1)
        else:
            m = torch.full((n + 8,), 3, dtype=torch.int8, device="cuda")
            v = torch.full((n + 8,), 3, dtype=torch.uint8, device="cuda")
            s = torch.ones(2, 6, device="cuda")
            trnfft_amd.adamw_step([p[4:-4]], [g], [m[4:-4]], [v[4:-4]], step=1, exp_avg_scales=[s[0, 1:-1]],
                                  exp_avg_sq_scales=[s[1, 1:-1]])
            assert (s[:, 0] == 1).all() and (s[:, -1] == 1).all() and (s[:, 1:-1] != 1).all()
        for t in (p, m, v):
            assert (t[:4] == 3).all() and (t[-4:] == 3).all() and (t[4:-4] != 3).any()


def test_graph_and_stream():
    params, grads, ms, vs = make(SIZES, torch.float32, seed=2)
    saved = [[t.clone() for t in x] for x in (params, ms, vs)]
    trnfft_amd.adamw_step(params, grads, ms, vs, step=3, **HYPER)
    expected = [[t.clone() for t in x] for x in (params, ms, vs)]

    def reset():
        for x, y in zip((params, ms, vs), saved):
            for a, b in zip(x, y):
                a.copy_(b)

    reset()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        trnfft_amd.adamw_step(params, grads, ms, vs, step=3, **HYPER)
    for _ in range(3):
        reset()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for x, y in zip((params, ms, vs), expected) for a, b in zip(x, y))
    reset()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        trnfft_amd.adamw_step(params, grads, ms, vs, step=3, **HYPER)
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(a, b) for x, y in zip((params, ms, vs), expected) for a, b in zip(x, y))


def test_optimizer_follows_torch():
    torch.manual_seed(0)
    shapes = [(64, 65), (33,), (5, 4, 3)]
    ours = [torch.nn.Parameter(torch.randn(s, device="cuda")) for s in shapes]
    theirs = [torch.nn.Parameter(p.detach().double().cpu()) for p in ours]
    a = AdamW(ours, lr=1e-2, weight_decay=0.05)
    b = torch.optim.AdamW(theirs, lr=1e-2, weight_decay=0.05)
    for i in range(5):
        for p, q in zip(ours, theirs):
            g = torch.randn(p.shape)
            p.grad, q.grad = (None, None) if i == 2 and p.dim() == 1 else (g.cuda(), g.double())
        a.step()
        b.step()
    for p, q in zip(ours, theirs):
        assert rel(p.detach(), q.detach()) <= 2e-6


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_optimizer_state_goes_through_a_checkpoint(bits, dtype):
    def fresh():
        torch.manual_seed(1)
        return [torch.nn.Parameter(torch.randn(s, device="cuda").to(dtype)) for s in ((100, 90), (7,))]

    def grads(params, i):
        r = torch.Generator().manual_seed(i)
        for p in params:
            p.grad = torch.randn(p.shape, generator=r).to(dtype).cuda()

    straight, first = fresh(), fresh()
    a, b = AdamW(straight, lr=1e-2, state_bits=bits), AdamW(first, lr=1e-2, state_bits=bits)
    for i in range(4):
        grads(straight, i)
        a.step()
    for i in range(2):
        grads(first, i)
        b.step()
    second = [torch.nn.Parameter(p.detach().clone()) for p in first]
    c = AdamW(second, lr=1e-2, state_bits=bits)
    c.load_state_dict(b.state_dict())
    big = c.state[second[0]]
    assert big["exp_avg"].dtype == (torch.int8 if bits == 8 else torch.float32)
    for i in range(2, 4):
        grads(second, i)
        c.step()
    assert all(torch.equal(p, q) for p, q in zip(straight, second))


def test_8_bit_states_train_as_well():
    # a least-squares problem of 100 steps: the loss with 8-bit states ends within 5 % of the one with 32
    losses = []
    for bits in (32, 8):
        torch.manual_seed(0)
        x, w = torch.randn(512, 128, device="cuda"), torch.randn(128, 64, device="cuda")
        y = x @ w
        p = torch.nn.Parameter(torch.zeros(128, 64, device="cuda"))
        opt = AdamW([p], lr=2e-2, weight_decay=0.0, state_bits=bits)
        for _ in range(100):
            p.grad = x.t() @ (x @ p.detach() - y) / 512
            opt.step()
        losses.append(float((x @ p.detach() - y).square().mean()))
    start = float(y.square().mean())
    assert losses[0] < 0.2 * start and losses[1] < 1.05 * losses[0] + 1e-3 * start
    assert math.isfinite(losses[1])
