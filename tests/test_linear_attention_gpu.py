"""Linear attention with decays against its definition in 64 bits (all pairs, on the CPU), its gradients against those
of the definition and against differences, and the step against the whole sequence.

Tolerances (relative 2-norm): fp32 results sum at most a few hundred fp32 products in each of two nested sums, random
rounding of 2^-24 each, so 2e-6 leaves a factor of several.  16-bit results are rounded once to nearest, 2^-9 (2^-12)
of the power of two below a value at most, 1.7e-3 (2.1e-4) in the mean square; scores and states may be
rounded once more to pieces of 16 bits on the way, which a factor of 1.5 covers.  (A mean square is one over many values: results of
fewer than 16 get the largest error of one rounding instead, 2^-8 or 2^-11.)  The decays' gradient is a sum with signs:
it is held to 5e-6 of the sum of its terms' magnitudes."""

from __future__ import annotations

import math

import pytest
import torch

import trnfft_amd

pytestmark = pytest.mark.gpu

TOL = {torch.float32: 2e-6, torch.bfloat16: 2.6e-3, torch.float16: 3.2e-4}


def reference(q, k, v, g, scale, state=None, lengths=None):
    """o, the end state and the decays' gradient terms' magnitudes' ingredients, from all pairs, in float64."""
    h, (b, t) = g.numel(), q.shape[:2]
    q, k, v = (x.repeat_interleave(h // x.shape[2], dim=2).transpose(1, 2) for x in (q, k, v))
    ends = torch.full((b,), t) if lengths is None else lengths.clamp(0, t)
    at = torch.arange(t)
    live = (at < ends[:, None])[:, None, :, None]
    q, k, v = (torch.where(live, x, 0.0) for x in (q, k, v))
    lag = (at[:, None] - at).double()
    w = torch.where(lag >= 0, torch.exp(g[:, None, None] * lag.clamp(min=0)), 0.0)
    o = ((q @ k.transpose(-1, -2)) * w) @ v
    left = (ends[:, None] - 1 - at).clamp(min=0).double()
    last = (k * torch.exp(g[:, None] * left[:, None])[..., None]).transpose(-1, -2) @ v
    if state is not None:
        o = o + torch.exp(g[:, None] * (at + 1))[..., None] * (q @ state)
        last = last + torch.exp(g * ends[:, None])[..., None, None] * state
    return (scale * o).transpose(1, 2), last


def make(b, t, heads, dk, dv, dtype, seed=0, lengths=False, state=False, g=None):
    h, hq, hk, hv = heads
    r = torch.Generator().manual_seed(seed)
    q, k, v = (torch.randn(b, t, n, d, generator=r).to(dtype) for n, d in ((hq, dk), (hk, dk), (hv, dv)))
    if g is None:
        g = -torch.rand(h, generator=r) * 0.5
        g[0] = -1e-3
    s = torch.randn(b, h, dk, dv, generator=r) if state else None
    n = torch.randint(0, t + 1, (b,), generator=r) if lengths else None
    if lengths and b > 1:
        n[0], n[1] = t, 0
    return q, k, v, g, s, n


def tol(ref, dtype):
    few = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
    return few.get(dtype, TOL[dtype]) if ref.numel() < 16 else TOL[dtype]


def rel(got, ref):
    got, ref = got.detach().double().cpu(), ref.detach().double()
    d, n = float((got - ref).norm()), float(ref.norm())
    return d / n if n else d


def cuda(*ts):
    return [None if t is None else t.cuda() for t in ts]


SHAPES = [
    # b, t, (h, hq, hk, hv), dk, dv
    (1, 1, (1, 1, 1, 1), 1, 1),
    (2, 2, (2, 2, 2, 2), 64, 64),
    (3, 15, (4, 2, 1, 4), 8, 16),
    (2, 16, (2, 2, 2, 2), 128, 128),
    (2, 17, (3, 3, 1, 3), 17, 33),
    (1, 31, (2, 2, 2, 2), 48, 80),
    (2, 33, (2, 1, 2, 2), 64, 32),
    (2, 63, (2, 2, 2, 2), 64, 64),
    (2, 64, (4, 4, 2, 1), 64, 64),
    (2, 65, (2, 2, 2, 2), 128, 64),
    (1, 127, (2, 2, 2, 2), 100, 128),
    (3, 129, (2, 2, 2, 2), 96, 96),
    (2, 200, (6, 6, 2, 3), 40, 128),
    (2, 300, (2, 2, 2, 2), 3, 128),
    (1, 301, (2, 2, 2, 2), 128, 5),
    (1, 1001, (2, 2, 2, 2), 64, 128),
    (1, 70, (2, 2, 1, 2), 129, 144),
    (1, 40, (1, 1, 1, 1), 256, 256),
]


@pytest.mark.parametrize("dtype", list(TOL))
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("extra", [False, True])
def test_forward(shape, dtype, extra):
    b, t, heads, dk, dv = shape
    q, k, v, g, s, n = make(b, t, heads, dk, dv, dtype, seed=t, lengths=extra, state=extra)
    ref, ref_last = reference(q.double(), k.double(), v.double(), g.double(), dk**-0.5, None if s is None else s.double(), n)
    o, last = trnfft_amd.linear_attention(*cuda(q, k, v, g), initial_state=cuda(s)[0], lengths=cuda(n)[0], return_state=True)
    assert o.dtype == dtype and o.shape == ref.shape and last.dtype == torch.float32
    assert rel(o, ref) <= tol(ref, dtype)
    assert rel(last, ref_last) <= 2e-6
    if n is not None:
        for i, end in enumerate(n.tolist()):
            assert not o[i, end:].any()


@pytest.mark.parametrize("dtype", list(TOL))
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("extra", [False, True])
def test_gradients(shape, dtype, extra):
    b, t, heads, dk, dv = shape
    q, k, v, g, s, n = make(b, t, heads, dk, dv, dtype, seed=100 + t, lengths=extra, state=extra)
    r = torch.Generator().manual_seed(7)
    do = torch.randn(b, t, heads[0], dv, generator=r).to(dtype)
    ds = torch.randn(b, heads[0], dk, dv, generator=r) if extra else None
    wrt = [x for x in (q, k, v, g, s) if x is not None]
    ref_in = [x.double().requires_grad_() for x in wrt]
    ref, ref_last = reference(*ref_in[:4], dk**-0.5, ref_in[4] if extra else None, n)
    outs, seeds = ([ref, ref_last], [do.double(), ds.double()]) if extra else ([ref], [do.double()])
    expected = torch.autograd.grad(outs, ref_in, seeds)
    leaves = [x.requires_grad_() for x in cuda(*wrt)]
    o, last = trnfft_amd.linear_attention(*leaves[:4], initial_state=leaves[4] if extra else None, lengths=cuda(n)[0],
                                          return_state=True)
    outs, seeds = ([o, last], cuda(do, ds)) if extra else ([o], cuda(do))
    got = torch.autograd.grad(outs, leaves, seeds)
    # the magnitudes that the decays' gradient sums: all pairs, by the same definition on absolute values
    a = [x.detach().abs() for x in ref_in]
    a[3] = ref_in[3].detach().clone().requires_grad_()
    oa, la = reference(*a[:4], dk**-0.5, a[4] if extra else None, n)
    size = torch.autograd.grad([oa, la] if extra else [oa], a[3], [do.double().abs(), ds.double().abs()] if extra else [do.double().abs()])[0]
    for name, x, y in zip(("q", "k", "v", "g", "s"), got, expected):
        assert x.shape == y.shape
        if name == "g":
            # (terms of random sign: their sum's error grows with the root of their number, their magnitudes with it)
            assert ((x.cpu().double() - y).abs() <= 5e-6 * size + 1e-30).all(), (x.cpu(), y, size)
        else:
            assert rel(x, y) <= (2e-6 if name == "s" else tol(y, dtype)), name
            assert x.dtype == (torch.float32 if name == "s" else dtype)


@pytest.mark.parametrize("name", ["q", "k", "v", "g", "s"])
def test_gradients_against_differences(name):
    # the loss is linear in q, k, v and the state one at a time, so central differences of it have no error of their own there;
    # by the decays they are off by eps^2/6 of the third derivative (T^3 times the sum at most)
    b, t, dk, dv = 2, 70, 16, 24
    q, k, v, g, s, n = make(b, t, (2, 2, 1, 2), dk, dv, torch.float32, seed=5, lengths=True, state=True)
    n = torch.tensor([70, 41])
    parts = dict(zip("qkvgs", cuda(q, k, v, g, s)))
    r = torch.Generator().manual_seed(3)
    do, ds = cuda(torch.randn(b, t, 2, dv, generator=r), torch.randn(b, 2, dk, dv, generator=r))
    u = torch.randn(parts[name].shape, generator=r).cuda()

    def loss(values):
        o, last = trnfft_amd.linear_attention(values["q"], values["k"], values["v"], values["g"],
                                              initial_state=values["s"], lengths=n.cuda(), return_state=True)
        return o, last

    leaf = {key: x.clone().requires_grad_(key == name) for key, x in parts.items()}
    o, last = loss(leaf)
    (grad,) = torch.autograd.grad([o, last], [leaf[name]], [do, ds])
    slope = float((grad.double() * u.double()).sum())
    eps = 1e-3 if name == "g" else 0.5
    values = []
    for sign in (1, -1):
        moved = dict(parts)
        moved[name] = parts[name] + sign * eps * u
        o2, last2 = loss(moved)
        values.append(float((o2.double() * do).sum() + (last2.double() * ds).sum()))
    noise = 1e-6 * (float(o.norm() * do.norm()) + float(last.norm() * ds.norm())) / eps
    curve = eps**2 / 6 * 70**2 * abs(slope) * float(u.abs().max()) ** 2 if name == "g" else 0.0
    assert abs((values[0] - values[1]) / (2 * eps) - slope) <= noise + curve


@pytest.mark.parametrize("dtype", list(TOL))
def test_padding_may_hold_anything(dtype):
    b, t, d = 3, 150, 64
    q, k, v, g, s, _ = make(b, t, (2, 2, 2, 2), d, d, dtype, seed=9, state=True)
    n = torch.tensor([0, 77, 150])
    clean = cuda(q, k, v)
    dirty = [x.clone() for x in clean]
    for x in dirty:
        for i, end in enumerate(n.tolist()):
            x[i, end:] = float("nan")
            if end + 1 < t:
                x[i, end + 1:] = float("inf")
    results = []
    for parts in (clean, dirty):
        leaves = [x.clone().requires_grad_() for x in parts] + [g.cuda().requires_grad_(), s.cuda().requires_grad_()]
        o, last = trnfft_amd.linear_attention(*leaves[:4], initial_state=leaves[4], lengths=n.cuda(), return_state=True)
        do = torch.ones_like(o)
        if parts is dirty:
            for i, end in enumerate(n.tolist()):
                do[i, end:] = float("nan")
        results.append([o, last, *torch.autograd.grad([o, last], leaves, [do, torch.ones_like(last)])])
    for x, y in zip(*results):
        assert torch.equal(x, y)
    assert torch.equal(results[0][1][0], s[0].cuda())  # a sequence of no frames leaves its state


@pytest.mark.parametrize("t", [1, 40, 200])
@pytest.mark.parametrize("dtype", list(TOL))
def test_decays_at_their_ends(t, dtype):
    # 0: nothing is forgotten; -inf: o_t = scale (q_t . k_t) v_t and the state is the last outer product
    q, k, v, _, s, _ = make(2, t, (3, 3, 3, 3), 32, 48, dtype, seed=t, state=True)
    g = torch.tensor([0.0, -math.inf, -200.0])
    ref, ref_last = reference(q.double(), k.double(), v.double(), torch.tensor([0.0, -1e4, -200.0]).double(), 0.5, s.double())
    leaves = [x.requires_grad_() for x in cuda(q, k, v, g, s)]
    o, last = trnfft_amd.linear_attention(*leaves[:4], scale=0.5, initial_state=leaves[4], return_state=True)
    assert rel(o, ref) <= TOL[dtype] and rel(last, ref_last) <= 2e-6
    assert rel(o[:, :, 1], ref[:, :, 1]) <= TOL[dtype]
    grads = torch.autograd.grad([o, last], leaves, [torch.ones_like(o), torch.ones_like(last)])
    assert all(torch.isfinite(x).all() for x in grads)
    assert grads[3][1] == 0


@pytest.mark.parametrize("dtype", list(TOL))
def test_strided_operands(dtype):
    b, t, h, d = 2, 100, 4, 32
    r = torch.Generator().manual_seed(2)
    packed = torch.randn(b, t, 3 * h * d + 5, generator=r).to(dtype).cuda()
    q, k, v = (packed[..., 3 + i * h * d:3 + (i + 1) * h * d].unflatten(-1, (h, d)) for i in range(3))
    g = (-torch.rand(h, generator=r)).cuda()
    dense = trnfft_amd.linear_attention(q.contiguous(), k.contiguous(), v.contiguous(), g)
    assert torch.equal(trnfft_amd.linear_attention(q, k, v, g), dense) or rel(trnfft_amd.linear_attention(q, k, v, g), dense.double().cpu()) <= TOL[dtype]
    # heads first in memory, features not contiguous, one key for every frame and head
    qh = q.transpose(1, 2).contiguous().transpose(1, 2)
    vt = v.transpose(2, 3).contiguous().transpose(2, 3)
    ke = k[:, :1, :1].expand(b, t, h, d)
    a = trnfft_amd.linear_attention(qh, ke, vt, g)
    e = trnfft_amd.linear_attention(q.contiguous(), ke.contiguous(), v.contiguous(), g)
    assert rel(a, e.double().cpu()) <= TOL[dtype]
    # a broadcast input gets the sum of its uses
    one = k[:, :1, :1].detach().clone().requires_grad_()
    full = k[:, :1, :1].expand(b, t, h, d).contiguous().requires_grad_()
    do = torch.randn(b, t, h, d, generator=r).to(dtype).cuda()
    (d1,) = torch.autograd.grad(trnfft_amd.linear_attention(q, one.expand(b, t, h, d), v, g), one, do)
    (d2,) = torch.autograd.grad(trnfft_amd.linear_attention(q, full, v, g), full, do)
    expect = d2.double().cpu().sum((1, 2), keepdim=True)
    size = d2.double().abs().sum((1, 2), keepdim=True).cpu()
    assert ((d1.double().cpu() - expect).abs() <= (1e-6 if dtype == torch.float32 else 2.0**-7) * size).all()


@pytest.mark.parametrize("dtype", list(TOL))
def test_a_long_sequence_in_one_head_and_in_pieces(dtype):
    # long and alone: its axis is shared out over the chip; a cut with the state carried on gives the same
    t, d = 5000, 64
    q, k, v, g, s, _ = make(1, t, (2, 2, 2, 2), d, d, dtype, seed=1, state=True, g=torch.tensor([-1e-3, -0.02]))
    ref, ref_last = reference(q.double(), k.double(), v.double(), g.double(), d**-0.5, s.double())
    q, k, v, g, s = cuda(q, k, v, g, s)
    o, last = trnfft_amd.linear_attention(q, k, v, g, initial_state=s, return_state=True)
    assert rel(o, ref) <= TOL[dtype] and rel(last, ref_last) <= 2e-6
    at, parts = 0, []
    for n in (1, 63, 64, 1000, 3, 3869):
        part, s = trnfft_amd.linear_attention(q[:, at:at + n], k[:, at:at + n], v[:, at:at + n], g, initial_state=s,
                                              return_state=True)
        parts.append(part)
        at += n
    assert at == t and rel(torch.cat(parts, 1), ref) <= TOL[dtype] and rel(s, ref_last) <= 2e-6


def test_gradients_of_a_long_sequence():
    b, t, d = 1, 3000, 64
    for dtype in TOL:
        q, k, v, g, s, _ = make(b, t, (2, 2, 2, 2), d, d, dtype, seed=11, state=True, g=torch.tensor([-1e-3, -0.1]))
        r = torch.Generator().manual_seed(1)
        do, ds = torch.randn(b, t, 2, d, generator=r).to(dtype), torch.randn(b, 2, d, d, generator=r)
        ref_in = [x.double().requires_grad_() for x in (q, k, v, g, s)]
        expected = torch.autograd.grad(reference(*ref_in[:4], d**-0.5, ref_in[4]), ref_in, [do.double(), ds.double()])
        leaves = [x.requires_grad_() for x in cuda(q, k, v, g, s)]
        out = trnfft_amd.linear_attention(*leaves[:4], initial_state=leaves[4], return_state=True)
        got = torch.autograd.grad(out, leaves, cuda(do, ds))
        for name, x, y in zip("qkvgs", got, expected):
            # (two heads' sums of some 1e6 terms of random sign: 1e-5 of the sum is 1e-8 of the terms' magnitudes)
            assert rel(x, y) <= (2e-5 if name == "g" else 2e-6 if name == "s" else TOL[dtype]), (name, dtype)


def test_no_frames_and_no_rows():
    g = torch.tensor([-0.1]).cuda()
    s = torch.randn(2, 1, 8, 8).cuda()
    q = torch.empty(2, 0, 1, 8).cuda()
    o, last = trnfft_amd.linear_attention(q, q, q, g, initial_state=s, return_state=True)
    assert o.shape == (2, 0, 1, 8) and torch.equal(last, s)
    o, last = trnfft_amd.linear_attention(q, q, q, g, return_state=True)
    assert not last.any()
    e = torch.empty(0, 5, 1, 8).cuda()
    leaf = e.clone().requires_grad_()
    gg = g.clone().requires_grad_()
    o, last = trnfft_amd.linear_attention(leaf, e, e, gg, return_state=True)
    assert o.shape == (0, 5, 1, 8) and last.shape == (0, 1, 8, 8)
    d = torch.autograd.grad(o, [leaf, gg], torch.empty_like(o))
    assert d[0].shape == leaf.shape and d[1] == 0


@pytest.mark.parametrize("dtype", list(TOL))
@pytest.mark.parametrize("b,heads,dk,dv", [(1, (1, 1, 1, 1), 1, 1), (3, (4, 2, 1, 4), 64, 64), (2, (2, 2, 2, 2), 100, 30),
                                           (5, (6, 3, 6, 2), 128, 128), (2, (2, 1, 1, 2), 200, 256), (64, (8, 8, 8, 8), 64, 64)])
def test_step_is_a_sequence_of_one(b, heads, dk, dv, dtype):
    q, k, v, g, s, _ = make(b, 3, heads, dk, dv, dtype, seed=dk, state=True)
    ref, ref_last = reference(q.double(), k.double(), v.double(), g.double(), dk**-0.5, s.double())
    q, k, v, g, s = cuda(q, k, v, g, s)
    outs = [trnfft_amd.linear_attention_step(q[:, i], k[:, i], v[:, i], g, s) for i in range(3)]
    assert rel(torch.stack(outs, 1), ref) <= tol(ref, dtype) and rel(s, ref_last) <= 2e-6


def test_step_leaves_an_odd_state_and_its_neighbours_alone():
    # a state at 4 bytes past a 16-byte boundary, with guards around it
    buf = torch.full((2 * 3 * 20 * 12 + 8,), 7.0, device="cuda")
    state = buf[1:1 + 2 * 3 * 20 * 12].view(2, 3, 20, 12)
    r = torch.Generator().manual_seed(0)
    fresh = torch.randn(2, 3, 20, 12, generator=r)
    state.copy_(fresh)
    q, k, v = (torch.randn(2, 3, d, generator=r) for d in (20, 20, 12))
    g = -torch.rand(3, generator=r)
    version = state._version
    o = trnfft_amd.linear_attention_step(*cuda(q, k, v, g), state)
    new = torch.exp(g.double())[:, None, None] * fresh.double() + k.double()[..., None] * v.double()[..., None, :]
    assert rel(state, new) <= 1e-6 and rel(o, (q.double()[..., None] * new).sum(2) * 20**-0.5) <= 1e-6
    assert buf[0] == 7 and (buf[1 + 2 * 3 * 20 * 12:] == 7).all()
    assert state._version > version


def test_other_streams_and_graphs():
    q, k, v, g, s, n = cuda(*make(2, 700, (4, 4, 2, 4), 64, 64, torch.bfloat16, seed=4, lengths=True, state=True))
    expected = trnfft_amd.linear_attention(q, k, v, g, initial_state=s, lengths=n, return_state=True)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = trnfft_amd.linear_attention(q, k, v, g, initial_state=s, lengths=n, return_state=True)
        step_state = s.clone()
        step = trnfft_amd.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g, step_state)
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(x, y) for x, y in zip(got, expected))
    graph_state, graph = s.clone(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, last = trnfft_amd.linear_attention(q, k, v, g, initial_state=s, lengths=n, return_state=True)
        first = trnfft_amd.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g, graph_state)
    for _ in range(3):
        graph_state.copy_(s)
        o.fill_(0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, expected[0]) and torch.equal(last, expected[1])
        assert torch.equal(first, step) and torch.equal(graph_state, step_state)
        q.sum().item()


def test_results_do_not_change_from_run_to_run():
    q, k, v, g, s, n = cuda(*make(2, 1000, (4, 2, 1, 4), 64, 80, torch.bfloat16, seed=6, lengths=True, state=True))
    runs = []
    for _ in range(2):
        leaves = [x.clone().requires_grad_() for x in (q, k, v, g, s)]
        o, last = trnfft_amd.linear_attention(*leaves[:4], initial_state=leaves[4], lengths=n, return_state=True)
        runs.append([o, last, *torch.autograd.grad([o, last], leaves, [torch.ones_like(o), torch.ones_like(last)])])
    assert all(torch.equal(x, y) for x, y in zip(*runs))


def test_cpu_inputs_come_back_to_the_cpu():
    q, k, v, g, s, n = make(2, 50, (2, 2, 2, 2), 16, 16, torch.float32, lengths=True, state=True)
    leaf = q.clone().requires_grad_()
    o, last = trnfft_amd.linear_attention(leaf, k, v, g, initial_state=s, lengths=n, return_state=True)
    assert o.device.type == "cpu" and last.device.type == "cpu"
    o.sum().backward()
    assert leaf.grad.device.type == "cpu"
    ref, _ = reference(q.double(), k.double(), v.double(), g.double(), 0.25, s.double(), n)
    assert rel(o, ref) <= 2e-6


def test_second_derivatives_are_refused():
    q, k, v, g, _, _ = cuda(*make(1, 20, (1, 1, 1, 1), 8, 8, torch.float32))
    leaf = q.clone().requires_grad_()
    (d,) = torch.autograd.grad(trnfft_amd.linear_attention(leaf, k, v, g).square().sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        d.sum().backward()
