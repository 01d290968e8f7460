"""Linear attention where its inputs are at an end: values that are not finite in live frames, decays that are NaN, no frames,
long streams.  What a value that is not finite reaches is what the recurrence in 64 bits says; all else is equal bits to the same call
without it."""

from __future__ import annotations

import math

import pytest
import torch

import trnfft_amd

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def recurrence(a, b, c, g, reverse=False):
    """out_t = sum gamma^|t - s| (a_t . b_s) c_s over s <= t (or s >= t) and the end state, token by token, (batch, token, head, feature)."""
    a, b, c = (x.double() for x in (a, b, c))
    gamma = torch.exp(g.double())[:, None, None]
    order = range(a.shape[1])
    m = torch.zeros(*b.shape[:1], *b.shape[2:], c.shape[-1], dtype=torch.float64)
    out = [None] * a.shape[1]
    for t in reversed(order) if reverse else order:
        m = gamma * m + b[:, t, :, :, None] * c[:, t, :, None, :]
        out[t] = (a[:, t, :, None, :] @ m)[..., 0, :]
    return torch.stack(out, 1), m


def same_but_where_not_finite(got, clean, ref):
    """got is not finite exactly where ref is not, and clean's bits elsewhere."""
    bad = ~torch.isfinite(ref)
    got, clean = got.detach().cpu(), clean.detach().cpu()
    assert torch.equal(~torch.isfinite(got), bad)
    assert torch.equal(torch.where(bad, 0.0, got), torch.where(bad, 0.0, clean))


def run(parts, g, do, decays):
    leaves = [x.cuda().requires_grad_() for x in parts]
    g = g.cuda().requires_grad_(decays)
    o, last = trnfft_amd.linear_attention(*leaves, g, scale=1.0, return_state=True)
    grads = torch.autograd.grad(o, leaves + ([g] if decays else []), do.cuda())
    return o, last, *grads


# (a head of 160 features goes token by token; 600 frames of one sequence are shared out over segments)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,dk,dv", [(150, 32, 48), (600, 64, 128), (130, 128, 128), (90, 160, 16)])
@pytest.mark.parametrize("where", ["first", "middle", "last"])
@pytest.mark.parametrize("name,value", [("k", math.nan), ("v", math.inf), ("v", math.nan), ("q", -math.inf), ("do", math.inf)])
def test_what_is_not_finite_does_not_reach_back(dtype, t, dk, dv, where, name, value):
    r = torch.Generator().manual_seed(t + dk)
    q, k, v, do = (torch.randn(1, t, 2, d, generator=r).to(dtype) for d in (dk, dk, dv, dv))
    g = torch.tensor([-0.02, -0.3])
    clean = {decays: run((q, k, v), g, do, decays) for decays in (False, True)}
    at = {"first": 0, "middle": t // 2 + 2, "last": t - 1}[where]
    dirty = {"q": q.clone(), "k": k.clone(), "v": v.clone(), "do": do.clone()}
    dirty[name][0, at, 0, 5 if name in "qk" else dv - 2] = value
    q, k, v, do = (dirty[n] for n in ("q", "k", "v", "do"))
    o, last = recurrence(q, k, v, g)
    refs = [o, last, recurrence(do, v, k, g)[0], recurrence(v, do, q, g, True)[0], recurrence(k, q, do, g, True)[0]]
    for decays in (False, True):
        got = run((q, k, v), g, do, decays)
        for x, y, ref in zip(got, clean[decays], refs):
            same_but_where_not_finite(x, y, ref)
        if decays:
            assert torch.equal(got[5][1], clean[True][5][1])  # the other head's decay


@pytest.mark.parametrize("dtype", DTYPES)
def test_values_near_the_largest_stay_in_their_frames(dtype):
    # the largest finite value of the type, in a value that later frames alone may see
    q, k, v = (torch.randn(1, 100, 1, 32, generator=torch.Generator().manual_seed(i)).to(dtype) for i in range(3))
    g = torch.tensor([-0.1])
    clean = trnfft_amd.linear_attention(*(x.cuda() for x in (q, k, v, g)))
    v[0, 40, 0, 3] = torch.finfo(dtype).max
    got = trnfft_amd.linear_attention(*(x.cuda() for x in (q, k, v, g)))
    assert torch.equal(got[:, :40], clean[:, :40])
    assert torch.equal(got[..., :3], clean[..., :3]) and torch.equal(got[..., 4:], clean[..., 4:])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,d", [(1, 64), (100, 64), (600, 32), (20, 160)])
def test_a_decay_that_is_nan_shows(dtype, t, d):
    r = torch.Generator().manual_seed(t)
    parts = [torch.randn(2, t, 3, d, generator=r).to(dtype) for _ in range(3)]
    do = torch.randn(2, t, 3, d, generator=r).to(dtype)
    g = torch.tensor([-0.1, math.nan, -math.inf])
    got, clean = run(parts, g, do, True), run(parts, torch.tensor([-0.1, -0.2, -math.inf]), do, True)
    for i, (x, y) in enumerate(zip(got, clean)):
        axis = {1: 1, 5: 0}.get(i, 2)  # (of the heads)
        x, y = x.movedim(axis, 0), y.movedim(axis, 0)
        nan = x[1][:, :-1] if i in (3, 4) else x[1]  # (the last frame's keys and values reach its output undecayed)
        assert nan.isnan().all()
        assert torch.equal(x[0], y[0]) and torch.equal(x[2], y[2])
    state = torch.zeros(2, 3, d, d, device="cuda")
    o = trnfft_amd.linear_attention_step(*(x[:, 0].cuda() for x in parts), g.cuda(), state)
    assert o[:, 1].isnan().all() and state[:, 1].isnan().all()
    assert torch.isfinite(o[:, ::2]).all() and torch.isfinite(state[:, ::2]).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads", [(2, 2, 2), (2, 1, 1), (1, 2, 1)])
def test_gradients_of_no_frames(dtype, heads):
    # the state goes through: its gradient is the end state's (divided by the scale and multiplied again: three roundings), the
    # decays' has no lag to count
    q, k, v = (torch.empty(2, 0, n, d, device="cuda", dtype=dtype, requires_grad=True) for n, d in zip(heads, (8, 8, 16)))
    g = torch.tensor([-0.1, -0.2], device="cuda", requires_grad=True)
    s = torch.randn(2, 2, 8, 16, device="cuda", requires_grad=True)
    ds = torch.randn(2, 2, 8, 16, device="cuda")
    o, last = trnfft_amd.linear_attention(q, k, v, g, initial_state=s, return_state=True)
    got = torch.autograd.grad([o, last], [q, k, v, g, s], [torch.empty_like(o), ds])
    assert all(x.shape == y.shape for x, y in zip(got, (q, k, v, g, s)))
    assert not got[3].any() and ((got[4] - ds).abs() <= 2.0**-22 * ds.abs()).all()
    (only,) = torch.autograd.grad(trnfft_amd.linear_attention(q, k, v, g.detach(), initial_state=s, return_state=True)[1], s, ds)
    assert torch.equal(only, got[4])


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_long_stream_keeps_the_precision_of_its_state(dtype):
    # 3000 steps: each rounds a state twice, to 2^-24 of it at most and 3.7e-8 in the mean square together, which adds up to 40 (the root of
    # half their number) times that, 1.5e-6, where nothing is forgotten; a factor of 2.7 above.  (A decay rounded to one fp32 would be off by
    # up to 3e-8 of it at every step in one direction, 9e-5 at the end.)
    t, d = 3000, 16
    g = torch.tensor([-1e-4, -2e-4, -4e-4, -7e-4, -1e-3, -1.7e-3, -2.3e-3, -1 / 256])
    r = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(t, 1, len(g), d, generator=r).to(dtype) for _ in range(3))
    state, ref = torch.zeros(1, len(g), d, d, device="cuda"), torch.zeros(1, len(g), d, d, dtype=torch.float64)
    gamma = torch.exp(g.double())[:, None, None]
    for x in zip(k.double(), v.double()):
        ref = gamma * ref + x[0][..., None] * x[1][..., None, :]
    qc, kc, vc, gc = (x.cuda() for x in (q, k, v, g))
    for i in range(t):
        trnfft_amd.linear_attention_step(qc[i], kc[i], vc[i], gc, state)
    off = (state.double().cpu() - ref).flatten(2).norm(dim=2) / ref.flatten(2).norm(dim=2)
    assert (off <= 4e-6).all(), off


def test_views_that_negate_what_they_read():
    # one value each: contiguous, and still the negative of its memory
    one = torch.ones(1, 1, 1, 1, device="cuda")
    minus = torch.complex(one, one).conj().imag
    assert minus.is_neg() and minus.is_contiguous()
    g = torch.complex(torch.zeros(1, device="cuda"), torch.ones(1, device="cuda")).conj().imag
    o, last = trnfft_amd.linear_attention(one, one, one, g, initial_state=minus, return_state=True)
    expect = 1.0 - math.exp(-1.0)
    assert abs(float(o) - expect) < 1e-6 and abs(float(last) - expect) < 1e-6
    assert abs(float(trnfft_amd.linear_attention_step(one[0], minus[0], one[0], g, one.clone())) - (math.exp(-1.0) - 1.0)) < 1e-6
    with pytest.raises(ValueError):
        trnfft_amd.linear_attention_step(one[0], one[0], one[0], g, minus)
    leaves = [x.clone().requires_grad_() for x in (one, one, one, one)]
    out = trnfft_amd.linear_attention(*leaves[:3], g, initial_state=leaves[3], return_state=True)
    grads = torch.autograd.grad(out, leaves, [minus, minus])
    # d(o + last) with o = q (v k + gamma s), last = v k + gamma s, all ones, times -1
    for x, expect in zip(grads, (-1.0 - math.exp(-1.0), -2.0, -2.0, -2.0 * math.exp(-1.0))):
        assert abs(float(x) - expect) < 1e-6


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_step_takes_its_operands_where_they_lie(dtype):
    # three heads of 20 features in a row of a projection, at odd addresses: no copies, the output is all that is allocated
    r = torch.Generator().manual_seed(0)
    packed = torch.randn(2, 1 + 3 * 3 * 20, generator=r).to(dtype)
    g, s = torch.tensor([-0.1, -0.2, -0.3]), torch.randn(2, 3, 20, 20, generator=r)
    q, k, v = (x.unflatten(-1, (3, 20)) for x in packed.cuda()[:, 1:].split(60, dim=-1))
    assert all(x.data_ptr() % 16 for x in (q, k, v))
    gc, state, dense = g.cuda(), s.cuda(), s.cuda()
    expected = trnfft_amd.linear_attention_step(q.contiguous(), k.contiguous(), v.contiguous(), gc, dense)
    before = torch.cuda.memory_stats()["allocation.all.allocated"]
    o = trnfft_amd.linear_attention_step(q, k, v, gc, state)
    assert torch.cuda.memory_stats()["allocation.all.allocated"] == before + 1
    assert torch.equal(o, expected) and torch.equal(state, dense)
