"""The operators of a state space layer behind 32-bit offsets and past one launch's workgroups, and values at the ends of what they take.

Tolerances as in test_state_space_gpu.py: the same frames computed from a state instead of behind a long sequence are the same
operations but for the tile that a frame falls into, so fp32 states agree to some roundings and 16-bit outputs but for one that
falls on the other side now and then."""

from __future__ import annotations

import pytest
import torch

import trnfft_amd

pytestmark = pytest.mark.gpu


def test_past_32_bit_offsets():
    """2.3e9 values: the last frames, and the first ones' gradients, are those of a short call."""
    t, ch, n, tail = 1_100_003, 2080, 1, 40
    g = torch.Generator("cuda").manual_seed(0)
    x = torch.empty(1, t, ch, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    w = torch.randn(ch, 4, generator=g, device="cuda")
    y, last = trnfft_amd.causal_conv(x, w, activation="silu", return_state=True)
    want = trnfft_amd.causal_conv(x[:, -tail:], w, activation="silu", initial_state=x[:, -tail - 3:-tail].contiguous())
    assert torch.equal(y[:, -tail:], want) and torch.equal(last, x[:, -3:])
    del y
    a = -torch.rand(ch, n, generator=g, device="cuda") - 0.5
    b, c = (torch.randn(1, t, 1, n, generator=g, device="cuda").bfloat16() for _ in range(2))
    cut = t - tail
    with torch.no_grad():
        y, last = trnfft_amd.selective_scan(x, x, a, b, c, return_state=True)
        _, state = trnfft_amd.selective_scan(x[:, cut - 400:cut], x[:, cut - 400:cut], a, b[:, cut - 400:cut], c[:, cut - 400:cut],
                                             return_state=True)  # (older frames have decayed to nothing)
        want, end = trnfft_amd.selective_scan(x[:, cut:], x[:, cut:], a, b[:, cut:], c[:, cut:], initial_state=state, return_state=True)
    assert float((last - end).norm()) <= 2e-6 * float(end.norm())
    assert float((y[:, cut:].float() - want.float()).norm()) <= 1e-3 * float(want.float().norm())
    leaves = [x.requires_grad_(), b.requires_grad_()]
    dy = torch.zeros_like(y)
    dy[:, cut:] = 1.0
    del y, want
    dx, db = torch.autograd.grad(trnfft_amd.selective_scan(x, x.detach(), a, b, c), leaves, dy)
    short = [v[:, cut - 400:].detach().clone().requires_grad_() for v in (x, b)]
    out = trnfft_amd.selective_scan(short[0], short[0].detach(), a, short[1], c[:, cut - 400:])
    wx, wb = torch.autograd.grad(out, short, dy[:, cut - 400:])
    for got, want in ((dx, wx), (db, wb)):
        assert float((got[:, -tail:].float() - want[:, -tail:].float()).norm()) <= 2e-3 * float(want[:, -tail:].float().norm())
    assert not dx[:, :1000].any()


def test_more_rows_than_one_launch():
    """2^24 + 3 rows of one frame: a launch holds 2^24 - 1 workgroups."""
    rows = 2**24 + 3
    g = torch.Generator("cuda").manual_seed(1)
    x, b, c = (torch.randn(rows, 1, 1, generator=g, device="cuda") for _ in range(3))
    dt = torch.rand(rows, 1, 1, generator=g, device="cuda")
    a, d = torch.full((1, 1), -0.5, device="cuda"), torch.full((1,), 2.0, device="cuda")
    state = torch.randn(rows, 1, 1, generator=g, device="cuda")
    h = torch.exp(dt.double() * -0.5) * state.double() + (dt * 1.0).double() * x.double() * b.double()
    want = (c.double() * h + 2.0 * x.double()).float()
    leaves = [x.requires_grad_(), a.requires_grad_()]
    y, last = trnfft_amd.selective_scan(x, dt, a, b[..., None], c[..., None], d=d, softplus=False, initial_state=state, return_state=True)
    assert float((y - want).abs().max()) <= 2e-5 and float((last - h).abs().max()) <= 1e-5
    dx, da = torch.autograd.grad(y, leaves, torch.ones_like(y))
    assert float((dx - (c * dt * b + 2.0)).abs().max()) <= 2e-5
    terms = c.double() * dt.double() * torch.exp(dt.double() * -0.5) * state.double()
    assert abs(float(da) - float(terms.sum())) <= 1e-5 * float(terms.abs().sum())
    with torch.no_grad():
        got = trnfft_amd.selective_scan_step(x[:, 0], dt[:, 0], a, b, c, state, d=d, softplus=False)
        assert float((got - want[:, 0]).abs().max()) <= 2e-5 and float((state - h).abs().max()) <= 1e-5
        w = torch.tensor([[0.5, 2.0]], device="cuda")
        before = torch.randn(rows, 1, 1, generator=g, device="cuda")
        assert torch.equal(trnfft_amd.causal_conv(x, w, initial_state=before), torch.addcmul(before * 0.5, x, torch.full_like(x, 2.0)))
        held = before.clone()
        assert torch.equal(trnfft_amd.causal_conv_step(x[:, 0], held, w), torch.addcmul(before * 0.5, x, torch.full_like(x, 2.0))[:, 0])
        assert torch.equal(held, x)


def test_no_memory_and_much_memory():
    """Rates of -inf and 0: outputs are those of the frame alone, and sums over all frames; padding changes neither state."""
    g = torch.Generator("cuda").manual_seed(2)
    x, dt, b, c = (torch.randn(2, 37, k, generator=g, device="cuda") for k in (20, 20, 4, 4))
    dt = dt.abs() + 0.1
    lengths = torch.tensor([37, 21], device="cuda")
    for rate in (float("-inf"), -3e38, 0.0):
        a = torch.full((20, 4), rate, device="cuda", requires_grad=True)
        y, last = trnfft_amd.selective_scan(x, dt, a, b[:, :, None], c[:, :, None], softplus=False, lengths=lengths, return_state=True)
        terms = (dt * x).double()[..., None] * b.double()[:, :, None]
        terms[1, 21:] = 0.0
        h = terms.cumsum(1) if rate == 0.0 else terms
        want = (h * c.double()[:, :, None]).sum(-1)
        want[1, 21:] = 0.0
        end = torch.stack([h[0, 36], h[1, 20]])
        assert float((y - want).norm()) <= 2e-6 * float(want.norm()) and float((last - end).norm()) <= 2e-6 * float(end.norm())
        da, = torch.autograd.grad(y.sum() + last.sum(), a)
        assert torch.isfinite(da).all() and (rate == 0.0 or not da.any())
        step = torch.ones(2, 20, 4, device="cuda")
        with torch.no_grad():
            trnfft_amd.selective_scan_step(x[:, 0], dt[:, 0], a, b[:, 0, None], c[:, 0, None], step, softplus=False)
        want = terms[:, 0] + (1.0 if rate == 0.0 else 0.0)
        assert float((step - want).norm()) <= 1e-6 * float(want.norm())


def test_frames_far_apart():
    """Frames 2^24 and more values apart are laid out anew."""
    flat = torch.randn(3 * (1 << 24) + 100, device="cuda")
    x = flat.as_strided((1, 3, 16), (0, 1 << 24, 1))
    a, b = -torch.ones(16, 4, device="cuda"), torch.randn(1, 3, 1, 4, device="cuda")
    assert torch.equal(trnfft_amd.selective_scan(x, x, a, b, b), trnfft_amd.selective_scan(*[x.contiguous()] * 2, a, b, b))


@pytest.mark.parametrize("order", ["up", "down", "one", "all", "none"])
@pytest.mark.parametrize("rows", [5, 70, 300])
def test_ragged_rows_in_any_order(rows, order):
    """Rows are worked on in the order of their lengths: each comes out in its own place."""
    t = 50
    lengths = torch.arange(rows) % (t + 1)
    if order != "up":
        lengths = {"down": lengths.flip(0), "one": torch.ones(rows), "all": torch.full((rows,), t), "none": torch.zeros(rows)}[order].long()
    g = torch.Generator("cuda").manual_seed(3)
    x, dt = (torch.randn(rows, t, 24, generator=g, device="cuda") for _ in range(2))
    b, c = (torch.randn(rows, t, 1, 8, generator=g, device="cuda") for _ in range(2))
    a = -torch.rand(24, 8, generator=g, device="cuda")
    y, last = trnfft_amd.selective_scan(x, dt, a, b, c, lengths=lengths.cuda(), return_state=True)
    for i in range(0, rows, max(1, rows // 7)):
        n = int(lengths[i])
        one, end = trnfft_amd.selective_scan(*[v[i:i + 1, :n] for v in (x, dt)], a, *[v[i:i + 1, :n] for v in (b, c)], return_state=True)
        assert torch.equal(y[i, :n], one[0]) and torch.equal(last[i], end[0]) and not y[i, n:].any()
