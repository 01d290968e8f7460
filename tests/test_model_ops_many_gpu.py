"""More rows than one launch's 2^32 threads: what lies past them equals the same rows taken alone, bit for bit (rows do not depend on each
other), and group norm its definition.

Tolerances: an fp32 norm of three values is some ten operations of 2^-24 each (1e-6 of a value of order 1, ten times that where three
values are close together); the weights' gradients are sums of 2^24 terms in 2^8 runs, whose rounding is far below 1e-5 of their magnitudes."""

import pytest
import torch

import trnfft_amd

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("ragged", [False, True])
def test_group_norm(ragged):
    n = (1 << 24) + 1001
    x = torch.randn(n, 1, 3, device="cuda")
    dy = torch.randn(n, 1, 3, device="cuda")
    lengths = torch.arange(n, device="cuda") % 3 if ragged else None
    w, b = torch.tensor([0.5, 1.0, 2.0], device="cuda"), torch.tensor([0.1, 0.0, -0.3], device="cuda")
    leaves = [t.requires_grad_() for t in (x, w, b)]
    y = trnfft_amd.group_norm(x, 1, w, b, eps=0.1, lengths=lengths)
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    live = torch.ones(n, 1, 1, device="cuda") if lengths is None else (lengths > 0).view(n, 1, 1)
    with torch.no_grad():
        d = x.double()
        d = d - d.mean(-1, keepdim=True)
        rstd = (d.square().mean(-1, keepdim=True) + 0.1).rsqrt()
        xh, g = d * rstd, dy.double() * live
        assert float((y - (xh * w + b) * live).abs().max()) <= 1e-5
        e = g * w
        ref = rstd * (e - e.mean(-1, keepdim=True) - xh * (e * xh).mean(-1, keepdim=True))
        assert float((dx - ref * live).abs().max()) <= 2e-5
        for got, terms in ((dw, g * xh), (db, g)):
            assert ((got - terms.sum((0, 1))).abs() <= 1e-5 * terms.abs().sum((0, 1))).all()


def tail_alone(q, k, v, g, do, rows=37):
    """The call on all batch rows and on the last ones."""
    results = []
    for cut in (slice(None), slice(-rows, None)):
        leaves = [x[cut].detach().requires_grad_() for x in (q, k, v)]
        o, last = trnfft_amd.linear_attention(*leaves, g, return_state=True)
        grads = torch.autograd.grad(o, leaves, do[cut])
        results.append([x[-rows:].detach().clone() for x in (o, last, *grads)])
    for whole, alone in zip(*results):
        assert torch.equal(whole, alone) and alone.any()


def test_linear_attention_in_blocks():
    # two heads that share keys and values: copies of odd operands, passes, sums over the shared heads
    b, t = (1 << 25) + 39, 4
    q, k, v, do = (torch.randn(b, t, h, 3, device="cuda") for h in (2, 1, 1, 2))
    tail_alone(q, k, v, torch.tensor([-0.1, -0.5], device="cuda"), do)


def test_linear_attention_token_by_token():
    b, t, h, d = (1 << 20) + 39, 2, 4, 129
    q, k, v, do = (torch.randn(b, t, h, d, device="cuda", dtype=torch.bfloat16) for _ in range(4))
    tail_alone(q, k, v, torch.full((h,), -0.1, device="cuda"), do)


def test_linear_attention_step():
    b, h = (1 << 20) + 39, 16
    q, k, v = (torch.randn(b, h, 1, device="cuda") for _ in range(3))
    state = torch.randn(b, h, 1, 1, device="cuda")
    g = torch.full((h,), -0.1, device="cuda")
    alone = state[-37:].clone()
    o = trnfft_amd.linear_attention_step(q, k, v, g, state)
    assert torch.equal(o[-37:], trnfft_amd.linear_attention_step(q[-37:], k[-37:], v[-37:], g, alone))
    assert torch.equal(state[-37:], alone)
