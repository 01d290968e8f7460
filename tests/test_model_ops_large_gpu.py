"""Operands of more than 2^31 elements: what lies behind the 32-bit offsets equals the same data taken alone.

Tolerances: two bf16 results of one value, each rounded from fp32 sums in its own order, differ by sqrt(2) of one rounding's
1.7e-3 in the mean square at most: 2.4e-3, a factor of 1.25 above.  AdamW's blocks do not depend on where they lie: equal bits.
"""

import pytest
import torch

import trnfft_amd

pytestmark = pytest.mark.gpu

TOL = 3e-3


def rel(got, ref):
    return float((got.double() - ref.double()).norm() / ref.double().norm())


def test_linear_attention():
    frames, heads, dim = (1 << 31) // (16 * 128) + 4160, 16, 128
    q, k, v = (torch.randn(1, frames, heads, dim, device="cuda", dtype=torch.bfloat16) for _ in range(3))
    decay = torch.full((heads,), -0.1, device="cuda")  # nothing is left of a frame after 4096: e^-409
    o, state = trnfft_amd.linear_attention(q, k, v, decay, return_state=True)
    assert o.numel() > 1 << 31
    tail, tail_state = trnfft_amd.linear_attention(q[:, -4160:], k[:, -4160:], v[:, -4160:], decay, return_state=True)
    assert rel(o[:, -64:], tail[:, -64:]) <= TOL
    # fp32 states of sums of some ten frames' products in another order
    assert rel(state, tail_state) <= 1e-5


def test_group_norm():
    x = torch.randn(3, 11_300_000, 64, device="cuda", dtype=torch.bfloat16)
    assert x[:2].numel() < 1 << 31 < x.numel()
    y = trnfft_amd.group_norm(x, 8, activation="silu")
    alone = trnfft_amd.group_norm(x[2:].clone(), 8, activation="silu")
    assert rel(y[2, -5000:], alone[0, -5000:]) <= TOL


def test_adamw():
    n, tail = (1 << 31) + 256 * 40 + 77, 256 * 64 + 77
    p = torch.randn(n, device="cuda", dtype=torch.bfloat16)
    g = torch.randn(n, device="cuda", dtype=torch.bfloat16)
    m, v = torch.randint(-127, 128, (n,), device="cuda", dtype=torch.int8), torch.randint(128, 256, (n,), device="cuda", dtype=torch.uint8)
    ms, vs = (torch.rand(-(-n // 256), device="cuda") + 0.1 for _ in range(2))
    small = [t[-tail:].clone() for t in (p, g, m, v)]
    scales = [t[-65:].clone() for t in (ms, vs)]
    trnfft_amd.adamw_step([p], [g], [m], [v], step=3, exp_avg_scales=[ms], exp_avg_sq_scales=[vs])
    trnfft_amd.adamw_step(*([t] for t in small), step=3, exp_avg_scales=[scales[0]], exp_avg_sq_scales=[scales[1]])
    for whole, alone in zip((p, m, v), (small[0], small[2], small[3])):
        assert torch.equal(whole[-tail:], alone)
    assert torch.equal(ms[-65:], scales[0]) and torch.equal(vs[-65:], scales[1])
