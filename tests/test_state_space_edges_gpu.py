"""The state space operators where steps are zero or there is no memory.  References and tolerances are those of
test_state_space_gpu.py: what is not masked passes the same operations, and what is masked is zero or the same bits."""

from __future__ import annotations

import pytest
import torch

import trnfft_amd
from test_state_space_gpu import SUMS, TOL, cuda, rel, scan, scan_inputs, scan_reference, tol

pytestmark = pytest.mark.gpu

# rows, t, channels, groups, states: 1, 2 and 4 states a lane, two waves a channel, segments, 8 and 16 lanes a channel
SHAPES = [(2, 37, 24, 1, 4), (2, 21, 12, 2, 7), (2, 50, 70, 2, 12), (1, 600, 20, 1, 16), (2, 35, 12, 1, 20), (2, 33, 9, 1, 40)]
INF = float("inf")


def check(v, lengths, dlast_scale=1.0, of_reference=None):
    """Outputs and all gradients against the definition; returns y, the last state and the gradients."""
    dtype, names = v["x"].dtype, list(v)
    ref = {**{k: x.double() for k, x in v.items()}, **(of_reference or {})}
    ref = {k: x.requires_grad_() for k, x in ref.items()}
    y_ref, last_ref = scan_reference(**ref, softplus=True, lengths=lengths)
    own = {k: cuda(x).requires_grad_() for k, x in v.items()}
    y, last = scan(own, cuda(lengths))
    assert rel(y, y_ref) <= tol(y_ref, dtype) and rel(last, last_ref) <= 2e-6
    g = torch.Generator().manual_seed(1)
    dy, dlast = torch.randn(y.shape, generator=g).to(dtype), torch.randn(last.shape, generator=g) * dlast_scale
    want = torch.autograd.grad([y_ref, last_ref], list(ref.values()), [dy.double(), dlast.double()])
    got = torch.autograd.grad([y, last], list(own.values()), [cuda(dy), cuda(dlast)])
    for name, w, d in zip(names, want, got):
        assert torch.isfinite(w).all(), name
        bound = SUMS if name in ("a", "d", "dt_bias") else 2e-6 if name == "state" else tol(w, dtype)
        if dtype == torch.float32 and name in ("dt", "b", "c", "z", "x"):
            bound = 4e-6
        assert rel(d, w) <= bound, name
    return y, last, dict(zip(names, got))


@pytest.mark.parametrize("dtype", list(TOL))
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_a_step_before_softplus_of_minus_infinity_is_none(shape, dtype):
    """Frames masked by dt, for a channel or for all of them, and channels masked by dt_bias leave the state."""
    v, _ = scan_inputs(*shape, dtype, 3)
    t = shape[1]
    lengths = torch.tensor([t, t - 5][:shape[0]])
    v["dt"][0, t // 2, 1] = v["dt"][:, 3] = v["dt"][-1, t - 7:] = -INF
    v["dt_bias"][2] = -INF
    y, last, grads = check(v, lengths)
    assert torch.equal(last[:, 2].cpu(), v["state"][:, 2])
    for at in ((0, t // 2, 1), (slice(None), 3), (slice(None), slice(None), 2)):
        assert not grads["dt"][at].any()
    assert not grads["dt_bias"][2].any()


@pytest.mark.parametrize("value", [-INF, torch.finfo(torch.float32).min, -200.0, 200.0, 1.8e38, 3e38])
def test_softplus_far_out(value):
    """Zero on one side and the value itself on the other, up to the type's ends."""
    one = torch.ones(1, 3, 16, device="cuda")
    b = torch.ones(1, 3, 1, 4, device="cuda")
    a = torch.zeros(16, 4, device="cuda")
    want = max(value, 0.0)
    for dt, bias in ((one * value, None), (one * 0.0, torch.full((16,), value, device="cuda"))):
        y, last = trnfft_amd.selective_scan(one * 2.0**-8, dt, a, b, b, dt_bias=bias, return_state=True)
        assert torch.equal(last, torch.full_like(last, 3 * 2.0**-8 * torch.tensor(want).item()))
        state = torch.zeros(1, 16, 4, device="cuda")
        trnfft_amd.selective_scan_step(one[:, 0] * 2.0**-8, dt[:, 0], a, b[:, 0], b[:, 0], state, dt_bias=bias)
        assert torch.equal(state, torch.full_like(state, 2.0**-8 * torch.tensor(want).item()))


@pytest.mark.parametrize("dtype", list(TOL))
@pytest.mark.parametrize("states", [4, 7, 16, 20, 40])
def test_masked_steps_leave_the_state_of_a_stream(states, dtype):
    v, _ = scan_inputs(5, 1, 24, 2, states, dtype, 4)
    one = {k: cuda(x)[:, 0] for k, x in v.items() if k in ("x", "dt", "b", "c", "z")}
    a, d, bias, state = (cuda(v[k]) for k in ("a", "d", "dt_bias", "state"))
    one["dt"][1], one["dt"][3, 7], bias[5] = -INF, -INF, -INF
    before = state.clone()
    y = trnfft_amd.selective_scan_step(one["x"], one["dt"], a, one["b"], one["c"], state, d=d, z=one["z"], dt_bias=bias)
    assert torch.isfinite(y).all() and torch.isfinite(state).all()
    assert torch.equal(state[1], before[1]) and torch.equal(state[3, 7], before[3, 7]) and torch.equal(state[:, 5], before[:, 5])
    assert not torch.equal(state[0], before[0])


@pytest.mark.parametrize("dtype", list(TOL))
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_padding_has_no_gradient_where_there_is_no_memory(shape, dtype):
    """Rates of -inf (in 64 bits, of -1e300: the same without 0 times infinity) before padding that ends inside a tile, and a large
    gradient of a large last state: the steps' bias sums up frames, not padding."""
    v, _ = scan_inputs(*shape, dtype, 5)
    lengths = torch.tensor([shape[1], shape[1] - 9][:shape[0]])
    v["state"] *= 30.0
    v["b"] *= 30.0
    far = v["a"].double()
    v["a"][1], v["a"][3, 0] = -INF, -INF
    far[1], far[3, 0] = -1e300, -1e300
    _, _, grads = check(v, lengths, dlast_scale=30.0, of_reference={"a": far})
    assert not grads["a"][1].any() and not grads["a"][3, 0].any()


@pytest.mark.parametrize("dtype", list(TOL))
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_masked_steps_have_no_gradient_where_there_is_no_memory(shape, dtype):
    """Frames of no step keep the state at rates of -inf too, and give steps no gradient, however large state and gradient are."""
    v, _ = scan_inputs(*shape, dtype, 6)
    t = shape[1]
    lengths = torch.tensor([t, t - 9][:shape[0]])
    v["state"] *= 30.0
    v["b"] *= 30.0
    far = v["a"].double()
    v["a"][1], v["a"][3, 0] = -INF, -INF
    far[1], far[3, 0] = -1e300, -1e300
    v["dt"][:, t - 12:] = v["dt"][:, 2] = -INF
    _, _, grads = check(v, lengths, dlast_scale=30.0, of_reference={"a": far})
    assert not grads["dt"][:, t - 12:].any() and not grads["dt"][:, 2].any()


@pytest.mark.parametrize("states", [4, 16, 20, 40])
def test_no_memory_for_gradients_that_are_not_wanted(states):
    """Fixed b and c: the others' gradients are the same, and the room that adds up b's and c's is not taken."""
    v, _ = scan_inputs(2, 1024, 512, 1, states, torch.bfloat16, 8, extra=False)
    own = {k: cuda(x) for k, x in v.items() if x is not None}
    peaks, grads = [], []  # (bytes as they are asked for: blocks that the allocator has at hand may be larger)
    for names in (("x", "dt", "a", "b", "c"), ("x", "dt", "a")):
        leaves = {k: x.detach().requires_grad_(k in names) for k, x in own.items()}
        y, _ = scan(leaves)
        dy = torch.ones_like(y)
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_stats()["requested_bytes.all.current"]
        grads.append(torch.autograd.grad(y, [leaves[k] for k in names], dy))
        peaks.append(torch.cuda.memory_stats()["requested_bytes.all.peak"] - before)
    for name, one, two in zip(("x", "dt", "a"), *grads):
        assert torch.equal(one, two), name
    # values of two sets of states for every token and 64 (16 above 32 states) channels, and the gradients of b and c themselves
    filled, channels = (64, 16) if states > 32 else (32, 64) if states > 16 else (16, 64) if states > 8 else (4, 64)
    assert peaks[0] - peaks[1] >= 2 * 1024 * 2 * filled * 4 * (512 // channels)
