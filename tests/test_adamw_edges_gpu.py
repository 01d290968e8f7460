"""The AdamW step where its callers and its 8-bit states are at an end: captures, outliers in a block."""

from __future__ import annotations

import pytest
import torch

import trnfft_amd
from trnfft_amd.optim import AdamW

pytestmark = pytest.mark.gpu


def test_the_optimizer_refuses_to_be_captured():
    # (replays would repeat the captured step's bias correction and leave the count where it is)
    def fresh():
        torch.manual_seed(0)
        p = torch.nn.Parameter(torch.randn(300, device="cuda"))
        p.grad = torch.randn(300, device="cuda")
        return p, AdamW([p], lr=1e-2)

    p, opt = fresh()
    opt.step()
    held, graph = p.detach().clone(), torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="captured"):
        with torch.cuda.graph(graph):
            opt.step()
    torch.cuda.synchronize()
    assert torch.equal(p, held) and opt.state[p]["step"] == 1
    opt.step()
    q, straight = fresh()
    straight.step()
    straight.step()
    assert torch.equal(p, q)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("ratio", [1e5, 5e5, 1e6, 1e8])
@pytest.mark.parametrize("on", [1, 200])
@pytest.mark.parametrize("stop", [False, True])
def test_an_outlier_in_a_block_does_not_blow_up_its_neighbours(dtype, ratio, on, stop):
    # One value's gradients are `ratio` times its neighbours' for `on` steps; the neighbours' stop 20 steps later, or go on.  fp32 states keep
    # updates of the neighbours within 1.1 lr.  Codes to nearest hold second moments still that grow slowly, worth 11 lr at most
    # by the same steps in 64 bits with these codes; moments kept beside second moments lost would be worth thousands.
    n, steps, lr = 512, 600, 1e-3
    r = torch.Generator().manual_seed(1)
    p = [torch.zeros(n, device="cuda", dtype=dtype)]
    mc, vc = [torch.zeros(n, dtype=torch.int8, device="cuda")], [torch.zeros(n, dtype=torch.uint8, device="cuda")]
    ms, vs = [torch.zeros(2, device="cuda")], [torch.zeros(2, device="cuda")]
    worst = torch.zeros((), device="cuda")
    for t in range(steps):
        g = torch.randn(n, generator=r) * 1e-4
        if stop and t >= on + 20:
            g[:] = 0
        if t < on:
            g[7] = 1e-4 * ratio
        p[0].zero_()
        trnfft_amd.adamw_step(p, [g.to("cuda", dtype)], mc, vc, step=t + 1, lr=lr, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0,
                              exp_avg_scales=ms, exp_avg_sq_scales=vs)
        p[0][7] = 0
        worst = torch.maximum(worst, p[0].abs().max().float())
    assert float(worst) <= 15 * lr


def test_second_moments_that_are_not_zero_keep_a_code():
    g = torch.full((256,), 1e-12, device="cuda")
    g[0], g[1], g[2] = 1.0, 0.0, 1e-5
    p = [torch.zeros(256, device="cuda")]
    mc, vc = [torch.zeros(256, dtype=torch.int8, device="cuda")], [torch.zeros(256, dtype=torch.uint8, device="cuda")]
    ms, vs = [torch.zeros(1, device="cuda")], [torch.zeros(1, device="cuda")]
    trnfft_amd.adamw_step(p, [g], mc, vc, step=1, exp_avg_scales=ms, exp_avg_sq_scales=vs)
    assert vc[0].tolist() == [255, 0, 1] + [1] * 253
    assert mc[0][:4].tolist() == [127, 0, 0, 0]


def test_a_gradient_that_negates_what_it_reads():
    # autograd hands the imaginary part of a conjugated tensor on as a view with the negative bit, contiguous where it has one value
    for bits in (32, 8):
        w = torch.nn.Parameter(torch.ones(1, device="cuda"))
        z = torch.complex(torch.ones(1, device="cuda"), w)
        (z.conj() * torch.tensor([1 + 2j], device="cuda")).abs().sum().backward()
        assert w.grad.is_neg() and float(w.grad) > 0
        AdamW([w], lr=0.1, weight_decay=0.0, state_bits=bits).step()
        assert abs(float(w) - 0.9) < 1e-6
        with pytest.raises(ValueError, match="negating"):
            trnfft_amd.adamw_step([w.detach()], [w.grad], [torch.zeros(1, device="cuda")], [torch.zeros(1, device="cuda")], step=1)


def test_lists_that_can_be_read_once():
    n = 600
    p, g = torch.ones(n, device="cuda", dtype=torch.bfloat16), torch.ones(n, device="cuda")
    mc, vc = torch.zeros(n, dtype=torch.int8, device="cuda"), torch.zeros(n, dtype=torch.uint8, device="cuda")
    ms, vs = torch.zeros(3, device="cuda"), torch.zeros(3, device="cuda")
    master, values = p.float(), torch.zeros(n, device="cuda")
    versions = master._version, values._version
    trnfft_amd.adamw_step(*(iter([t]) for t in (p, g, mc, vc)), step=1, exp_avg_scales=iter([ms]), exp_avg_sq_scales=iter([vs]),
                          masters=iter([master]))
    out = trnfft_amd.adamw_state_values(iter([mc]), iter([ms]), iter([values]))
    assert (master != 1).all() and torch.equal(p, master.to(p.dtype))
    assert len(out) == 1 and out[0] is values and (values != 0).all()
    assert master._version > versions[0] and values._version > versions[1]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_parameters_written_between_steps_keep_what_was_written(dtype):
    # as with torch's optimizer, which has no masters: weights that are loaded or clamped are where the next step starts
    torch.manual_seed(0)
    p = torch.nn.Parameter(torch.randn(300, device="cuda").to(dtype))
    opt = AdamW([p], lr=1e-3, weight_decay=0.0)
    r = torch.Generator().manual_seed(0)
    for _ in range(3):
        p.grad = torch.randn(300, generator=r).to("cuda", dtype)
        opt.step()
    kept, before = opt.state[p]["master"][100:].clone(), p.detach().clone()
    with torch.no_grad():
        p[:100] = 7.0
    p.grad = torch.zeros(300, device="cuda", dtype=dtype)
    opt.step()
    # (a zero gradient moves by the momentum alone: 3 lr at most)
    assert ((p[:100].float() - 7.0).abs() <= 7.0 * 2.0**-8).all()
    assert ((opt.state[p]["master"][:100] - 7.0).abs() <= 3e-3).all()
    assert ((opt.state[p]["master"][100:] - kept).abs() <= 3e-3).all() and (kept != before[100:].float()).any()
    # and what a checkpoint brings back is its own
    saved, weights = opt.state_dict(), p.detach().clone()
    again = torch.nn.Parameter(weights)
    other = AdamW([again], lr=1e-3, weight_decay=0.0)
    other.load_state_dict(saved)
    for q, o in ((p, opt), (again, other)):
        q.grad = torch.ones(300, device="cuda", dtype=dtype)
        o.step()
    assert torch.equal(opt.state[p]["master"], other.state[again]["master"]) and torch.equal(p, again)
