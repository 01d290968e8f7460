"""The gradients' global norm and their clipping against 64 bits.

Tolerances: squares are summed in fp64, so a norm is off by its rounding to fp32, 2^-24, and by n 2^-53 at most.  A clipped value is
the factor's rounding, the product's and, in 16 bits, the result's: 2 2^-24 + 2^-9 (2^-12) of it."""

from __future__ import annotations

import math

import pytest
import torch

import trnfft_amd
from trnfft_amd.optim import AdamW, clip_grad_norm_

pytestmark = pytest.mark.gpu

HALF = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
SIZES = [(1,), (3, 5), (16383,), (16384,), (16385,), (128, 300), (0,), (7,), (100_001,), (2, 3, 4)]


def gradients(dtypes, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(s, generator=g) * scale).to(dtypes[i % len(dtypes)]).cuda() for i, s in enumerate(SIZES)]


def norm_of(grads):
    return math.sqrt(sum(float(x.double().square().sum()) for x in grads))


@pytest.mark.parametrize("dtypes", [(torch.float32,), (torch.bfloat16,), (torch.float16,), (torch.bfloat16, torch.float32, torch.float16)], ids=str)
@pytest.mark.parametrize("share", [0.25, 4.0])
def test_clip(dtypes, share):
    grads = gradients(dtypes)
    before, want = [x.clone() for x in grads], norm_of(grads)
    versions = [x._version for x in grads]
    assert abs(float(trnfft_amd.grad_norm(grads)) - want) <= 2.0**-23 * want
    norm = trnfft_amd.clip_grads(grads, share * want)
    assert norm.shape == () and norm.dtype == torch.float32 and norm.is_cuda
    assert abs(float(norm) - want) <= 2.0**-23 * want
    factor = min(1.0, share * want / (want + 1e-6))
    for x, old, version in zip(grads, before, versions):
        if share > 1:
            assert torch.equal(x, old)
        else:
            assert ((x.double() - old.double() * factor).abs() <= (HALF[x.dtype] + 2.0**-23) * (old.double() * factor).abs() + 1e-7).all()
        assert x._version > version


def test_odd_addresses_and_rest_of_a_buffer():
    flat = torch.full((200_003,), 3.0, device="cuda")
    grads = [flat[1:50_002], flat[50_003:50_004], flat[100_001:]]
    norm = trnfft_amd.clip_grads(grads, 1.0)
    assert abs(float(norm) - 3.0 * math.sqrt(sum(x.numel() for x in grads))) <= 1e-6 * float(norm)
    inside = torch.zeros_like(flat, dtype=torch.bool)
    inside[1:50_002] = inside[50_003] = inside[100_001:] = True
    assert (flat[~inside] == 3.0).all() and (flat[inside] < 1.0).all()


def test_squares_neither_overflow_nor_vanish():
    for value in (1e30, 1e-30, 3e38):
        x = torch.full((20_000,), value, device="cuda")
        want = float(x[0]) * math.sqrt(20_000)
        got = float(trnfft_amd.grad_norm([x]))
        assert got == float("inf") if want > 3.4e38 else abs(got - want) <= 2.0**-23 * want
    x = torch.full((20_000,), 1e30, device="cuda")
    trnfft_amd.clip_grads([x], 1.0)
    assert abs(norm_of([x]) - 1.0) <= 1e-6


@pytest.mark.parametrize("value", [float("inf"), float("nan")])
def test_what_is_not_finite(value):
    grads = gradients((torch.float32,))
    grads[3][5] = value
    assert not math.isfinite(float(trnfft_amd.clip_grads(grads, 1.0)))
    flat = torch.cat([x.flatten() for x in grads])
    if math.isnan(value):
        assert flat.isnan().all()
    else:
        assert flat.isnan().sum() == 1 and not flat[~flat.isnan()].any()
    p = torch.nn.Parameter(torch.zeros(4, device="cuda"))
    p.grad = torch.tensor([1.0, value, 2.0, 3.0], device="cuda")
    with pytest.raises(RuntimeError, match="not finite"):
        clip_grad_norm_(p, 1.0, error_if_nonfinite=True)
    assert p.grad[0] == 1.0


def test_the_norm_does_not_depend_on_timing():
    grads = [torch.randn(1 << 20, device="cuda", generator=torch.Generator("cuda").manual_seed(i)) for i in range(20)]
    first = trnfft_amd.grad_norm(grads)
    assert all(torch.equal(first, trnfft_amd.grad_norm(grads)) for _ in range(5))


def test_parameters():
    torch.manual_seed(0)
    m = torch.nn.Sequential(torch.nn.Linear(30, 40), torch.nn.Linear(40, 7)).cuda()
    m[1].weight.grad = torch.randn(40, 7, device="cuda").t()  # as a transposed weight's
    m[0].weight.grad, m[0].bias.grad = torch.randn(40, 30, device="cuda"), torch.randn(40, device="cuda")
    params = [*m.parameters(), *m.parameters()]  # listed twice: taken once
    before = [None if p.grad is None else p.grad.clone() for p in m.parameters()]
    want = norm_of([x for x in before if x is not None])
    assert abs(float(clip_grad_norm_(params, 0.5)) - want) <= 2.0**-23 * want
    for p, old in zip(m.parameters(), before):
        assert (p.grad is None) == (old is None)
        if old is not None:
            torch.testing.assert_close(p.grad, old * (0.5 / (want + 1e-6)), rtol=1e-6, atol=0)
    assert float(clip_grad_norm_([], 1.0)) == 0.0
    AdamW(m.parameters(), lr=1e-3).step()


def test_captured_and_replayed():
    source = [torch.randn(s, device="cuda") for s in (40_000, 333)]
    grads = [x.clone() for x in source]
    trnfft_amd.clip_grads(grads, 1.0)  # (loads the kernels)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = trnfft_amd.clip_grads(grads, 1.0)
    for i in range(3):
        for x, s in zip(grads, source):
            x.copy_(s * (i + 1))
        want = norm_of(grads)
        graph.replay()
        torch.cuda.synchronize()
        assert abs(float(norm) - want) <= 2.0**-23 * want and abs(norm_of(grads) - 1.0) <= 1e-5


def test_refusals_of_the_native_call():
    good = torch.ones(8, device="cuda")
    for bad, error, text in ((torch.ones(8, device="cuda", dtype=torch.float64), TypeError, "got torch.float64"),
                             (torch.ones(4, 4, device="cuda").t()[1:], ValueError, "contiguous"),
                             (torch.ones(8), ValueError, "GPU of the first"), (3, TypeError, "tensors")):
        version = good._version
        for call in (lambda g: trnfft_amd.grad_norm(g), lambda g: trnfft_amd.clip_grads(g, 0.5)):
            with pytest.raises(error, match=text):
                call([good, bad])
        assert good._version == version and torch.equal(good, torch.ones_like(good))
    version = good._version
    assert float(trnfft_amd.clip_grads([good], 100.0)) == pytest.approx(8.0**0.5, rel=1e-6) and good._version > version
