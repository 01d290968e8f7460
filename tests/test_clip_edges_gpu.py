"""The gradients' norm and their clipping over more tensors than a launch's table holds, over more parts than every workgroup adds up by
itself, and over workgroups' stretches longer than the shortest.

Tolerances: squares are summed in fp64, so a norm is off by its rounding to fp32, 2^-24, and by some n 2^-53; the reference by the
latter.  A clipped value is off by the factor's rounding to fp32, 2^-24 of it, and the product's: in fp32 the result's own, 2^-24; in 16 bits
2^-24 and the result's, 2^-8 (2^-11), of fp16 subnormals 2^-25 by themselves."""

from __future__ import annotations

import math

import pytest
import torch

import trnfft_amd

pytestmark = pytest.mark.gpu

HALF = {torch.float32: 0.0, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
TYPES = tuple(HALF)


def check(flat, lists):
    """lists: [(dtype, places in its flat buffer)].  The norm, what is scaled, and that nothing else is written."""
    grads = [flat[d][begin:end] for d, places in lists for begin, end in places]
    before = {d: v.clone() for d, v in flat.items()}
    want = math.sqrt(sum(float(g.double().square().sum()) for g in grads)) if len(grads) < 1000 else None
    if want is None:  # (sums of running sums: a few calls for many tensors)
        total = 0.0
        for d, places in lists:
            sums = torch.cat([torch.zeros(1, dtype=torch.float64, device="cuda"), flat[d].double().square().cumsum(0)])
            at = torch.tensor(places, device="cuda")
            total += float((sums[at[:, 1]] - sums[at[:, 0]]).sum())
        want = math.sqrt(total)
    norm = trnfft_amd.grad_norm(grads)
    assert abs(float(norm) - want) <= 2.0**-23 * want
    factor = 0.25 * want / (want + 1e-6)
    assert torch.equal(trnfft_amd.clip_grads(grads, 0.25 * want), norm)
    for d, places in lists:
        edges = torch.zeros(flat[d].numel() + 1, dtype=torch.int32, device="cuda")
        at = torch.tensor(places, device="cuda").flatten()
        edges.index_add_(0, at, torch.tensor([1, -1], dtype=torch.int32, device="cuda").repeat(len(places)))
        inside = edges.cumsum(0)[:-1] == 1
        scaled = before[d].double() * factor
        bound = (HALF[d] + 2.0**-23) * scaled.abs() + (2.0**-25 if d == torch.float16 else 0.0)
        assert torch.where(inside, (flat[d].double() - scaled).abs() <= bound, flat[d] == before[d]).all()
    # within the bound nothing is written
    held = {d: v.clone() for d, v in flat.items()}
    trnfft_amd.clip_grads(grads, want)
    assert all(torch.equal(v, held[d]) for d, v in flat.items())


def layout(sizes, gap):
    places, end = [], 0
    for i, n in enumerate(sizes):
        begin = end + gap + i % 3  # odd addresses, values between the tensors
        end = begin + n
        places.append((begin, end))
    return places


def buffers(lists, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    return {d: torch.randn(places[-1][1] + 5, generator=g, device="cuda").to(d) for d, places in lists}


def test_more_tensors_than_a_launch_holds():
    """Of one type 400 tensors, of the others fewer; some are empty."""
    lists = [(d, layout([(37 * i * i + i) % 5003 if i % 11 else 0 for i in range(n)], 1)) for d, n in zip(TYPES, (190, 400, 45))]
    check(buffers(lists, 1), lists)


def test_more_parts_than_are_added_everywhere():
    """17000 small tensors, a part each."""
    lists = [(d, layout([1 + (7 * i) % 13 for i in range(n)], 0)) for d, n in zip(TYPES, (1000, 15000, 1000))]
    check(buffers(lists, 2), lists)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("values", [8_400_001, 17_000_003, 70_000_001, 134_300_001])
def test_longer_stretches(values, dtype):
    """Up to 64 Ki values a workgroup, the last of each tensor's odd."""
    lists = [(dtype, layout([values // 3 * 2 + 1, 0, 77, values // 3 - 65], 1))]
    check(buffers(lists, 3), lists)
