"""Group norm with an activation against its definition in 64 bits, its gradients against the definition's and against
differences.

Tolerances (relative 2-norm): fp32 results are a handful of fp32 operations on statistics of up to a million terms summed
in blocks, 2e-6; 16-bit results are rounded once from such, 1.7e-3 (2.1e-4) in the mean square, a factor of 1.2 above."""

from __future__ import annotations

import math

import pytest
import torch
import torch.nn.functional as F

import trnfft_amd
from trnfft_amd.nn import GroupNorm

pytestmark = pytest.mark.gpu

TOL = {torch.float32: 2e-6, torch.bfloat16: 2.1e-3, torch.float16: 2.6e-4}
ACT = {None: lambda z: z, "silu": F.silu, "gelu": F.gelu, "relu": F.relu}


def reference(x, groups, w, b, eps, act, lengths=None):
    """Sample by sample over its live positions, in float64; eps under the root."""
    parts = []
    for i in range(x.shape[0]):
        end = x.shape[1] if lengths is None else int(lengths[i].clamp(0, x.shape[1]))
        live = x[i, :end] if x.dim() > 2 else x[i]
        r = live.reshape(-1, groups, x.shape[-1] // groups)
        if r.numel() == 0:
            parts.append(torch.zeros_like(x[i]) + 0.0 * x[i].nan_to_num(0.0, 0.0, 0.0))
            continue
        d = r - r.mean((0, 2), keepdim=True)
        z = d / torch.sqrt((d * d).mean((0, 2), keepdim=True) + eps)
        z = z.flatten(1)
        z = z if w is None else z * w
        z = z if b is None else z + b
        y = ACT[act](z).reshape(live.shape)
        if x.dim() > 2 and end < x.shape[1]:
            y = torch.cat([y, torch.zeros(x.shape[1] - end, *x.shape[2:], dtype=y.dtype)])
        parts.append(y)
    return torch.stack(parts)


def rel(got, ref):
    got, ref = got.detach().double().cpu(), ref.detach().double()
    d, n = float((got - ref).norm()), float(ref.norm())
    return d / n if n else d


SHAPES = [
    # shape, groups
    ((2, 16), 2),
    ((1, 1, 64), 4),
    ((3, 7, 12), 3),
    ((2, 33, 5), 1),
    ((2, 33, 5), 5),
    ((4, 100, 64), 8),
    ((2, 65, 33, 32), 8),
    ((2, 9, 257, 8), 2),
    ((1, 1001, 48), 6),
    ((2, 50, 96), 32),
    ((1, 20, 2304), 3),
    ((2, 17, 4100), 4),
    ((1, 3000, 512), 32),
    ((1, 40000, 24), 3),
    ((300, 3, 40), 5),
    ((2, 700, 1024), 1),
]


def make(shape, dtype, seed, affine=True):
    r = torch.Generator().manual_seed(seed)
    x = (torch.randn(shape, generator=r) * 1.5 + torch.randn(shape[-1], generator=r)).to(dtype)
    w = 1 + 0.3 * torch.randn(shape[-1], generator=r) if affine else None
    b = 0.3 * torch.randn(shape[-1], generator=r) if affine else None
    return x, w, b, torch.randn(shape, generator=r).to(dtype)


@pytest.mark.parametrize("dtype", list(TOL))
@pytest.mark.parametrize("act", list(ACT))
@pytest.mark.parametrize("shape,groups", SHAPES, ids=str)
def test_forward_and_gradients(shape, groups, act, dtype):
    x, w, b, dy = make(shape, dtype, seed=len(shape) + shape[-1])
    ref_in = [t.double().requires_grad_() for t in (x, w, b)]
    ref = reference(ref_in[0], groups, ref_in[1], ref_in[2], 1e-5, act)
    expected = torch.autograd.grad(ref, ref_in, dy.double())
    leaves = [t.cuda().requires_grad_() for t in (x, w, b)]
    y = trnfft_amd.group_norm(leaves[0], groups, leaves[1], leaves[2], activation=act)
    got = torch.autograd.grad(y, leaves, dy.cuda())
    assert y.dtype == dtype and rel(y, ref) <= TOL[dtype]
    assert got[0].dtype == dtype and rel(got[0], expected[0]) <= TOL[dtype]
    # (sums over a channel: fp32 sums of their terms' magnitudes' error)
    for g, e in zip(got[1:], expected[1:]):
        assert rel(g, e) <= 3e-6
    with torch.no_grad():
        assert torch.equal(trnfft_amd.group_norm(leaves[0], groups, leaves[1], leaves[2], activation=act), y)


@pytest.mark.parametrize("dtype", list(TOL))
@pytest.mark.parametrize("shape,groups", [((4, 37, 24), 3), ((3, 50, 9, 16), 4), ((3, 2500, 64), 8), ((3, 21, 7), 7)], ids=str)
def test_padding_may_hold_anything(shape, groups, dtype):
    x, w, b, dy = make(shape, dtype, seed=3)
    n = torch.tensor([0, shape[1], shape[1] // 2, 5][:shape[0]])
    ref_in = [t.double().requires_grad_() for t in (x, w, b)]
    ref = reference(ref_in[0], groups, ref_in[1], ref_in[2], 1e-5, "silu", n)
    expected = torch.autograd.grad(ref, ref_in, dy.double())
    for dirty in (False, True):
        xd, dyd = x.clone(), dy.clone()
        if dirty:
            for i, end in enumerate(n.tolist()):
                xd[i, end:], dyd[i, end:] = float("inf"), float("nan")
        leaves = [t.cuda().requires_grad_() for t in (xd, w, b)]
        y = trnfft_amd.group_norm(leaves[0], groups, leaves[1], leaves[2], activation="silu", lengths=n.cuda())
        got = torch.autograd.grad(y, leaves, dyd.cuda())
        assert rel(y, ref) <= TOL[dtype] and rel(got[0], expected[0]) <= TOL[dtype]
        for g, e in zip(got[1:], expected[1:]):
            assert rel(g, e) <= 3e-6
        for i, end in enumerate(n.tolist()):
            assert not y[i, end:].any() and not got[0][i, end:].any()


@pytest.mark.parametrize("shape", [(1, 64, 64), (2, 5000, 32)], ids=str)
def test_a_mean_far_from_zero(shape):
    # deviations of 1 around 1000: the inputs' own fp32 spacing is 6e-5, exact in both; a mean rounded to fp32 is off by up to
    # 3e-5 of a deviation, and xhat by as much
    r = torch.Generator().manual_seed(0)
    x = (1000 + torch.randn(shape, generator=r)).float()
    y = trnfft_amd.group_norm(x.cuda(), 4)
    assert rel(y, reference(x.double(), 4, None, None, 1e-5, None)) <= 4e-5


def test_constant_groups_and_infinite_inputs():
    x = torch.full((2, 30, 16), 3.0).cuda()
    w, b = torch.randn(16).cuda(), torch.randn(16).cuda()
    y = trnfft_amd.group_norm(x, 4, w, b)
    assert torch.equal(y, b.expand_as(y))
    x = torch.randn(2, 30, 16).cuda()
    x[0, 3, 1] = float("inf")
    y = trnfft_amd.group_norm(x, 4, w, b)
    assert y[0, :, :4].isnan().any() and torch.isfinite(y[0, :, 4:]).all() and torch.isfinite(y[1]).all()


@pytest.mark.parametrize("which", ["x", "w", "b"])
def test_gradients_against_differences(which):
    # central differences in a direction: truncation eps^2 / 6 of a third derivative of order one a value, noise 1e-6 / eps
    x, w, b, dy = (t.cuda() for t in make((2, 40, 24), torch.float32, seed=8))
    parts = {"x": x, "w": w, "b": b}
    u = torch.randn(parts[which].shape, generator=torch.Generator().manual_seed(1)).cuda()

    def loss(p):
        return trnfft_amd.group_norm(p["x"], 4, p["w"], p["b"], activation="gelu")

    leaf = {k: t.clone().requires_grad_(k == which) for k, t in parts.items()}
    y = loss(leaf)
    (g,) = torch.autograd.grad(y, leaf[which], dy)
    slope, eps, values = float((g.double() * u.double()).sum()), 1e-2, []
    for sign in (1, -1):
        p = dict(parts)
        p[which] = p[which] + sign * eps * u
        values.append(float((loss(p).double() * dy.double()).sum()))
    size = float(y.norm() * dy.norm())
    assert abs((values[0] - values[1]) / (2 * eps) - slope) <= 1e-6 * size / eps + eps**2 * 10 * size


def test_without_affine_and_with_16_bit_weights():
    x, w, b, _ = make((2, 30, 16), torch.bfloat16, seed=2)
    y = trnfft_amd.group_norm(x.cuda(), 2, activation="relu")
    assert rel(y, reference(x.double(), 2, None, None, 1e-5, "relu")) <= TOL[torch.bfloat16]
    w, b = w.bfloat16(), b.bfloat16()
    leaf = w.cuda().requires_grad_()
    y = trnfft_amd.group_norm(x.cuda(), 2, leaf, b.cuda(), eps=1e-3)
    assert rel(y, reference(x.double(), 2, w.double(), b.double(), 1e-3, None)) <= TOL[torch.bfloat16]
    y.float().sum().backward()
    assert leaf.grad.dtype == torch.bfloat16


def test_strides_unaligned_views_and_empty_inputs():
    x, w, b, _ = make((3, 20, 32), torch.bfloat16, seed=1)
    ref = reference(x.double(), 4, w.double(), b.double(), 1e-5, "silu")
    w, b = w.cuda(), b.cuda()
    first = x.transpose(1, 2).contiguous().cuda().transpose(1, 2)  # channels first in memory
    assert rel(trnfft_amd.group_norm(first, 4, w, b, activation="silu"), ref) <= TOL[torch.bfloat16]
    buf = torch.zeros(x.numel() + 8, dtype=x.dtype, device="cuda")
    odd = buf[1:1 + x.numel()].view(x.shape)
    odd.copy_(x)
    assert rel(trnfft_amd.group_norm(odd, 4, w, b, activation="silu"), ref) <= TOL[torch.bfloat16]
    for shape in ((0, 5, 32), (2, 0, 32)):
        leaf, wl = torch.empty(shape).cuda().requires_grad_(), w.clone().requires_grad_()
        y = trnfft_amd.group_norm(leaf, 4, wl, b)
        assert y.shape == shape
        gx, gw = torch.autograd.grad(y, [leaf, wl], torch.empty_like(y))
        assert gx.shape == shape and not gw.any()


def test_streams_graphs_and_repeats():
    x, w, b, dy = (t.cuda() for t in make((4, 626, 64), torch.bfloat16, seed=4))
    n = torch.tensor([626, 100, 0, 625]).cuda()

    def train():
        leaves = [t.clone().requires_grad_() for t in (x, w, b)]
        y = trnfft_amd.group_norm(leaves[0], 8, leaves[1], leaves[2], activation="silu", lengths=n)
        return [y, *torch.autograd.grad(y, leaves, dy)]

    expected = train()
    assert all(torch.equal(p, q) for p, q in zip(train(), expected))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = train()
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(p, q) for p, q in zip(got, expected))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = trnfft_amd.group_norm(x, 8, w, b, activation="silu", lengths=n)
    for _ in range(3):
        y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, expected[0])
        x.sum().item()


def test_module_and_cpu_inputs():
    layer = GroupNorm(4, 32, activation="silu")
    x, _, _, _ = make((2, 30, 32), torch.float32, seed=6)
    with torch.no_grad():
        layer.weight.normal_()
        layer.bias.normal_()
    y = layer(x)
    assert y.device.type == "cpu"
    assert rel(y, reference(x.double(), 4, layer.weight.double(), layer.bias.double(), 1e-5, "silu")) <= 2e-6
    y.sum().backward()
    assert layer.weight.grad.shape == (32,) and math.isfinite(float(layer.weight.grad.sum()))
    layer = layer.cuda()
    assert rel(layer(x.cuda()), y.detach().double()) <= 2e-6


# many samples of few positions: groups of one vector and of 64, of sizes that are no power of two, fewer groups than a tile holds
FEW = [((700, 1, 64), 4), ((300, 2, 120), 5), ((40, 7, 144), 3), ((5000, 1, 512), 1), ((33, 13, 64), 2), ((65, 30, 48), 3),
       ((9, 3, 5, 16), 1), ((2100, 1, 256), 8)]


@pytest.mark.parametrize("dtype", list(TOL))
@pytest.mark.parametrize("shape,groups", FEW, ids=str)
def test_samples_of_few_positions(shape, groups, dtype):
    x, w, b, dy = make(shape, dtype, seed=11)
    n = torch.randint(0, shape[1] + 1, (shape[0],), generator=torch.Generator().manual_seed(12)) if shape[1] > 1 else None
    ref_in = [t.double().requires_grad_() for t in (x, w, b)]
    ref = reference(ref_in[0], groups, ref_in[1], ref_in[2], 1e-5, "silu", n)
    expected = torch.autograd.grad(ref, ref_in, dy.double())
    if n is not None:
        for i, end in enumerate(n.tolist()):
            x[i, end:], dy[i, end:] = float("nan"), float("inf")
    leaves = [t.cuda().requires_grad_() for t in (x, w, b)]
    y = trnfft_amd.group_norm(leaves[0], groups, leaves[1], leaves[2], activation="silu", lengths=None if n is None else n.cuda())
    got = torch.autograd.grad(y, leaves, dy.cuda())
    assert rel(y, ref) <= TOL[dtype] and rel(got[0], expected[0]) <= TOL[dtype]
    for g, e in zip(got[1:], expected[1:]):
        assert rel(g, e) <= 3e-6
