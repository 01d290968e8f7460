"""The operators of a state space layer against their definitions in 64 bits (frame by frame, on the CPU), their gradients
against those of the definitions and against differences, the steps against whole sequences, and a run of them together.

Tolerances (relative 2-norm).  fp32: a value passes some ten operations, a rounding of 2^-24 (6e-8) each, and exponentials whose
argument of up to 8 is rounded too, 5e-7; a state sums up over its memory of up to some hundred frames with random roundings,
ten times one rounding: 2e-6.  16-bit results are rounded once to nearest, 2^-9 (2^-12) of the power of two below a value at
most, 1.7e-3 (2.1e-4) in the mean square; half as much again covers what comes before.  That is a mean over values of many sizes: a
norm may lie in a few values just above powers of two, where a rounding is off by 2^-8 (2^-11) of the value.  No value is off by more,
so neither is any norm: results of fewer than 1000 values get that bound, and the fp32 one for what comes before.  Gradients of a, d, dt_bias and filters sum N terms of both signs: the sum is
about sqrt(N) terms, its error about 3 2^-24 sqrt(N) of them by their own roundings and 2^-24 N / 4 by the sum's in the worst
order that is used (N / 16 terms at once): for N up to 1300 together below 1e-5 of the result."""

from __future__ import annotations

import math

import pytest
import torch

import trnfft_amd

pytestmark = pytest.mark.gpu

TOL = {torch.float32: 2e-6, torch.bfloat16: 2.6e-3, torch.float16: 3.2e-4}
SUMS = 1e-5


def tol(ref, dtype):
    few = {torch.bfloat16: 2.0**-8 + TOL[torch.float32], torch.float16: 2.0**-11 + TOL[torch.float32]}
    return few.get(dtype, TOL[dtype]) if ref.numel() < 1000 else TOL[dtype]


def rel(got, ref):
    got, ref = got.detach().double().cpu(), ref.detach().double()
    d, n = float((got - ref).norm()), float(ref.norm())
    return d / n if n else d


def cuda(v):
    return v.detach().cuda() if torch.is_tensor(v) else v


def activate(z, act):
    if act == "silu":
        return z * torch.sigmoid(z)
    if act == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z / math.sqrt(2.0)))
    return torch.relu(z) if act == "relu" else z


# ---------------------------------------------------------------------------------------------
# causal convolution
# ---------------------------------------------------------------------------------------------


def conv_reference(x, weight, bias, act, state, lengths):
    """Row by row, tap by tap, in float64."""
    (b, t, c), width = x.shape, weight.shape[1]
    ys, lasts = [], []
    for i in range(b):
        end = t if lengths is None else min(max(int(lengths[i]), 0), t)
        before = torch.zeros(width - 1, c, dtype=torch.float64) if state is None else state[i]
        seq = torch.cat([before, x[i, :end]])
        pre = sum(weight[:, j] * seq[j:j + end] for j in range(width))
        pre = pre if bias is None else pre + bias
        ys.append(torch.cat([activate(pre, act), torch.zeros(t - end, c, dtype=torch.float64)]))
        lasts.append(seq[end:])
    return torch.stack(ys), torch.stack(lasts)


def conv_inputs(b, t, c, width, dtype, seed, bias=True, state=True, lengths=True):
    g = torch.Generator().manual_seed(seed)
    n = torch.randint(0, t + 1, (b,), generator=g) if lengths else None
    if lengths and b > 1:
        n[0], n[1] = t, 0
    return dict(x=torch.randn(b, t, c, generator=g).to(dtype), weight=torch.randn(c, width, generator=g) * width**-0.5,
                bias=torch.randn(c, generator=g) * 0.3 if bias else None,
                state=torch.randn(b, width - 1, c, generator=g).to(dtype) if state else None, lengths=n)


CONVS = [
    # b, t, c, width
    (1, 1, 1, 1),
    (1, 1, 8, 4),
    (2, 2, 5, 4),
    (3, 3, 16, 8),
    (3, 31, 64, 4),
    (2, 33, 24, 3),
    (2, 64, 7, 2),
    (4, 65, 40, 4),
    (2, 130, 256, 5),
    (3, 300, 520, 4),
    (2, 77, 12, 6),
    (2, 40, 1000, 7),
]


@pytest.mark.parametrize("dtype", list(TOL))
@pytest.mark.parametrize("shape", CONVS, ids=str)
@pytest.mark.parametrize("extra", [False, True])
def test_conv(shape, dtype, extra):
    b, t, c, width = shape
    act = ("silu", None, "gelu", "relu")[t % 4]
    v = conv_inputs(*shape, dtype, t, bias=extra, state=extra, lengths=extra)
    names = [k for k in ("x", "weight", "bias", "state") if v[k] is not None]
    ref = {k: v[k].double().requires_grad_() for k in names}
    y_ref, last_ref = conv_reference(ref["x"], ref["weight"], ref.get("bias"), act, ref.get("state"), v["lengths"])
    own = {k: cuda(v[k]).requires_grad_() for k in names}
    y, last = trnfft_amd.causal_conv(own["x"], own["weight"], own.get("bias"), activation=act, initial_state=own.get("state"),
                                     lengths=cuda(v["lengths"]), return_state=True)
    assert y.dtype == dtype and y.shape == y_ref.shape and last.dtype == dtype and last.shape == last_ref.shape
    assert rel(y, y_ref) <= tol(y_ref, dtype)
    assert torch.equal(last.cpu().double(), last_ref.detach())
    if extra:
        for i, end in enumerate(v["lengths"].tolist()):
            assert not y[i, end:].any()
    g = torch.Generator().manual_seed(1)
    dy, dlast = torch.randn(y.shape, generator=g).to(dtype), torch.randn(last.shape, generator=g).to(dtype)
    want = torch.autograd.grad([y_ref, last_ref], list(ref.values()), [dy.double(), dlast.double()], allow_unused=True)
    got = torch.autograd.grad([y, last], list(own.values()), [cuda(dy), cuda(dlast)])
    for name, w, d in zip(names, want, got):
        w = torch.zeros_like(ref[name]) if w is None else w
        assert d.dtype == own[name].dtype and d.shape == w.shape
        assert rel(d, w) <= (SUMS if name in ("weight", "bias") else tol(w, dtype)), name


@pytest.mark.parametrize("dtype", list(TOL))
@pytest.mark.parametrize("c,width", [(64, 4), (7, 3), (520, 8), (16, 1)])
def test_conv_steps_are_the_sequence(c, width, dtype):
    v = {k: cuda(x) for k, x in conv_inputs(3, 20, c, width, dtype, 3, lengths=False).items()}
    whole, last = trnfft_amd.causal_conv(v["x"], v["weight"], v["bias"], activation="silu", initial_state=v["state"],
                                         return_state=True)
    state = v["state"].clone()
    frames = [trnfft_amd.causal_conv_step(v["x"][:, t], state, v["weight"], v["bias"], activation="silu") for t in range(20)]
    assert torch.equal(torch.stack(frames, 1), whole) and torch.equal(state, last)


def test_conv_takes_views_and_odd_addresses():
    g = torch.Generator().manual_seed(0)
    big = torch.randn(3, 50, 70, generator=g).bfloat16().cuda()
    w = torch.randn(24, 4, generator=g).cuda()
    for at in (0, 1, 8, 46):
        x = big[:, 3:40, at:at + 24]
        assert torch.equal(trnfft_amd.causal_conv(x, w), trnfft_amd.causal_conv(x.contiguous(), w))
    turned = big.transpose(1, 2)[..., :32]  # frames contiguous: copied
    w = torch.randn(32, 4, generator=g).cuda()
    assert torch.equal(trnfft_amd.causal_conv(turned, w), trnfft_amd.causal_conv(turned.contiguous(), w))
    same = big[:1, :, :24].expand(3, 50, 24)  # one row for all
    w = torch.randn(24, 4, generator=g).cuda()
    assert torch.equal(trnfft_amd.causal_conv(same, w), trnfft_amd.causal_conv(same.contiguous(), w))


def test_conv_keeps_what_is_not_finite_inside_the_filter():
    x = torch.ones(1, 12, 16, device="cuda")
    x[0, 5, 3] = float("inf")
    x[0, 8:, 5] = float("nan")
    w = torch.ones(16, 3, device="cuda")
    y = trnfft_amd.causal_conv(x, w, lengths=torch.tensor([8], device="cuda"))
    assert y[0, 5:8, 3].isinf().all() and torch.isfinite(y[0, :5]).all() and not y[0, 8:].any()
    assert torch.isfinite(torch.cat([y[..., :3], y[..., 4:]], -1)).all()


# ---------------------------------------------------------------------------------------------
# selective scan
# ---------------------------------------------------------------------------------------------


def scan_reference(x, dt, a, b, c, d, z, dt_bias, state, softplus, lengths):
    """Frame by frame in float64; frames past a row's length leave its state and give zeros."""
    rows, t, ch = x.shape
    each = ch // b.shape[2]
    s = dt if dt_bias is None else dt + dt_bias
    s = torch.logaddexp(s, torch.zeros_like(s)) if softplus else s
    h = torch.zeros(rows, ch, a.shape[1], dtype=torch.float64) if state is None else state
    ys = []
    for i in range(t):
        new = torch.exp(s[:, i, :, None] * a) * h + (s * x)[:, i, :, None] * b[:, i].repeat_interleave(each, dim=1)
        y = (new * c[:, i].repeat_interleave(each, dim=1)).sum(-1)
        y = y if d is None else y + d * x[:, i]
        y = y if z is None else y * activate(z[:, i], "silu")
        if lengths is not None:
            live = (i < lengths)[:, None]
            new, y = torch.where(live[..., None], new, h), torch.where(live, y, 0.0)
        h = new
        ys.append(y)
    return (torch.stack(ys, 1) if ys else x * 0.0), h


def scan_inputs(rows, t, ch, groups, n, dtype, seed, extra=True, softplus=True):
    g = torch.Generator().manual_seed(seed)
    size = torch.rand(ch, generator=g) * 0.3 + 0.01
    v = dict(x=torch.randn(rows, t, ch, generator=g).to(dtype),
             dt=(torch.randn(rows, t, ch, generator=g) if softplus else size * torch.rand(rows, t, ch, generator=g)).to(dtype),
             a=-torch.rand(ch, n, generator=g) * 4.0,
             b=torch.randn(rows, t, groups, n, generator=g).to(dtype), c=torch.randn(rows, t, groups, n, generator=g).to(dtype),
             d=torch.randn(ch, generator=g) if extra else None, z=torch.randn(rows, t, ch, generator=g).to(dtype) if extra else None,
             # (without softplus it has to leave steps positive: one of -4 at a rate of -4 multiplies states by e^16 a frame, which is past
             # fp32's range, e^88, in six)
             dt_bias=None if not extra else torch.log(torch.expm1(size)) if softplus else size,
             state=torch.randn(rows, ch, n, generator=g) if extra else None)
    lengths = torch.randint(0, t + 1, (rows,), generator=g) if extra else None
    if extra and rows > 1:
        lengths[0], lengths[1] = t, 0
    return v, lengths


def scan(v, lengths=None, softplus=True, return_state=True):
    return trnfft_amd.selective_scan(v["x"], v["dt"], v["a"], v["b"], v["c"], d=v.get("d"), z=v.get("z"), dt_bias=v.get("dt_bias"),
                                     softplus=softplus, initial_state=v.get("state"), lengths=lengths, return_state=return_state)


SCANS = [
    # rows, t, channels, groups, n
    (1, 1, 1, 1, 1),
    (2, 2, 3, 1, 4),
    (2, 15, 64, 1, 3),
    (3, 16, 65, 1, 5),
    (2, 17, 32, 2, 8),
    (3, 33, 48, 1, 16),
    (2, 48, 16, 1, 16),
    (2, 50, 70, 2, 12),
    (2, 31, 24, 3, 17),
    (2, 40, 40, 1, 32),
    (2, 35, 130, 2, 16),
    (1, 64, 12, 4, 64),
    (2, 20, 9, 1, 49),
    (2, 100, 260, 1, 4),
]


def check_scan(shape, dtype, extra, softplus, seed=0):
    v, lengths = scan_inputs(*shape, dtype, seed, extra, softplus)
    names = [k for k, x in v.items() if x is not None]
    ref = {k: v[k].double().requires_grad_() for k in names}
    full = {k: ref.get(k) for k in v}
    y_ref, last_ref = scan_reference(**full, softplus=softplus, lengths=lengths)
    own = {k: cuda(v[k]).requires_grad_() for k in names}
    y, last = scan(own, cuda(lengths), softplus)
    assert y.dtype == dtype and y.shape == y_ref.shape and last.dtype == torch.float32 and last.shape == last_ref.shape
    assert rel(y, y_ref) <= tol(y_ref, dtype)
    assert rel(last, last_ref) <= 2e-6
    if extra:
        for i, end in enumerate(lengths.tolist()):
            assert not y[i, end:].any()
    with torch.no_grad():  # without gradients: the same
        y2, last2 = scan(own, cuda(lengths), softplus)
        assert torch.equal(y2, y) and torch.equal(last2, last)
    g = torch.Generator().manual_seed(1)
    dy, dlast = torch.randn(y.shape, generator=g).to(dtype), torch.randn(last.shape, generator=g)
    want = torch.autograd.grad([y_ref, last_ref], list(ref.values()), [dy.double(), dlast.double()], allow_unused=True)
    got = torch.autograd.grad([y, last], list(own.values()), [cuda(dy), cuda(dlast)])
    for name, w, d in zip(names, want, got):
        w = torch.zeros_like(ref[name]) if w is None else w
        assert d.dtype == own[name].dtype and d.shape == w.shape
        bound = SUMS if name in ("a", "d", "dt_bias") else 2e-6 if name == "state" else tol(w, dtype)
        if dtype == torch.float32 and name in ("dt", "b", "c", "z", "x"):
            bound = 4e-6  # (two nested sums of such states)
        assert rel(d, w) <= bound, name


@pytest.mark.parametrize("dtype", list(TOL))
@pytest.mark.parametrize("shape", SCANS, ids=str)
@pytest.mark.parametrize("extra", [False, True])
def test_scan(shape, dtype, extra):
    check_scan(shape, dtype, extra, softplus=True)


@pytest.mark.parametrize("shape", SCANS[3:8], ids=str)
@pytest.mark.parametrize("extra", [False, True])
def test_scan_of_steps_as_they_are(shape, extra):
    check_scan(shape, torch.float32, extra, softplus=False, seed=5)


@pytest.mark.parametrize("dtype", list(TOL))
@pytest.mark.parametrize("shape", [(2, 45, 33, 1, 9), (3, 33, 40, 2, 11), (2, 130, 18, 1, 15), (1, 255, 17, 1, 10), (2, 64, 32, 1, 16),
                                   (2, 32, 130, 1, 14)], ids=str)
def test_scan_of_two_waves_a_channel(shape, dtype):
    """9 to 16 states: half of them to a wave each, with odd and even numbers of tiles and halves of one state to eight."""
    for extra in (False, True):
        check_scan(shape, dtype, extra, softplus=True, seed=11)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(161, 8, 250, 1, 16), (41, 31, 1000, 8, 16)], ids=str)
def test_scan_of_many_rows_and_channels(shape, dtype):
    """More waves than that is done for."""
    check_scan(shape, dtype, True, softplus=True, seed=12)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(1, 1300, 20, 1, 16), (2, 700, 5, 1, 6), (3, 513, 36, 2, 40)], ids=str)
def test_scan_in_segments(shape, dtype):
    """Long sequences of few channels are shared out over time."""
    check_scan(shape, dtype, True, softplus=True, seed=7)


@pytest.mark.parametrize("shape", [(257, 3, 20, 1, 16), (600, 2, 40, 5, 3), (640, 2, 17, 1, 33)], ids=str)
def test_gradients_over_many_rows(shape):
    """Sums over rows in two passes."""
    check_scan(shape, torch.float32, True, softplus=True, seed=13)


@pytest.mark.parametrize("t,end", [(1056, 1056), (1090, 1071), (1090, 300)])
def test_scan_in_long_segments(t, end):
    """Two segments backwards, whose sums are made in halves (the definition on the GPU, in float64)."""
    ch = 16400
    v, _ = scan_inputs(1, t, ch, 1, 1, torch.float32, 8, extra=False)
    names = list(k for k in v if v[k] is not None)
    ref = {k: v[k].double().cuda().requires_grad_() for k in names}
    h, ys = torch.zeros(1, ch, 1, dtype=torch.float64, device="cuda"), []
    for x, dt, b, c in list(zip(*(ref[k].unbind(1) for k in ("x", "dt", "b", "c"))))[:end]:
        s = torch.logaddexp(dt, torch.zeros_like(dt))
        h = torch.exp(s[..., None] * ref["a"]) * h + (s * x)[..., None] * b
        ys.append((h * c).sum(-1))
    y_ref = torch.nn.functional.pad(torch.stack(ys, 1), (0, 0, 0, t - end))
    own = {k: cuda(v[k]).requires_grad_() for k in names}
    y, last = scan(own, torch.tensor([end]))
    dy, dlast = torch.randn_like(y), torch.randn_like(last)
    want = torch.autograd.grad([y_ref, h], list(ref.values()), [dy.double(), dlast.double()])
    got = torch.autograd.grad([y, last], list(own.values()), [dy, dlast])
    assert rel(y, y_ref.cpu()) <= 2e-6 and rel(last, h.cpu()) <= 2e-6
    for name, w, g in zip(names, want, got):
        assert rel(g, w.cpu()) <= (SUMS if name == "a" else 4e-6), name


@pytest.mark.parametrize("dtype", list(TOL))
@pytest.mark.parametrize("ch,groups,n,softplus", [(48, 1, 16, True), (10, 2, 3, True), (7, 1, 21, False), (33, 3, 64, True),
                                                  (260, 1, 8, True)])
def test_scan_steps_are_the_sequence(ch, groups, n, softplus, dtype):
    v, _ = scan_inputs(3, 12, ch, groups, n, dtype, 2, True, softplus)
    v = {k: cuda(x) for k, x in v.items()}
    whole, last = scan(v, softplus=softplus)
    state = v["state"].clone()
    frames = [trnfft_amd.selective_scan_step(v["x"][:, t], v["dt"][:, t], v["a"], v["b"][:, t], v["c"][:, t], state, d=v["d"],
                                             z=v["z"][:, t], dt_bias=v["dt_bias"], softplus=softplus) for t in range(12)]
    assert rel(state, last.cpu()) <= 5e-7
    got = torch.stack(frames, 1)
    if dtype == torch.float32:
        assert rel(got, whole.cpu()) <= 1e-6
    else:  # sums in another order: a rounding apart now and then
        eps = torch.finfo(dtype).eps
        assert (got.float() - whole.float()).abs().le(eps * whole.float().abs() + 1e-5).all()


def test_scan_takes_views_and_odd_addresses():
    g = torch.Generator().manual_seed(0)
    rows, t, ch, n = 2, 40, 24, 5
    v, _ = scan_inputs(rows, t, ch, 1, n, torch.bfloat16, 4)
    v = {k: cuda(x) for k, x in v.items()}
    proj = torch.randn(rows, t, 3 + 2 * n, generator=g).bfloat16().cuda()
    xz = torch.randn(rows, t, 2 * ch + 1, generator=g).bfloat16().cuda()
    v.update(b=proj[..., 3:3 + n].unsqueeze(2), c=proj[..., 3 + n:].unsqueeze(2), x=xz[..., 1:1 + ch], z=xz[..., 1 + ch:])
    dense = {k: x.contiguous() for k, x in v.items()}
    for got, want in zip(scan(v), scan(dense)):
        assert torch.equal(got, want)
    shared = {**dense, "b": dense["b"][:1].expand(rows, -1, -1, -1), "dt": dense["dt"][:, :1].expand(-1, t, -1)}
    for got, want in zip(scan(shared), scan({k: x.contiguous() for k, x in shared.items()})):
        assert torch.equal(got, want)


def test_gradients_of_broadcast_inputs_are_summed():
    v, _ = scan_inputs(3, 20, 16, 1, 16, torch.float32, 9)
    v = {k: cuda(x) for k, x in v.items()}
    one = v["b"][:1].clone().requires_grad_()
    y = scan({**v, "b": one.expand(3, -1, -1, -1)}, return_state=False)
    got, = torch.autograd.grad(y.square().sum(), one)
    full = v["b"][:1].expand(3, -1, -1, -1).contiguous().requires_grad_()
    want, = torch.autograd.grad(scan({**v, "b": full}, return_state=False).square().sum(), full)
    assert rel(got, want.sum(0, keepdim=True).cpu()) <= 1e-6


def test_scan_gradients_against_differences():
    """A central difference of step 2^-5 along a direction of fp32 inputs is off by the third derivative, measured by halving the
    step, and by fp32 values of the loss, 2^-24 of it over the step."""
    v, lengths = scan_inputs(2, 21, 18, 1, 7, torch.float32, 11)
    v = {k: cuda(x) for k, x in v.items()}
    g = torch.Generator().manual_seed(2)
    wy, wl = torch.randn(2, 21, 18, generator=g).cuda().double(), torch.randn(2, 18, 7, generator=g).cuda().double()

    def loss(v):
        y, last = scan(v, cuda(lengths))
        return (y.double() * wy).sum() + (last.double() * wl).sum()

    leaves = {k: x.clone().requires_grad_() for k, x in v.items()}
    grads = dict(zip(leaves, torch.autograd.grad(loss(leaves), list(leaves.values()))))
    for name in v:
        way = torch.randn(v[name].shape, generator=g).cuda()
        want = float((grads[name].double() * way).sum())

        def difference(step):
            with torch.no_grad():
                up, down = (loss({**v, name: v[name] + sign * step * way}) for sign in (1.0, -1.0))
                return float(up - down) / (2.0 * step)

        fine, coarse = difference(2.0**-6), difference(2.0**-5)
        scale = float(grads[name].double().norm())
        assert abs(fine - want) <= abs(fine - coarse) + 1e-4 * scale, name


def test_scan_keeps_what_is_not_finite_to_its_channel_and_later_frames():
    v, _ = scan_inputs(2, 40, 40, 1, 16, torch.float32, 6)
    v = {k: cuda(x) for k, x in v.items()}
    clean, _ = scan(v)
    for name, value in (("x", float("nan")), ("dt", float("inf")), ("z", float("nan"))):
        bad = {**v, name: v[name].clone()}
        bad[name][0, 20, 17] = value
        y, _ = scan(bad)
        assert torch.equal(y[1], clean[1]) and torch.equal(y[0, :20], clean[0, :20])
        others = torch.arange(40, device="cuda") != 17
        assert torch.equal(y[0][:, others], clean[0][:, others])
        assert not torch.isfinite(y[0, 20, 17])
    # padding is not read, whatever it holds
    lengths = torch.tensor([20, 40], device="cuda")
    bad = {k: x.clone() for k, x in v.items()}
    for name in ("x", "dt", "z", "b", "c"):
        bad[name][0, 20:] = float("nan")
    leaves = {k: x.requires_grad_() for k, x in bad.items()}
    y, last = scan(leaves, lengths)
    assert torch.isfinite(y).all() and torch.isfinite(last).all() and not y[0, 20:].any()
    grads = torch.autograd.grad(y.sum() + last.sum(), list(leaves.values()))
    assert all(torch.isfinite(d).all() for d in grads)
    for name, d in zip(leaves, grads):
        if name in ("x", "dt", "z", "b", "c"):
            assert not d[0, 20:].any(), name


def test_steps_called_natively_and_from_python_agree(monkeypatch):
    """Operands as the C ABI takes them go to it directly, others are converted or refused first: the same call either way."""
    from trnfft_amd import state_space

    rows, ch, groups, n = 5, 24, 2, 6
    v = {k: cuda(w) for k, w in scan_inputs(rows, 1, ch, groups, n, torch.float32, 3)[0].items()}
    frame = {k: v[k][:, 0] for k in ("x", "dt", "b", "c", "z")}
    x2, weight, bias = torch.randn(2 * rows, ch, device="cuda")[::2], torch.randn(ch, 4, device="cuda"), torch.randn(ch, device="cuda")

    def steps(x, dt, a, weight):
        state, taps = v["state"].clone(), torch.ones(rows, 3, ch, device="cuda")
        versions = state._version, taps._version
        y = trnfft_amd.selective_scan_step(x, dt, a, frame["b"], frame["c"], state, d=v["d"], z=frame["z"], dt_bias=v["dt_bias"])
        u = trnfft_amd.causal_conv_step(x2, taps, weight, bias, activation="silu")
        assert state._version > versions[0] and taps._version > versions[1]
        return y, state, u, taps

    taken = []
    direct = state_space._step
    monkeypatch.setattr(state_space, "_step", lambda *args: taken.append(direct(*args)) or taken[-1])
    want = steps(frame["x"], frame["dt"], v["a"], weight)
    assert len(taken) == 2 and all(torch.is_tensor(t) for t in taken)
    taken.clear()
    wide = torch.zeros(rows, 2 * ch, device="cuda")
    wide[:, ::2] = frame["dt"]
    got = steps(frame["x"], wide[:, ::2], v["a"].t().contiguous().t(), weight.t().contiguous().t())
    assert taken == [None, None]
    for g, w in zip(got, want):
        assert torch.equal(g, w)
    monkeypatch.setattr(state_space, "_step", lambda *args: None)
    for g, w in zip(steps(frame["x"], frame["dt"], v["a"], weight), want):
        assert torch.equal(g, w)
    monkeypatch.undo()
    with pytest.raises(RuntimeError, match="no gradients"):
        steps(frame["x"].clone().requires_grad_(), frame["dt"], v["a"], weight)
    with pytest.raises(ValueError, match="state must be"):
        trnfft_amd.causal_conv_step(x2, torch.ones(rows, 2, ch, device="cuda"), weight, bias)
    with pytest.raises(TypeError, match="state must be"):
        trnfft_amd.causal_conv_step(x2, torch.ones(rows, 3, ch, device="cuda", dtype=torch.float16), weight, bias)
    with torch.inference_mode():
        got = trnfft_amd.causal_conv_step(x2, torch.ones(rows, 3, ch, device="cuda"), weight, bias, activation="silu")
    assert torch.equal(got, want[2])


@pytest.mark.parametrize("extra", [False, True])
def test_sequences_called_natively_and_from_python_agree(extra, monkeypatch):
    """The same for whole sequences, with and without gradients: what has to be converted goes through Python."""
    from trnfft_amd import state_space

    v, lengths = scan_inputs(3, 21, 24, 2, 6, torch.float32, 4, extra)
    v, lengths = {k: cuda(w) for k, w in v.items()}, cuda(lengths)
    conv = conv_inputs(3, 21, 24, 4, torch.float32, 5, bias=extra, state=extra, lengths=False)
    conv = {k: cuda(conv.get(k)) for k in ("x", "weight", "bias", "state")}

    def passes(v, conv, lengths):
        leaves = [w.detach().requires_grad_() for w in (*v.values(), *conv.values()) if torch.is_tensor(w)]
        own = iter(leaves)
        v = {k: next(own) if torch.is_tensor(w) else None for k, w in v.items()}
        conv = {k: next(own) if torch.is_tensor(w) else None for k, w in conv.items()}
        outs = []
        for grads in (True, False):
            with torch.set_grad_enabled(grads):
                y, last = scan(v, lengths)
                u, end = trnfft_amd.causal_conv(conv["x"], conv["weight"], conv["bias"], activation="gelu", initial_state=conv["state"],
                                                lengths=lengths, return_state=True)
                alone = scan(v, lengths, return_state=False)
                assert torch.is_tensor(alone) and torch.equal(alone, y)
            outs += [y, last, u, end]
            assert y.requires_grad == grads and end.requires_grad == grads
        return [*outs, *torch.autograd.grad([outs[0].sum(), outs[2].square().sum(), outs[3].sum()], leaves, allow_unused=True)]

    taken = []
    direct = state_space._direct
    monkeypatch.setattr(state_space, "_direct", lambda *args: taken.append(direct(*args)) or taken[-1])
    want = passes(v, conv, lengths)
    assert len(taken) == 6 and all(t is not None for t in taken)
    taken.clear()
    turned = {**v, "a": v["a"].t().contiguous().t()}
    got = passes(turned, {**conv, "weight": conv["weight"].t().contiguous().t()}, None if lengths is None else lengths.int())
    assert taken == [None] * 6
    monkeypatch.setattr(state_space, "_direct", lambda *args: None)
    for other in (got, passes(v, conv, lengths)):
        for a, b in zip(other, want):
            assert (a is None and b is None) or torch.equal(a, b)
    with pytest.raises(NotImplementedError, match="64 states"):
        monkeypatch.undo()
        trnfft_amd.selective_scan(v["x"], v["dt"], torch.zeros(24, 65, device="cuda"), *(torch.zeros(3, 21, 2, 65, device="cuda"),) * 2)


@pytest.mark.parametrize("rows,t", [(0, 5), (3, 0), (0, 0)])
def test_nothing_to_do(rows, t):
    v, _ = scan_inputs(rows, t, 6, 1, 4, torch.float32, 0, extra=False)
    leaves = {k: cuda(x).requires_grad_() for k, x in v.items() if x is not None}
    state = torch.randn(rows, 6, 4, device="cuda", requires_grad=True)
    y, last = scan({**leaves, "state": state})
    assert y.shape == (rows, t, 6) and (torch.equal(last, state) or t)
    grads = torch.autograd.grad(y.sum() + last.sum(), [*leaves.values(), state], allow_unused=True)
    assert all(not d.any() for d in grads[:-1]) and (grads[-1] == 1).all()
    x, w = torch.zeros(rows, t, 6, device="cuda"), torch.ones(6, 4, device="cuda", requires_grad=True)
    before = torch.randn(rows, 3, 6, device="cuda")
    y, last = trnfft_amd.causal_conv(x, w, initial_state=before, return_state=True)
    assert y.shape == (rows, t, 6) and (torch.equal(last, before) or t)
    assert not torch.autograd.grad(y.sum() + last.sum() if last.requires_grad else y.sum(), w)[0].any()
