"""The operators of a state space layer together, as they are used: nn.StateSpace trained with clipped gradients and AdamW,
served frame by frame and block by block, captured in graphs, on other streams; and in the denoiser example.

Tolerances: fp32 with sums in other orders, through the layer's products of up to 128 features, convolution, scan and gate: each is off
by a few 2^-24 sqrt(128) of its result, together below 1e-5 of the largest output."""

import os
import sys

import pytest
import torch
import torch.utils.checkpoint

import trnfft_amd
from trnfft_amd.nn import StateSpace
from trnfft_amd.optim import AdamW, clip_grad_norm_

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "examples"))

pytestmark = pytest.mark.gpu


def layer(features=32, seed=0, dtype=torch.float32, **options):
    torch.manual_seed(seed)
    return StateSpace(features, **options).to("cuda", dtype)


def near(got, want, tol=1e-5):
    return float((got.double() - want.double()).abs().max()) <= tol * float(want.double().abs().max())


@pytest.mark.parametrize("options", [{}, dict(states=5, width=3, expand=1, rank=3), dict(states=40, width=1)], ids=str)
def test_streams_and_blocks_equal_the_whole(options):
    m = layer(**options)
    x = torch.randn(3, 50, 32, device="cuda")
    with torch.no_grad():
        whole, (conv, scan) = m(x, return_state=True)
        state = m.state(3)
        frames = torch.stack([m.step(x[:, t], state) for t in range(50)], 1)
        assert near(frames, whole)
        assert near(state[1], scan)
        if conv.numel():
            assert near(state[0], conv)
        parts, state = [], m.state(3)
        for block in x.split([17, 1, 32], dim=1):  # blocks of a stream, one of a single frame
            y, state = m(block, state=state, return_state=True)
            parts.append(y)
        assert near(torch.cat(parts, 1), whole) and near(state[1], scan)


def test_padding_does_not_matter():
    m = layer()
    x, lengths = torch.randn(3, 40, 32, device="cuda"), torch.tensor([40, 0, 23], device="cuda")
    with torch.no_grad():
        alone, end = m(x[2:, :23], return_state=True)
        x[1:, 23:] = 1e4
        y, state = m(x, lengths, return_state=True)
    assert near(y[2, :23], alone[0]) and near(state[1][2], end[1][0])
    assert not y[1].any() and not y[2, 23:].any() and not state[1][1].any()


def test_training_with_clipped_gradients_in_16_bits():
    m = layer(dtype=torch.bfloat16)
    opt = AdamW(m.parameters(), lr=1e-3)
    before = [p.detach().clone() for p in m.parameters()]
    x = torch.randn(4, 60, 32, device="cuda", dtype=torch.bfloat16)
    for _ in range(3):
        opt.zero_grad()
        m(x, torch.tensor([60, 7, 0, 33], device="cuda")).float().square().sum().backward()
        norm = clip_grad_norm_(m.parameters(), 1.0)
        assert torch.isfinite(norm) and norm > 0
        assert all(p.grad is not None and torch.isfinite(p.grad.float()).all() for p in m.parameters())
        opt.step()
    assert any(not torch.equal(p, b) for p, b in zip(m.parameters(), before))


def test_gradients_against_differences():
    """A difference over 2^-6 of a direction is off by its curvature, which halving the step measures, and by the two losses' roundings:
    an output passes some eight fp32 operations in line, 2^-24 each, and the losses' errors, at most 8 2^-24 sum |w y| each, are divided
    by the distance of 2^-5 between them."""
    m = layer(features=8, states=6)
    x = torch.randn(2, 19, 8, device="cuda")
    w = torch.randn(2, 19, 8, device="cuda").double()

    def loss():
        return (m(x).double() * w).sum()

    grads = torch.autograd.grad(loss(), list(m.parameters()))
    g = torch.Generator("cuda").manual_seed(3)
    with torch.no_grad():
        rounding = 2.0 * 8.0 * 2.0**-24 * float((m(x).double() * w).abs().sum()) / 2.0**-5
    for (name, p), d in zip(m.named_parameters(), grads):
        way = torch.randn(p.shape, generator=g, device="cuda")
        way *= p.detach().norm().clamp(min=0.1) / way.norm()

        def difference(step):
            with torch.no_grad():
                old = p.clone()
                ends = []
                for sign in (1.0, -1.0):
                    p.copy_(old + sign * step * way)
                    ends.append(float(loss()))
                p.copy_(old)
                return (ends[0] - ends[1]) / (2.0 * step)

        fine, coarse, want = difference(2.0**-6), difference(2.0**-5), float((d.double() * way.double()).sum())
        assert abs(fine - want) <= abs(fine - coarse) + rounding + 1e-3 * float(d.double().norm() * way.double().norm()), name


def test_a_stream_of_its_own():
    m = layer()
    x = torch.randn(2, 600, 32, device="cuda")
    with torch.no_grad():
        want, _ = m(x), torch.cuda.synchronize()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = [m(x) for _ in range(3)]
        torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(g, want) for g in got)


def test_a_captured_step_serves_a_stream():
    m = layer()
    x = torch.randn(12, 2, 32, device="cuda")
    with torch.no_grad():
        state = m.state(2)
        want = [m.step(f, state) for f in x]
        frame, held = x[0].clone(), m.state(2)
        m.step(frame, m.state(2))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = m.step(frame, held)
        for part in held:
            part.zero_()
        for i, f in enumerate(x):
            frame.copy_(f)
            graph.replay()
            if i % 3 == 0:  # the program's own work between replays
                m.step(f, m.state(2))
            torch.cuda.synchronize()
            assert torch.equal(out, want[i])


def operands(rows=2, t=300, ch=24, n=16, seed=0):
    g = torch.Generator("cuda").manual_seed(seed)

    def r(*s):
        return torch.randn(*s, generator=g, device="cuda")

    return [r(rows, t, ch), r(rows, t, ch), -r(ch, n).abs(), r(rows, t, 1, n), r(rows, t, 1, n)]


def test_two_captured_graphs_share_nothing():
    """Workspaces are a call's own: two graphs' replays in any order give the eager results."""
    cases = [operands(seed=1), operands(t=700, seed=2)]  # both in segments
    with torch.no_grad():
        want = [trnfft_amd.selective_scan(*v) for v in cases]
        graphs, outs = [], []
        for v in cases:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                outs.append(trnfft_amd.selective_scan(*v))
            graphs.append(graph)
        for order in ((0, 1), (1, 0), (0, 0)):
            for out in outs:
                out.zero_()
            for i in order:
                graphs[i].replay()
            eager = trnfft_amd.selective_scan(*cases[0])
            torch.cuda.synchronize()
            assert torch.equal(eager, want[0])
            for i in set(order):
                assert torch.equal(outs[i], want[i])


def test_a_captured_training_pass():
    leaves = [v.requires_grad_() for v in operands(seed=3)]
    w = torch.randn(24, 4, device="cuda", requires_grad=True)

    def run():
        y = trnfft_amd.selective_scan(trnfft_amd.causal_conv(leaves[0], w, activation="silu"), *leaves[1:])
        return torch.autograd.grad(y, [*leaves, w], torch.ones_like(y))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    want = [g.clone() for g in run()]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    for _ in range(3):
        for g in got:
            g.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_a_capture_refuses_leaves_whose_eager_graph_lives():
    """(Its backward pass would end the process.)  Leaves that are used through other nodes are found as well."""
    v = operands(t=40)
    x = v[0].requires_grad_()
    w = torch.randn(24, 4, device="cuda", dtype=torch.float64, requires_grad=True)
    eager = trnfft_amd.selective_scan(trnfft_amd.causal_conv(x * 2.0, w.float()), *v[1:])
    eager.sum().backward(retain_graph=True)
    graph, mark = torch.cuda.CUDAGraph(), torch.zeros(3, device="cuda")
    with torch.cuda.graph(graph):
        mark.add_(1.0)
        with pytest.raises(RuntimeError, match="eager pass"):
            trnfft_amd.selective_scan(x, *v[1:])
        with pytest.raises(RuntimeError, match="eager pass"):
            trnfft_amd.causal_conv(v[1], w.float())
        with pytest.raises(RuntimeError, match="eager pass"):
            trnfft_amd.causal_conv(x.tanh(), w.detach().float())
        with torch.no_grad():
            y = trnfft_amd.selective_scan(x, *v[1:])
    graph.replay()
    torch.cuda.synchronize()
    with torch.no_grad():
        assert torch.equal(y, trnfft_amd.selective_scan(x, *v[1:])) and torch.equal(mark, torch.ones_like(mark))
    want = torch.autograd.grad(trnfft_amd.selective_scan(x, *v[1:]).square().sum(), x)[0]
    del eager
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = trnfft_amd.selective_scan(x, *v[1:])
        g, = torch.autograd.grad(y, x, 2.0 * y.detach())
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(g, want)


def test_threads_and_streams_do_not_share():
    """Calls of several threads, each on a stream of its own: the native calls give up Python's lock."""
    import threading

    cases = [[v.requires_grad_() for v in operands(rows=2, t=t, ch=ch, seed=seed)] for seed, (t, ch) in enumerate([(300, 24), (700, 40), (33, 130)])]

    def passes(leaves):
        y, last = trnfft_amd.selective_scan(*leaves, return_state=True)
        u = trnfft_amd.causal_conv(y, torch.ones(y.shape[2], 3, device="cuda"), activation="relu")
        grads = torch.autograd.grad([u, last], leaves, [torch.ones_like(u), torch.ones_like(last)])
        norm = trnfft_amd.grad_norm([g.contiguous() for g in grads])
        return [y.detach(), last.detach(), u.detach(), *grads, norm]

    want = [passes(leaves) for leaves in cases]
    torch.cuda.synchronize()
    wrong = []

    def work(leaves, expected):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(20):
                    got = passes(leaves)
                    stream.synchronize()
                    if not all(torch.equal(a, b) for a, b in zip(got, expected)):
                        wrong.append("results differ")
        except Exception as e:  # (of the thread)
            wrong.append(repr(e))

    threads = [threading.Thread(target=work, args=pair) for pair in zip(cases, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_results_do_not_depend_on_timing():
    leaves = [v.requires_grad_() for v in operands(rows=3, t=900, ch=130, seed=4)]

    def run():
        y = trnfft_amd.selective_scan(*leaves)
        return (y, *torch.autograd.grad(y, leaves, torch.ones_like(y)))

    first = run()
    assert all(all(torch.equal(a, b) for a, b in zip(run(), first)) for _ in range(3))


def test_tensors_on_the_cpu_come_back_there():
    v = [x.cpu() for x in operands(t=20)]
    y, last = trnfft_amd.selective_scan(*v, return_state=True)
    assert not y.is_cuda and not last.is_cuda
    assert torch.equal(y, trnfft_amd.selective_scan(*[x.cuda() for x in v]).cpu())
    x, w = v[0].requires_grad_(), torch.randn(24, 4, requires_grad=True)
    y = trnfft_amd.causal_conv(x, w)
    y.sum().backward()
    assert not y.is_cuda and not x.grad.is_cuda and not w.grad.is_cuda


def test_gradients_are_not_differentiated_again_and_states_are_seen_to_change():
    v = operands(t=10)
    x = v[0].requires_grad_()
    y = trnfft_amd.selective_scan(*v)
    g, = torch.autograd.grad(y.square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()
    state = torch.zeros(2, 24, 16, device="cuda")
    version = state._version
    with torch.no_grad():
        trnfft_amd.selective_scan_step(v[0][:, 0], v[1][:, 0], v[2], v[3][:, 0], v[4][:, 0], state)
    assert state._version > version


def test_nodes_of_the_graph_are_kept_freed_hooked_and_recomputed():
    v = operands(rows=2, t=70, ch=24)
    leaves = [v[0].requires_grad_(), v[2].requires_grad_()]
    weight = torch.randn(24, 4, device="cuda", requires_grad=True)

    def layer():
        return trnfft_amd.selective_scan(trnfft_amd.causal_conv(v[0], weight, activation="silu"), *v[1:])

    wanted = [*leaves, weight]
    y = layer()
    dy = torch.randn_like(y)
    want = torch.autograd.grad(y, wanted, dy, retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, wanted, dy), want))
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(y, wanted, dy)
    # one gradient at a time, and one that is made to be differentiated and then is not
    for i, leaf in enumerate(wanted):
        assert torch.equal(torch.autograd.grad(layer(), leaf, dy, create_graph=i == 1)[0], want[i])
    moved = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: moved.append(t.device.type) or t.cpu(), lambda t: t.cuda()):
        y = layer()
    assert len(moved) >= 7 and all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, wanted, dy), want))
    y = torch.utils.checkpoint.checkpoint(layer, use_reentrant=False)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, wanted, dy), want))
    y = layer()
    with torch.no_grad():
        weight.mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, wanted, dy)

    def broken(_):
        raise ValueError("of a hook")

    with torch.autograd.graph.saved_tensors_hooks(broken, lambda t: t), pytest.raises(ValueError, match="of a hook"):
        layer()


def test_the_example_with_this_layer():
    import denoise

    torch.manual_seed(1)
    model = denoise.Denoiser(features=32, blocks=2, mixer="state-space").to("cuda")
    losses = denoise.train(model, 2, 3, 8000, 8, max_norm=1.0)
    assert len(losses) == 2
    assert all(p.grad is not None and bool(torch.isfinite(p.grad).all()) for p in model.parameters())
    total = torch.sqrt(sum(p.grad.double().square().sum() for p in model.parameters()))
    assert float(total) <= 1.0 + 1e-5
    with torch.no_grad():
        _, noisy, _ = denoise.signals(3, 8000, torch.Generator(device="cuda").manual_seed(2), torch.device("cuda"))
        frames = model.features(denoise.spectrum_of(noisy))
        whole, streamed = model(frames), denoise.stream(model, frames)
    assert float((whole - streamed).abs().max()) < 1e-4
