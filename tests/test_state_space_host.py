"""What the operators of a state space layer and the clipping of gradients refuse, without a GPU: shapes, types and values, in
Python and at the C entry points."""

from __future__ import annotations

import ctypes

import pytest
import torch

import trnfft_amd
from trnfft_amd import _lib
from trnfft_amd.optim import clip_grad_norm_


def test_conv_refusals():
    f, x, w = trnfft_amd.causal_conv, torch.zeros(2, 5, 12), torch.zeros(12, 4)
    for args, kwargs, error in [
        ((x[0], w), {}, ValueError),
        ((x.double(), w), {}, TypeError),
        ((x, w[:11]), {}, ValueError),
        ((x, w[0]), {}, ValueError),
        ((x, w[:, :0]), {}, ValueError),
        ((x, w.half()), {}, TypeError),
        ((x, w, torch.zeros(11)), {}, ValueError),
        ((x, w, torch.zeros(12).half()), {}, TypeError),
        ((x, w), dict(activation="tanh"), ValueError),
        ((x, w), dict(initial_state=torch.zeros(2, 4, 12)), ValueError),
        ((x, w), dict(initial_state=torch.zeros(2, 3, 12).half()), TypeError),
        ((x, w), dict(lengths=torch.zeros(3, dtype=torch.int64)), ValueError),
        ((x, w), dict(lengths=torch.zeros(2)), TypeError),
    ]:
        with pytest.raises(error):
            f(*args, **kwargs)
    step, state = trnfft_amd.causal_conv_step, torch.zeros(2, 3, 12)
    with pytest.raises(ValueError):
        step(x, state, w)
    with pytest.raises(ValueError):
        step(x[:, 0], state[:, :2], w)
    with pytest.raises(TypeError):
        step(x[:, 0], state.half(), w)
    with pytest.raises(RuntimeError, match="no gradients"):
        step(x[:, 0], state, w.clone().requires_grad_())


def _scan(dtype=torch.float32, lead=(2, 5)):
    return dict(x=torch.zeros(*lead, 12, dtype=dtype), dt=torch.zeros(*lead, 12, dtype=dtype), a=torch.zeros(12, 4),
                b=torch.zeros(*lead, 3, 4, dtype=dtype), c=torch.zeros(*lead, 3, 4, dtype=dtype))


def test_scan_refusals():
    f, good = trnfft_amd.selective_scan, _scan()
    for change, error in [
        (dict(x=good["x"][0]), ValueError),
        (dict(x=good["x"].double()), TypeError),
        (dict(dt=good["dt"][:, :4]), ValueError),
        (dict(dt=good["dt"].half()), TypeError),
        (dict(a=good["a"][:11]), ValueError),
        (dict(a=good["a"][:, :0]), ValueError),
        (dict(a=good["a"].bfloat16()), TypeError),
        (dict(b=good["b"][..., :3]), ValueError),
        (dict(b=good["b"][:, :, 0]), ValueError),
        (dict(b=torch.zeros(2, 5, 5, 4), c=torch.zeros(2, 5, 5, 4)), ValueError),
        (dict(b=good["b"][:, :, :0], c=good["c"][:, :, :0]), ValueError),
        (dict(c=good["c"][:, :, :1]), ValueError),
        (dict(c=good["c"].bfloat16()), TypeError),
        (dict(z=good["x"][:1]), ValueError),
        (dict(z=good["x"].half()), TypeError),
        (dict(d=torch.zeros(11)), ValueError),
        (dict(dt_bias=torch.zeros(12).half()), TypeError),
        (dict(initial_state=torch.zeros(2, 12, 5)), ValueError),
        (dict(initial_state=torch.zeros(2, 12, 4).half()), TypeError),
        (dict(lengths=torch.zeros(3, dtype=torch.int64)), ValueError),
        (dict(lengths=torch.zeros(2)), TypeError),
    ]:
        with pytest.raises(error):
            f(**{**good, **change})
    step, one = trnfft_amd.selective_scan_step, _scan(lead=(2,))
    with pytest.raises(ValueError):
        step(**one, state=torch.zeros(2, 12, 5))
    with pytest.raises(TypeError):
        step(**one, state=torch.zeros(2, 12, 4, dtype=torch.bfloat16))
    with pytest.raises(RuntimeError, match="no gradients"):
        step(**{**one, "a": one["a"].requires_grad_()}, state=torch.zeros(2, 12, 4))


def test_clip_refusals():
    with pytest.raises(ValueError):
        trnfft_amd.clip_grads([torch.zeros(3)], -1.0)
    with pytest.raises(ValueError):
        trnfft_amd.clip_grads([torch.zeros(3)], float("nan"))
    with pytest.raises(TypeError):
        trnfft_amd.grad_norm([torch.zeros(3).double()])
    assert float(trnfft_amd.grad_norm([])) == 0.0 and float(clip_grad_norm_([], 1.0)) == 0.0


def test_forward_mode_tangents_are_refused():
    import torch.autograd.forward_ad as fwd

    one = _scan()
    with fwd.dual_level():
        x = fwd.make_dual(one["x"], torch.ones_like(one["x"]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            trnfft_amd.selective_scan(**{**one, "x": x})
        with pytest.raises(NotImplementedError, match="forward-mode"):
            trnfft_amd.causal_conv(x, torch.zeros(12, 4))


@pytest.mark.skipif(torch.cuda.is_available(), reason="checks the no-GPU behaviour")
def test_operators_fail_loudly_without_a_gpu():
    for call in (lambda: trnfft_amd.selective_scan(**_scan()), lambda: trnfft_amd.causal_conv(torch.zeros(1, 2, 3), torch.zeros(3, 4)),
                 lambda: trnfft_amd.clip_grads([torch.zeros(3)], 1.0), lambda: trnfft_amd.grad_norm([torch.zeros(3)])):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()


def test_native_calls_are_bound_to_the_library():
    from trnfft_amd import _lib

    native = _lib.state_space()
    assert native is _lib.state_space() and set(native.ENTRIES) - {"tfa_last_error"} <= set(_lib.EXPORTS)
    with pytest.raises(RuntimeError, match="tensor or None"):
        native.causal_conv(1, None, None, None, None, 0, False, True)
    with pytest.raises(TypeError):
        native.selective_scan()
    x, state = torch.zeros(2, 8), torch.zeros(2, 3, 8)  # on the CPU: left to Python
    assert native.conv_step(0, x, state, torch.zeros(8, 4), None, 0) is None
    assert native.scan_step(0, x, x, torch.zeros(8, 2), x, x, state, None, None, None, True) is None
    assert native.conv_step(0, 3, state, None, None, 0) is None
    assert native.causal_conv(x[None], torch.zeros(8, 4), None, None, None, 0, False, False) is None
    assert native.selective_scan(3, x, x, x, x, None, None, None, None, None, True, False, False) is None


def test_c_entries_refuse_bad_descriptors():
    # by the arguments alone: no pointer is followed
    lib, far, size = _lib.lib(), 4096, ctypes.c_size_t()

    def conv(**changes):
        return _lib.ConvDesc(**{**dict(dtype=0, channels=8, width=4, activation=0, batch=1, tokens=4), **changes})

    for desc, rc in [
        (conv(dtype=3), _lib.TFA_ERR_INVALID),
        (conv(channels=0), _lib.TFA_ERR_INVALID),
        (conv(width=0), _lib.TFA_ERR_INVALID),
        (conv(width=9), _lib.TFA_ERR_UNSUPPORTED),
        (conv(activation=4), _lib.TFA_ERR_INVALID),
        (conv(tokens=-1), _lib.TFA_ERR_INVALID),
        (conv(batch=2**40), _lib.TFA_ERR_UNSUPPORTED),
        (conv(tokens=2**31), _lib.TFA_ERR_UNSUPPORTED),
        (conv(channels=2**21), _lib.TFA_ERR_UNSUPPORTED),
    ]:
        assert lib.tfa_causal_conv(desc, far, far, None, None, None, far, None, None) == rc
        assert lib.tfa_causal_conv_workspace_size(desc, size) == rc
        assert lib.tfa_causal_conv_backward(desc, far, far, None, None, None, far, None, far, far, far, None, far, None) == rc
    assert lib.tfa_causal_conv(conv(), None, far, None, None, None, far, None, None) == _lib.TFA_ERR_INVALID
    assert lib.tfa_causal_conv(conv(), far, far, None, None, far, far, far, None) == _lib.TFA_ERR_INVALID
    assert lib.tfa_causal_conv(conv(batch=0), None, None, None, None, None, None, None, None) == _lib.TFA_OK
    assert lib.tfa_causal_conv_step(conv(), far, far, None, far, far, None) == _lib.TFA_ERR_INVALID
    assert lib.tfa_causal_conv_step(conv(tokens=1), far, far, None, None, far, None) == _lib.TFA_ERR_INVALID
    assert lib.tfa_causal_conv_backward(conv(), far, far, None, None, None, far, None, far, far, None, None, None, None) == _lib.TFA_ERR_INVALID

    def scan(**changes):
        return _lib.ScanDesc(**{**dict(dtype=0, channels=8, groups=2, states=4, softplus=1, batch=1, tokens=4), **changes})

    sizes = [ctypes.c_size_t() for _ in range(3)]
    grads = _lib.ScanGrads(far)
    for desc, rc in [
        (scan(dtype=-1), _lib.TFA_ERR_INVALID),
        (scan(groups=3), _lib.TFA_ERR_INVALID),
        (scan(groups=0), _lib.TFA_ERR_INVALID),
        (scan(states=0), _lib.TFA_ERR_INVALID),
        (scan(states=65), _lib.TFA_ERR_UNSUPPORTED),
        (scan(batch=-1), _lib.TFA_ERR_INVALID),
        (scan(batch=2**29), _lib.TFA_ERR_UNSUPPORTED),
        (scan(batch=2**25, tokens=2**30), _lib.TFA_ERR_UNSUPPORTED),
        (scan(tokens=2**31), _lib.TFA_ERR_UNSUPPORTED),
    ]:
        assert lib.tfa_selective_scan_sizes(desc, *sizes) == rc
        assert lib.tfa_selective_scan(desc, far, far, far, far, far, None, None, None, None, None, far, None, None, None, None) == rc
        assert lib.tfa_selective_scan_backward(desc, far, far, far, far, far, None, None, None, None, None, far, grads, far, None) == rc
    call = lib.tfa_selective_scan
    assert call(scan(), far, far, None, far, far, None, None, None, None, None, far, None, None, None, None) == _lib.TFA_ERR_INVALID
    assert call(scan(), far, far, far, far, far, None, None, None, None, far, far, far, None, None, None) == _lib.TFA_ERR_INVALID
    assert call(scan(), far, far, far, far, far, None, None, None, None, None, far, None, far + 8, None, None) == _lib.TFA_ERR_INVALID
    for strides in (dict(x_stride_token=2**24), dict(b_stride_token=-1)):
        assert call(scan(**strides), far, far, far, far, far, None, None, None, None, None, far, None, None, None, None) == _lib.TFA_ERR_UNSUPPORTED
    assert call(scan(batch=0), *[None] * 15) == _lib.TFA_OK
    assert lib.tfa_selective_scan_step(scan(), far, far, far, far, far, None, None, None, far, far, None) == _lib.TFA_ERR_INVALID
    back = lib.tfa_selective_scan_backward
    assert back(scan(tokens=40), far, far, far, far, far, None, None, None, None, None, None, grads, far, None) == _lib.TFA_ERR_INVALID  # no states
    gate = _lib.ScanGrads(far, None, None, None, None, None, far)
    assert back(scan(), far, far, far, far, far, None, None, None, None, None, None, gate, far, None) == _lib.TFA_ERR_INVALID

    def lists(*rows, dtype=0):
        g = _lib.GradLists()
        g.tensors[dtype] = b"".join(ctypes.c_int64(v).value.to_bytes(8, "little", signed=True) for r in rows for v in r)
        g.count[dtype] = len(rows)
        return g

    assert lib.tfa_grad_norm_workspace_size(lists((far, -1)), size) == _lib.TFA_ERR_INVALID
    assert lib.tfa_grad_norm_workspace_size(lists((0, 3)), size) == _lib.TFA_ERR_INVALID
    assert lib.tfa_grad_norm_workspace_size(lists((far, 20000), (far, 1)), size) == _lib.TFA_OK and size.value >= 8 * 2
    assert lib.tfa_grad_norm(lists((far, 3)), None, far, None) == _lib.TFA_ERR_INVALID
    assert lib.tfa_grad_norm(lists((far, 3)), far, far + 4, None) == _lib.TFA_ERR_INVALID
    assert lib.tfa_clip_grads(lists((far, 3)), -1.0, far, far, None) == _lib.TFA_ERR_INVALID
    assert lib.tfa_clip_grads(lists((far, 3), (far + 8, 3)), 1.0, far, far, None) == _lib.TFA_ERR_INVALID  # overlap
    assert b"overlap" in lib.tfa_last_error()


def test_the_layer_refuses_sizes_below_one():
    from trnfft_amd.nn import StateSpace

    for bad in (dict(features=0), dict(features=4, states=0), dict(features=4, width=0), dict(features=4, expand=0),
                dict(features=4, rank=0)):
        with pytest.raises(ValueError):
            StateSpace(**bad)
    m = StateSpace(20)
    assert m.rank == 2 and [s.shape for s in m.state(3)] == [(3, 3, 40), (3, 40, 16)]
