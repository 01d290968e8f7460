"""What the operators of models refuse, without a GPU: shapes, types and values, in Python and at the C entry points."""

from __future__ import annotations

import ctypes

import pytest
import torch

import trnfft_amd
from trnfft_amd import _lib
from trnfft_amd.nn import GroupNorm
from trnfft_amd.optim import AdamW


def _qkv(t=4, hq=2, hk=2, hv=2, dk=8, dv=8, dtype=torch.float32):
    return [torch.zeros(1, t, h, d, dtype=dtype) for h, d in ((hq, dk), (hk, dk), (hv, dv))]


def test_linear_attention_refusals():
    f, g = trnfft_amd.linear_attention, torch.zeros(2)
    q, k, v = _qkv()
    for args, error in [
        ((q[0], k, v, g), ValueError),
        ((q.double(), k.double(), v.double(), g), TypeError),
        ((q, k.bfloat16(), v, g), TypeError),
        ((q, k[..., :4], v, g), ValueError),
        ((q, k[:, :3], v, g), ValueError),
        ((q, k, v, g.double()), TypeError),
        ((q, k, v, torch.zeros(2, 1)), TypeError),
        ((q, k, v, torch.zeros(3)), ValueError),
        ((q, k, v, torch.zeros(0)), ValueError),
        ((q, k[..., :0], v, g), ValueError),
    ]:
        with pytest.raises(error):
            f(*args)
    for kwargs, error in [
        (dict(scale=0.0), ValueError),
        (dict(scale=float("nan")), ValueError),
        (dict(initial_state=torch.zeros(1, 2, 8, 7)), ValueError),
        (dict(initial_state=torch.zeros(1, 2, 8, 8, dtype=torch.bfloat16)), TypeError),
        (dict(lengths=torch.zeros(2, dtype=torch.int64)), ValueError),
        (dict(lengths=torch.zeros(1)), TypeError),
    ]:
        with pytest.raises(error):
            f(q, k, v, g, **kwargs)


def test_linear_attention_step_refusals():
    f, g = trnfft_amd.linear_attention_step, torch.zeros(2)
    q, k, v = (x[:, 0] for x in _qkv())
    with pytest.raises(ValueError):
        f(q, k, v, g, torch.zeros(1, 2, 8, 9))
    with pytest.raises(TypeError):
        f(q, k, v, g, torch.zeros(1, 2, 8, 8, dtype=torch.float16))
    with pytest.raises(RuntimeError):
        f(q.requires_grad_(), k, v, g, torch.zeros(1, 2, 8, 8))


def test_group_norm_refusals():
    f, x = trnfft_amd.group_norm, torch.zeros(2, 5, 12)
    for args, kwargs, error in [
        ((x.double(), 3), {}, TypeError),
        ((x[0, 0], 3), {}, ValueError),
        ((x, 5), {}, ValueError),
        ((x, 0), {}, ValueError),
        ((x, 3, torch.zeros(11)), {}, ValueError),
        ((x, 3, torch.zeros(12, dtype=torch.float16)), {}, TypeError),
        ((x, 3), dict(activation="tanh"), ValueError),
        ((x, 3), dict(eps=-1.0), ValueError),
        ((x, 3), dict(lengths=torch.zeros(3, dtype=torch.int64)), ValueError),
        ((x, 3), dict(lengths=torch.zeros(2)), TypeError),
        ((x[:, 0], 3), dict(lengths=torch.zeros(2, dtype=torch.int64)), ValueError),
    ]:
        with pytest.raises(error):
            f(*args, **kwargs)
    with pytest.raises(ValueError):
        GroupNorm(5, 12)


def test_adamw_refusals():
    f = trnfft_amd.adamw_step
    p = [torch.zeros(300)]
    with pytest.raises(TypeError):
        f([p[0].double()], p, p, p, step=1)
    with pytest.raises(TypeError):
        f(p, [p[0].half()], p, p, step=1)
    with pytest.raises(ValueError):
        f(p, p, p, p, step=0)
    with pytest.raises(ValueError):
        f(p, p, p, p, step=1, exp_avg_scales=p)
    with pytest.raises(TypeError):
        trnfft_amd.adamw_state_values(p, p)
    for bad in (dict(state_bits=4), dict(betas=(1.0, 0.9)), dict(lr=-1.0)):
        with pytest.raises(ValueError):
            AdamW([torch.nn.Parameter(torch.zeros(3))], **bad)
    f([], [], [], [], step=1)


@pytest.mark.skipif(torch.cuda.is_available(), reason="checks the no-GPU behaviour")
def test_operators_fail_loudly_without_a_gpu():
    q, k, v = _qkv()
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        trnfft_amd.linear_attention(q, k, v, torch.zeros(2))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        trnfft_amd.group_norm(torch.zeros(2, 4), 2)
    p = [torch.zeros(3)]
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        trnfft_amd.adamw_step(p, p, p, p, step=1)


def _attn(**changes):
    d = dict(dtype=0, heads=2, q_heads=2, k_heads=1, v_heads=2, key_dim=8, value_dim=8, scale=1.0, batch=1, tokens=4)
    d.update(changes)
    return _lib.AttnDesc(**d)


def test_c_entries_refuse_bad_descriptors():
    # by the arguments alone: no pointer is followed
    lib, size, far = _lib.lib(), ctypes.c_size_t(), 4096
    for desc, rc in [
        (_attn(dtype=3), _lib.TFA_ERR_INVALID),
        (_attn(heads=0), _lib.TFA_ERR_INVALID),
        (_attn(k_heads=3), _lib.TFA_ERR_INVALID),
        (_attn(tokens=-1), _lib.TFA_ERR_INVALID),
        (_attn(scale=0.0), _lib.TFA_ERR_INVALID),
        (_attn(scale=float("inf")), _lib.TFA_ERR_INVALID),
        (_attn(key_dim=257), _lib.TFA_ERR_UNSUPPORTED),
        (_attn(batch=2**40), _lib.TFA_ERR_UNSUPPORTED),
        (_attn(tokens=2**31), _lib.TFA_ERR_UNSUPPORTED),
    ]:
        assert lib.tfa_linear_attention_workspace_size(desc, 0, size) == rc
        assert lib.tfa_linear_attention(desc, far, far, far, far, None, None, far, None, None, None) == rc
        assert lib.tfa_linear_attention_backward(desc, far, far, far, far, None, None, far, None, far, far, far, None, None,
                                                 far, None) == rc
    assert lib.tfa_linear_attention(_attn(), None, far, far, far, None, None, far, None, None, None) == _lib.TFA_ERR_INVALID
    assert lib.tfa_linear_attention(_attn(), far, far, far, far, None, far, far, far, None, None) == _lib.TFA_ERR_INVALID
    assert lib.tfa_linear_attention(_attn(batch=0), None, None, None, None, None, None, None, None, None, None) == _lib.TFA_OK
    assert lib.tfa_linear_attention_step(_attn(), far, far, far, far, far, far, None) == _lib.TFA_ERR_INVALID
    assert lib.tfa_linear_attention_workspace_size(None, 0, size) == _lib.TFA_ERR_INVALID

    def norm(**changes):
        d = dict(dtype=0, channels=8, groups=2, activation=0, batch=1, positions=4, inner=1, eps=1e-5)
        d.update(changes)
        return _lib.NormDesc(**d)

    for desc, rc in [
        (norm(dtype=-1), _lib.TFA_ERR_INVALID),
        (norm(groups=3), _lib.TFA_ERR_INVALID),
        (norm(groups=0), _lib.TFA_ERR_INVALID),
        (norm(inner=3), _lib.TFA_ERR_INVALID),
        (norm(inner=0), _lib.TFA_ERR_INVALID),
        (norm(activation=4), _lib.TFA_ERR_INVALID),
        (norm(eps=float("nan")), _lib.TFA_ERR_INVALID),
        (norm(batch=2**31), _lib.TFA_ERR_UNSUPPORTED),
        (norm(channels=2**21, groups=1), _lib.TFA_ERR_UNSUPPORTED),
    ]:
        assert lib.tfa_group_norm_workspace_size(desc, 0, size) == rc
        assert lib.tfa_group_norm(desc, far, None, None, None, far, far, far, far, None) == rc
        assert lib.tfa_group_norm_backward(desc, far, far, None, None, None, far, far, far, None, None, far, None) == rc
    assert lib.tfa_group_norm(norm(), None, None, None, None, far, far, far, far, None) == _lib.TFA_ERR_INVALID

    def adam(**changes):
        d = dict(param_dtype=0, grad_dtype=0, state_bits=32, step=1, lr=1e-3, beta1=0.9, beta2=0.99, eps=1e-8)
        d.update(changes)
        return _lib.AdamDesc(**d)

    row = (ctypes.c_int64 * 8)(far, far, far, far, 0, 0, 0, 5)
    for desc in (adam(param_dtype=7), adam(state_bits=16), adam(step=0), adam(beta1=1.0), adam(lr=float("inf")), adam(eps=-1.0)):
        assert lib.tfa_adamw_step(1, row, desc, None) == _lib.TFA_ERR_INVALID
    assert lib.tfa_adamw_step(1, row, adam(state_bits=8), None) == _lib.TFA_ERR_INVALID  # no scales
    assert lib.tfa_adamw_step(-1, row, adam(), None) == _lib.TFA_ERR_INVALID
    assert lib.tfa_adamw_step(0, None, adam(), None) == _lib.TFA_OK
    assert lib.tfa_adamw_state_values(1, (ctypes.c_int64 * 4)(far, 0, far, 5), 0, None) == _lib.TFA_ERR_INVALID
    assert lib.tfa_last_error()


def test_tensor_table_refusals():
    """The builder of AdamW's tables reads the lists itself: what it refuses it names, without a GPU."""
    from trnfft_amd import _lib

    table = _lib.tensor_table()
    x, f32 = torch.zeros(3), torch.float32
    with pytest.raises(TypeError, match="op: states must be torch.int8, got torch.float32"):
        table("op", ("states",), ([x],), (torch.int8,), 0)
    with pytest.raises(ValueError, match="op: states must be on the GPU"):
        table("op", ("states",), ([x],), (f32,), 0)
    with pytest.raises(TypeError, match="op: states must be tensors"):
        table("op", ("states",), ([3],), (f32,), 0)
    with pytest.raises(ValueError, match="op: 0 a, but 1 b"):
        table("op", ("a", "b"), ([], [x]), (f32, f32), 0)
    with pytest.raises(ValueError, match="must agree"):
        table("op", ("a",), (), (), 0)
    with pytest.raises(TypeError, match="lists of tensors"):
        table("op", ("a", "b"), ([], (x,)), (f32, f32), 0)
    with pytest.raises(TypeError, match="lists of tensors"):
        table("op", ("a",), ([x],), ("float32",), 0)
    assert table("op", ("a", "b"), ([], None), (f32, f32), 0) == b""
