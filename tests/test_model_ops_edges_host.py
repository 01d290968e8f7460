"""What the operators of models refuse at their ends, without a GPU."""

from __future__ import annotations

import ctypes

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import trnfft_amd
from trnfft_amd import _lib
from trnfft_amd.optim import AdamW


def test_the_optimizer_refuses_to_be_captured(monkeypatch):
    p = torch.nn.Parameter(torch.zeros(5))
    p.grad = torch.ones(5)
    opt = AdamW([p])
    monkeypatch.setattr(torch.cuda, "is_initialized", lambda: True)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="captured"):
        opt.step()
    assert not opt.state[p]


def test_lists_of_tensors_hold_no_negating_views():
    minus = torch.complex(torch.ones(1), torch.ones(1)).conj().imag
    assert minus.is_neg() and minus.is_contiguous()
    with pytest.raises(ValueError, match="negating"):
        _lib.tensor_table()("op", ("states",), ([minus],), (torch.float32,), 0)


def test_forward_mode_tangents_are_not_dropped():
    q, g, s, x, w = (torch.zeros(n) for n in ((1, 4, 2, 8), (2,), (1, 2, 8, 8), (2, 5, 4), (4,)))
    with forward_ad.dual_level():
        for i in range(5):
            a = [forward_ad.make_dual(t, torch.ones_like(t)) if i == j else t for j, t in enumerate((q, q, q, g, s))]
            with pytest.raises(NotImplementedError, match="forward-mode"):
                trnfft_amd.linear_attention(*a[:4], initial_state=a[4])
            with pytest.raises(NotImplementedError, match="forward-mode"):
                trnfft_amd.linear_attention_step(*(t[:, 0] for t in a[:3]), a[3], a[4])
        for i in range(3):
            a = [forward_ad.make_dual(t, torch.ones_like(t)) if i == j else t for j, t in enumerate((x, w, w))]
            with pytest.raises(NotImplementedError, match="forward-mode"):
                trnfft_amd.group_norm(a[0], 2, a[1], a[2])


def test_the_c_library_is_built_where_the_table_cannot_be(monkeypatch, tmp_path):
    from trnfft_amd.csrc import build

    linked = []

    def no_headers():
        raise RuntimeError("Python.h: No such file or directory")

    monkeypatch.setattr(build, "HERE", str(tmp_path))
    monkeypatch.setattr(build, "_build_table", no_headers)
    monkeypatch.setattr(build, "_compile", lambda src, obj: None)
    monkeypatch.setattr(build, "_link", lambda objs, out: linked.append(out))
    with pytest.raises(RuntimeError, match="Python.h"):
        build.build()
    assert linked == [build.LIB, build.COPY_LIB]


@pytest.mark.parametrize("tokens,states", [(1, 0), (64, 0), (256, 0), (512, 1), (1024, 3)])
def test_the_decays_gradient_keeps_states_between_tokens_alone(tokens, states):
    # (many short sequences: a state for each, 64 KB of no use, was more than the card holds)
    batch, heads, dim = 40064, 16, 128
    desc = _lib.AttnDesc(_lib.DTYPE_BF16, heads, heads, heads, heads, dim, dim, 1.0, batch, tokens,
                         *((tokens * heads * dim, heads * dim, dim) * 3))
    size = {}
    for kind in (1, 2):
        out = ctypes.c_size_t()
        assert _lib.lib().tfa_linear_attention_workspace_size(desc, kind, out) == _lib.TFA_OK
        size[kind] = out.value
    assert size[2] - size[1] == states * batch * heads * dim * dim * 4


@pytest.mark.parametrize("bad", [dict(state_bits=4), dict(betas=(1.0, 0.9)), dict(lr=-1.0), dict(eps=-1.0), dict(weight_decay=-1.0)])
def test_a_group_of_parameters_with_options_of_its_own_is_checked(bad):
    p, q = (torch.nn.Parameter(torch.zeros(3)) for _ in range(2))
    with pytest.raises(ValueError):
        AdamW([{"params": [p], **bad}])
    opt = AdamW([{"params": [p], "state_bits": 8, "lr": 0.5}])
    assert opt.param_groups[0]["state_bits"] == 8 and opt.param_groups[0]["lr"] == 0.5
    with pytest.raises(ValueError):
        opt.add_param_group({"params": [q], **bad})


def test_a_refused_step_does_not_count():
    # (on the CPU: there is no GPU, or the parameters are not on it; not contiguous anywhere)
    p = torch.nn.Parameter(torch.zeros(4, 6).t())
    p.grad = torch.ones(6, 4)
    opt = AdamW([p])
    for _ in range(2):
        with pytest.raises((RuntimeError, ValueError)):
            opt.step()
    assert opt.state[p]["step"] == 0
