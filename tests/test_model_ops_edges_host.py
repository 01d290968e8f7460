"""What the operators of models refuse at their ends, without a GPU."""

from __future__ import annotations

import pytest
import torch

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
