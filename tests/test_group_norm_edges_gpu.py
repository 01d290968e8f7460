"""Group norm where its inputs are at an end: views that negate what they read."""

from __future__ import annotations

import pytest
import torch

import trnfft_amd

pytestmark = pytest.mark.gpu


def test_views_that_negate_what_they_read():
    # one value each: contiguous, and still the negative of its memory
    one = torch.ones(1, device="cuda")
    minus = torch.complex(one, one).conj().imag
    assert minus.is_neg() and minus.is_contiguous()
    x = torch.randn(3, 7, 1, device="cuda")
    y = trnfft_amd.group_norm(x, 1, minus, minus)
    assert torch.equal(y, trnfft_amd.group_norm(x, 1, -one, -one))
    w, b = one.clone().requires_grad_(), one.clone().requires_grad_()
    dw, db = torch.autograd.grad(trnfft_amd.group_norm(minus.view(1, 1), 1, w, b, eps=1.0), [w, b], minus.view(1, 1))
    assert float(dw) == 0.0 and float(db) == -1.0
