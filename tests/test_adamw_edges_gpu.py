"""The AdamW step where its callers are at an end: captures."""

from __future__ import annotations

import pytest
import torch

from trnfft_amd.optim import AdamW

pytestmark = pytest.mark.gpu


def test_the_optimizer_refuses_to_be_captured():
    # (replays would repeat the captured step's bias correction and leave the count where it is)
    def fresh():
        torch.manual_seed(0)
        p = torch.nn.Parameter(torch.randn(300, device="cuda"))
        p.grad = torch.randn(300, device="cuda")
        return p, AdamW([p], lr=1e-2)

    p, opt = fresh()
    opt.step()
    held, graph = p.detach().clone(), torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="captured"):
        with torch.cuda.graph(graph):
            opt.step()
    torch.cuda.synchronize()
    assert torch.equal(p, held) and opt.state[p]["step"] == 1
    opt.step()
    q, straight = fresh()
    straight.step()
    straight.step()
    assert torch.equal(p, q)
