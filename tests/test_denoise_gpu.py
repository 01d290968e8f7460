"""The denoiser example: the frame operators trained and served together (examples/denoise.py)."""

import os
import sys

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "examples"))

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,bits", [(torch.float32, 32), (torch.bfloat16, 8)])
def test_training_lowers_the_loss(dtype, bits):
    import denoise

    torch.manual_seed(0)
    model = denoise.Denoiser(features=64, heads=2, key_dim=16, blocks=2).to("cuda", dtype)
    losses = denoise.train(model, 30, 4, 8000, bits)
    # masks begin at 1/2 everywhere, where noise and lost signal both count: any that follow the harmonics do better
    assert sum(losses[-5:]) < 0.8 * sum(losses[:5]), losses
    assert all(p.grad is not None and bool(torch.isfinite(p.grad.float()).all()) for p in model.parameters())


def test_stream_equals_the_whole_signal():
    import denoise

    torch.manual_seed(1)
    model = denoise.Denoiser(features=64, heads=2, key_dim=16, blocks=2).to("cuda")
    _, noisy, _ = denoise.signals(3, 8000, torch.Generator(device="cuda").manual_seed(2), torch.device("cuda"))
    with torch.no_grad():
        frames = model.features(denoise.spectrum_of(noisy))
        whole, streamed = model(frames), denoise.stream(model, frames)
    # fp32 throughout, other orders of summation; the matrix cores take three bf16 pieces of a value (2^-24 of it).
    # A mask moves by a quarter of what its logit does, and logits are of order 1 through two blocks: 1e-4 is 400 roundings.
    assert whole.shape == (3, denoise.frames_of(8000), denoise.BINS)
    assert float((whole - streamed).abs().max()) < 1e-4


def test_padding_does_not_reach_the_masks():
    import denoise

    torch.manual_seed(3)
    model = denoise.Denoiser(features=64, heads=2, key_dim=16, blocks=1).to("cuda")
    frames = torch.randn(2, 40, denoise.BINS, device="cuda")
    lengths = torch.tensor([40, 23], device="cuda")
    with torch.no_grad():
        alone = model(frames[1:, :23])
        frames[1, 23:] = 1e4
        padded = model(frames, lengths)
    assert float((padded[1, :23] - alone[0]).abs().max()) < 1e-4
