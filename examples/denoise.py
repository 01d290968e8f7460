"""A denoiser on STFT frames that is trained on whole signals and then runs on a stream, frame by frame.

    python examples/denoise.py [--steps 60] [--batch 16] [--seconds 2] [--dtype bfloat16] [--state-bits 8]
                               [--mixer attention] [--max-norm 1]

Signals are synthetic: gliding harmonics in white noise.  Frames-major spectra go through blocks of group norm and linear attention
with learned decays, or with ``--mixer state-space`` of group norm and a selective state space layer; a mask per bin comes out and
the inverse STFT gives the waveform back.  Training runs whole, ragged signals through ``linear_attention`` (``causal_conv`` and
``selective_scan``) and its gradient, clips the gradients where it is told to, and steps with ``AdamW``.  Serving keeps one state a
block and takes each new frame through ``linear_attention_step`` (the other layer's steps); its masks equal those of the whole
signal.
"""

from __future__ import annotations

import argparse
import math
import os
import sys

import torch
import torch.nn as nn
import torch.nn.functional as F

if __package__ in (None, ""):
    sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import trnfft_amd
from trnfft_amd.nn import GroupNorm, StateSpace
from trnfft_amd.optim import AdamW, clip_grad_norm_

N_FFT, HOP, RATE = 512, 160, 16000
BINS = N_FFT // 2 + 1


class FrameNorm(GroupNorm):
    """Group norm of every frame by itself: a stream's frame gets the statistics that it gets in a whole signal."""

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return super().forward(x.reshape(-1, x.shape[-1])).view(x.shape)


class Block(nn.Module):
    def __init__(self, features: int, heads: int, key_dim: int):
        super().__init__()
        self.heads, self.key_dim, self.value_dim = heads, key_dim, features // heads
        self.norm = FrameNorm(1, features)
        # one projection for queries and keys that all heads share, and each head's values
        self.project = nn.Linear(features, 2 * key_dim + features, bias=False)
        self.mix = nn.Linear(features, features, bias=False)
        self.norm2 = FrameNorm(heads, features, activation="silu")
        self.out = nn.Linear(features, features)
        # memories of 4 to 64 frames to begin with: exp(log_decay) = 1 - 1 / memory
        memory = 2.0 ** torch.linspace(2.0, 6.0, heads)
        self.rate = nn.Parameter(torch.log(-torch.log1p(-1.0 / memory)))

    def _split(self, x: torch.Tensor):
        q, k, v = self.project(self.norm(x)).split([self.key_dim, self.key_dim, self.heads * self.value_dim], dim=-1)
        own = (1, 1, self.heads)
        return tuple(F.normalize(t.float(), dim=-1).to(t.dtype).unflatten(-1, (n, -1)) if n == 1 else t.unflatten(-1, (n, -1))
                     for t, n in zip((q, k, v), own))

    def _log_decay(self) -> torch.Tensor:
        return -torch.exp(self.rate.float())

    def _join(self, x: torch.Tensor, o: torch.Tensor) -> torch.Tensor:
        return x + self.out(self.norm2(self.mix(o.flatten(-2))))

    def forward(self, x: torch.Tensor, lengths: torch.Tensor | None = None) -> torch.Tensor:
        q, k, v = self._split(x)
        return self._join(x, trnfft_amd.linear_attention(q, k, v, self._log_decay(), scale=1.0, lengths=lengths))

    def step(self, x: torch.Tensor, state: torch.Tensor) -> torch.Tensor:
        q, k, v = self._split(x)
        return self._join(x, trnfft_amd.linear_attention_step(q, k, v, self._log_decay(), state, scale=1.0))

    def state(self, streams: int, device) -> torch.Tensor:
        return torch.zeros(streams, self.heads, self.key_dim, self.value_dim, device=device)


class StateSpaceBlock(nn.Module):
    """The block with a selective state space layer in the attention's place."""

    def __init__(self, features: int):
        super().__init__()
        self.norm = FrameNorm(1, features)
        self.mix = StateSpace(features)

    def forward(self, x: torch.Tensor, lengths: torch.Tensor | None = None) -> torch.Tensor:
        return x + self.mix(self.norm(x), lengths)

    def step(self, x: torch.Tensor, state) -> torch.Tensor:
        return x + self.mix.step(self.norm(x), state)

    def state(self, streams: int, device):
        return self.mix.state(streams, device)


MIXERS = ("attention", "state-space")


class Denoiser(nn.Module):
    def __init__(self, features: int = 256, heads: int = 4, key_dim: int = 32, blocks: int = 2, mixer: str = "attention"):
        super().__init__()
        self.enter = nn.Linear(BINS, features)
        self.blocks = nn.ModuleList(Block(features, heads, key_dim) if mixer == "attention" else StateSpaceBlock(features)
                                    for _ in range(blocks))
        self.leave = nn.Linear(features, BINS)

    def features(self, spectrum: trnfft_amd.ComplexTensor) -> torch.Tensor:
        power = spectrum.real * spectrum.real + spectrum.imag * spectrum.imag
        return torch.log(power + 1e-5).to(self.enter.weight.dtype)

    def forward(self, frames: torch.Tensor, lengths: torch.Tensor | None = None) -> torch.Tensor:
        """Masks (batch, frames, bins) of feature frames."""
        x = self.enter(frames)
        for block in self.blocks:
            x = block(x, lengths)
        return torch.sigmoid(self.leave(x).float())

    def states(self, streams: int, device) -> list:
        return [b.state(streams, device) for b in self.blocks]

    def step(self, frame: torch.Tensor, states: list) -> torch.Tensor:
        """Masks (streams, bins) of every stream's next frame; the states are updated."""
        x = self.enter(frame)
        for block, state in zip(self.blocks, states):
            x = block.step(x, state)
        return torch.sigmoid(self.leave(x).float())


def spectrum_of(signal: torch.Tensor) -> trnfft_amd.ComplexTensor:
    """Frames-major spectrum (batch, frames, bins)."""
    return trnfft_amd.stft(signal, N_FFT, hop_length=HOP, frames_major=True).transpose(-1, -2)


def frames_of(length: int) -> int:
    return 1 + length // HOP  # centred frames


def waveform(spectrum: trnfft_amd.ComplexTensor, mask: torch.Tensor, length: int) -> torch.Tensor:
    masked = trnfft_amd.ComplexTensor(spectrum.real * mask, spectrum.imag * mask)
    return trnfft_amd.istft(masked.transpose(-1, -2), N_FFT, hop_length=HOP, length=length)


def signals(batch: int, length: int, g: torch.Generator, device):
    """Clean and noisy signals (batch, length) and their lengths in frames: the first whole, others end early."""
    t = torch.arange(length, device=device) / RATE
    base = 120.0 + 300.0 * torch.rand(batch, 1, generator=g, device=device)
    glide = 60.0 * (torch.rand(batch, 1, generator=g, device=device) - 0.5)
    phase = 2.0 * math.pi * (base * t + 0.5 * glide * t * t)
    clean = sum(torch.sin(k * phase) / k for k in (1, 2, 3, 5))
    clean = clean * (0.6 + 0.4 * torch.sin(2.0 * math.pi * 3.0 * t))
    frames = frames_of(length)
    ends = (frames * (0.5 + 0.5 * torch.rand(batch, generator=g, device=device))).long()
    ends[0] = frames
    clean = clean * (t < (ends[:, None] - 1) * (HOP / RATE))
    return clean, clean + 0.5 * torch.randn(batch, length, generator=g, device=device), ends


def train(model: Denoiser, steps: int, batch: int, length: int, state_bits: int, seed: int = 0,
          max_norm: float | None = None) -> list[float]:
    device = model.enter.weight.device
    g = torch.Generator(device=device).manual_seed(seed)
    optimizer = AdamW(model.parameters(), lr=2e-3, state_bits=state_bits)
    losses = []
    for _ in range(steps):
        clean, noisy, ends = signals(batch, length, g, device)
        spectrum = spectrum_of(noisy)
        mask = model(model.features(spectrum), ends)
        live = torch.arange(mask.shape[1], device=device) < ends[:, None]
        error = waveform(spectrum, mask * live[:, :, None], length) - clean
        loss = error.square().mean()
        optimizer.zero_grad()
        loss.backward()
        if max_norm is not None:
            clip_grad_norm_(model.parameters(), max_norm)
        optimizer.step()
        losses.append(loss.detach())
    return torch.stack(losses).tolist() if losses else []


@torch.no_grad()
def stream(model: Denoiser, frames: torch.Tensor) -> torch.Tensor:
    """Masks of feature frames (streams, frames, bins) that arrive one by one."""
    states = model.states(frames.shape[0], frames.device)
    return torch.stack([model.step(frames[:, t], states) for t in range(frames.shape[1])], dim=1)


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=60)
    ap.add_argument("--batch", type=int, default=16)
    ap.add_argument("--seconds", type=float, default=2.0)
    ap.add_argument("--dtype", choices=("float32", "bfloat16"), default="bfloat16")
    ap.add_argument("--state-bits", type=int, choices=(8, 32), default=8)
    ap.add_argument("--mixer", choices=MIXERS, default="attention")
    ap.add_argument("--max-norm", type=float, default=None)
    a = ap.parse_args()
    torch.manual_seed(0)
    model = Denoiser(mixer=a.mixer).to("cuda", getattr(torch, a.dtype))
    length = int(a.seconds * RATE)
    losses = train(model, a.steps, a.batch, length, a.state_bits, max_norm=a.max_norm)
    if losses:
        print(f"loss {losses[0]:.4f} -> {losses[-1]:.4f} in {a.steps} steps")
    clean, noisy, _ = signals(2, length, torch.Generator(device="cuda").manual_seed(1), torch.device("cuda"))
    with torch.no_grad():
        spectrum = spectrum_of(noisy)
        frames = model.features(spectrum)
        whole, streamed = model(frames), stream(model, frames)
        out = waveform(spectrum, streamed, length)
    ratio = [10.0 * math.log10(float(clean.square().sum() / (x - clean).square().sum())) for x in (noisy, out)]
    print(f"stream of {frames.shape[1]} frames: signal to noise {ratio[0]:.1f} -> {ratio[1]:.1f} dB, "
          f"masks differ from the whole signal's by at most {float((whole - streamed).abs().max()):.1e}")


if __name__ == "__main__":
    main()
