#!/usr/bin/env python
"""Distil an ALPHABET teacher into a feed-forward student, then serve the student in 8 bits.

    python examples/distill_feedforward.py [--steps 30] [--batch 64] [--hidden 256]

The teacher is a ``B200Alphabet`` on 4x4 patch tokens of (synthetic) uint8 images.  Its largest
logits are what a data set of stored teacher outputs would hold.  The student sees the mean of the
image's tokens through feed-forward blocks and a linear head: residual RMSNorm, products with bias,
activation and residual in their epilogues, and the distillation loss with hard labels mixed in.
"""

from __future__ import annotations

import argparse
import sys
from pathlib import Path

ROOT = Path(__file__).resolve().parents[1]
sys.path.insert(0, str(ROOT / "lnet-h200-imagenet1k-pg-ab_b200"))

import torch  # noqa: E402
from torch import Tensor, nn  # noqa: E402

from lnet_b200 import (AlphabetConfig, B200Alphabet, B200FeedForward,  # noqa: E402
                       distillation_loss, linear_act, residual_rms_norm)
from lnet_b200.images import patchify_images  # noqa: E402


class Student(nn.Module):
    """Token features -> feed-forward blocks -> class logits."""

    def __init__(self, channels: int, dim: int, hidden: int, classes: int, depth: int = 2) -> None:
        super().__init__()
        self.stem = nn.Linear(channels, dim, dtype=torch.bfloat16)
        self.blocks = nn.ModuleList(B200FeedForward(dim, hidden) for _ in range(depth))
        self.norm_weight = nn.Parameter(torch.ones(dim))
        self.head = nn.Linear(dim, classes, dtype=torch.bfloat16)

    def forward(self, tokens: Tensor) -> Tensor:
        x = linear_act(tokens.mean(1), self.stem.weight, self.stem.bias, activation="silu")
        for block in self.blocks:
            x = block(x)
        y, _ = residual_rms_norm(x, self.norm_weight)
        return linear_act(y, self.head.weight, self.head.bias)

    def quantize_(self) -> "Student":
        self.eval()
        for block in self.blocks:
            block.quantize_()
        return self


def run(steps: int = 30, batch: int = 64, hidden: int = 256, classes: int = 100, top: int = 8,
        temperature: float = 2.0, alpha: float = 0.7, log=print) -> dict:
    """Trains and serves; returns the losses and how far the 8-bit logits are from the others."""
    torch.manual_seed(0)
    dev = torch.device("cuda")
    images = torch.randint(0, 256, (batch, 32, 32, 3), dtype=torch.uint8, device=dev)
    tokens = patchify_images(images)  # [B, 64, 48] bf16
    config = AlphabetConfig(raw_input_dim=48, model_dim=96, modes=48, output_dim=classes)
    teacher = B200Alphabet(config, classes).eval().to(dev)
    with torch.no_grad():
        logits = teacher(tokens).float()
        logits = 3 * (logits - logits.mean(0)) / logits.std(0).clamp(min=1e-6)
        kept, indices = torch.topk(logits, top, dim=-1)
        labels = indices[:, 0].contiguous()
    student = Student(48, 96, hidden, classes).to(dev)
    # bf16 parameters take steps of 1e-2 of their size at least
    optimizer = torch.optim.AdamW(student.parameters(), lr=4e-3)
    losses = []
    for step in range(steps):
        loss = distillation_loss(student(tokens), indices, kept, labels=labels,
                                 temperature=temperature, alpha=alpha)
        optimizer.zero_grad(set_to_none=True)
        loss.backward()
        optimizer.step()
        losses.append(float(loss.detach()))
        if step % 10 == 0 or step == steps - 1:
            log(f"step {step:4d}  loss {losses[-1]:.4f}")
    with torch.no_grad():
        full = student.eval()(tokens).float()
        served = student.quantize_()(tokens).float()
        one = student(tokens[:1]).float()  # a single row takes the kernels for few rows
    off = float((served - full).norm() / full.norm())
    single = float((one - served[:1]).norm() / served[:1].norm())
    log(f"8-bit logits differ from bf16's by {off:.3f} (relative), one row alone by {single:.4f}")
    return {"losses": losses, "fp8": off, "single": single}


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__)
    ap.add_argument("--steps", type=int, default=30)
    ap.add_argument("--batch", type=int, default=64)
    ap.add_argument("--hidden", type=int, default=256)
    a = ap.parse_args()
    run(a.steps, a.batch, a.hidden)
