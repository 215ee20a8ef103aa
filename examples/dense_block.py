"""A residual block around a sparse-pooling layer, trained for a few steps on one GPU.

    x -> group norm + SiLU -> linear + GELU -> sparse pooling (mean of ReLU neurons) -> linear + x

The dense operators come from ``granulelayer_b200.dense``; with ``--checkpoint int8`` they keep what their backward
passes read in 8 bits.  Parameter gradients accumulate in fp32 ``main_grad`` buffers and ``FusedAdamW`` applies them.

    python examples/dense_block.py [--checkpoint int8] [--dtype bf16] [--steps 20]
"""
import argparse
import sys
from pathlib import Path

import torch
from torch import nn

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

from granulelayer_b200 import FusedAdamW, GroupNormAct, LinearAct, SparsePoolingLayer  # noqa: E402


class DenseBlock(nn.Module):
    """norm -> linear -> sparse pooling -> linear + residual over token rows [batch, width]."""

    def __init__(self, width: int, neurons: int, groups: int, norm_groups: int = 8, checkpoint: str = "none",
                 dtype=torch.float32, device="cuda", seed: int = 0):
        super().__init__()
        kw = dict(dtype=dtype, device=device)
        self.norm = GroupNormAct(width, norm_groups, activation="silu", checkpoint=checkpoint, **kw)
        self.mix = LinearAct(width, width, activation="gelu", checkpoint=checkpoint, seed=seed, **kw)
        self.pool = SparsePoolingLayer(width, neurons, groups, shared_neurons=None, pooling="mean", seed=seed, **kw)
        self.out = LinearAct(groups, width, checkpoint=checkpoint, seed=seed + 1, **kw)
        for m in (self.norm, self.mix, self.pool, self.out):
            m.enable_main_grad()

    def forward(self, x):
        pooled = self.pool(self.mix(self.norm(x)))
        return self.out(pooled.to(x.dtype), residual=x)


def train(checkpoint="none", dtype=torch.float32, steps=20, batch=256, width=512, neurons=65536, groups=256, seed=0,
          lr=2e-3):
    """The losses of `steps` steps on one random regression batch."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    block = DenseBlock(width, neurons, groups, checkpoint=checkpoint, dtype=dtype, seed=seed)
    opt = FusedAdamW(block.parameters(), lr=lr, moments="fp32")
    x = torch.randn(batch, width, generator=gen, device="cuda").to(dtype)
    target = torch.randn(batch, width, generator=gen, device="cuda").to(dtype)
    losses = []
    for _ in range(steps):
        y = block(x)
        loss = (y.float() - target.float()).square().mean()
        loss.backward()
        opt.step()
        losses.append(loss.detach())
    return torch.stack(losses).tolist()


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--checkpoint", choices=("none", "int8"), default="none")
    ap.add_argument("--dtype", choices=("f32", "bf16"), default="f32")
    ap.add_argument("--steps", type=int, default=20)
    a = ap.parse_args()
    losses = train(a.checkpoint, torch.float32 if a.dtype == "f32" else torch.bfloat16, a.steps)
    for i, v in enumerate(losses):
        print(f"step {i:3d}  loss {v:.5f}")


if __name__ == "__main__":
    main()
