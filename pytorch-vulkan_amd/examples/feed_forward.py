"""Trains a stack of residual feed-forward blocks on the "vulkan" device and
then serves single tokens from it.

A block is ``h + down(gelu(up(layer_norm(h))))``: the layer norm, the two
linear layers (bias, GELU and the residual in the products' epilogues) and
their gradients run on the backend's kernels, the matrices step with Muon and
the vectors with AdamW.  The task is synthetic: regress a fixed random
nonlinear map of Gaussian tokens.

    python pytorch-vulkan_amd/examples/feed_forward.py --width 1024 --steps 50
"""
from __future__ import annotations

import argparse
import os
import sys
import time

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import torch
import torch.nn.functional as F

import torch_vulkan
from torch_vulkan.nn import Linear
from torch_vulkan.optim import AdamW, Muon


class Block(torch.nn.Module):
    def __init__(self, width, hidden):
        super().__init__()
        self.norm = torch.nn.LayerNorm(width)
        self.up = Linear(width, hidden, activation="gelu")
        self.down = Linear(hidden, width)

    def forward(self, h):
        return self.down(self.up(self.norm(h)), residual=h)


def build(width, hidden, blocks, seed=0):
    torch.manual_seed(seed)
    return torch.nn.Sequential(*[Block(width, hidden) for _ in range(blocks)])


def train(model, x, target, steps, lr=0.02):
    """Losses of `steps` full-batch steps."""
    matrices = [p for p in model.parameters() if p.dim() == 2]
    vectors = [p for p in model.parameters() if p.dim() != 2]
    optimizers = [Muon(matrices, lr=lr, weight_decay=0.0), AdamW(vectors, lr=lr / 10, weight_decay=0.0)]
    losses = []
    for _ in range(steps):
        loss = F.mse_loss(model(x), target)
        model.zero_grad(set_to_none=True)
        loss.backward()
        for opt in optimizers:
            opt.step()
        losses.append(loss.detach())
    return [float(v) for v in losses]


def main():
    ap = argparse.ArgumentParser(description=__doc__)
    ap.add_argument("--width", type=int, default=256)
    ap.add_argument("--blocks", type=int, default=2)
    ap.add_argument("--tokens", type=int, default=2048)
    ap.add_argument("--steps", type=int, default=30)
    args = ap.parse_args()
    model = build(args.width, 4 * args.width, args.blocks).to("vulkan")
    g = torch.Generator().manual_seed(1)
    x = torch.randn(args.tokens, args.width, generator=g)
    target = torch.tanh(x @ torch.randn(args.width, args.width, generator=g) / args.width ** 0.5)
    x, target = x.to("vulkan"), target.to("vulkan")
    train(model, x, target, 2)
    torch_vulkan.synchronize()
    t0 = time.perf_counter()
    losses = train(model, x, target, args.steps)
    torch_vulkan.synchronize()
    print(f"loss {losses[0]:.4f} -> {losses[-1]:.4f}, {(time.perf_counter() - t0) / args.steps * 1e3:.2f} ms a step")
    with torch.no_grad():
        token = x[:1]
        model(token)
        torch_vulkan.synchronize()
        t0 = time.perf_counter()
        for _ in range(100):
            out = model(token)
        torch_vulkan.synchronize()
        print(f"one token: {(time.perf_counter() - t0) * 1e4:.1f} us, |out| {float(out.cpu().norm()):.4f}")


if __name__ == "__main__":
    main()
