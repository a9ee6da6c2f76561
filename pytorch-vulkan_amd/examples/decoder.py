"""Trains a small decoder on packed sequences on the "vulkan" device and then serves
tokens from a paged cache.

A block is attention (norm and rotation of queries and keys, a window with first
tokens that stay visible, shared key heads) and a feed-forward block, each behind a
layer norm and around the residual stream.  The task is synthetic: each token's
target is a fixed linear map of the token three places before it in its sequence, which only
attention can reach.

    python pytorch-vulkan_amd/examples/decoder.py --width 256 --steps 30
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
from torch_vulkan.nn import Attention, KVCache, Linear
from torch_vulkan.optim import AdamW, Muon

PAGE = 16


class Block(torch.nn.Module):
    def __init__(self, width, heads, kv_heads, window, sinks):
        super().__init__()
        self.norm1, self.norm2 = torch.nn.LayerNorm(width), torch.nn.LayerNorm(width)
        self.attention = Attention(width, heads, kv_heads, window=window, sinks=sinks)
        self.up = Linear(width, 4 * width, activation="gelu")
        self.down = Linear(4 * width, width)

    def forward(self, h, positions, **batch):
        h = self.attention(self.norm1(h), positions, residual=h, **batch)
        return self.down(self.up(self.norm2(h)), residual=h)


class Decoder(torch.nn.Module):
    def __init__(self, width, heads, kv_heads, blocks, window, sinks):
        super().__init__()
        self.blocks = torch.nn.ModuleList(Block(width, heads, kv_heads, window, sinks) for _ in range(blocks))

    def forward(self, h, positions, starts=None, caches=None, **batch):
        for block, cache in zip(self.blocks, caches or [None] * len(self.blocks)):
            h = block(h, positions, starts=starts, **(dict(batch, cache=cache) if cache is not None else {}))
        return h


def build(width, heads=4, kv_heads=2, blocks=2, window=32, sinks=2, seed=0):
    torch.manual_seed(seed)
    return Decoder(width, heads, kv_heads, blocks, window, sinks)


def data(lengths, width, seed=1):
    """(tokens, positions, starts, targets) of packed sequences, on the CPU."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(sum(lengths), width, generator=g)
    m = torch.randn(width, width, generator=g) / width ** 0.5
    positions = torch.cat([torch.arange(n) for n in lengths])
    starts = torch.tensor([0] + list(lengths)).cumsum(0).to(torch.int32)
    before = torch.arange(len(x)) - 3
    target = torch.where((positions >= 3)[:, None], x[before.clamp_min(0)] @ m, torch.zeros(()))
    return x, positions, starts, target


def train(model, x, positions, starts, target, steps, lr=0.02):
    """Losses of `steps` full-batch steps."""
    matrices = [p for p in model.parameters() if p.dim() == 2]
    vectors = [p for p in model.parameters() if p.dim() != 2]
    optimizers = [Muon(matrices, lr=lr, weight_decay=0.0), AdamW(vectors, lr=lr / 10, weight_decay=0.0)]
    losses = []
    for _ in range(steps):
        loss = F.mse_loss(model(x, positions, starts), target)
        model.zero_grad(set_to_none=True)
        loss.backward()
        for opt in optimizers:
            opt.step()
        losses.append(loss.detach())
    return [float(v) for v in losses]


def serve(model, prompts, new, dtype=torch.int8):
    """The rows that follow `prompts` (a list of [tokens, width] on the CPU), each step's output the next
    step's token: the prompts in one call, then a token of every sequence a step."""
    attention = model.blocks[0].attention
    count, lengths = len(prompts), [len(p) for p in prompts]
    width = -(-(max(lengths) + new) // PAGE)
    caches = [KVCache(count * width, attention.kv_heads, PAGE, attention.head_dim, dtype) for _ in model.blocks]
    table = torch.arange(count * width, dtype=torch.int32).view(count, width).to("vulkan")
    held = torch.tensor(lengths, dtype=torch.int32)
    starts = torch.tensor([0] + lengths).cumsum(0).to(torch.int32)
    with torch.no_grad():
        h = model(torch.cat(prompts).to("vulkan"), torch.cat([torch.arange(n) for n in lengths]).to("vulkan"),
                  starts.to("vulkan"), caches, table=table, lengths=held.to("vulkan"))
        h = h.cpu()[starts[1:].long() - 1]
        outs = [h]
        for _ in range(new - 1):
            positions, held = held.long(), held + 1
            h = model(h.to("vulkan"), positions.to("vulkan"), None, caches, table=table, lengths=held.to("vulkan")).cpu()
            outs.append(h)
    return torch.stack(outs, 1)


def main():
    ap = argparse.ArgumentParser(description=__doc__)
    ap.add_argument("--width", type=int, default=256)
    ap.add_argument("--tokens", type=int, default=2048)
    ap.add_argument("--steps", type=int, default=30)
    args = ap.parse_args()
    model = build(args.width).to("vulkan")
    lengths = [args.tokens // 2, args.tokens // 3, args.tokens - args.tokens // 2 - args.tokens // 3]
    batch = [t.to("vulkan") for t in data(lengths, args.width)]
    train(model, *batch, 2)
    torch_vulkan.synchronize()
    t0 = time.perf_counter()
    losses = train(model, *batch, args.steps)
    torch_vulkan.synchronize()
    print(f"loss {losses[0]:.4f} -> {losses[-1]:.4f}, {(time.perf_counter() - t0) / args.steps * 1e3:.2f} ms a step")
    prompts = [torch.randn(n, args.width) for n in (40, 7, 100)]
    serve(model, prompts, 4)
    t0 = time.perf_counter()
    out = serve(model, prompts, 32)
    print(f"served {out.shape[1]} tokens of {out.shape[0]} sequences: {(time.perf_counter() - t0) / out.shape[1] * 1e3:.2f} ms a token")


if __name__ == "__main__":
    main()
