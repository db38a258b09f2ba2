"""Trains two Laplacian blocks for a few steps on synthetic data and then serves them with 8-bit projections:
norms, products with fused epilogues, gated feed-forward blocks, gradient clipping and the 8-bit path together.

    python examples/train_block.py [--steps 20] [--batch 32]
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from laplacianformer_b200 import ops  # noqa: E402
from laplacianformer_b200.block import LaplacianBlock  # noqa: E402


def train(steps: int = 20, batch: int = 32, dim: int = 64, heads: int = 2, grid: int = 14, lr: float = 0.05, max_norm: float = 1.0):
    """Losses of `steps` steps of regression to a fixed random block's outputs, and the trained blocks."""
    torch.manual_seed(0)
    kw = {"heads": heads, "grid": grid, "device": "cuda"}
    blocks = torch.nn.Sequential(LaplacianBlock(dim, **kw), LaplacianBlock(dim, **kw))
    teacher = LaplacianBlock(dim, **kw)
    params = list(blocks.parameters())
    master = [p.detach().float() for p in params]  # fp32 copies that the updates accumulate in
    losses = []
    for _ in range(steps):
        x = torch.randn(batch, grid * grid, dim, device="cuda", dtype=torch.bfloat16)
        with torch.no_grad():
            target = teacher(x)
        loss = (blocks(x).float() - target.float()).square().mean()
        loss.backward()
        grads = [p.grad for p in params]
        ops.clip_grad_norm(grads, max_norm, out=grads)
        with torch.no_grad():
            for p, m, g in zip(params, master, grads):
                m.sub_(g.float(), alpha=lr)
                p.copy_(m)
                p.grad = None
        losses.append(loss.detach())
    return [float(v) for v in losses], blocks


def serve(blocks, batch: int = 8):
    """The blocks' outputs on one batch, with 16-bit and with 8-bit query-key-value projections."""
    x = torch.randn(batch, blocks[0].grid ** 2, blocks[0].norm1.numel(), device="cuda", dtype=torch.bfloat16)
    with torch.no_grad():
        full = blocks(x)
        for b in blocks:
            b.quantize_()
        return full, blocks(x)


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=20)
    ap.add_argument("--batch", type=int, default=32)
    a = ap.parse_args()
    losses, blocks = train(a.steps, a.batch)
    print("loss: first %.4f, last %.4f" % (losses[0], losses[-1]))
    full, quant = serve(blocks)
    print("8-bit projections change the output by %.2f %%" % (100 * float((quant.float() - full.float()).norm() / full.float().norm())))
