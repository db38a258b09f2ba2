"""Trains two causal blocks for a few steps to tell the next vector of a synthetic sequence, then takes a prompt and goes on
from it token by token: decayed linear attention, rotary positions and sandwich norms together.

    python examples/train_causal.py [--steps 20] [--batch 8] [--tokens 512]
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from laplacianformer_b200 import ops  # noqa: E402
from laplacianformer_b200.block import DecayBlock  # noqa: E402


def waves(batch: int, tokens: int, dim: int):
    """Sequences of sines of random frequency and phase per channel."""
    t = torch.arange(tokens, device="cuda")[:, None]
    turn, phase = torch.rand(2, batch, 1, dim, device="cuda").unbind(0)
    return torch.sin(0.3 * turn * t + 6.28 * phase).bfloat16()


def train(steps: int = 20, batch: int = 8, tokens: int = 512, dim: int = 128, heads: int = 2, lr: float = 0.05, max_norm: float = 1.0):
    """Losses of `steps` steps on sequences of up to `tokens` tokens, and the trained blocks."""
    torch.manual_seed(0)
    blocks = torch.nn.ModuleList(DecayBlock(dim, heads, residual_scale=0.7, device="cuda") for _ in range(2))
    params = list(blocks.parameters())
    master = [p.detach().float() for p in params]  # fp32 copies that the updates accumulate in
    losses = []
    for _ in range(steps):
        x = waves(batch, tokens + 1, dim)
        lengths = torch.randint(tokens // 2, tokens + 1, (batch,), device="cuda")
        live = torch.arange(tokens, device="cuda") < lengths[:, None]
        y = x[:, :-1]
        for b in blocks:
            y = b(y, lengths=lengths)
        error = (y.float() - x[:, 1:].float()).square().mean(-1)
        loss = (error * live).sum() / live.sum()
        for p in params:
            p.grad = None
        loss.backward()
        grads = [p.grad for p in params]
        ops.clip_grad_norm(grads, max_norm, out=grads)
        with torch.no_grad():
            for p, m, g in zip(params, master, grads):
                m.sub_(g.float(), alpha=lr)
                p.copy_(m)
        losses.append(loss.detach())
    return [float(v) for v in losses], blocks


@torch.no_grad()
def generate(blocks, batch: int = 4, prompt: int = 256, tokens: int = 16):
    """What follows prompts, one token at a time, each the input of the next: [batch, tokens, dim]."""
    y, states = waves(batch, prompt, blocks[0].norm1.numel()), []
    for b in blocks:
        y, s = b(y, return_state=True)
        states.append(s)
    y, out = y[:, -1], []
    positions = torch.full((batch,), prompt, dtype=torch.int64, device="cuda")
    for _ in range(tokens):
        out.append(y)
        for b, s in zip(blocks, states):
            y = b.step(y, s, positions)
        positions += 1
    return torch.stack(out, 1)


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=20)
    ap.add_argument("--batch", type=int, default=8)
    ap.add_argument("--tokens", type=int, default=512)
    a = ap.parse_args()
    losses, blocks = train(a.steps, a.batch, a.tokens)
    print("loss: first %.4f, last %.4f" % (losses[0], losses[-1]))
    print("16 tokens after a prompt, 2-norm per token:", [round(float(v), 2) for v in generate(blocks).float().norm(dim=-1).mean(0)])
