"""The block operators run together: LaplacianBlock against a 64-bit restatement, its 8-bit form, and the training example."""
import importlib.util
import math
import os

import pytest
import torch

from laplacianformer_b200.block import LaplacianBlock

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def block64(b, x, p):
    """The block in 64 bits on the parameters p (a dict by name)."""
    def norm(t, w):
        return t / torch.sqrt((t * t).mean(-1, keepdim=True) + 1e-6) * w

    B, N, C = x.shape
    h, D, g, s = b.heads, C // b.heads, b.grid, b.grid // b.pool
    qkv = norm(x, p["norm1"]) @ p["w_qkv"].T + p["b_qkv"]
    q, k, v = qkv.view(B, N, 3, h, D).permute(2, 0, 3, 1, 4)
    L = k.reshape(B, h, s, b.pool, s, b.pool, D).mean((3, 5)).reshape(B, h, s * s, D)
    dist = lambda u, w: (u[..., :, None, :] - w[..., None, :, :]).abs().sum(-1)  # noqa: E731
    sigma = math.sqrt(D)
    A = torch.exp(-dist(L, L) / sigma) + 0.01 * torch.eye(s * s, dtype=torch.float64, device=x.device)
    V = 1.8 / A.sum(-1).amax(-1)[..., None, None] ** 2 * A
    for _ in range(b.iters):
        V = 2 * V - V @ A @ V
    a = torch.exp(-dist(q, L) / sigma) @ (V @ (torch.exp(-dist(L, k) / sigma) @ v))
    t = x + a.transpose(1, 2).reshape(B, N, C) @ p["w_proj"].T + p["b_proj"]
    z = norm(t, p["norm2"]) @ p["w_in"].T
    f = z.shape[-1] // 2
    return (torch.nn.functional.silu(z[..., :f]) * z[..., f:]) @ p["w_out"].T + t


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_block_forward_backward(dtype):
    torch.manual_seed(0)
    b = LaplacianBlock(64, heads=2, grid=8, hidden=172, dtype=dtype, device="cuda")
    x = torch.randn(3, 64, 64, device="cuda").to(dtype).requires_grad_()
    dy = torch.randn(3, 64, 64, device="cuda").to(dtype)
    names, params = zip(*b.named_parameters())
    y = b(x)
    grads = torch.autograd.grad(y, (x, *params), dy)
    x64 = x.detach().double().requires_grad_()
    p64 = {n: t.detach().double().requires_grad_() for n, t in zip(names, params)}
    y64 = block64(b, x64, p64)
    g64 = torch.autograd.grad(y64, (x64, *p64.values()), dy.double())
    # About ten roundings in a row between x and y, twice as many to a gradient, each of unit roundoff u, and an
    # inverse whose condition number is below 20 on these landmarks: 2-norm errors within 20 u and 80 u.
    u = {torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}[dtype]
    assert float((y.double() - y64).norm() / y64.norm()) <= 20 * u
    for n, a, r in zip(("x", *names), grads, g64):
        assert float((a.double() - r).norm() / r.norm()) <= 80 * u, n


def test_block_quantized():
    torch.manual_seed(1)
    b = LaplacianBlock(64, heads=2, grid=8, device="cuda")
    x = torch.randn(2, 64, 64, device="cuda").bfloat16()
    with torch.no_grad():
        full = b(x)
        quant = b.quantize_()(x)
    # 8-bit operands carry 2^-4 per value at most, averaged over 64 products
    assert 0 < float((quant.float() - full.float()).norm() / full.float().norm()) <= 2.0**-4
    x.requires_grad_()
    y = b(x)  # with gradients: the 16-bit weights
    assert torch.equal(y, full)
    y.sum().backward()
    assert torch.isfinite(x.grad).all()


def test_training_example():
    spec = importlib.util.spec_from_file_location("train_block", os.path.join(ROOT, "examples", "train_block.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    losses, blocks = m.train(steps=30, batch=8)
    assert all(map(math.isfinite, losses)) and sum(losses[-5:]) < sum(losses[:5])
    full, quant = m.serve(blocks, batch=2)
    assert torch.isfinite(full).all() and torch.isfinite(quant).all()
