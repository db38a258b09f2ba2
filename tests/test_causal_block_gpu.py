"""The causal operators run together: DecayBlock against a 64-bit restatement (training, prompts in pieces, single tokens, captured),
and what the operators refuse on the GPU."""
import copy
import importlib.util
import math
import os

import pytest
import torch

from laplacianformer_b200 import capi, ops
from laplacianformer_b200.block import DecayBlock

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
U = {F16: 2.0**-11, BF16: 2.0**-8}
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def gen(seed=0):
    return torch.Generator(device="cuda").manual_seed(seed)


def rand(g, *shape, dtype=F32):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def rel(a, b):
    d, n = (a.detach().double() - b.detach().double()).norm(), b.detach().double().norm()
    return float(d / n) if n > 0 else float(d)


def block(dim, heads, dtype=BF16, seed=0, **kw):
    """A block whose vectors are not the ones and zeros that they start from."""
    torch.manual_seed(seed)
    b = DecayBlock(dim, heads, dtype=dtype, device="cuda", **kw)
    with torch.no_grad():
        for p in b.parameters():
            if p.dim() == 1:
                p.add_(0.3 * torch.randn_like(p))
    return b


def block64(b, x, p, state=None, lengths=None, offset=0):
    """The block in 64 bits on the parameters p (a dict by name), and the state after it, token by token."""
    def norm(t, w):
        return t / torch.sqrt((t * t).mean(-1, keepdim=True) + 1e-6) * w

    B, N, C = x.shape
    h, D, pairs = b.heads, C // b.heads, b.frequencies.numel()
    n = norm(x, p["norm1"])
    q, k, v = (n @ p["w_qkv"].T + p["b_qkv"]).view(B, N, 3, h, D).unbind(2)
    angle = (offset + torch.arange(N, device=x.device)).double()[:, None, None] * b.frequencies.to(x.device)
    c, s = angle.cos(), angle.sin()
    turn = lambda t: torch.cat((t[..., :pairs] * c - t[..., pairs:2 * pairs] * s, t[..., :pairs] * s + t[..., pairs:2 * pairs] * c,  # noqa: E731
                                t[..., 2 * pairs:]), -1)
    q, k = turn(q), turn(k)
    S = torch.zeros(B, h, D, D, dtype=torch.float64, device=x.device) if state is None else state
    l, outs = b.log_decay.double().exp()[:, None, None], []
    for i in range(N):
        live = (torch.full((B,), N, device=x.device) if lengths is None else lengths) > i
        live = live[:, None, None, None]
        S = torch.where(live, l * S + k[:, i, :, :, None] * v[:, i, :, None, :], S)
        outs.append(torch.where(live, D**-0.5 * q[:, i, :, None, :] @ S, 0.0).reshape(B, C))
    gate = torch.sigmoid(n @ p["w_gate"].T + p["b_gate"])
    t = x + b.residual_scale * gate * norm(torch.stack(outs, 1) @ p["w_proj"].T + p["b_proj"], p["norm1_out"])
    z = norm(t, p["norm2"]) @ p["w_in"].T
    f = z.shape[-1] // 2
    y = (torch.nn.functional.silu(z[..., :f]) * z[..., f:]) @ p["w_out"].T
    return t + b.residual_scale * p["channels"] * norm(y, p["norm2_out"]), S


def params64(b):
    return {n: t.detach().double() for n, t in b.named_parameters()}


# As for the other block: about ten roundings in a row between x and y and twice as many to a gradient, each of unit roundoff u;
# a norm passes a relative error on, and the sums that a gate or a projection makes of rounded values average theirs.
FORWARD, BACKWARD = 20, 80


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("B, N, dim, heads, kw", [(3, 150, 64, 2, {}), (2, 131, 96, 3, {"rotary_dim": 20, "residual_scale": 0.5}), (1, 1, 64, 1, {}),
                                                  (2, 40, 192, 2, {"decays": [1.0, 0.5]}), (2, 33, 48, 3, {"rotary_dim": 0})])
def test_block_forward_backward(B, N, dim, heads, kw, dtype):
    g, b = gen(N), block(dim, heads, dtype, **kw)
    x, dy = (rand(g, B, N, dim, dtype=dtype) for _ in range(2))
    x.requires_grad_()
    names, params = zip(*b.named_parameters())
    y = b(x)
    grads = torch.autograd.grad(y, (x, *params), dy)
    x64 = x.detach().double().requires_grad_()
    p64 = {n: t.requires_grad_() for n, t in params64(b).items()}
    y64, _ = block64(b, x64, p64)
    g64 = torch.autograd.grad(y64, (x64, *p64.values()), dy.double())
    assert rel(y, y64) <= FORWARD * U[dtype]
    for n, a, r in zip(("x", *names), grads, g64):
        assert a.shape == r.shape and rel(a, r) <= BACKWARD * U[dtype], n


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_prompt_then_tokens(dtype):
    """A padded batch of prompts in two pieces and four tokens each: the outputs and states of whole sequences."""
    g, b = gen(1), block(64, 2, dtype)
    n = torch.tensor([200, 131, 1, 0], device="cuda")
    x = rand(g, 4, 204, 64, dtype=dtype)
    whole = torch.stack([torch.cat((x[i, :n[i]], x[i, 200:], x[i, n[i]:200])) for i in range(4)])  # without the padding
    want, s64 = block64(b, whole.double(), params64(b), lengths=n + 4)
    with torch.no_grad():
        head, state = b(x[:, :130], lengths=n, return_state=True)
        tail, state = b(x[:, 130:200], state, (n - 130).clamp(min=0), offset=130, return_state=True)
        y = torch.cat((head, tail), 1)
        for i in range(4):
            assert n[i] == 0 or rel(y[i, :n[i]], want[i, :n[i]]) <= FORWARD * U[dtype]
        for j in range(4):
            out = b.step(x[:, 200 + j], state, n + j)
            assert out.shape == (4, 64)
            assert rel(out, want[torch.arange(4), n + j]) <= FORWARD * U[dtype]
    # the state is a sum of products of keys and values that went through four roundings
    assert rel(state, s64) <= 8 * U[dtype]


def test_tokens_captured():
    """A graph that takes a token and moves on, replayed: the bits of eager steps; two blocks on one state list."""
    g, blocks = gen(2), [block(64, 2, seed=i) for i in range(2)]
    states = [b.new_state(3) for b in blocks]
    x, pos = rand(g, 3, 64, dtype=BF16), torch.zeros(3, dtype=torch.int64, device="cuda")

    def run(states, pos):
        y = x
        for b, s in zip(blocks, states):
            y = b.step(y, s, pos)
        pos += 1
        return y

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        run([t.clone() for t in states], pos.clone())
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(states, pos)
    eager, at = [b.new_state(3) for b in blocks], torch.zeros_like(pos)
    for _ in range(5):
        x.copy_(rand(g, 3, 64, dtype=BF16))
        graph.replay()
        assert torch.equal(out, run(eager, at))
    assert all(torch.equal(a, c) for a, c in zip(states, eager)) and torch.equal(pos, at)


def test_training_step_captured():
    """Forward and backward of a stack on a padded batch, captured and replayed on other values."""
    g, blocks = gen(3), torch.nn.Sequential(block(64, 2, seed=1), block(64, 2, seed=2))
    x, n = rand(g, 2, 140, 64, dtype=BF16).requires_grad_(), torch.tensor([140, 70], device="cuda")
    params = [p for p in blocks.parameters()]

    def step():
        y = x
        for b in blocks:
            y = b(y, lengths=n)
        return torch.autograd.grad(y.float().square().mean(), (x, *params))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    with torch.no_grad():
        x.copy_(rand(g, 2, 140, 64, dtype=BF16))
        n.copy_(torch.tensor([3, 140], device="cuda"))
    graph.replay()
    assert all(torch.equal(a, c) for a, c in zip(out, step()))


def test_block_conversions():
    b = DecayBlock(64, 2, dtype=BF16, device="cuda")
    kept = b.log_decay.clone()
    for c in (b.half(), copy.deepcopy(b), b.to(BF16).float().to(F16)):
        assert c.log_decay.dtype == F32 and torch.equal(c.log_decay, kept)
        assert c(torch.ones(1, 3, 64, dtype=F16, device="cuda")).shape == (1, 3, 64)
    other = DecayBlock(64, 2, decays=[0.25, 0.5], dtype=F16, device="cuda")
    other.load_state_dict(b.state_dict())
    assert torch.equal(other.log_decay, kept)
    for bad in ({"heads": 3}, {"heads": 2, "decays": [0.5]}, {"heads": 2, "decays": [0.5, 1.5]}, {"heads": 2, "rotary_dim": 34}):
        with pytest.raises(ValueError):
            DecayBlock(64, **bad)


def test_example():
    spec = importlib.util.spec_from_file_location("train_causal", os.path.join(ROOT, "examples", "train_causal.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    losses, blocks = m.train(steps=3, batch=2, tokens=140)
    assert len(losses) == 3 and all(map(math.isfinite, losses))
    assert all(p.grad is not None and torch.isfinite(p.grad).all() and p.grad.any() for p in blocks.parameters())
    y = m.generate(blocks, prompt=130, tokens=4)
    assert y.shape[1] == 4 and torch.isfinite(y).all()


# ------------------------------------------------------------------ refusals


def operands():
    z = lambda *s, dt=BF16: torch.zeros(*s, dtype=dt, device="cuda")  # noqa: E731
    return z, z(2, 3, 5, 16), z(2, 3, 5, 8), z(3, dt=F32), z(2, 3, 16, 8, dt=F32)


def test_refusals():
    z, q, v, g, s = operands()
    n, f = torch.zeros(2, dtype=torch.int64, device="cuda"), ops.rotary_frequencies(8)
    a, st, ro, sw = ops.decay_attention, ops.decay_attention_step, ops.rotary, ops.sandwich_norm
    x, w = z(2, 5, 32), z(32)
    q1, v1 = q[:, :, 0], v[:, :, 0]
    bad = [
        lambda: a(q.float(), q.float(), v.float(), g), lambda: a(q, q.half(), v, g), lambda: a(q, q[:, :2], v, g), lambda: a(q[0], q[0], v[0], g),
        lambda: a(q, q, v[:, :, :4], g), lambda: a(q, q, v, g.double()), lambda: a(q, q, v, g[:2]), lambda: a(q, q, v, g.cpu()),
        lambda: a(q, q, v, g, s.bfloat16()), lambda: a(q, q, v, g, s[:1]), lambda: a(q, q, v, g, s.mT), lambda: a(q, q, v, g, lengths=n.int()),
        lambda: a(q, q, v, g, lengths=n.cpu()), lambda: a(q, q, v, g, lengths=n[:1]), lambda: a(q, q, v, g, scale=0.0), lambda: a(q, q, v, g, scale=-1.0),
        lambda: a(q, q, v, g, scale=math.inf), lambda: a(q, q, v, g, scale=math.nan), lambda: a(z(1, 1, 2, 129), z(1, 1, 2, 129), z(1, 1, 2, 8), g[:1]),
        lambda: st(q1, q1, v1, g, s.half()), lambda: st(q1, q1, v1, g, s[:, :, :, :4]), lambda: st(q1, q1, v1, g, s.transpose(0, 1).contiguous().transpose(0, 1)),
        lambda: st(q1, q1, v1, g, s[:1].expand(2, 3, 16, 8)), lambda: st(q, q, v, g, s), lambda: st(q1, q1.half(), v1, g, s), lambda: st(q1, q1, v1, g.cpu(), s),
        lambda: st(q1, q1, v1, g, s, scale=0.0),
        lambda: ro(q, None, f.float()), lambda: ro(q, None, f.cuda()), lambda: ro(q, None, ops.rotary_frequencies(18)), lambda: ro(q, q[:, :, :3], f),
        lambda: ro(q, q.half(), f), lambda: ro(q, None, f, positions=torch.arange(5)), lambda: ro(q, None, f, positions=torch.arange(5, device="cuda").int()),
        lambda: ro(q, None, f, positions=torch.arange(4, device="cuda")), lambda: ro(q, None, f, positions=torch.zeros(3, 5, dtype=torch.int64, device="cuda")),
        lambda: ro(q[0], None, f), lambda: ro(q.double(), None, f),
        lambda: sw(x, w[:16], x), lambda: sw(x, w, x[:1]), lambda: sw(x, w.float(), x), lambda: sw(x, w, x.half()), lambda: sw(x, w, x, z(3, 1, 32)),
        lambda: sw(x, w, x, z(1, 5, 32)), lambda: sw(x, w, x, z(2, 5, 1)), lambda: sw(x, w, x, z(2, 5, 32).cpu()), lambda: sw(x, w, x, None, w[:8]),
        lambda: sw(x.double(), w.double(), x.double()),
    ]
    for i, call in enumerate(bad):
        with pytest.raises((RuntimeError, TypeError)):
            call()
            pytest.fail(f"call {i} was taken")
    assert capi.device_status() == 0


def forms():
    g = gen(5)
    z, q, v, dec, s = operands()
    q, v, x, w = rand(g, 1, 2, 5, 16, dtype=BF16), rand(g, 1, 2, 5, 8, dtype=BF16), rand(g, 5, 16, dtype=BF16), rand(g, 16, dtype=BF16)
    f = ops.rotary_frequencies(8)
    return {"attention": lambda t: ops.decay_attention(t.view(1, 1, 5, 16).expand(1, 2, 5, 16), q, v, dec[:2]),
            "state": lambda t: ops.decay_attention(q, q, v, dec[:2], t.view(-1)[:32].float().view(1, 2, 16, 1).expand(1, 2, 16, 8)),
            "rotary": lambda t: ops.rotary(t.view(1, 1, 5, 16), q, f)[0], "sandwich": lambda t: ops.sandwich_norm(t, w, x, t, w)[0]}


@pytest.mark.parametrize("form", ["attention", "state", "rotary", "sandwich"])
def test_other_derivatives_are_refused(form):
    from torch.autograd import forward_ad

    f, x = forms()[form], rand(gen(6), 5, 16, dtype=BF16)
    for tracked in (False, True):
        with forward_ad.dual_level():
            dual = forward_ad.make_dual(x.clone().requires_grad_(tracked), torch.ones_like(x))
            with pytest.raises(RuntimeError, match="forward"):
                f(dual)
    y = f(x.requires_grad_())
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(y, x, torch.ones_like(y), create_graph=True)
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda t: f(t).float().sum())(x.detach())


def test_no_gradient_where_there_is_none():
    z, q, v, g, s = operands()
    q, v, s = q.requires_grad_(), v.requires_grad_(), s.requires_grad_()
    with pytest.raises(RuntimeError, match="log_decay"):
        ops.decay_attention(q, q, v, g.requires_grad_())
    g = g.detach()
    with pytest.raises(RuntimeError, match="no_grad"):
        ops.decay_attention_step(q[:, :, 0], q[:, :, 0], v[:, :, 0], g, s.detach())
    # a state that a backward pass saved may not be overwritten in between
    t = torch.zeros(2, 3, 16, 8, device="cuda").requires_grad_() * 1.0
    o = ops.decay_attention(q, q, v, g, t)
    with torch.no_grad():
        ops.decay_attention_step(q[:, :, 0], q[:, :, 0], v[:, :, 0], g, t)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        o.sum().backward()
    f = ops.rotary_frequencies(8)
    y = ops.rotary(q, None, f)
    f.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()


def test_broadcast_inputs():
    """Keys shared by the heads and a state shared by the sequences: their gradients are sums of the copies'."""
    g, dec = gen(7), torch.tensor([-0.1, -0.5, -0.01], device="cuda")
    q, v = rand(g, 2, 3, 140, 64, dtype=F16), rand(g, 2, 3, 140, 64, dtype=F16)
    k, s = rand(g, 2, 1, 140, 64, dtype=F16).requires_grad_(), rand(g, 1, 3, 64, 64).requires_grad_()
    do = rand(g, 2, 3, 140, 64, dtype=F16)
    a = torch.autograd.grad(ops.decay_attention(q, k.expand(2, 3, 140, 64), v, dec, s.expand(2, 3, 64, 64)), (k, s), do)
    kk, ss = k.detach().expand(2, 3, 140, 64).contiguous().requires_grad_(), s.detach().repeat(2, 1, 1, 1).requires_grad_()
    b = torch.autograd.grad(ops.decay_attention(q, kk, v, dec, ss), (kk, ss), do)
    # (sums of three 16-bit and of two fp32 gradients)
    assert rel(a[0], b[0].double().sum(1, keepdim=True)) <= U[F16] and rel(a[1], b[1].double().sum(0, keepdim=True)) <= 2.0**-23
