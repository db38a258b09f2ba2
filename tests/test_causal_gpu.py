"""The causal operators against their definitions in 64 bits: decayed linear attention (prompts, training, single tokens),
rotary positions and the sandwich norm, at the sizes, strides and values where they can go wrong.

Tolerances.  u is a rounding's largest relative size (half a step) of the 16-bit type, E of fp32.  A rounding is uniform
within its step, so over many values its errors have a 2-norm of at most u / sqrt(3) of the values'.

Attention: an output is rounded once, and what it sums is rounded once before (each weighted score, or each state entry
that a query meets): two independent errors, together sqrt(2 / 3) u = 0.82 u of the norm; 1.25 u leaves room for the
scatter of small outputs.  Per element the two are bounded by u |o| + u B, with B the sum of the terms' sizes
scale sum_j w |q| . |k_j| |v_j|, plus 300 E B for sums of up to 300 terms in a row in fp32, and in fp16 half its smallest
step for each score.  States: each term l^n k v is held in parts that leave u^2 of it (two) or less, and the sums are
fp32: (u^2 + 300 E) of the terms' sizes per element."""
import math

import pytest
import torch

from laplacianformer_b200 import ops

pytestmark = pytest.mark.gpu
U = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0**-25, torch.float32: 0.0}  # half the smallest step (bf16, fp32: below all sizes here)
E = 2.0**-24
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def gen(seed=0):
    return torch.Generator(device="cuda").manual_seed(seed)


def rand(g, *shape, dtype=F32, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def heads(g, b, h, t, d, dtype, scale=1.0):
    return rand(g, b, t, h, d, dtype=dtype, scale=scale).transpose(1, 2)


def rel(a, b):
    d, n = (a.detach().double() - b.detach().double()).norm(), b.detach().double().norm()
    return float(d / n) if n > 0 else float(d)


def within(a, b, tol, what=""):
    a, b = a.detach().double(), b.detach().double()
    bad = ~((a - b).abs() <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float(((a - b).abs() - tol)[bad].max()):.3g}"


# ------------------------------------------------------------------ attention: the definition


def powers(g, n):
    """l^n for integers n [..] per head, [H, *n.shape]; l^0 = 1 for every l."""
    g = g.double().view(-1, *[1] * n.dim())
    return torch.where(n == 0, 1.0, torch.exp(torch.where(n == 0, 0.0, g) * n.double()))


def attention64(q, k, v, g, state=None, lengths=None, scale=None, absolute=False):
    """(o, state) by the quadratic form; with `absolute` the sums of the terms' sizes."""
    B, H, T, dk = q.shape
    scale = dk**-0.5 if scale is None else scale
    i = torch.arange(T, device=q.device)
    n = torch.full((B,), T, device=q.device) if lengths is None else lengths.clamp(0, T)
    live = (i < n[:, None])[:, None, :, None]
    q, k, v = (torch.where(live, x, 0.0) for x in (q, k, v))
    if absolute:
        q, k, v, state = q.abs(), k.abs(), v.abs(), None if state is None else state.abs()
    gap = i[:, None] - i[None, :]
    w = torch.where(gap >= 0, powers(g, gap.clamp(min=0)), 0.0)
    o = ((q @ k.mT) * w) @ v
    left = (n[:, None] - 1 - i).clamp(min=0)
    end = (k * powers(g, left).transpose(0, 1)[..., None]).mT @ v
    if state is not None:
        o = o + powers(g, i + 1)[None, :, :, None] * (q @ state)
        end = end + powers(g, n).transpose(0, 1)[..., None, None] * state
    return scale * o, end


def check_attention(q, k, v, g, state=None, lengths=None, scale=None, grads=True, seed=9):
    """o, the last state and all gradients of one call."""
    dtype, (B, H, T, dk), dv = q.dtype, q.shape, v.shape[-1]
    u, r = U[dtype], gen(seed)
    leaves = [x.detach().requires_grad_() for x in (q, k, v)] + ([state.detach().requires_grad_()] if state is not None else [])
    o, end = ops.decay_attention(*leaves[:3], g, leaves[3] if state is not None else None, lengths, scale, return_state=True)
    assert o.shape == (B, H, T, dv) and o.dtype == dtype and end.shape == (B, H, dk, dv) and end.dtype == F32
    assert o.transpose(1, 2).is_contiguous()
    l64 = [x.detach().double().requires_grad_() for x in leaves]
    args = (l64[0], l64[1], l64[2], g, l64[3] if state is not None else None, lengths, scale)
    o64, end64 = attention64(*args)
    with torch.no_grad():
        size, end_size = attention64(*args, absolute=True)
        scores = TINY[dtype] * (v.double().abs().sum(2, keepdim=True) + 1)
    within(o, o64, u * o64.abs() + (1.05 * u + 300 * E) * size + scores, "o")
    within(end, end64, (1.1 * u * u + 300 * E) * end_size + TINY[dtype] * v.double().abs().sum(2)[..., None, :], "state")
    if T * B > 64:
        assert rel(o, o64) <= 1.25 * u
    if not grads:
        return o, end
    do, dend = heads(r, B, H, T, dv, dtype), rand(r, B, H, dk, dv)
    got = torch.autograd.grad((o, end), leaves, (do, dend))
    want = torch.autograd.grad((o64, end64), l64, (do.double(), dend.double()))
    for name, a, b, x in zip(("dq", "dk", "dv", "dstate"), got, want, leaves):
        assert a.shape == x.shape and a.dtype == x.dtype
        bound = 1.25 * u if name != "dstate" else 1.5 * u * u + 40 * E
        assert rel(a, b) <= bound or float(b.norm()) == 0 or T * B <= 64 and rel(a, b) <= 2 * u, (name, rel(a, b))
    if lengths is not None:
        for x in (o, *got[:3]):
            for b in range(B):
                assert not x[b, :, int(lengths[b].clamp(0, T)):].any()
    return o, end


def decays(h):
    """From a token that sees itself alone over usual ones to no decay at all."""
    return torch.tensor([[-0.1], [-0.02, -1.0], [-float("inf"), -0.05, 0.0]][min(h, 3) - 1] + [-0.3, -6.0, -1e-4, -0.01, -90.0] * 4, device="cuda")[:h]


# ------------------------------------------------------------------ attention


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("b, h, t, dk, dv", [
    (1, 1, 1, 64, 64), (2, 3, 2, 32, 32), (1, 2, 127, 64, 64), (2, 1, 128, 64, 64), (1, 3, 129, 64, 64), (3, 2, 300, 64, 64), (1, 5, 700, 128, 128),
    (2, 3, 260, 128, 40), (1, 2, 333, 50, 37), (2, 2, 140, 1, 1), (1, 3, 257, 7, 128), (1, 1, 1030, 16, 64), (40, 8, 5, 64, 64), (400, 1, 150, 32, 32)])
def test_attention_sizes(b, h, t, dk, dv, dtype):
    g = gen(t + dk)
    check_attention(heads(g, b, h, t, dk, dtype), heads(g, b, h, t, dk, dtype), heads(g, b, h, t, dv, dtype), decays(h))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("b, h, t, dk, dv", [(2, 3, 1, 64, 64), (3, 2, 200, 64, 64), (1, 2, 2000, 64, 64), (2, 3, 600, 128, 96), (1, 1, 1500, 128, 128),
                                             (2, 2, 131, 33, 65)])
def test_attention_states(b, h, t, dk, dv, dtype):
    g = gen(t)
    check_attention(heads(g, b, h, t, dk, dtype), heads(g, b, h, t, dk, dtype), heads(g, b, h, t, dv, dtype), decays(h), state=rand(g, b, h, dk, dv, scale=3.0))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("t, dk, dv, lengths", [(300, 64, 64, [0, 1, 300, 128, 129, 250]), (1, 64, 64, [0, 1]), (130, 32, 50, [130, 2, 0]),
                                                (2100, 64, 64, [2100, 3]), (1100, 128, 128, [0, 1027, 640]), (200, 64, 64, [-5, 1 << 40, 77])])
@pytest.mark.parametrize("with_state", [False, True])
def test_attention_lengths(t, dk, dv, lengths, with_state, dtype):
    """Sequences padded at their end: what lies there, NaN included, enters nothing."""
    g, b, h = gen(t), len(lengths), 2
    n = torch.tensor(lengths, device="cuda")
    q, k, v = heads(g, b, h, t, dk, dtype), heads(g, b, h, t, dk, dtype), heads(g, b, h, t, dv, dtype)
    state = rand(g, b, h, dk, dv) if with_state else None
    o, end = check_attention(q, k, v, decays(h), state, n)
    for i in range(b):
        for x in (q, k, v):
            x[i, :, int(n[i].clamp(0, t)):] = float("nan")
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    p, last = ops.decay_attention(*leaves, decays(h), state, n, return_state=True)
    assert torch.equal(p, o) and torch.equal(last, end)
    do = heads(g, b, h, t, dv, dtype)
    clean = torch.autograd.grad(p, leaves, do, retain_graph=True)
    for i in range(b):
        do[i, :, int(n[i].clamp(0, t)):] = float("nan")
    for a, c in zip(torch.autograd.grad(p, leaves, do), clean):
        assert torch.equal(a, c)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_attention_strides(dtype):
    """Views of a joint projection, other orders of the dimensions, heads off 16-byte boundaries, expanded and reversed operands."""
    g, b, h, t, d = gen(1), 2, 3, 200, 64
    qkv = rand(g, b, t, 3, h, d, dtype=dtype)
    a = qkv.permute(2, 0, 3, 1, 4)
    dec = decays(h)
    base = ops.decay_attention(*a, dec)
    assert torch.equal(ops.decay_attention(*(x.contiguous() for x in a), dec), base)
    assert torch.equal(ops.decay_attention(*(x.permute(3, 1, 0, 2).contiguous().permute(2, 1, 3, 0) for x in a), dec), base)
    odd = torch.zeros(3, b, h, t, d + 3, dtype=dtype, device="cuda")
    odd[..., 1 : d + 1] = a
    assert torch.equal(ops.decay_attention(*odd[..., 1 : d + 1], dec), base)
    q, k, v = a
    check_attention(q[:, :1].expand(-1, h, -1, -1), k, v[:1].expand(b, -1, -1, -1), dec)
    x, y = q.detach().requires_grad_(), k.detach().requires_grad_()
    o = ops.decay_attention(x, y, v, dec)
    do = heads(g, b, h, t, d, dtype)
    want = torch.autograd.grad(o, (x, y), do, retain_graph=True)
    for other in (do.contiguous(), do.mT.contiguous().mT, torch.cat((do, do), -1)[..., d:]):
        for m, n in zip(torch.autograd.grad(o, (x, y), other, retain_graph=True), want):
            assert torch.equal(m, n)
    one = torch.autograd.grad(o, (x, y), torch.ones((), dtype=dtype, device="cuda").expand(o.shape))
    full = torch.autograd.grad(ops.decay_attention(x, y, v, dec), (x, y), torch.ones_like(o))
    assert all(torch.equal(m, n) for m, n in zip(one, full))


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_attention_ranges(dtype):
    """States far above fp16's range that queries bring back, tiny ones, and no decay over many tokens."""
    g, b, h, t, d = gen(2), 1, 2, 640, 64
    dec = torch.zeros(h, device="cuda")
    q, k, v = heads(g, b, h, t, d, dtype, 2.0**-9), heads(g, b, h, t, d, dtype).abs() + 1, heads(g, b, h, t, d, dtype).abs() + 1
    state = rand(g, b, h, d, d).abs() * 1e6
    o, end = ops.decay_attention(q, k, v, dec, state, return_state=True)
    o64, end64 = attention64(q.double(), k.double(), v.double(), dec, state.double())
    assert float(end.max()) > 1e6 and rel(o, o64) <= 1.25 * U[dtype] and rel(end, end64) <= 40 * E + U[dtype] ** 2
    state = rand(g, b, h, d, d) * 1e-6
    zero = torch.zeros_like(k)
    o = ops.decay_attention(q * 2.0**9, zero, zero, decays(2), state, scale=2.0**15)
    o64, _ = attention64(q.double() * 2.0**9, zero.double(), zero.double(), decays(2), state.double(), scale=2.0**15)
    assert rel(o, o64) <= 1.25 * U[dtype]


def test_attention_not_finite():
    """A NaN reaches nothing before its chunk of 128 tokens, and no other head."""
    g, b, h, t, d = gen(3), 1, 2, 400, 64
    q, k, v = (heads(g, b, h, t, d, BF16) for _ in range(3))
    want = ops.decay_attention(q, k, v, decays(h))
    v[0, 1, 300, 5] = float("nan")
    got = ops.decay_attention(q, k, v, decays(h))
    assert torch.equal(got[:, 0], want[:, 0]) and torch.equal(got[:, 1, :256], want[:, 1, :256]) and torch.isnan(got[0, 1, 300:, 5]).all()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("t, cuts", [(700, [1, 130, 131, 512]), (400, [128, 256])])
def test_attention_in_pieces(t, cuts, dtype):
    """A prompt in pieces, each from the last one's state, is the prompt; so are its tokens one by one."""
    g, b, h, d = gen(4), 2, 3, 64
    q, k, v, dec = heads(g, b, h, t, d, dtype), heads(g, b, h, t, d, dtype), heads(g, b, h, t, d, dtype), decays(h)
    o64, end64 = attention64(q.double(), k.double(), v.double(), dec)
    state, parts = None, []
    for a, z in zip([0, *cuts], [*cuts, t]):
        o, state = ops.decay_attention(q[:, :, a:z], k[:, :, a:z], v[:, :, a:z], dec, state, return_state=True)
        parts.append(o)
    assert rel(torch.cat(parts, 2), o64) <= 1.25 * U[dtype] and rel(state, end64) <= U[dtype] ** 2 + 40 * E
    _, state = ops.decay_attention(q[:, :, : t - 3], k[:, :, : t - 3], v[:, :, : t - 3], dec, return_state=True)
    for i in range(t - 3, t):
        o = ops.decay_attention_step(q[:, :, i], k[:, :, i], v[:, :, i], dec, state)
        assert rel(o, o64[:, :, i]) <= 1.25 * U[dtype]
    assert rel(state, end64) <= U[dtype] ** 2 + 40 * E


def test_attention_gradients_by_differences():
    """Along random directions the gradients are the slope of the 64-bit definition's differences."""
    g, b, h, t, d = gen(5), 2, 2, 150, 32
    leaves = [heads(g, b, h, t, d, F16).requires_grad_() for _ in range(3)] + [rand(g, b, h, d, d).requires_grad_()]
    dec = decays(h)
    o, end = ops.decay_attention(*leaves[:3], dec, leaves[3], return_state=True)
    do, dend = heads(g, b, h, t, d, F16), rand(g, b, h, d, d)
    grads = torch.autograd.grad((o, end), leaves, (do, dend))
    f = lambda *x: sum((y * w.double()).sum() for y, w in zip(attention64(*x[:3], dec, x[3]), (do, dend)))  # noqa: E731
    base = [x.detach().double() for x in leaves]
    for i, x in enumerate(base):
        step = torch.randn(x.shape, generator=g, device="cuda", dtype=torch.float64) * 1e-4
        up, down = ([y + s * step if j == i else y for j, y in enumerate(base)] for s in (1, -1))
        slope, mine = (f(*up) - f(*down)) / 2, (grads[i].double() * step).sum()
        # The function is linear in each operand: differences are exact to 64 bits.  1.25 u of the gradient's norm, times the step's.
        assert abs(float(slope - mine)) <= 1.25 * U[F16] * float(grads[i].double().norm() * step.norm())


@pytest.mark.parametrize("want", [(True, False, False, False), (False, True, False, False), (False, False, True, False), (False, False, False, True)])
def test_attention_gradients_of_some(want):
    g, b, h, t, d = gen(6), 2, 2, 140, 64
    x = [heads(g, b, h, t, d, BF16) for _ in range(3)] + [rand(g, b, h, d, d)]
    do = heads(g, b, h, t, d, BF16)

    def grads(flags):
        y = [a.detach().requires_grad_(f) for a, f in zip(x, flags)]
        o = ops.decay_attention(y[0], y[1], y[2], decays(h), y[3])
        o.backward(do)
        return [a.grad for a in y]

    every, some = grads((True,) * 4), grads(want)
    for a, b_, w in zip(some, every, want):
        assert torch.equal(a, b_) if w else a is None


def test_attention_gradient_of_the_state_alone():
    g, b, h, t, d = gen(7), 2, 2, 300, 64
    k, v, q = (heads(g, b, h, t, d, BF16).requires_grad_() for _ in range(3))
    _, end = ops.decay_attention(q, k, v, decays(h), return_state=True)
    dend = rand(g, b, h, d, d)
    got = torch.autograd.grad(end, (q, k, v), dend)
    l64 = [x.detach().double().requires_grad_() for x in (q, k, v)]
    _, end64 = attention64(*l64, decays(h))
    want = torch.autograd.grad(end64, l64[1:], dend.double())
    assert not got[0].any() and all(rel(a, c) <= 1.25 * U[BF16] for a, c in zip(got[1:], want))


def test_attention_empty():
    dec = decays(2)
    z = lambda *s, dt=BF16: torch.zeros(*s, dtype=dt, device="cuda")  # noqa: E731
    state = rand(gen(), 3, 2, 16, 8)
    o, end = ops.decay_attention(z(3, 2, 0, 16), z(3, 2, 0, 16), z(3, 2, 0, 8), dec, state, return_state=True)
    assert o.shape == (3, 2, 0, 8) and torch.equal(end, state)
    _, end = ops.decay_attention(z(3, 2, 0, 16), z(3, 2, 0, 16), z(3, 2, 0, 8), dec, return_state=True)
    assert not end.any()
    o, end = ops.decay_attention(z(0, 2, 7, 16), z(0, 2, 7, 16), z(0, 2, 7, 8), dec, return_state=True)
    assert o.shape == (0, 2, 7, 8) and end.shape == (0, 2, 16, 8)
    s = state.clone().requires_grad_()
    x = z(3, 2, 0, 16).requires_grad_()
    _, end = ops.decay_attention(x, x, z(3, 2, 0, 8), dec, s, return_state=True)
    dx, ds = torch.autograd.grad(end, (x, s), torch.ones_like(end))
    assert dx.shape == x.shape and torch.equal(ds, torch.ones_like(s))
    assert ops.decay_attention_step(z(0, 2, 16), z(0, 2, 16), z(0, 2, 8), dec, z(0, 2, 16, 8, dt=F32)).shape == (0, 2, 8)


def test_attention_repeats_and_streams():
    """The same bits each time; on a side stream; two calls at once; captured, and replayed on new inputs."""
    g, b, h, t, d = gen(8), 3, 4, 900, 64
    q, k, v = (heads(g, b, h, t, d, BF16) for _ in range(3))
    state, dec, n = rand(g, b, h, d, d), decays(h), torch.tensor([900, 500, 0], device="cuda")
    run = lambda: ops.decay_attention(q, k, v, dec, state, n, return_state=True)  # noqa: E731
    want = run()
    assert all(torch.equal(a, c) for a, c in zip(run(), want))
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for s in streams:
        with torch.cuda.stream(s):
            got.append(run())
    torch.cuda.synchronize()
    for r in got:
        assert all(torch.equal(a, c) for a, c in zip(r, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    new = [heads(g, b, h, t, d, BF16) for _ in range(3)]
    for x, y in zip((q, k, v), new):
        x.copy_(y)
    n.copy_(torch.tensor([10, 900, 300], device="cuda"))
    graph.replay()
    assert all(torch.equal(a, c) for a, c in zip(out, run()))


def test_attention_training_step_captured():
    g, b, h, t, d = gen(9), 2, 2, 300, 64
    x = [heads(g, b, h, t, d, BF16).requires_grad_() for _ in range(3)]
    do, dec = heads(g, b, h, t, d, BF16), decays(h)

    def step():
        return torch.autograd.grad(ops.decay_attention(*x, dec), x, do)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    with torch.no_grad():
        for y in x:
            y.copy_(heads(g, b, h, t, d, BF16))
    graph.replay()
    assert all(torch.equal(a, c) for a, c in zip(out, step()))


@pytest.mark.parametrize("b, d", [(296, 32), (148, 128), (3, 64)])
def test_attention_states_of_slow_heads(b, d):
    """States that remember 4096 tokens, over 64 chunks in one block or over segments.  In units of E of the state: a chunk's sum is
    cut off at most 8 times by 2 (its products of the second parts are small), added with a rounding to a state that remembers 32
    chunks, whose weights l^128 are off by at most 3 each: 16 + 32 + 96, besides u^2 of each term."""
    g, t, dtype = gen(4), 8192, F16
    q, k, v, do = (heads(g, b, 1, t, d, dtype) for _ in range(4))
    dec = torch.full((1,), -(2.0**-12), device="cuda")
    state = torch.zeros(b, 1, d, d, device="cuda").requires_grad_()
    o, end = ops.decay_attention(q, k, v, dec, state, return_state=True)
    (ds,) = torch.autograd.grad(o, state, do)
    i = torch.arange(t, device="cuda").double()
    want = torch.stack([(k[j].double() * torch.exp(-(2.0**-12) * (t - 1 - i))[:, None]).mT @ v[j].double() for j in range(b)])
    want_ds = torch.stack([(q[j].double() * torch.exp(-(2.0**-12) * (i + 1))[:, None]).mT @ do[j].double() for j in range(b)]) * d**-0.5
    u = U[dtype]
    assert rel(end, want) <= u * u + 144 * E and rel(ds, want_ds) <= u * u + 144 * E


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("t, dk, dv, lengths", [(5000, 64, 48, [5000, 2111]), (4000, 128, 128, [1, 2500]), (3840, 64, 64, [3839, 0])])
def test_attention_many_segments(t, dk, dv, lengths, dtype):
    """Few heads of long sequences, dealt to many blocks whose sums are joined before them."""
    g = gen(t)
    check_attention(heads(g, 2, 1, t, dk, dtype), heads(g, 2, 1, t, dk, dtype), heads(g, 2, 1, t, dv, dtype), torch.tensor([-0.003], device="cuda"),
                    state=rand(g, 2, 1, dk, dv, scale=3.0), lengths=torch.tensor(lengths, device="cuda"))


def test_attention_many_sequences_long_offsets():
    """Elements past 2^31: the last sequences of a large batch are their own calls' results."""
    b, h, t, d = 530, 8, 8192, 64
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB")
    x = torch.empty(b, t, h, d, dtype=BF16, device="cuda").normal_(generator=gen(1)).transpose(1, 2)
    o, end = ops.decay_attention(x, x, x, decays(h), return_state=True)
    p, last = ops.decay_attention(x[-1:], x[-1:], x[-1:], decays(h), return_state=True)
    # (other cuts of the sequence: equal to the roundings)
    assert rel(o[-1:], p.double()) <= 2 * U[BF16] and rel(end[-1:], last.double()) <= 2 * U[BF16] ** 2 + 40 * E


# ------------------------------------------------------------------ single tokens


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("b, h, dk, dv", [(1, 1, 64, 64), (3, 2, 32, 32), (200, 3, 64, 64), (2, 2, 128, 128), (1, 3, 1, 1), (2, 2, 7, 50), (1, 1, 128, 3), (2, 1, 5, 128)])
def test_step(b, h, dk, dv, dtype):
    g = gen(dk + dv)
    q, k, v = rand(g, b, h, dk, dtype=dtype), rand(g, b, h, dk, dtype=dtype), rand(g, b, h, dv, dtype=dtype)
    state, dec = rand(g, b, h, dk, dv), decays(h)
    s64 = powers(dec, torch.ones((), device="cuda"))[:, None, None] * state.double() + k.double()[..., None] * v.double()[..., None, :]
    o64 = dk**-0.5 * torch.einsum("bhd,bhde->bhe", q.double(), s64)
    size = (k.double()[..., None] * v.double()[..., None, :]).abs() + state.double().abs()
    version = state._version
    o = ops.decay_attention_step(q, k, v, dec, state)
    assert state._version > version and o.dtype == dtype and o.shape == (b, h, dv)
    within(state, s64, 8 * E * size, "state")  # the power, a product and a fused sum
    within(o, o64, U[dtype] * o64.abs() + (dk + 16) * E * dk**-0.5 * torch.einsum("bhd,bhde->bhe", q.double().abs(), size) + TINY[dtype], "o")


def test_step_strides_graph_and_views():
    g, b, h, d = gen(1), 4, 3, 64
    qkv = rand(g, b, 3, h, d, dtype=BF16)
    dec, state = decays(h), rand(g, b, h, d, d)
    one, two = state.clone(), torch.zeros(b * h * d * d + 1, device="cuda")[1:].view(b, h, d, d).copy_(state)  # off 16-byte boundaries
    want = ops.decay_attention_step(*(x.contiguous() for x in qkv.unbind(1)), dec, one)
    assert torch.equal(ops.decay_attention_step(*qkv.unbind(1), dec, two), want) and torch.equal(one, two)
    three = state.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = ops.decay_attention_step(*qkv.unbind(1), dec, three)
    for _ in range(3):
        graph.replay()
    for _ in range(2):
        want = ops.decay_attention_step(*qkv.unbind(1), dec, one)
    assert torch.equal(three, one) and torch.equal(o, want)


# ------------------------------------------------------------------ rotary positions


def rotary64(x, f, pos, interleaved, magnitude):
    """Complex multiplication in 64 bits; pos [B, N] (angles of far positions reduced with integers where they are exact)."""
    r = 2 * f.numel()
    unit = torch.polar(torch.full((), magnitude, dtype=torch.float64, device=x.device), pos.double()[:, None, :, None] * f.cuda())
    z = x[..., :r].double()
    z = torch.complex(z[..., ::2], z[..., 1::2]) if interleaved else torch.complex(z[..., : r // 2], z[..., r // 2 :])
    z = z * unit
    y = torch.stack((z.real, z.imag), -1).flatten(-2) if interleaved else torch.cat((z.real, z.imag), -1)
    return torch.cat((y, x[..., r:].double()), -1), torch.cat([z.abs()] * 2, -1) if not interleaved else z.abs().repeat_interleave(2, -1)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("b, h, hk, t, d, rot", [(2, 3, 3, 50, 64, 64), (1, 8, 1, 1, 128, 96), (3, 2, 2, 33, 50, 34), (2, 1, 4, 17, 7, 2), (1, 2, 2, 300, 32, 16),
                                                (2, 2, 2, 9, 16, 0), (1, 1, 1, 5, 300, 256), (2, 16, 16, 40, 64, 24), (5000, 2, 1, 1, 8, 8)])
def test_rotary(b, h, hk, t, d, rot, interleaved, dtype):
    g = gen(d + rot)
    q, k = heads(g, b, h, t, d, dtype).requires_grad_(), heads(g, b, hk, t, d, dtype).requires_grad_()
    f = ops.rotary_frequencies(rot)
    pos = torch.randint(-3000, 100000, (b, t), generator=g, device="cuda")
    y, z = ops.rotary(q, k, f, pos, interleaved=interleaved, magnitude=1.25)
    dy, dz = heads(g, b, h, t, d, dtype), heads(g, b, hk, t, d, dtype)
    grads = torch.autograd.grad((y, z), (q, k), (dy, dz))
    for x, w, dw, dx in ((q, y, dy, grads[0]), (k, z, dz, grads[1])):
        assert w.shape == x.shape and w.dtype == dtype and w.transpose(1, 2).is_contiguous()
        for a, c, p in ((w, x, pos), (dx, dw, -pos)):
            want, size = rotary64(c.detach(), f, p, interleaved, 1.25)
            # The angle's fraction in fp32 (2 pi 2^-25), the sine and cosine, and two products and a sum: below 16 E of the pair's length.
            size = torch.cat((size, torch.zeros_like(want[..., rot:])), -1)
            within(a, want, U[dtype] * want.abs() + 16 * E * size + TINY[dtype])
    assert torch.equal(y[..., rot:], q[..., rot:])


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_positions(interleaved):
    """Offsets, shared positions, far ones (2^40), none for k, and scaled frequencies."""
    g, b, h, t, d = gen(1), 2, 2, 20, 64
    q = heads(g, b, h, t, d, F32)
    f = ops.rotary_frequencies(d)
    run = lambda *a, **kw: ops.rotary(q, None, *a, interleaved=interleaved, **kw)  # noqa: E731
    at = torch.arange(t, device="cuda")
    assert torch.equal(run(f), run(f, at)) and torch.equal(run(f, offset=7), run(f, (at + 7).expand(b, t)))
    # Whole turns: a frequency of 2 pi / 64 at position 2^40 + p is that at p (the quotient by 2 pi is exact to 2^-53 of 2^34 turns).
    turns = torch.full((d // 2,), 2 * math.pi / 64, dtype=torch.float64)
    assert rel(run(turns, at + (1 << 40)), run(turns, at).double()) <= 2 * math.pi * 2.0**-53 * 2.0**35 + 16 * E
    for scaling, kw in (("linear", {}), ("base", {}), ("by_parts", {"original_length": 2048})):
        s = ops.rotary_frequencies(d, scaling=scaling, factor=4.0, **kw)
        want, size = rotary64(q, s, at.expand(b, t) * 1000, interleaved, 1.0)
        within(run(s, at * 1000), want, 17 * E * size)


def test_rotary_frequencies():
    f = ops.rotary_frequencies(64, base=500.0)
    assert f.dtype == torch.float64 and f.device.type == "cpu"
    assert torch.allclose(f, torch.tensor([500.0 ** (-2 * i / 64) for i in range(32)], dtype=torch.float64), rtol=1e-14)
    s = ops.rotary_frequencies(64, base=500.0, scaling="base", factor=8.0)
    assert abs(float(s[0] / f[0]) - 1) < 1e-14 and abs(float(s[-1] / f[-1]) - 1 / 8) < 1e-12
    assert torch.allclose(ops.rotary_frequencies(64, base=500.0, scaling="linear", factor=8.0) * 8, f, rtol=1e-14)
    p = ops.rotary_frequencies(64, scaling="by_parts", factor=8.0, original_length=4096)
    f = ops.rotary_frequencies(64)
    turns = 4096 * f / (2 * math.pi)
    assert torch.equal(p[turns >= 32], f[turns >= 32]) and torch.allclose(p[turns <= 1], f[turns <= 1] / 8, rtol=1e-14)
    mid = (turns > 1) & (turns < 32)
    assert mid.any() and (p[mid] < f[mid]).all() and (p[mid] > f[mid] / 8).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rotary_strides_and_graph(dtype):
    g, b, h, t, d = gen(2), 2, 3, 40, 64
    qkv = rand(g, b, t, 3, h, d, dtype=dtype).permute(2, 0, 3, 1, 4)
    f, pos = ops.rotary_frequencies(d), torch.arange(t, device="cuda")
    q, k, _ = qkv
    want = ops.rotary(q, k, f, pos)
    for change in (lambda x: x.contiguous(), lambda x: x.mT.contiguous().mT, lambda x: torch.nn.functional.pad(x, (1, 2))[..., 1:-2]):
        assert all(torch.equal(a, c) for a, c in zip(ops.rotary(change(q), change(k), f, pos), want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.rotary(q, k, f, pos)
    pos += 1000
    graph.replay()
    assert all(torch.equal(a, c) for a, c in zip(out, ops.rotary(q, k, f, pos)))
    x, y = q.detach().requires_grad_(), k.detach().requires_grad_()
    one, ones = ops.rotary(x, y, f, pos), torch.ones_like(x)
    both = torch.autograd.grad(one, (x, y), (ones, ones), retain_graph=True)
    assert torch.equal(torch.autograd.grad(one[1], y, ones)[0], both[1])  # k's gradient alone
    assert ops.rotary(q[:, :, :0], k[:, :, :0], f)[0].shape == (b, h, 0, d)


# ------------------------------------------------------------------ sandwich norm


def sandwich64(x, w, r, gate, wn, act, scale, eps=1e-6):
    norm = lambda t, v: t / torch.sqrt((t * t).mean(-1, keepdim=True) + eps) * v  # noqa: E731
    a = {"none": lambda z: z, "sigmoid": torch.sigmoid, "silu": torch.nn.functional.silu, "tanh": torch.tanh}[act]
    s = r + scale * (norm(x, w) if gate is None else a(gate) * norm(x, w))
    return s, None if wn is None else norm(s, wn)


def check_sandwich(lead, c, gate_shape, act, nxt, dtype, scale=0.7, seed=0):
    """Values, and gradients in the 2-norm: each is rounded once, and the backward reads the rounded sum (its normalised
    value is off by one rounding): sqrt(2 / 3) u = 0.82 u, 1.5 u with the scatter of small ones.  fp32: sums of up to 4096
    terms in groups of 8 or 32, below 40 E."""
    g, u = gen(seed), U[dtype]
    x, r, w = rand(g, *lead, c, dtype=dtype), rand(g, *lead, c, dtype=dtype), rand(g, c, dtype=dtype)
    gate = None if gate_shape is None else rand(g, *gate_shape, c, dtype=dtype)
    wn = rand(g, c, dtype=dtype) if nxt else None
    leaves = [t.requires_grad_() for t in (x, w, r, gate, wn) if t is not None]
    out = ops.sandwich_norm(x, w, r, gate, wn, act, scale)
    y, s = out if nxt else (None, out)
    d = [t.detach().double().requires_grad_() if t is not None else None for t in (x, w, r, gate, wn)]
    s64, y64 = sandwich64(*d, act, scale)
    part = (s64 - d[2]).abs() + d[2].abs()
    within(s, s64, u * s64.abs() + 24 * E * part + TINY[dtype], "s")
    if nxt:
        rt = 1 / torch.sqrt((s64 * s64).mean(-1, keepdim=True) + 1e-6)
        within(y, y64, u * y64.abs() + 40 * E * part * rt * d[4].abs() + TINY[dtype], "y")
    ds, dy = rand(g, *lead, c, dtype=dtype), rand(g, *lead, c, dtype=dtype)
    got = torch.autograd.grad((s, y) if nxt else s, leaves, (ds, dy) if nxt else ds)
    total = (s64 * ds.double()).sum() + ((y64 * dy.double()).sum() if nxt else 0)
    want = torch.autograd.grad(total, [t for t in d if t is not None])
    names = [n for n, t in zip(("dx", "dw", "dr", "dgate", "dnext"), (x, w, r, gate, wn)) if t is not None]
    # dx = rx (e - xh mean(e xh)) is a difference of two terms that nearly cancel in narrow rows (with one channel xh is
    # 1 - 5e-7 / x^2): each carries up to 40 E of its own size in fp32, whatever is left of them.
    dt = want[names.index("dr")]
    e = scale * dt * d[1] * (1.0 if gate is None else {"none": lambda z: z, "sigmoid": torch.sigmoid, "silu": torch.nn.functional.silu, "tanh": torch.tanh}[act](d[3]))
    rx = 1 / torch.sqrt((d[0] * d[0]).mean(-1, keepdim=True) + 1e-6)
    terms = rx * (e.abs() + (d[0] * rx * (e * d[0] * rx).mean(-1, keepdim=True)).abs())
    for n, a, b, t in zip(names, got, want, leaves):
        assert a.shape == t.shape and a.dtype == dtype
        bound = (1.5 * u if dtype != F32 else 40 * E) * float(b.norm()) + (40 * E * float(terms.norm()) + TINY[dtype] * b.numel() ** 0.5 if n == "dx" else 0)
        assert float((a.double() - b).norm()) <= bound, (n, rel(a, b))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("lead, c", [((1,), 64), ((3, 5), 64), ((7, 33), 96), ((2, 50), 771), ((300,), 256), ((2, 9), 1024), ((4, 3), 1536), ((5,), 2050),
                                     ((3,), 4096), ((2, 3), 33), ((3,), 1), ((2, 5), 20001), ((2, 2), 20480), ((2000, 2), 40)])
def test_sandwich_sizes(lead, c, dtype):
    check_sandwich(lead, c, lead, "silu", True, dtype, seed=c)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("act", ["none", "sigmoid", "silu", "tanh"])
@pytest.mark.parametrize("nxt", [False, True])
@pytest.mark.parametrize("lead, gate", [((4, 70), None), ((4, 70), (4, 70)), ((4, 70), (4, 1)), ((4, 70), ()), ((4, 70), (1, 1)), ((3, 2, 40), (3, 1, 1)), ((3, 2, 40), (3, 2, 1)),
                                        ((600, 3), (600, 1)), ((2, 4000), (2, 1))])
@pytest.mark.parametrize("c", [128, 77])
def test_sandwich_gates(lead, gate, c, nxt, act, dtype):
    check_sandwich(lead, c, gate, act, nxt, dtype)


@pytest.mark.parametrize("c", [1024, 20001])
@pytest.mark.parametrize("gate", [(3, 1), (), (3, 30)])
def test_sandwich_wide_shared_gates(c, gate):
    check_sandwich((3, 30), c, gate, "silu", True, BF16)


def test_sandwich_gradients_of_some():
    """Each gradient alone, and one output's gradient alone, are those of the whole call."""
    g, lead, c = gen(1), (3, 20), 128
    x = [rand(g, *lead, c, dtype=BF16), rand(g, c, dtype=BF16), rand(g, *lead, c, dtype=BF16), rand(g, 3, 1, c, dtype=BF16), rand(g, c, dtype=BF16)]
    ds, dy = rand(g, *lead, c, dtype=BF16), rand(g, *lead, c, dtype=BF16)

    def grads(flags, outs=(True, True)):
        z = [t.detach().requires_grad_(f) for t, f in zip(x, flags)]
        y, s = ops.sandwich_norm(z[0], z[1], z[2], z[3], z[4], "silu", 0.5)
        return torch.autograd.grad([o for o, f in zip((s, y), outs) if f], [t for t, f in zip(z, flags) if f],
                                   [d for d, f in zip((ds, dy), outs) if f], allow_unused=True)

    every = grads([True] * 5)
    for i in range(5):
        assert torch.equal(grads([j == i for j in range(5)])[0], every[i])
    for outs, zero in (((True, False), dy), ((False, True), ds)):
        keep = zero.clone()
        zero.zero_()
        want = grads([True] * 5)
        zero.copy_(keep)
        for a, b in zip(grads([True] * 5, outs), want):
            assert a is None and not b.any() or torch.equal(a, b)


@pytest.mark.parametrize("dtype", [F32, F16])
def test_sandwich_strides_streams_and_graph(dtype):
    g, lead, c = gen(2), (4, 30), 96
    wide = rand(g, *lead, 2 * c, dtype=dtype)
    x, gate, r, w, wn = wide[..., :c], wide[..., c:], rand(g, *lead, c, dtype=dtype), rand(g, c, dtype=dtype), rand(g, c, dtype=dtype)
    want = ops.sandwich_norm(x.contiguous(), w, r, gate.contiguous(), wn, "sigmoid")
    odd = lambda t: torch.nn.functional.pad(t, (1, 0))[..., 1:]  # noqa: E731
    for args in ((x, w, r, gate, wn), (odd(x), odd(w), odd(r), odd(gate), odd(wn)), (x, w, r.mT.contiguous().mT, gate, wn)):
        for a, b in zip(ops.sandwich_norm(*args, "sigmoid"), want):
            assert rel(a, b.double()) <= U[dtype]  # (scalar accesses: another order of the sums)
    with torch.cuda.stream(torch.cuda.Stream()):
        other = ops.sandwich_norm(x, w, r, gate, wn, "sigmoid")
        torch.cuda.current_stream().synchronize()
    assert all(torch.equal(a, b) for a, b in zip(other, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.sandwich_norm(x, w, r, gate, wn, "sigmoid")
    wide.copy_(rand(g, *lead, 2 * c, dtype=dtype))
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(out, ops.sandwich_norm(x, w, r, gate, wn, "sigmoid")))


def test_sandwich_empty_and_values():
    z = lambda *s: torch.zeros(*s, device="cuda")  # noqa: E731
    y, s = ops.sandwich_norm(z(0, 8), z(8), z(0, 8), None, z(8))
    assert y.shape == s.shape == (0, 8)
    w = torch.ones(8, device="cuda").requires_grad_()
    gate = torch.ones(8, device="cuda").requires_grad_()
    s = ops.sandwich_norm(z(0, 8), w, z(0, 8), gate)
    dw, dg = torch.autograd.grad(s, (w, gate), z(0, 8))
    assert not dw.any() and not dg.any()
    # a row of zeros is finite; a NaN stays in its row; infinite gates follow the formula
    x, r = torch.randn(3, 8, device="cuda"), torch.randn(3, 8, device="cuda")
    x[0], x[1, 3] = 0, float("nan")
    y, s = ops.sandwich_norm(x, w.detach(), r, None, w.detach())
    assert torch.equal(s[0], r[0]) and torch.isfinite(y[[0, 2]]).all() and torch.isnan(s[1]).all()
    big = torch.tensor([-float("inf"), -1e4, -100.0, 0.0, 100.0, 1e4, float("inf"), 1.0], device="cuda")
    for act in ("sigmoid", "tanh"):
        assert torch.isfinite(ops.sandwich_norm(x[2:], w.detach(), r[2:], big, None, act)).all()
