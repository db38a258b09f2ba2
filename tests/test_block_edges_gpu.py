"""Edges of the block operators on a GPU: the activations' tails, rows and sums that are empty, tiny or huge, strided
operands, gradients of some inputs only, graphs, refusals, and the extension's and the C ABI's own entry points."""
import ctypes
import math

import pytest
import torch
import test_block_gpu as base
from test_block_gpu import DT16, E, TINY, U, act64, gen, rand, slope64, slope_err, within

from laplacianformer_b200 import capi, ops

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ activations


def act_parts(z, name):
    """The gate p with act(z) = z p, the two terms of act'(z) = p + z p', and the relative error that p may have in 32
    bits: 8 E for the exponential, the reciprocal and the additions (16 E with a polynomial of seven terms), and what the
    rounding of the exponential's argument adds (1.5 units in 2^-24 of it for the sigmoid, 2.5 for z^2 / 2, 6 for the
    cubic).  z p' is formed of rounded 1 - p, so its error counts from its size without that factor."""
    if name == "silu":
        p, q = torch.sigmoid(z), torch.sigmoid(-z)
        return p, z * p * q, (z * p).abs(), (8 + z.abs()) * E
    if name == "gelu_tanh":
        k = 2 * math.sqrt(2 / math.pi)
        a, da = k * (z + 0.044715 * z**3), k * (1 + 3 * 0.044715 * z * z)
        p, q = torch.sigmoid(a), torch.sigmoid(-a)
        return p, z * p * q * da, (z * p).abs() * da, (8 + 3 * a.abs()) * E
    t = z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    return 0.5 * torch.erfc(-z / math.sqrt(2)), t, t.abs(), (16 + z * z) * E


@pytest.mark.parametrize("dtype", DT16)
@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_activation_tails(dtype, act):
    """Values and slopes keep their leading digits where they are small: z itself through an identity weight."""
    n = 64
    z = torch.linspace(-8 if act == "gelu_tanh" else -12, 12, 700 * n, dtype=torch.float64).to(dtype).cuda().reshape(-1, n)
    x, eye = z.clone().requires_grad_(), torch.eye(n, dtype=dtype, device="cuda")
    y = ops.linear(x, eye, activation=act)
    (dx,) = torch.autograd.grad(y, x, torch.ones_like(y))  # the slope, rounded once as the product's operand
    z = z.double()
    p, zdp, steep, rel = act_parts(z, act)
    u, tiny = U[dtype], TINY[dtype]
    within(y.detach(), z * p, u * (z * p).abs() + 1.01 * rel * (z * p).abs() + tiny, "value")
    s = p + zdp
    within(dx, s, u * s.abs() + 1.01 * (2 * rel + 4 * E) * (p + steep) + tiny, "slope")


# ------------------------------------------------------------------ rows without values, tiny rows


def poison(n):
    """Leaves NaN where the caching allocator takes the next small tensors from."""
    torch.cuda.synchronize()
    keep = [torch.full((n,), float("nan"), device="cuda") for _ in range(8)]
    torch.cuda.synchronize()
    del keep


@pytest.mark.parametrize("dtype", list(U))
def test_scales_of_empty_rows(dtype):
    """A row without values is a row of zeros: its scale is 1."""
    z = lambda *s: torch.zeros(*s, device="cuda", dtype=dtype)  # noqa: E731
    for call in (lambda: ops.quantize_rows(z(5, 0)), lambda: ops.rms_norm_quant(z(5, 0), z(0)),
                 lambda: ops.rms_norm_quant(z(5, 0), z(0), residual=z(5, 0))):
        poison(5)
        q, scale = call()[:2]
        assert q.shape == (5, 0) and torch.equal(scale, torch.ones(5, device="cuda"))
    assert ops.quantize_rows(z(0, 8))[1].shape == (0,)


@pytest.mark.parametrize("dtype", DT16)
@pytest.mark.parametrize("m", [1, 5, 200])
def test_linear_quant_of_empty_sums(dtype, m):
    b, r = rand(gen("k0 quant"), dtype, 24), rand(gen("r0 quant", m), dtype, m, 24)
    poison(m)
    q, sx = ops.quantize_rows(torch.zeros(m, 0, device="cuda"))
    poison(24)
    wq, sw = ops.quantize_rows(torch.zeros(24, 0, device="cuda"))
    y = ops.linear_quant(q, sx, wq, sw, b, residual=r, dtype=dtype)
    within(y, b.double() + r.double(), (U[dtype] + E) * (b.double().abs() + r.double().abs()), "k = 0")


@pytest.mark.parametrize("cols", [5, 64, 771, 20000])
def test_scale_of_tiny_rows(cols):
    """fp32 rows whose largest value divided by 448 is zero: scale 1 and zeros, as a row of zeros has."""
    x = torch.zeros(4, cols, device="cuda")
    x[0, 1], x[1, :], x[2, 3], x[3, 0] = 1.4e-45, 2.0e-43, -1e-42, 1.0
    q, scale = ops.quantize_rows(x)
    assert torch.equal(scale[:2], torch.ones(2, device="cuda")) and (q[:2].float() == 0).all()
    assert (scale > 0).all() and q.float().isfinite().all()
    w = torch.full((cols,), 1e-44, device="cuda")
    q, scale = ops.rms_norm_quant(torch.ones(2, cols, device="cuda"), w)
    assert torch.equal(scale, torch.ones(2, device="cuda")) and (q.float() == 0).all()


# ------------------------------------------------------------------ clipping


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("where", [0, 3, 70000, 200000])
def test_clip_grad_norm_of_huge_values(dtype, where):
    """Squares that pass the largest fp32 number: the norm is finite, so gradients are scaled and not erased."""
    g = gen("huge", dtype, where)
    flat = rand(g, dtype, 200001, scale=1e20)
    flat[where] = 1e25
    grads = list(flat.split([1001, 100000, 99000]))
    n64 = float(flat.double().norm())
    norm, out = ops.clip_grad_norm(grads, 2.0)
    assert abs(float(norm) - n64) <= 300 * E * n64
    ref = flat.double() * (2.0 / (n64 + 1e-6))
    within(torch.cat(out), ref, (U[dtype] + 310 * E) * ref.abs() + TINY[dtype], "clipped")


def test_clip_grad_norm_of_shared_memory():
    """Gradients that are only read may be the same one or overlap; written ones may not."""
    g = rand(gen("shared"), torch.float32, 1000)
    for grads in ([g, g], [g, g[100:300]]):
        n64 = math.sqrt(sum(float(t.double().square().sum()) for t in grads))
        norm, out = ops.clip_grad_norm(grads, 0.5)
        assert abs(float(norm) - n64) <= 300 * E * n64
        for a, b in zip(grads, out):
            ref = a.double() * (0.5 / (n64 + 1e-6))
            within(b, ref, (U[torch.float32] + 310 * E) * ref.abs() + TINY[torch.float32], "shared")
        before = g.clone()
        with pytest.raises(RuntimeError, match="overlap"):
            ops.clip_grad_norm(grads, 0.5, out=grads)
        assert torch.equal(g, before)


def test_clip_grad_norm_counts_as_a_write():
    """Written tensors get a new version, so that autograd refuses to use what it saved before."""
    a, b = (torch.ones(40, device="cuda") for _ in range(2))
    x = torch.ones(40, device="cuda", requires_grad=True)
    y = (x * a).sum()
    va, vb = a._version, b._version
    ops.clip_grad_norm([a], 0.5, out=[b])
    assert a._version == va and b._version > vb
    ops.clip_grad_norm([a], 0.5, out=[a])
    assert a._version > va
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with torch.inference_mode():
        c = torch.full((4,), 2.0, device="cuda")
        assert abs(float(ops.clip_grad_norm([c], 1.0, out=[c])[0]) - 4) < 1e-5 and abs(float(c[0]) - 0.5) < 1e-5


# ------------------------------------------------------------------ other kinds of differentiation


def forms(dtype=torch.bfloat16):
    """Each differentiable operator as a function of x."""
    g = gen("forms", dtype)
    w, wi, wo = rand(g, dtype, 24, 32, scale=0.2), rand(g, dtype, 80, 32, scale=0.2), rand(g, dtype, 32, 40, scale=0.2)
    wn, r = rand(g, dtype, 32), rand(g, dtype, 12, 32)
    return {"rms_norm": lambda x: ops.rms_norm(x, wn), "rms_norm residual": lambda x: ops.rms_norm(r, wn, residual=x)[0],
            "rms_norm weight": lambda x: ops.rms_norm(r, x[0]), "linear": lambda x: ops.linear(x, w),
            "linear weight": lambda x: ops.linear(r, x, activation="gelu"), "linear residual": lambda x: ops.linear(r, wi[:32], residual=x),
            "gated_feed_forward": lambda x: ops.gated_feed_forward(x, wi, wo),
            "gated_feed_forward residual": lambda x: ops.gated_feed_forward(r, wi, wo, residual=x)}


@pytest.mark.parametrize("form", ["rms_norm", "rms_norm residual", "rms_norm weight", "linear", "linear weight", "linear residual",
                                  "gated_feed_forward", "gated_feed_forward residual"])
def test_forward_mode_is_refused(form):
    """There is no forward-mode derivative, and a tangent is not dropped in silence."""
    from torch.autograd import forward_ad

    f = forms()[form]
    x, t = (rand(gen("dual", k), torch.bfloat16, 12, 32) for k in "xt")
    for tracked in (False, True):
        with forward_ad.dual_level():
            dual = forward_ad.make_dual(x.clone().requires_grad_(tracked), t)
            with pytest.raises(RuntimeError, match="forward"):
                f(dual)
        f(x)
