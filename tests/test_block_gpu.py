"""The block operators on a GPU against their definitions in 64 bits.

Bounds are worst-case bounds, element by element: u is the unit roundoff of the
storage type (one rounding per output, and one per value that a later product
takes as an operand), E = 2^-23 covers one fp32 operation with room for the
tensor core's accumulation and the fast exponential, and a sum of n terms may
be off by (n + 16) E times the sum of the terms' sizes.
"""
import math
import zlib

import pytest
import torch

from laplacianformer_b200 import capi, ops

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
TINY = {torch.float32: 2.0**-140, torch.float16: 2.0**-25, torch.bfloat16: 2.0**-130}
E = 2.0**-23
DT16 = [torch.float16, torch.bfloat16]
ACTS = ["none", "relu", "gelu", "gelu_tanh", "silu"]


def rand(g, dtype, *shape, scale=1.0):
    return (torch.randn(*shape, generator=g, dtype=torch.float64) * scale).to(dtype).cuda()


def gen(*key):
    return torch.Generator().manual_seed(zlib.crc32("/".join(map(str, key)).encode()))


def within(got, ref, bound, what):
    assert got.shape == ref.shape, what
    err = (got.double() - ref).abs()
    bad = ~(err <= bound)
    assert not bool(bad.any()), (what, int(bad.sum()), float((err / bound)[bad].max()) if bad.any() else 0)


def act64(z, name):
    return {"none": lambda t: t, "relu": torch.relu, "silu": lambda t: t * torch.sigmoid(t),
            "gelu": lambda t: 0.5 * t * (1 + torch.erf(t / math.sqrt(2))),
            "gelu_tanh": lambda t: 0.5 * t * (1 + torch.tanh(math.sqrt(2 / math.pi) * (t + 0.044715 * t**3)))}[name](z)


def slope64(z, name):
    with torch.enable_grad():
        t = z.detach().requires_grad_()
        return torch.autograd.grad(act64(t, name).sum(), t)[0]


def slope_err(z, ez, name):
    """How far act'(z) may be off for |z - z_true| <= ez: |act''| <= 1.2 for the smooth ones, a jump of relu at 0."""
    if name == "none":
        return torch.zeros_like(z)
    if name == "relu":
        return (z.abs() <= ez).double()
    return 1.2 * ez + 32 * E


# ------------------------------------------------------------------ norm


def norm64(x, w, r, eps):
    s = x.double() + (r.double() if r is not None else 0)
    return s / torch.sqrt((s * s).mean(-1, keepdim=True) + eps) * w.double(), s


@pytest.mark.parametrize("dtype", list(U))
@pytest.mark.parametrize("shape", [(1, 1), (3, 7), (1, 64), (37, 64), (5, 200), (300, 256), (33, 512), (64, 771), (19, 1024), (7, 1031),
                                   (9, 2048), (700, 768), (5, 1400), (6, 1536), (400, 1288), (5, 3008), (5, 4104), (3, 8192), (2, 5000), (2, 20000), (2, 16390)])
@pytest.mark.parametrize("residual", [False, True])
def test_rms_norm_forward_backward(dtype, shape, residual):
    g = gen("norm", dtype, shape, residual)
    m, c = shape
    x, w = rand(g, dtype, m, c).requires_grad_(), (1 + 0.1 * rand(g, torch.float64, c)).to(dtype).requires_grad_()
    r = rand(g, dtype, m, c).requires_grad_() if residual else None
    dy, ds = rand(g, dtype, m, c), rand(g, dtype, m, c)
    u, tiny = U[dtype], TINY[dtype]
    y64, s64 = norm64(x, w, r, 1e-6)
    out = ops.rms_norm(x, w, residual=r)
    y, s = out if residual else (out, None)
    within(y, y64, u * y64.abs() + (c + 16) * E * y64.abs() + tiny, "y")
    if residual:
        within(s, s64, u * s64.abs() + E * s64.abs() + tiny, "s")
    # gradients from their formula
    rstd = 1 / torch.sqrt((s64 * s64).mean(-1, keepdim=True) + 1e-6)
    xh, a = s64 * rstd, dy.double() * w.double()
    mean = (a * xh).mean(-1, keepdim=True)
    dx64 = rstd * (a - xh * mean) + (ds.double() if residual else 0)
    dw64 = (dy.double() * xh).sum(0)
    ins = (x, w) + ((r,) if residual else ())
    got = torch.autograd.grad((y, s) if residual else y, ins, (dy, ds) if residual else dy)
    k = (u + (c + 16) * E) * (1 if residual else 0) + (c + 16) * E  # the stored sum is rounded, x itself is not
    small = rstd * (k * xh.abs() * mean.abs() + xh.abs() * (k * (a * xh).abs().mean(-1, keepdim=True)) + (c + 16) * E * a.abs())
    within(got[0], dx64, u * dx64.abs() + small + (ds.double().abs() * E if residual else 0) + tiny, "dx")
    within(got[1], dw64, u * dw64.abs() + (k + (m + c + 16) * E) * (dy.double() * xh).abs().sum(0) + tiny, "dw")
    if residual:
        assert torch.equal(got[2], got[0])


def test_rms_norm_gradient_against_differences():
    g = gen("norm differences")
    x, w, r = (rand(g, torch.float32, *s) for s in ((6, 40), (40,), (6, 40)))
    dy, ds = rand(g, torch.float32, 6, 40), rand(g, torch.float32, 6, 40)

    def loss(x, w, r):
        y, s = ops.rms_norm(x, w, residual=r)
        return float((y.double() * dy.double()).sum() + (s.double() * ds.double()).sum())

    leaves = [t.clone().requires_grad_() for t in (x, w, r)]
    y, s = ops.rms_norm(*leaves[:2], residual=leaves[2])
    grads = torch.autograd.grad((y, s), leaves, (dy, ds))
    h = 2.0**-6
    for i, gr in enumerate(grads):
        d = rand(g, torch.float32, *gr.shape).sign()
        plus, minus = [[t + k * h * d if j == i else t for j, t in enumerate((x, w, r))] for k in (1, -1)]
        got = (loss(*plus) - loss(*minus)) / (2 * h)
        want = float((gr.double() * d.double()).sum())
        # rounding of 240 outputs of size ~1 over 2h, and the third-order term h^2 times a few times the sum of the terms
        assert abs(got - want) <= 240 * 40 * E / h + 4 * h * h * float((gr.abs()).sum() + 40)


@pytest.mark.parametrize("dtype", list(U))
@pytest.mark.parametrize("shape", [(1, 1), (5, 12), (196, 512), (33, 771), (4, 4096), (3, 5001), (2, 20000)])
@pytest.mark.parametrize("residual", [False, True])
def test_rms_norm_quant(dtype, shape, residual):
    g = gen("quant", dtype, shape, residual)
    m, c = shape
    x, w = rand(g, dtype, m, c), (1 + 0.1 * rand(g, torch.float64, c)).to(dtype)
    r = rand(g, dtype, m, c) if residual else None
    y64, s64 = norm64(x, w, r, 1e-6)
    out = ops.rms_norm_quant(x, w, residual=r)
    q, scale = out[:2]
    assert q.dtype == torch.float8_e4m3fn and scale.dtype == torch.float32 and scale.shape == (m,)
    sc64 = y64.abs().amax(-1) / 448
    within(scale, sc64, (c + 16) * E * sc64, "scale")
    v = y64 / sc64[:, None]
    within(q.float(), v, (2.0**-4 + (c + 16) * E) * v.abs() + 2.0**-10, "q")
    if residual:
        within(out[2], s64, (U[dtype] + E) * s64.abs() + TINY[dtype], "s")
    q2, sc2 = ops.quantize_rows(x)
    mx = x.double().abs().amax(-1)
    within(sc2, mx / 448, E * mx, "row scale")
    v = x.double() / (mx / 448)[:, None]
    within(q2.float(), v, (2.0**-4 + 4 * E) * v.abs() + 2.0**-10, "row q")


def test_norm_special_rows():
    """A row of zeros, one with an infinity, one with a NaN beside ordinary ones: each keeps to itself."""
    x = torch.ones(5, 96, device="cuda", dtype=torch.bfloat16)
    x[1] = 0
    x[2, 3] = float("inf")
    x[3, 5] = float("nan")
    w = torch.ones(96, device="cuda", dtype=torch.bfloat16)
    y = ops.rms_norm(x, w)
    assert torch.equal(y[0], torch.ones_like(y[0])) and torch.equal(y[4], y[0]) and torch.equal(y[1], torch.zeros_like(y[1]))
    assert y[2, 3].isnan() and (y[2, :3] == 0).all() and y[3].isnan().all()
    q, scale = ops.rms_norm_quant(x, w)
    assert float(scale[1]) == 1 and (q[1].float() == 0).all() and (q[0].float() == 448).all()
    assert scale[2].isnan() and scale[3].isnan() and q[3].float().isnan().all()


def test_norm_offsets_beyond_31_bits():
    m, c = (1 << 21) + 3, 1024
    x = torch.zeros(m, c, device="cuda", dtype=torch.bfloat16)
    x[-2:] = rand(gen("far"), torch.bfloat16, 2, c)
    w = torch.ones(c, device="cuda", dtype=torch.bfloat16)
    y = ops.rms_norm(x, w)
    y64, _ = norm64(x[-2:], w, None, 1e-6)
    within(y[-2:], y64, (2.0**-8 + (c + 16) * E) * y64.abs() + 1e-30, "last rows")
    assert not bool(y[: m - 2].any())


# ------------------------------------------------------------------ linear


def linear64(x, w, b, act, r):
    z = x.double() @ w.double().T + (b.double() if b is not None else 0)
    mag = x.double().abs() @ w.double().abs().T + (b.double().abs() if b is not None else 0)
    return z, mag, act64(z, act) + (r.double() if r is not None else 0)


def check_linear(x, w, b, act, r, y):
    u, tiny = U[x.dtype], TINY[x.dtype]
    z, mag, y64 = linear64(x, w, b, act, r)
    ez = (x.shape[-1] + 16) * E * mag
    within(y, y64, u * y64.abs() + 1.2 * ez + 64 * E * (z.abs() + 1) + tiny, "y")
    return z, ez


LINEAR_SHAPES = [(1, 1, 1), (1, 96, 64), (2, 130, 1031), (3, 7, 8), (5, 1000, 512), (8, 4096, 1024), (9, 65, 63), (64, 64, 64),
                 (127, 129, 191), (128, 256, 128), (129, 257, 136), (200, 96, 40), (300, 1027, 515), (1000, 768, 512),
                 (2500, 24, 16), (130, 512, 4100)]


@pytest.mark.parametrize("dtype", DT16)
@pytest.mark.parametrize("shape", LINEAR_SHAPES)
@pytest.mark.parametrize("kind", ["plain", "bias gelu", "bias relu residual", "silu residual", "bias gelu_tanh"])
def test_linear_forward_backward(dtype, shape, kind):
    m, n, k = shape
    act = next((a for a in ACTS[1:][::-1] if a in kind.split()), "none")
    g = gen("linear", dtype, shape, kind)
    x, w = rand(g, dtype, m, k).requires_grad_(), rand(g, dtype, n, k, scale=k**-0.5).requires_grad_()
    b = rand(g, dtype, n).requires_grad_() if "bias" in kind else None
    r = rand(g, dtype, m, n).requires_grad_() if "residual" in kind else None
    y = ops.linear(x, w, b, activation=act, residual=r)
    with torch.no_grad():
        assert torch.equal(ops.linear(x, w, b, activation=act, residual=r), y)
    z, ez = check_linear(x.detach(), w.detach(), None if b is None else b.detach(), act, None if r is None else r.detach(), y.detach())
    dy = rand(g, dtype, m, n)
    ins = [t for t in (x, w, b, r) if t is not None]
    got = dict(zip(["x", "w"] + (["b"] if b is not None else []) + (["r"] if r is not None else []),
                   torch.autograd.grad(y, ins, dy)))
    u, tiny = U[dtype], TINY[dtype]
    dz = dy.double() * slope64(z, act)
    edz = (0 if act == "none" else u) * dz.abs() + dy.double().abs() * slope_err(z, ez, act) + tiny
    xd, wd = x.detach().double(), w.detach().double()
    for name, a, bm, ea in (("x", dz, wd, edz), ("w", dz.T, xd, edz.T)):
        ref = a @ bm
        bound = u * ref.abs() + ea @ bm.abs() * 1.01 + (a.shape[1] + 16) * E * (a.abs() @ bm.abs()) + tiny
        within(got[name], ref, bound, "d" + name)
    if b is not None:
        ref = dz.sum(0)
        within(got["b"], ref, u * ref.abs() + edz.sum(0) * 1.01 + (m + 16) * E * dz.abs().sum(0) + tiny, "db")
    if r is not None:
        assert torch.equal(got["r"], dy)


@pytest.mark.parametrize("op", ["linear", "ffn"])
def test_product_gradients_against_differences(op):
    """The operators' own forward passes, differenced along a direction, against their gradients.  The inputs are
    multiples of 1/16 and the step is 1/4, so stepped inputs are exact; what is left is the outputs' rounding (bounded
    element by element) and the curvature (taken from the same differences in 64 bits)."""
    g = gen("differences", op)
    dtype, h = torch.float16, 0.25
    m, c, f = 40, 48, 56
    q = lambda t: (t * 16).round() / 16  # noqa: E731
    x = q(rand(g, torch.float64, m, c))
    win, wout = q(rand(g, torch.float64, 2 * f, c, scale=0.3)), q(rand(g, torch.float64, c, f, scale=0.3))
    dy = q(rand(g, torch.float64, m, c if op == "ffn" else 2 * f))
    if op == "linear":
        run = lambda x: ops.linear(x, win.to(dtype), activation="silu")  # noqa: E731
        ref = lambda x: act64(x @ win.T, "silu")  # noqa: E731
    else:
        run = lambda x: ops.gated_feed_forward(x, win.to(dtype), wout.to(dtype), activation="silu")  # noqa: E731
        ref = lambda x: (act64(x @ win[:f].T, "silu") * (x @ win[f:].T)) @ wout.T  # noqa: E731
    leaf = x.to(dtype).requires_grad_()
    grad = torch.autograd.grad(run(leaf), leaf, dy.to(dtype))[0].double()
    d = rand(g, torch.float64, m, c).sign()
    own = [(run((x + s * h * d).to(dtype)).double() * dy).sum() for s in (1, -1)]
    r64 = [ref(x + s * h * d) for s in (1, -1)]
    fd64 = float(((r64[0] - r64[1]) * dy).sum() / (2 * h))
    xl = x.clone().requires_grad_()
    slope = float((torch.autograd.grad((ref(xl) * dy).sum(), xl)[0] * d).sum())
    u = U[dtype]
    if op == "linear":
        room = sum(float(((u * t.abs() + 64 * E * (t.abs() + 1)) * dy.abs()).sum()) for t in r64) / (2 * h)
    else:
        hs = [(act64(t @ win[:f].T, "silu") * (t @ win[f:].T)).abs() @ wout.abs().T for t in (x + h * d, x - h * d)]
        room = sum(float(((u * t.abs() + (u + 200 * E) * k) * dy.abs()).sum()) for t, k in zip(r64, hs)) / (2 * h)
    assert abs(float(own[0] - own[1]) / (2 * h) - fd64) <= room
    assert abs(float((grad * d).sum()) - slope) <= 4 * u * float(grad.abs().sum())
    # and the 64-bit slope against a small step
    e = 2.0**-20
    fine = float(((ref(x + e * d) - ref(x - e * d)) * dy).sum() / (2 * e))
    assert abs(fine - slope) <= 1e-6 * (abs(slope) + 1)


@pytest.mark.parametrize("dtype", DT16)
@pytest.mark.parametrize("m", [1, 6, 50, 300])
def test_linear_strided_and_unaligned(dtype, m):
    """Slices of a joint projection, a transposed batch, an offset base: what callers hold, without copies or with."""
    g = gen("strides", dtype, m)
    joint = rand(g, dtype, m, 3 * 64)
    w = rand(g, dtype, 72, 64, scale=0.125)
    for x in (joint[:, 64:128], joint[:, 1:65], joint[:, 7:71]):
        check_linear(x, w, None, "none", None, ops.linear(x, w))
    wide = rand(g, dtype, 72, 80, scale=0.125)
    check_linear(joint[:, :64], wide[:, 8:72], None, "gelu", None, ops.linear(joint[:, :64], wide[:, 8:72], activation="gelu"))
    check_linear(joint[:, :64], wide[:, 3:67], None, "none", None, ops.linear(joint[:, :64], wide[:, 3:67]))
    x = rand(g, dtype, 4, m, 64).transpose(0, 1)
    y = ops.linear(x, w)
    assert y.shape == (m, 4, 72)
    check_linear(x.reshape(-1, 64), w, None, "none", None, y.reshape(-1, 72))
    r = rand(g, dtype, m, 144)[:, 72:]
    check_linear(joint[:, :64], w, None, "relu", r, ops.linear(joint[:, :64], w, activation="relu", residual=r))
    xg = joint[:, 64:128].detach().requires_grad_()
    dy = rand(g, dtype, m, 73)[:, 1:]
    (dx,) = torch.autograd.grad(ops.linear(xg, w), xg, dy)
    ref = dy.double() @ w.double()
    within(dx, ref, U[dtype] * ref.abs() + 100 * E * (dy.double().abs() @ w.double().abs()) + TINY[dtype], "dx of strided dy")


@pytest.mark.parametrize("dtype", DT16)
def test_expanded_operands(dtype):
    """Broadcast inputs and gradients have strides of zero: every operand expanded equals its dense copy."""
    g = gen("expanded", dtype)
    m, k, n, f = 40, 64, 48, 72
    x, w, b, r, dy = rand(g, dtype, 1, k).expand(m, k), rand(g, dtype, n, k, scale=0.1), rand(g, dtype, 1).expand(n), \
        rand(g, dtype, 1, n).expand(m, n), rand(g, dtype, 1, n).expand(m, n)
    wi, wo, dz = rand(g, dtype, 2 * f, k, scale=0.1), rand(g, dtype, k, f, scale=0.1), rand(g, dtype, m, 1).expand(m, k)
    wn, dr = rand(g, dtype, 1).expand(k), rand(g, dtype, 1, k).expand(m, k)

    def run(*t):
        x, w, b, r, dy, wi, wo, dz, wn, dr = t
        leaf = x.detach().requires_grad_()
        y = ops.linear(leaf, w, b, activation="silu", residual=r)
        h = ops.gated_feed_forward(leaf, wi, wo, residual=dz)
        q, s = ops.rms_norm(leaf, wn, residual=dr)
        return (y, h, q, s, *(torch.autograd.grad(o, leaf, d)[0] for o, d in ((y, dy), (h, dz), (q, dr))), *ops.rms_norm_quant(x, wn)[:1])

    expanded = (x, w, b, r, dy, wi, wo, dz, wn, dr)
    for a, c in zip(run(*expanded), run(*(t.contiguous() for t in expanded))):
        assert torch.equal(a.float(), c.float())
    assert torch.equal(ops.linear(x.view(1, m, k).expand(3, m, k), w), ops.linear(x.contiguous(), w).expand(3, m, n))


@pytest.mark.parametrize("dtype", DT16)
@pytest.mark.parametrize("shape", [(1, 64, 64), (1, 1000, 512), (7, 33, 96), (128, 256, 128), (200, 96, 144), (300, 515, 1040),
                                   (65, 40, 131), (1000, 1536, 512)])
@pytest.mark.parametrize("kind", ["plain", "bias silu residual"])
def test_linear_quant(dtype, shape, kind):
    m, n, k = shape
    g = gen("linear quant", dtype, shape, kind)
    q, sx = ops.quantize_rows(rand(g, torch.float32, m, k))
    wq, sw = ops.quantize_rows(rand(g, torch.float32, n, k, scale=k**-0.5))
    b = rand(g, dtype, n) if "bias" in kind else None
    r = rand(g, dtype, m, n) if "residual" in kind else None
    act = "silu" if "silu" in kind else "none"
    y = ops.linear_quant(q, sx, wq, sw, b, activation=act, residual=r, dtype=dtype)
    x64, w64 = q.double() * sx.double()[:, None], wq.double() * sw.double()[:, None]
    z, mag, y64 = linear64(x64, w64, b, act, r)
    within(y, y64, U[dtype] * y64.abs() + 1.2 * (k + 16) * E * mag + 64 * E * (z.abs() + 1) + TINY[dtype], "y")


def test_linear_offsets_beyond_31_bits():
    m, n, k = (1 << 20) + 5, 2056, 64
    x = torch.zeros(m, k, device="cuda", dtype=torch.bfloat16)
    g = gen("far product")
    x[-3:] = rand(g, torch.bfloat16, 3, k)
    w = rand(g, torch.bfloat16, n, k, scale=0.125)
    y = ops.linear(x, w)
    check_linear(x[-3:], w, None, "none", None, y[-3:])
    assert not bool(y[(1 << 20) - 2: -3].any())


# ------------------------------------------------------------------ gated feed-forward block

FFN_SHAPES = [(1, 8, 8), (1, 64, 171), (3, 33, 65), (8, 512, 1365), (9, 64, 256), (130, 40, 72), (128, 64, 128), (197, 96, 200),
              (300, 130, 257), (1000, 64, 256), (257, 512, 1365), (20, 1031, 50),
              (18945, 64, 200), (19000, 128, 136), (38001, 40, 65), (19500, 100, 64), (56900, 24, 17)]


@pytest.mark.parametrize("dtype", DT16)
@pytest.mark.parametrize("shape", FFN_SHAPES)
@pytest.mark.parametrize("kind", ["silu", "gelu bias residual", "relu residual", "gelu_tanh bias", "none"])
def test_gated_feed_forward(dtype, shape, kind):
    m, c, f = shape
    act = kind.split()[0]
    g = gen("ffn", dtype, shape, kind)
    x = rand(g, dtype, m, c).requires_grad_()
    win, wout = rand(g, dtype, 2 * f, c, scale=c**-0.5).requires_grad_(), rand(g, dtype, c, f, scale=f**-0.5).requires_grad_()
    bin_ = rand(g, dtype, 2 * f, scale=0.5).requires_grad_() if "bias" in kind else None
    bout = rand(g, dtype, c, scale=0.5).requires_grad_() if "bias" in kind else None
    r = rand(g, dtype, m, c).requires_grad_() if "residual" in kind else None
    y = ops.gated_feed_forward(x, win, wout, bin_, bout, activation=act, residual=r)
    with torch.no_grad():
        assert torch.equal(ops.gated_feed_forward(x, win, wout, bin_, bout, activation=act, residual=r), y)
    u, tiny = U[dtype], TINY[dtype]
    d = lambda t: None if t is None else t.detach().double()  # noqa: E731
    X, Wi, Wo = d(x), d(win), d(wout)
    z, mag, _ = linear64(X, Wi, d(bin_), "none", None)
    ez = (c + 16) * E * mag
    G, Up, eg, eu = z[:, :f], z[:, f:], ez[:, :f], ez[:, f:]
    a, sl = act64(G, act), slope64(G, act)
    ea = 1.2 * eg + 64 * E * (G.abs() + 1) * (0 if act in ("none", "relu") else 1)
    h = a * Up
    eh = u * h.abs() + 1.01 * (ea * Up.abs() + a.abs() * eu) + E * h.abs() + tiny
    y64 = h @ Wo.T + (d(bout) if bout is not None else 0) + (d(r) if r is not None else 0)
    fwd = h.abs() @ Wo.abs().T + (d(bout).abs() if bout is not None else 0)
    within(y.detach(), y64, u * y64.abs() + 1.01 * eh @ Wo.abs().T + (f + 16) * E * fwd + tiny, "y")
    dy = rand(g, dtype, m, c)
    names = [k for k, t in (("x", x), ("win", win), ("wout", wout), ("bin", bin_), ("bout", bout), ("r", r)) if t is not None]
    got = dict(zip(names, torch.autograd.grad(y, [t for t in (x, win, wout, bin_, bout, r) if t is not None], dy)))
    D = dy.double()
    dh = D @ Wo
    edh = (c + 16) * E * (D.abs() @ Wo.abs())
    esl = slope_err(G, eg, act)
    dg, du = dh * Up * sl, dh * a
    edg = u * dg.abs() + 1.01 * (edh * (Up * sl).abs() + dh.abs() * eu * sl.abs() + (dh * Up).abs() * esl) + 4 * E * dg.abs() + tiny
    edu = u * du.abs() + 1.01 * (edh * a.abs() + dh.abs() * ea) + 4 * E * du.abs() + tiny
    dz, edz = torch.cat((dg, du), 1), torch.cat((edg, edu), 1)
    for name, p, q, ep, eq in (("x", dz, Wi, edz, None), ("win", dz.T, X, edz.T, None), ("wout", D.T, h, None, eh)):
        ref = p @ q
        bound = u * ref.abs() + (p.shape[1] + 16) * E * (p.abs() @ q.abs()) + tiny
        bound = bound + 1.01 * (ep @ q.abs() if ep is not None else p.abs() @ eq)
        within(got[name], ref, bound, "d" + name)
    if bin_ is not None:
        ref = dz.sum(0)
        within(got["bin"], ref, u * ref.abs() + 1.01 * edz.sum(0) + (m + 16) * E * dz.abs().sum(0) + tiny, "db_in")
        ref = D.sum(0)
        within(got["bout"], ref, u * ref.abs() + (m + 16) * E * D.abs().sum(0) + tiny, "db_out")
    if r is not None:
        assert torch.equal(got["r"], dy)


# ------------------------------------------------------------------ clipping


@pytest.mark.parametrize("dtype", list(U))
@pytest.mark.parametrize("sizes", [[1], [0, 5, 0], [7, 64, 1000, 3], [1 << 20, 33, 65537], [100] * 200, [100] * 700])
@pytest.mark.parametrize("clipped", [True, False])
def test_clip_grad_norm(dtype, sizes, clipped):
    g = gen("clip", dtype, len(sizes), clipped)
    flat = rand(g, dtype, sum(sizes), scale=0.01)
    grads = list(flat.split(sizes))
    n64 = float(flat.double().norm())
    max_norm = n64 * (0.5 if clipped else 2)
    before = flat.clone()
    norm, out = ops.clip_grad_norm(grads, max_norm)
    assert torch.equal(flat, before)
    assert abs(float(norm) - n64) <= 300 * E * n64
    c = min(1.0, max_norm / (n64 + 1e-6))
    got = torch.cat(out)
    ref = flat.double() * c
    if clipped:
        within(got, ref, (U[dtype] + 310 * E) * ref.abs() + TINY[dtype], "clipped")
    else:
        assert torch.equal(got, flat)
    norm2, same = ops.clip_grad_norm(grads, max_norm, out=grads)
    assert torch.equal(norm2, norm) and torch.equal(flat, got)


def test_clip_grad_norm_mixed_types_and_orders():
    g = gen("clip mixed")
    grads = [rand(g, torch.float32, 33, 7), rand(g, torch.bfloat16, 5, 64).T, rand(g, torch.float16, 3, 4, 5),
             rand(g, torch.float32, 1001)[1:]]
    n64 = math.sqrt(sum(float(t.double().square().sum()) for t in grads))
    norm, out = ops.clip_grad_norm(grads, 0.25)
    assert abs(float(norm) - n64) <= 300 * E * n64
    for a, b in zip(grads, out):
        ref = a.double() * (0.25 / (n64 + 1e-6))
        within(b, ref, (U[a.dtype] + 310 * E) * ref.abs() + TINY[a.dtype], "mixed")


def test_clip_grad_norm_not_finite():
    for bad in (float("nan"), float("inf")):
        a, b = torch.ones(50, device="cuda"), torch.ones(70, device="cuda")
        b[3] = bad
        norm, out = ops.clip_grad_norm([a, b], 1.0)
        assert not torch.isfinite(norm)
        assert out[1][3].isnan()
        if math.isnan(bad):
            assert out[0].isnan().all()
        else:
            assert (out[0] == 0).all()


# ------------------------------------------------------------------ together


@pytest.mark.parametrize("dtype", DT16)
def test_empty_sizes(dtype):
    z = lambda *s: torch.zeros(*s, device="cuda", dtype=dtype)  # noqa: E731
    assert ops.rms_norm(z(0, 64), z(64)).shape == (0, 64)
    assert ops.rms_norm(z(4, 0), z(0)).shape == (4, 0)
    assert ops.linear(z(0, 8), z(5, 8)).shape == (0, 5)
    assert ops.linear(z(3, 8), z(0, 8)).shape == (3, 0)
    b, r = rand(gen("k0"), dtype, 6), rand(gen("r0"), dtype, 20, 6)
    y = ops.linear(z(20, 0), z(6, 0), b, residual=r)  # an empty sum
    within(y, b.double() + r.double(), (U[dtype] + E) * (b.double().abs() + r.double().abs()), "k = 0")
    x, w = z(0, 8).requires_grad_(), z(5, 8).requires_grad_()
    dx, dw = torch.autograd.grad(ops.linear(x, w, activation="silu"), (x, w), z(0, 5))
    assert dx.shape == (0, 8) and dw.shape == (5, 8) and not bool(dw.any())
    x, wi, wo, bo = (t.requires_grad_() for t in (z(12, 8), z(0, 8), z(8, 0), rand(gen("f0"), dtype, 8)))
    y = ops.gated_feed_forward(x, wi, wo, None, bo)  # no hidden column
    assert torch.equal(y, bo.expand(12, 8))
    dx, dbo = torch.autograd.grad(y, (x, bo), torch.ones_like(y))
    assert not bool(dx.any()) and torch.equal(dbo, torch.full_like(dbo, 12))
    x, wi, wo = (t.requires_grad_() for t in (z(0, 8), z(6, 8), z(8, 3)))
    grads = torch.autograd.grad(ops.gated_feed_forward(x, wi, wo), (x, wi, wo), z(0, 8))
    assert [t.shape for t in grads] == [x.shape, wi.shape, wo.shape] and not any(bool(t.any()) for t in grads)


def test_nan_and_infinity_stay_in_their_rows():
    g = gen("nan rows")
    x, w = rand(g, torch.bfloat16, 300, 64), rand(g, torch.bfloat16, 200, 64)
    wi, wo = rand(g, torch.bfloat16, 144, 64), rand(g, torch.bfloat16, 64, 72)
    clean, ffn = ops.linear(x, w, activation="gelu"), ops.gated_feed_forward(x, wi, wo)
    x[17, 3], x[250, 60] = float("nan"), float("inf")
    keep = torch.ones(300, dtype=torch.bool, device="cuda")
    keep[17] = keep[250] = False
    for got, ref in ((ops.linear(x, w, activation="gelu"), clean), (ops.gated_feed_forward(x, wi, wo), ffn)):
        assert torch.equal(got[keep], ref[keep]) and got[17].isnan().all() and not got[250].isfinite().all()


@pytest.mark.parametrize("shape", [(3, 8, 40), (200, 8, 40), (200, 64, 200), (200, 100, 40)])
def test_infinite_row_of_the_feed_forward_block(shape):
    # all positive: an infinite row is infinite and not NaN, whatever a tile holds past the last hidden column
    m, c, f = shape
    g = gen("infinite row", shape)
    x, dy = rand(g, torch.bfloat16, m, c).abs(), rand(g, torch.bfloat16, m, c).abs()
    wi, wo = rand(g, torch.bfloat16, 2 * f, c).abs() + 0.1, rand(g, torch.bfloat16, c, f).abs() + 0.1
    run = lambda x: ops.gated_feed_forward(x, wi, wo, activation="relu")  # noqa: E731
    keep = torch.arange(m, device="cuda") != 1
    bad = torch.where(keep[:, None], x, float("inf"))
    clean, got = run(x), run(bad)
    assert clean.isfinite().all() and torch.equal(got[keep], clean[keep]) and (got[1] == float("inf")).all()
    leaves = [t.requires_grad_() for t in (x, wi, wo)]
    wi_run = lambda d: torch.autograd.grad(ops.gated_feed_forward(*leaves, activation="relu"), leaves, d)  # noqa: E731
    ref, grads = wi_run(dy), wi_run(torch.where(keep[:, None], dy, float("inf")))
    assert torch.equal(grads[0][keep], ref[0][keep]) and all((t == float("inf")).all() for t in (grads[0][1], *grads[1:]))


def test_other_stream_and_determinism():
    g = gen("stream")
    x, wi, wo = rand(g, torch.float16, 3000, 96), rand(g, torch.float16, 512, 96, scale=0.1), rand(g, torch.float16, 96, 256, scale=0.1)
    leaves = [t.requires_grad_() for t in (x, wi, wo)]

    def step():
        y = ops.gated_feed_forward(*leaves)
        return y, *torch.autograd.grad(y, leaves, torch.ones_like(y))

    first = step()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        second = step()
    side.synchronize()
    for a, b in zip(first, second):
        assert torch.equal(a, b)
    assert capi.device_status() == 0


def test_first_call_of_a_host_thread():
    """A thread that has made no CUDA call yet has no current context; its memory comes from the allocator's cache."""
    import threading

    g = gen("thread")
    x, w = rand(g, torch.bfloat16, 200, 64), rand(g, torch.bfloat16, 64, 64, scale=0.1)
    want = ops.linear(x, w)
    spare = [torch.empty_like(want) for _ in range(4)]
    torch.cuda.synchronize()
    del spare
    got = []
    t = threading.Thread(target=lambda: got.append(ops.linear(x, w)))
    t.start()
    t.join()
    assert got and torch.equal(got[0], want)


def test_runs_in_a_cuda_graph():
    g = gen("graph")
    x, w = rand(g, torch.bfloat16, 200, 64), rand(g, torch.bfloat16, 64, 64, scale=0.1)
    wn = torch.ones(64, device="cuda", dtype=torch.bfloat16)
    step = lambda: ops.linear(ops.rms_norm(x, wn), w, activation="silu", residual=x)  # noqa: E731
    want = step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = step()
    y.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, want)


def test_refusals():
    z = lambda *s, dt=torch.bfloat16: torch.zeros(*s, device="cuda", dtype=dt)  # noqa: E731
    with pytest.raises(RuntimeError, match="dtype"):
        ops.linear(z(4, 8, dt=torch.float32), z(3, 8, dt=torch.float32))
    with pytest.raises(RuntimeError, match="dtype"):
        ops.rms_norm(z(4, 8, dt=torch.float64), z(8, dt=torch.float64))
    with pytest.raises(RuntimeError, match="input's dtype"):
        ops.linear(z(4, 8), z(3, 8, dt=torch.float16))
    with pytest.raises(RuntimeError, match="weight must be"):
        ops.linear(z(4, 8), z(3, 9))
    with pytest.raises(RuntimeError, match="bias must have"):
        ops.linear(z(4, 8), z(3, 8), z(4))
    with pytest.raises(RuntimeError, match="residual"):
        ops.linear(z(4, 8), z(3, 8), residual=z(4, 4))
    with pytest.raises(ValueError, match="activation"):
        ops.linear(z(4, 8), z(3, 8), activation="swish2")
    with pytest.raises(RuntimeError, match="w_in must be"):
        ops.gated_feed_forward(z(4, 8), z(7, 8), z(8, 4))
    with pytest.raises(RuntimeError, match="weight must have"):
        ops.rms_norm(z(4, 8), z(9))
    with pytest.raises(RuntimeError, match="residual"):
        ops.rms_norm(z(4, 8), z(8), residual=z(5, 8))
    with pytest.raises(RuntimeError, match="float8_e4m3fn"):
        ops.linear_quant(z(4, 8), torch.ones(4, device="cuda"), z(3, 8), torch.ones(3, device="cuda"))
    with pytest.raises(RuntimeError, match="one value per row"):
        q, s = ops.quantize_rows(z(4, 8))
        ops.linear_quant(q, s[:3], q, s)
    with pytest.raises(RuntimeError, match="shape and strides"):
        ops.clip_grad_norm([z(4, 8)], 1.0, out=[z(8, 4).T])
    with pytest.raises(RuntimeError, match="at least one"):
        ops.clip_grad_norm([], 1.0)
    with pytest.raises(RuntimeError, match="max_norm"):
        ops.clip_grad_norm([z(4)], -1.0)
    a = capi.Linear(m=20, n=8, k=8, ldx=8, ldw=8, dtype=capi.LF_BF16)
    assert capi.lib().lf_linear_fwd(a, None, 0, None) == capi.LF_ERR_INVALID
