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


@pytest.mark.parametrize("act", ["relu", "silu", "gelu", "gelu_tanh"])
def test_activations_of_huge_values(act):
    """Finite values whose squares or cubes pass fp32's range: z or 0, with a slope of 1 or 0."""
    n = 64
    z = torch.tensor([s * v for v in (60000.0, 1e10, 1.2e13, 1e19, 2e19, 1e30, 3e38) for s in (1, -1)]).bfloat16().cuda()
    x = torch.zeros(z.numel(), n, dtype=torch.bfloat16, device="cuda")
    x[:, 5] = z
    x.requires_grad_()
    y = ops.linear(x, torch.eye(n, dtype=torch.bfloat16, device="cuda"), activation=act)
    (dx,) = torch.autograd.grad(y, x, torch.ones_like(y))
    assert torch.equal(y[:, 5], torch.relu(z)) and torch.equal(dx[:, 5].float(), (z > 0).float())


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


@pytest.mark.parametrize("form", ["rms_norm", "linear", "gated_feed_forward"])
def test_second_order_and_transforms_are_refused(form):
    f = forms()[form]
    x = rand(gen("second"), torch.bfloat16, 12, 32).requires_grad_()
    y = f(x)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(y, x, torch.ones_like(y), create_graph=True)
    with pytest.raises(RuntimeError):
        torch.func.vmap(f)(x.detach()[None])
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda t: f(t).float().sum())(x.detach())
    assert capi.device_status() == 0


# ------------------------------------------------------------------ gradients of some inputs, strided operands


def ffn64(x, wi, wo, bi, bo, act, r, dy):
    """The gated block's outputs and gradients in 64 bits with bounds: name -> (value, bound)."""
    dtype, (m, c), f = x.dtype, x.shape, wo.shape[1]
    u, tiny = U[dtype], TINY[dtype]
    d = lambda t: None if t is None else t.detach().double()  # noqa: E731
    X, Wi, Wo, D = d(x), d(wi), d(wo), d(dy)
    z, mag, _ = base.linear64(X, Wi, d(bi), "none", None)
    ez = (c + 16) * E * mag
    G, Up, eg, eu = z[:, :f], z[:, f:], ez[:, :f], ez[:, f:]
    a, sl = act64(G, act), slope64(G, act)
    ea = 1.2 * eg + 64 * E * (G.abs() + 1)
    h = a * Up
    eh = u * h.abs() + 1.01 * (ea * Up.abs() + a.abs() * eu) + E * h.abs() + tiny
    y = h @ Wo.T + (d(bo) if bo is not None else 0) + (d(r) if r is not None else 0)
    mag = h.abs() @ Wo.abs().T + (d(bo).abs() if bo is not None else 0)
    out = {"y": (y, u * y.abs() + 1.01 * eh @ Wo.abs().T + (f + 16) * E * mag + tiny)}
    dh, edh, esl = D @ Wo, (c + 16) * E * (D.abs() @ Wo.abs()), slope_err(G, eg, act)
    dg, du = dh * Up * sl, dh * a
    edg = u * dg.abs() + 1.01 * (edh * (Up * sl).abs() + dh.abs() * eu * sl.abs() + (dh * Up).abs() * esl) + 4 * E * dg.abs() + tiny
    edu = u * du.abs() + 1.01 * (edh * a.abs() + dh.abs() * ea) + 4 * E * du.abs() + tiny
    dz, edz = torch.cat((dg, du), 1), torch.cat((edg, edu), 1)
    for name, p, q, ep, eq in (("x", dz, Wi, edz, None), ("wi", dz.T, X, edz.T, None), ("wo", D.T, h, None, eh)):
        v = p @ q
        err = ep @ q.abs() if ep is not None else p.abs() @ eq
        out[name] = v, u * v.abs() + (p.shape[1] + 16) * E * (p.abs() @ q.abs()) + 1.01 * err + tiny
    v = dz.sum(0)
    out["bi"] = v, u * v.abs() + 1.01 * edz.sum(0) + (m + 16) * E * dz.abs().sum(0) + tiny
    v = D.sum(0)
    out["bo"] = v, u * v.abs() + (m + 16) * E * D.abs().sum(0) + tiny
    out["r"] = D, torch.zeros_like(D)
    return out


SUBSETS = ["x", "wi", "wo", "bi", "bo", "wi wo", "wi bi", "bi bo", "wo bo", "x bi", "x wo", "x wi wo", "wi wo bi bo", "r", "r bi", "x wi wo bi bo r"]


@pytest.mark.parametrize("dtype", DT16)
@pytest.mark.parametrize("shape", [(300, 64, 50), (130, 40, 100), (300, 64, 200), (20000, 64, 256), (2, 64, 64), (300, 128, 136), (257, 96, 333)])
def test_gradients_of_some_inputs_of_the_feed_forward_block(dtype, shape):
    """First layers need no dx, frozen weights no dw, fine-tuned biases nothing else: each choice alone."""
    m, c, f = shape
    g = gen("subsets", dtype, shape)
    t = {"x": rand(g, dtype, m, c), "wi": rand(g, dtype, 2 * f, c, scale=c**-0.5), "wo": rand(g, dtype, c, f, scale=f**-0.5),
         "bi": rand(g, dtype, 2 * f, scale=0.5), "bo": rand(g, dtype, c, scale=0.5), "r": rand(g, dtype, m, c)}
    dy = rand(g, dtype, m, c)
    want = ffn64(t["x"], t["wi"], t["wo"], t["bi"], t["bo"], "silu", t["r"], dy)
    for names in (s.split() for s in SUBSETS):
        a = {k: v.clone().requires_grad_(k in names) for k, v in t.items()}
        y = ops.gated_feed_forward(a["x"], a["wi"], a["wo"], a["bi"], a["bo"], residual=a["r"])
        within(y.detach(), *want["y"], "y")
        y.backward(dy)
        for k, v in a.items():
            assert (v.grad is not None) == (k in names), (k, names)
            if k in names:
                within(v.grad, *want[k], f"d{k} of {names}")
    assert capi.device_status() == 0


@pytest.mark.parametrize("dtype", list(U))
@pytest.mark.parametrize("shape", [(300, 64), (40, 771), (5, 20000)])
def test_gradients_of_some_inputs_of_the_norm(dtype, shape):
    """Any choice of inputs, and either output alone, as the whole backward gives them."""
    g = gen("norm subsets", dtype, shape)
    t = {"x": rand(g, dtype, *shape), "w": rand(g, dtype, shape[1]), "r": rand(g, dtype, *shape)}
    dy, ds, none = rand(g, dtype, *shape), rand(g, dtype, *shape), torch.zeros(shape, device="cuda", dtype=dtype)

    def run(names, dy, ds):
        a = {k: v.clone().requires_grad_(k in names) for k, v in t.items()}
        out = [(o, d) for o, d in zip(ops.rms_norm(a["x"], a["w"], residual=a["r"]), (dy, ds)) if d is not None and o.requires_grad]
        torch.autograd.backward(*zip(*out))
        assert all((v.grad is not None) == (k in names) for k, v in a.items())
        return {k: a[k].grad for k in names}

    for ups, same in (((dy, ds), (dy, ds)), ((dy, None), (dy, none))):
        want = run("xwr", *same)
        for names in ("x", "w", "r", "xw", "xr", "wr"):
            got = run(names, *ups)
            assert all(torch.equal(got[k], want[k]) for k in names), names
    got = run("xr", None, ds)
    assert torch.equal(got["x"], ds) and torch.equal(got["r"], ds)


@pytest.mark.parametrize("dtype", DT16)
@pytest.mark.parametrize("act", ["none", "gelu"])
@pytest.mark.parametrize("shape", [(300, 72, 96), (3, 64, 64), (4000, 256, 64), (129, 131, 65)])
def test_gradients_of_some_inputs_of_linear(dtype, act, shape):
    m, n, k = shape
    g = gen("linear subsets", dtype, act, shape)
    t = {"x": rand(g, dtype, m, k), "w": rand(g, dtype, n, k, scale=k**-0.5), "b": rand(g, dtype, n), "r": rand(g, dtype, m, n)}
    dy = rand(g, dtype, m, n)
    u, tiny = U[dtype], TINY[dtype]
    z, mag, _ = base.linear64(t["x"], t["w"], t["b"], act, None)
    ez = (k + 16) * E * mag
    dz = dy.double() * slope64(z, act)
    edz = (0 if act == "none" else u) * dz.abs() + dy.double().abs() * slope_err(z, ez, act) + tiny
    want = {"r": (dy.double(), torch.zeros_like(dz)), "b": (dz.sum(0), u * dz.sum(0).abs() + edz.sum(0) * 1.01 + (m + 16) * E * dz.abs().sum(0) + tiny)}
    for name, p, q, ep in (("x", dz, t["w"].double(), edz), ("w", dz.T, t["x"].double(), edz.T)):
        v = p @ q
        want[name] = v, u * v.abs() + ep @ q.abs() * 1.01 + (p.shape[1] + 16) * E * (p.abs() @ q.abs()) + tiny
    for names in ("x", "w", "b", "x w", "w b", "x b", "r", "x w b r"):
        a = {i: v.clone().requires_grad_(i in names.split()) for i, v in t.items()}
        ops.linear(a["x"], a["w"], a["b"], activation=act, residual=a["r"]).backward(dy)
        for i, v in a.items():
            assert (v.grad is not None) == (i in names.split()), (i, names)
            if v.grad is not None:
                within(v.grad, *want[i], f"d{i} of {names}")
    assert capi.device_status() == 0


@pytest.mark.parametrize("dtype", DT16)
@pytest.mark.parametrize("shape", [(1, 64, 64), (5, 64, 96), (300, 64, 200), (300, 40, 330), (20000, 64, 640), (300, 128, 136)])
@pytest.mark.parametrize("offset", [0, 8, 1])
def test_feed_forward_block_on_strided_rows(dtype, shape, offset):
    """x, residual and dy as slices of wider tensors: on a 16-byte boundary and off it."""
    m, c, f = shape
    g = gen("strided ffn", dtype, shape, offset)
    cut = lambda: rand(g, dtype, m, c + 24)[:, offset:offset + c]  # noqa: E731
    x, r, dy = cut(), cut(), cut()
    wi, wo = rand(g, dtype, 2 * f, c, scale=c**-0.5), rand(g, dtype, c, f, scale=f**-0.5)
    want = ffn64(x, wi, wo, None, None, "silu", r, dy)
    leaves = [t.detach().requires_grad_() for t in (x, wi, wo, r)]
    assert leaves[0].stride() == x.stride()
    y = ops.gated_feed_forward(*leaves[:3], residual=leaves[3])
    within(y.detach(), *want["y"], "y")
    for k, got in zip(("x", "wi", "wo", "r"), torch.autograd.grad(y, leaves, dy)):
        within(got, *want[k], "d" + k)
    assert capi.device_status() == 0


@pytest.mark.parametrize("dtype", list(U))
def test_norm_on_strided_rows(dtype):
    g = gen("strided norm", dtype)
    wide = rand(g, dtype, 40, 3, 72)
    w = rand(g, dtype, 64)
    x, r, dy, ds = wide[:, 0, 5:69], wide[:, 1, :64], wide[:, 2, 8:72], rand(g, dtype, 64, 40).T

    def run(x, r, dy, ds):
        a = [t.detach().requires_grad_() for t in (x, w, r)]
        y, s = ops.rms_norm(*a[:2], residual=a[2])
        return y, s, *torch.autograd.grad((y, s), a, (dy, ds)), *(t.float() for t in ops.rms_norm_quant(x, w, residual=r)), *(t.float() for t in ops.quantize_rows(x))

    for a, b in zip(run(x, r, dy, ds), run(*(t.contiguous() for t in (x, r, dy, ds)))):
        assert torch.equal(a, b)


# ------------------------------------------------------------------ graphs


def test_training_step_in_a_cuda_graph():
    """Forward and backward of all four operators, captured once and replayed on other values."""
    dtype, g = torch.bfloat16, gen("step graph")
    m, c, f = 300, 64, 200
    x, dy = rand(g, dtype, m, c), rand(g, dtype, m, c)
    params = [t.requires_grad_() for t in (rand(g, dtype, c), rand(g, dtype, c, c, scale=0.1), rand(g, dtype, c), rand(g, dtype, 2 * f, c, scale=0.1),
                                           rand(g, dtype, c, f, scale=0.1), rand(g, dtype, 2 * f), rand(g, dtype, c))]
    wn, w, b, wi, wo, bi, bo = params

    def step():
        y, s = ops.rms_norm(ops.linear(x, w, b, activation="gelu"), wn, residual=x)
        out = ops.gated_feed_forward(y, wi, wo, bi, bo, residual=s)
        grads = list(torch.autograd.grad(out, params, dy))
        norm, _ = ops.clip_grad_norm(grads, 0.5, out=grads)
        return out, norm, *grads

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for k in range(2):
        with torch.no_grad():
            x.copy_(rand(gen("replay", k), dtype, m, c))
        graph.replay()
        torch.cuda.synchronize()
        for a, b_ in zip(got, step()):
            assert torch.equal(a, b_)
    assert capi.device_status() == 0


# ------------------------------------------------------------------ entry points below the autograd nodes


@pytest.mark.parametrize("dtype", DT16)
@pytest.mark.parametrize("shape", [(300, 64, 200), (300, 128, 136), (2, 64, 64)])
def test_extension_entry_points(dtype, shape):
    """The extension's forward and backward functions give what the autograd nodes do."""
    e, act, g, (m, c, f) = ops.ext(), ops.ACTIVATIONS["gelu"], gen("entry", dtype, shape), shape
    x, r, dy, ds, wn, b = (rand(g, dtype, *s) for s in ((m, c), (m, c), (m, c), (m, c), (c,), (c,)))
    w, wi, wo, bi = rand(g, dtype, c, c, scale=0.1), rand(g, dtype, 2 * f, c, scale=0.1), rand(g, dtype, c, f, scale=0.1), rand(g, dtype, 2 * f)

    def same(got, want):
        assert len(got) == len(want) and all(torch.equal(p, q) for p, q in zip(got, want))

    def grads(f, leaves, up):
        a = [t.detach().requires_grad_() for t in leaves]
        out = f(*a)
        return out, torch.autograd.grad(out, a, up)

    (y, s), want = grads(lambda x, w, r: ops.rms_norm(x, w, residual=r), (x, wn, r), (dy, ds))
    y1, s1, rstd = e.RmsNorm_forward(x, wn, r, 1e-6, True)
    same((y1, s1), (y, s))
    assert rstd.dtype == torch.float32 and rstd.shape == (m,)
    assert e.RmsNorm_forward(x, wn, None, 1e-6, False)[1:] == (None, None)
    same(e.RmsNorm_backward(dy, ds, s1, rstd, wn, True, True), want[:2])
    dx, none = e.RmsNorm_backward(dy, ds, s1, rstd, wn, True, False)
    assert none is None and torch.equal(dx, want[0])

    y, want = grads(lambda x, w, b, r: ops.linear(x, w, b, activation="gelu", residual=r), (x, w, b, r), dy)
    assert torch.equal(e.Linear_forward(x, w, b, r, act), y)
    same(e.Linear_backward(dy, x, w, b, act, True, True, True), want[:3])
    assert e.Linear_backward(dy, x, w, b, act, False, False, False) == (None, None, None)

    y, want = grads(lambda *t: ops.gated_feed_forward(*t[:5], activation="gelu", residual=t[5]), (x, wi, wo, bi, b, r), dy)
    assert torch.equal(e.GatedFeedForward_forward(x, wi, wo, bi, b, r, act), y)
    same(e.GatedFeedForward_backward(dy, x, wi, wo, bi, act, True, True, True, True, True), want[:5])

    # and the C ABI with a workspace of exactly the size it asks for
    L, st = capi.lib(), torch.cuda.current_stream().cuda_stream
    ws = lambda n: torch.empty(max(n, 256), device="cuda", dtype=torch.uint8)  # noqa: E731
    code = capi.LF_F16 if dtype == torch.float16 else capi.LF_BF16
    p = lambda t: t.data_ptr()  # noqa: E731
    out = [torch.empty_like(t) for t in (x, wi, bi, wo, b)]
    a = capi.GatedFfn(p(x), p(wi), p(bi), p(wo), p(b), p(r), None, p(dy), *map(p, out), c, c, c, m, c, f, act, code)
    n = L.lf_gated_ffn_bwd_workspace_size(ctypes.byref(a))
    room = ws(n)
    assert L.lf_gated_ffn_bwd(ctypes.byref(a), p(room), n, st) == capi.LF_OK
    same(out, [want[k] for k in (0, 1, 3, 2, 4)])
    _, want = grads(lambda x, w, b: ops.linear(x, w, b, activation="gelu"), (x, w, b), dy)
    out = [torch.empty_like(t) for t in (x, w, b)]
    a = capi.Linear(p(x), p(w), p(b), None, None, None, None, p(dy), *map(p, out), c, c, 0, c, m, c, c, act, code)
    n = L.lf_linear_bwd_workspace_size(ctypes.byref(a))
    room = ws(n)
    assert L.lf_linear_bwd(ctypes.byref(a), p(room), n, st) == capi.LF_OK
    same(out, want)
    _, want = grads(lambda x, w: ops.rms_norm(x, w), (x, wn), dy)
    y, _, rstd = e.RmsNorm_forward(x, wn, None, 1e-6, True)
    out = [torch.empty_like(t) for t in (x, wn)]
    n = L.lf_rms_norm_bwd_workspace_size(m, c)
    room = ws(n)
    assert L.lf_rms_norm_bwd(p(dy), None, p(x), p(rstd), p(wn), *map(p, out), m, c, code, p(room), n, st) == capi.LF_OK
    same(out, want)
    assert capi.device_status() == 0
