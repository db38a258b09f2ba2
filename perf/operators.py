"""What the block operators are measured on: norm, matrix product, gated feed-forward and gradient clipping.

Each case is one pass through one operator, in the sizes of this repository's configurations (56x56 and 14x14 token
grids, the 16384-token long sequence, widths heads x head size = 64, 512 and 1024) or generic ones.  ``own`` selects
the elementary 32-bit torch form or the calls a user makes of :mod:`laplacianformer_b200.ops`.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6
E4M3_MAX = 448.0


def listed():
    return [
        # Norm before a sublayer in a training step of the long-sequence configuration (8 x 16384 tokens, width 1024).
        {"name": "norm_train_long", "op": "norm", "m": 131072, "c": 1024, "dtype": "bf16", "residual": True, "train": True},
        # The same in 32 bits on a 14x14 grid with a class token, at a width that no vector load divides.
        {"name": "norm_train_f32_ragged", "op": "norm", "m": 32 * 197, "c": 771, "dtype": "f32", "residual": True, "train": True},
        # One image of the 14x14 grid served with 8-bit activations.
        {"name": "norm_quant_serve", "op": "norm_quant", "m": 196, "c": 512, "dtype": "f16", "residual": True, "train": False},
        # One token through an expanding projection: latency.
        {"name": "linear_token", "op": "linear", "m": 1, "k": 1024, "n": 4096, "dtype": "bf16", "act": "gelu", "bias": True,
         "residual": False, "train": False},
        # The attention's output projection in training, 128 images of 196 tokens, width 512.
        {"name": "linear_proj_train", "op": "linear", "m": 25088, "k": 512, "n": 512, "dtype": "f16", "act": "none", "bias": True,
         "residual": True, "train": True},
        # A batch of those images through the query-key-value projection with 8-bit activations and weights.
        {"name": "linear_quant_qkv", "op": "linear_quant", "m": 25088, "k": 512, "n": 1536, "dtype": "bf16", "act": "none",
         "bias": True, "residual": False, "train": False},
        # One token through the whole feed-forward block: latency, weights read once.
        {"name": "ffn_token", "op": "ffn", "m": 1, "c": 1024, "f": 4096, "dtype": "bf16", "act": "silu", "bias": False,
         "residual": True, "train": False},
        # Eight images with a class token; hidden width 8/3 of 512, odd.
        {"name": "ffn_train_ragged", "op": "ffn", "m": 8 * 197, "c": 512, "f": 1365, "dtype": "f16", "act": "gelu", "bias": True,
         "residual": True, "train": True},
        # First pyramid stage: 32 images of 56x56 tokens, width 64.
        {"name": "ffn_train_stage1", "op": "ffn", "m": 100352, "c": 64, "f": 256, "dtype": "bf16", "act": "silu", "bias": False,
         "residual": True, "train": True},
        # The long-sequence configuration's feed-forward block: the largest.
        {"name": "ffn_train_long", "op": "ffn", "m": 131072, "c": 1024, "f": 4096, "dtype": "bf16", "act": "silu", "bias": False,
         "residual": True, "train": True},
        # Gradients of a small pyramid model in 32 bits: many tensors, few bytes.
        {"name": "clip_small", "op": "clip", "layers": 8, "c": 64, "f": 171, "dtype": "f32", "clipped": True},
        # Gradients of a 24-layer model of width 1024 in 16 bits.
        {"name": "clip_large", "op": "clip", "layers": 24, "c": 1024, "f": 2731, "dtype": "bf16", "clipped": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A width over a logarithmic range: a multiple of 64, of 8, or any number."""
    w = _log(rng, lo, hi)
    step = rng.choice((64, 64, 8, 1))
    w = max(step, w // step * step)
    return w - step if w in (1536, 3072) else w


def draw(rng):
    op = rng.choice(("norm", "norm", "norm_quant", "linear", "linear", "linear_quant", "ffn", "ffn", "ffn", "clip"))
    if op in ("norm", "norm_quant"):
        c = _width(rng, 32, 4096)
        m = min(_log(rng, 1, 200000), (1 << 27) // c)
        return {"op": op, "m": m, "c": c, "dtype": rng.choice(("f32", "f16", "bf16")), "residual": rng.random() < 0.7,
                "train": op == "norm" and rng.random() < 0.7}
    if op in ("linear", "linear_quant"):
        train = op == "linear" and rng.random() < 0.6
        return {"op": op, "m": _log(rng, 1, 60000), "k": _width(rng, 64, 2048), "n": _width(rng, 64, 4096),
                "dtype": rng.choice(("f16", "bf16")), "act": rng.choice(("none", "relu", "gelu", "gelu_tanh", "silu")),
                "bias": rng.random() < 0.5, "residual": rng.random() < 0.5, "train": train}
    if op == "ffn":
        c = _width(rng, 64, 1024)
        return {"op": op, "m": _log(rng, 1, 100000), "c": c, "f": _width(rng, c, 4 * c), "dtype": rng.choice(("f16", "bf16")),
                "act": rng.choice(("silu", "gelu", "gelu_tanh", "relu")), "bias": rng.random() < 0.5,
                "residual": rng.random() < 0.5, "train": rng.random() < 0.6}
    c = _width(rng, 64, 1024)
    return {"op": op, "layers": rng.randint(1, 24), "c": c, "f": _width(rng, c, 4 * c), "dtype": rng.choice(("f32", "f16", "bf16")),
            "clipped": rng.random() < 0.7}


# ------------------------------------------------------------------ inputs


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, dtype, *shape, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def _quant(x):
    scale = x.abs().amax(1) / E4M3_MAX
    return (x / scale[:, None]).to(torch.float8_e4m3fn), scale


def _clip_shapes(case):
    """Parameter shapes of one block: two norms, query, key-value and output projections with biases, both feed-forward weights."""
    c, f = case["c"], case["f"]
    return [(c,), (c, c), (c,), (2 * c, c), (2 * c,), (c, c), (c,), (c,), (2 * f, c), (c, f)] * case["layers"]


def prepare(case, seed):
    g, s = _gen(seed), {"case": case}
    dt = DTYPES[case["dtype"]]
    grad = bool(case.get("train"))
    op = case["op"]
    if op in ("norm", "norm_quant"):
        m, c = case["m"], case["c"]
        s["x"] = _randn(g, dt, m, c)
        s["w"] = (1.0 + 0.1 * torch.randn(c, generator=g, device="cuda")).to(dt)
        s["r"] = _randn(g, dt, m, c) if case["residual"] else None
        if grad:
            s["dy"], s["ds"] = _randn(g, dt, m, c), _randn(g, dt, m, c) if case["residual"] else None
    elif op == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        s["x"], s["w"] = _randn(g, dt, m, k), _randn(g, dt, n, k, scale=k ** -0.5)
        s["b"] = _randn(g, dt, n, scale=0.1) if case["bias"] else None
        s["r"] = _randn(g, dt, m, n) if case["residual"] else None
        if grad:
            s["dy"] = _randn(g, dt, m, n)
    elif op == "linear_quant":
        m, k, n = case["m"], case["k"], case["n"]
        s["q"], s["sx"] = _quant(torch.randn(m, k, generator=g, device="cuda"))
        s["wq"], s["sw"] = _quant(torch.randn(n, k, generator=g, device="cuda") * k ** -0.5)
        s["b"] = _randn(g, dt, n, scale=0.1) if case["bias"] else None
        s["r"] = _randn(g, dt, m, n) if case["residual"] else None
    elif op == "ffn":
        m, c, f = case["m"], case["c"], case["f"]
        s["x"] = _randn(g, dt, m, c)
        s["win"], s["wout"] = _randn(g, dt, 2 * f, c, scale=c ** -0.5), _randn(g, dt, c, f, scale=f ** -0.5)
        s["bin"] = _randn(g, dt, 2 * f, scale=0.1) if case["bias"] else None
        s["bout"] = _randn(g, dt, c, scale=0.1) if case["bias"] else None
        s["r"] = _randn(g, dt, m, c) if case["residual"] else None
        if grad:
            s["dy"] = _randn(g, dt, m, c)
    else:
        # One gradient buffer with a view per parameter, as a data-parallel trainer keeps it; odd widths leave the
        # views unaligned.  The norm is about sqrt(total) * 1e-3.
        shapes = _clip_shapes(case)
        sizes = [math.prod(t) for t in shapes]
        total = sum(sizes)
        s["flat"] = _randn(g, dt, total, scale=1e-3)
        s["out"] = torch.empty_like(s["flat"])
        s["grads"] = [v.view(t) for v, t in zip(s["flat"].split(sizes), shapes)]
        s["outs"] = [v.view(t) for v, t in zip(s["out"].split(sizes), shapes)]
        s["max_norm"] = (0.5 if case["clipped"] else 2.0) * 1e-3 * math.sqrt(total)
    if grad:
        for k in ("x", "w", "b", "r", "win", "wout", "bin", "bout"):
            if s.get(k) is not None:
                s[k].requires_grad_()
    return s


# ------------------------------------------------------------------ the framework's operators


def _run_own(s):
    from laplacianformer_b200 import ops

    case = s["case"]
    op = case["op"]
    if op == "norm":
        y = ops.rms_norm(s["x"], s["w"], residual=s["r"], eps=EPS)
        if s["r"] is None:
            if not case["train"]:
                return {"y": y}
            dx, dw = torch.autograd.grad(y, (s["x"], s["w"]), s["dy"])
            return {"y": y, "dx": dx, "dw": dw}
        y, t = y
        if not case["train"]:
            return {"y": y, "s": t}
        dx, dr, dw = torch.autograd.grad((y, t), (s["x"], s["r"], s["w"]), (s["dy"], s["ds"]))
        return {"y": y, "s": t, "dx": dx, "dr": dr, "dw": dw}
    if op == "norm_quant":
        out = ops.rms_norm_quant(s["x"], s["w"], residual=s["r"], eps=EPS)
        return dict(zip(("q", "scale", "s"), out))
    if op == "linear":
        y = ops.linear(s["x"], s["w"], s["b"], activation=case["act"], residual=s["r"])
        names = ("x", "w", "b", "r")
    elif op == "linear_quant":
        return {"y": ops.linear_quant(s["q"], s["sx"], s["wq"], s["sw"], s["b"], activation=case["act"], residual=s["r"],
                                      dtype=DTYPES[case["dtype"]])}
    elif op == "ffn":
        y = ops.gated_feed_forward(s["x"], s["win"], s["wout"], s["bin"], s["bout"], activation=case["act"], residual=s["r"])
        names = ("x", "win", "wout", "bin", "bout", "r")
    else:
        norm, _ = ops.clip_grad_norm(s["grads"], s["max_norm"], out=s["outs"])
        return {"norm": norm, "grads": s["out"]}
    if not case["train"]:
        return {"y": y}
    names = [k for k in names if s[k] is not None]
    return {"y": y} | dict(zip(["d" + k for k in names], torch.autograd.grad(y, [s[k] for k in names], s["dy"])))


# ------------------------------------------------------------------ the plain form


def _f(t):
    return None if t is None else t.float()


def _act(z, name):
    """The activation and its derivative."""
    if name == "none":
        return z, torch.ones_like(z)
    if name == "relu":
        return z.clamp(min=0), (z > 0).to(z.dtype)
    if name == "silu":
        p = 1 / (1 + torch.exp(-z))
        return z * p, p * (1 + z * (1 - p))
    if name == "gelu":
        p = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
        return z * p, p + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    a, b = math.sqrt(2 / math.pi), 0.044715
    t = torch.tanh(a * (z + b * z * z * z))
    return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * a * (1 + 3 * b * z * z)


def _run_plain(s):
    case = s["case"]
    dt = DTYPES[case["dtype"]]
    op = case["op"]
    if op in ("norm", "norm_quant"):
        t, w = _f(s["x"]), _f(s["w"])
        if s["r"] is not None:
            t = t + _f(s["r"])
        rstd = 1 / torch.sqrt((t * t).mean(1, keepdim=True) + EPS)
        y = t * rstd * w
        out = {"s": t.to(dt)} if s["r"] is not None else {}
        if op == "norm_quant":
            scale = y.abs().amax(1) / E4M3_MAX
            scale = torch.where(scale == 0, torch.ones_like(scale), scale)
            return out | {"q": (y / scale[:, None]).to(torch.float8_e4m3fn), "scale": scale}
        out["y"] = y.to(dt)
        if case["train"]:
            dy, xhat = _f(s["dy"]), t * rstd
            a = dy * w
            dx = rstd * (a - xhat * (a * xhat).mean(1, keepdim=True))
            if s["r"] is not None:
                dx = dx + _f(s["ds"])
                out["dr"] = dx.to(dt)
            out["dx"], out["dw"] = dx.to(dt), (dy * xhat).sum(0).to(dt)
        return out
    if op in ("linear", "linear_quant"):
        if op == "linear":
            x, w = _f(s["x"]), _f(s["w"])
        else:
            x, w = _f(s["q"]) * s["sx"][:, None], _f(s["wq"]) * s["sw"][:, None]
        z = x @ w.T
        if s["b"] is not None:
            z = z + _f(s["b"])
        y, slope = _act(z, case["act"])
        if s["r"] is not None:
            y = y + _f(s["r"])
        out = {"y": y.to(dt)}
        if case["train"]:
            dz = _f(s["dy"]) * slope
            out["dx"], out["dw"] = (dz @ w).to(dt), (dz.T @ x).to(dt)
            if s["b"] is not None:
                out["db"] = dz.sum(0).to(dt)
            if s["r"] is not None:
                out["dr"] = s["dy"]
        return out
    if op == "ffn":
        x, win, wout = _f(s["x"]), _f(s["win"]), _f(s["wout"])
        z = x @ win.T
        if s["bin"] is not None:
            z = z + _f(s["bin"])
        gate, up = z.chunk(2, 1)
        a, slope = _act(gate, case["act"])
        h = a * up
        y = h @ wout.T
        if s["bout"] is not None:
            y = y + _f(s["bout"])
        if s["r"] is not None:
            y = y + _f(s["r"])
        out = {"y": y.to(dt)}
        if case["train"]:
            dy = _f(s["dy"])
            dh = dy @ wout
            dz = torch.cat((dh * up * slope, dh * a), 1)
            out["dx"], out["dwin"], out["dwout"] = (dz @ win).to(dt), (dz.T @ x).to(dt), (dy.T @ h).to(dt)
            if s["bin"] is not None:
                out["dbin"], out["dbout"] = dz.sum(0).to(dt), dy.sum(0).to(dt)
            if s["r"] is not None:
                out["dr"] = s["dy"]
        return out
    flat = _f(s["flat"])
    norm = torch.sqrt((flat * flat).sum())
    return {"norm": norm, "grads": (flat * (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0)).to(dt)}


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return _run_plain(state)


# ------------------------------------------------------------------ 64 bits


def _phi(z, name):
    """The activation by its definition, differentiable."""
    if name == "silu":
        return z * torch.sigmoid(z)
    if name in ("gelu", "gelu_tanh"):
        return torch.nn.functional.gelu(z, approximate="tanh" if name == "gelu_tanh" else "none")
    return torch.relu(z) if name == "relu" else z


def exact(case, seed):
    s = prepare(case, seed)
    d = {k: v.detach().double().requires_grad_(v.requires_grad) for k, v in s.items()
         if isinstance(v, torch.Tensor) and k not in ("flat", "out")}
    op = case["op"]
    if op == "clip":
        flat = s["flat"].double()
        norm = torch.linalg.vector_norm(flat)
        return {"norm": norm, "grads": flat * min(1.0, s["max_norm"] / (float(norm) + 1e-6))}
    grads = {}
    if op in ("norm", "norm_quant"):
        t = d["x"] + d["r"] if case["residual"] else d["x"]
        y = torch.nn.functional.rms_norm(t, (case["c"],), d["w"], EPS)
        out = {"s": t.detach()} if case["residual"] else {}
        if op == "norm_quant":
            scale = y.abs().amax(1) / E4M3_MAX
            return out | {"q": y / scale[:, None], "scale": scale}
        out["y"], names = y.detach(), ("x", "r", "w")
        total = (y * d["dy"]).sum() + ((t * d["ds"]).sum() if case["residual"] else 0) if case["train"] else None
    else:
        if op == "linear_quant":
            y = torch.nn.functional.linear(d["q"] * d["sx"][:, None], d["wq"] * d["sw"][:, None], d.get("b"))
            names = ()
        elif op == "linear":
            y = torch.nn.functional.linear(d["x"], d["w"], d.get("b"))
            names = ("x", "w", "b", "r")
        if op == "ffn":
            f = case["f"]
            z = torch.nn.functional.linear(d["x"], d["win"], d.get("bin"))
            y = torch.nn.functional.linear(_phi(z[:, :f], case["act"]) * z[:, f:], d["wout"], d.get("bout"))
            names = ("x", "win", "wout", "bin", "bout", "r")
        else:
            y = _phi(y, case["act"])
        if case["residual"]:
            y = y + d["r"]
        out = {"y": y.detach()}
        total = (y * d["dy"]).sum() if case["train"] else None
    if case["train"]:
        names = [k for k in names if k in d]
        grads = dict(zip(["d" + k for k in names], torch.autograd.grad(total, [d[k] for k in names])))
    return out | grads


def work(case):
    e = {"f32": 4, "f16": 2, "bf16": 2}[case["dtype"]]
    op = case["op"]
    if op in ("norm", "norm_quant"):
        m, c, r = case["m"], case["c"], case["residual"]
        # x, residual in; y, sum out; training: dy, ds in and dx out.
        rows = (2 if r else 1) * e + (1 if op == "norm_quant" else e) + (e if r else 0)
        rows += (3 if r else 2) * e if case["train"] else 0
        return {"bytes": m * c * rows + c * e * (2 if case["train"] else 1) + (4 * m if op == "norm_quant" else 0),
                "flops": m * c * (16 if case["train"] else 5)}
    if op in ("linear", "linear_quant"):
        m, k, n, q = case["m"], case["k"], case["n"], 1 if op == "linear_quant" else e
        b = m * k * q + n * k * q + m * n * e * (2 if case["residual"] else 1) + (n * e if case["bias"] else 0)
        b += 4 * (m + n) if op == "linear_quant" else 0
        if not case["train"]:
            return {"bytes": b, "flops": 2 * m * n * k}
        b += m * n * e + m * k * e + n * k * e + (n * e if case["bias"] else 0)
        return {"bytes": b, "flops": 6 * m * n * k}
    if op == "ffn":
        m, c, f = case["m"], case["c"], case["f"]
        biases = (2 * f + c) * e if case["bias"] else 0
        b = m * c * e * (3 if case["residual"] else 2) + 3 * c * f * e + biases
        if not case["train"]:
            return {"bytes": b, "flops": 6 * m * c * f}
        b += m * c * e * 2 + 3 * c * f * e + biases
        return {"bytes": b, "flops": 18 * m * c * f}
    total = sum(math.prod(t) for t in _clip_shapes(case))
    return {"bytes": 2 * total * e, "flops": 3 * total}
