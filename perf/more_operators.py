"""What the causal operators are measured on: linear attention with a decay per head (prompts, training, single tokens),
rotary positions, and the norms before and after a sublayer with its gate and residual scale.

Each case is one pass through one operator, in the sizes of this repository's configurations (56x56 and 14x14 token
grids, the 16384- and 65536-token long sequences, widths heads x head size = 64, 512 and 1024) or generic ones.  ``own``
selects the elementary 32-bit torch form or the calls a user makes of :mod:`laplacianformer_b200.ops`.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6
TAU = 2 * math.pi
CHUNK = 64  # tokens per chunk of the plain form


def listed():
    return [
        # 128 images of 14x14 tokens, 8 heads of 64: many short sequences, the last chunk ragged.
        {"name": "decay_train_images", "op": "decay", "b": 128, "h": 8, "t": 196, "dk": 64, "dv": 64, "dtype": "bf16", "train": True,
         "state": False, "ragged": False},
        # First pyramid stage: 32 images of 56x56 tokens, 2 heads of 32.
        {"name": "decay_train_stage1", "op": "decay", "b": 32, "h": 2, "t": 3136, "dk": 32, "dv": 32, "dtype": "f16", "train": True,
         "state": False, "ragged": False},
        # The long-sequence configuration, 8 sequences of 16384 tokens, 16 heads of 64: the largest.
        {"name": "decay_train_long", "op": "decay", "b": 8, "h": 16, "t": 16384, "dk": 64, "dv": 64, "dtype": "bf16", "train": True,
         "state": False, "ragged": False},
        # The next pieces of a padded batch of prompts: lengths of their own, states carried in and out, an odd head size.
        {"name": "decay_prompt_ragged", "op": "decay", "b": 6, "h": 8, "t": 1333, "dk": 64, "dv": 50, "dtype": "f16", "train": False,
         "state": True, "ragged": True},
        # One prompt of 65536 tokens, 8 heads of 128: few rows, a long axis.
        {"name": "decay_prompt_long", "op": "decay", "b": 1, "h": 8, "t": 65536, "dk": 128, "dv": 128, "dtype": "bf16", "train": False,
         "state": True, "ragged": False},
        # One token of one sequence: latency.
        {"name": "decay_step_one", "op": "step", "b": 1, "h": 16, "dk": 64, "dv": 64, "dtype": "bf16"},
        # One token of 192 sequences: the states are read and written once.
        {"name": "decay_step_batch", "op": "step", "b": 192, "h": 16, "dk": 64, "dv": 64, "dtype": "f16"},
        # Queries and keys of the long-sequence configuration, forward and backward.
        {"name": "rotary_train_long", "op": "rotary", "b": 8, "h": 16, "hk": 16, "t": 16384, "d": 64, "rot": 64, "dtype": "bf16",
         "pairs": "halves", "scaling": "none", "far": False, "train": True},
        # One token of 64 sequences at far positions: pairs side by side in three quarters of the head, stretched for long contexts.
        {"name": "rotary_serve", "op": "rotary", "b": 64, "h": 8, "hk": 8, "t": 1, "d": 128, "rot": 96, "dtype": "f16",
         "pairs": "neighbours", "scaling": "by_parts", "far": True, "train": False},
        # Between two sublayers of the long-sequence configuration: a gate per token and channel, the next norm, training.
        {"name": "sandwich_train_long", "op": "sandwich", "groups": 8, "rows": 16384, "c": 1024, "dtype": "bf16", "gate": "tokens",
         "act": "silu", "next": True, "train": True},
        # 32 images of 14x14 tokens and a class token in 32 bits: one gate per image, a width that no vector load divides.
        {"name": "sandwich_train_f32_ragged", "op": "sandwich", "groups": 32, "rows": 197, "c": 771, "dtype": "f32", "gate": "groups",
         "act": "none", "next": True, "train": True},
        # One token served, with a gate per channel: latency.
        {"name": "sandwich_token", "op": "sandwich", "groups": 1, "rows": 1, "c": 1024, "dtype": "bf16", "gate": "channels",
         "act": "none", "next": True, "train": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _head(rng):
    return rng.choice((32, 64, 64, 128, rng.randrange(8, 129, 8), rng.randint(1, 128)))


def draw(rng):
    op = rng.choice(("decay", "decay", "decay", "decay", "step", "step", "rotary", "rotary", "sandwich", "sandwich"))
    if op == "decay":
        dk = _head(rng)
        dv = dk if rng.random() < 0.7 else _head(rng)
        b, h = _log(rng, 1, 128), rng.choice((1, 2, 3, 8, 16))
        t = min(_log(rng, 1, 65536), max(1, (1 << 27) // (b * h * max(dk, dv))))
        return {"op": op, "b": b, "h": h, "t": t, "dk": dk, "dv": dv, "dtype": rng.choice(("f16", "bf16")), "train": rng.random() < 0.6,
                "state": rng.random() < 0.5, "ragged": rng.random() < 0.3}
    if op == "step":
        return {"op": op, "b": _log(rng, 1, 512), "h": rng.choice((1, 2, 3, 8, 16)), "dk": _head(rng), "dv": _head(rng),
                "dtype": rng.choice(("f32", "f16", "bf16"))}
    if op == "rotary":
        d = max(2, _head(rng))
        rot = d // 2 * 2 if rng.random() < 0.5 else rng.randint(1, d // 2) * 2
        b, h = _log(rng, 1, 128), rng.choice((1, 2, 3, 8, 16))
        t = min(_log(rng, 1, 65536), max(1, (1 << 27) // (b * h * d)))
        return {"op": op, "b": b, "h": h, "hk": rng.choice((1, h)), "t": t, "d": d, "rot": rot, "dtype": rng.choice(("f32", "f16", "bf16")),
                "pairs": rng.choice(("halves", "neighbours")), "scaling": rng.choice(("none", "linear", "base", "by_parts")),
                "far": rng.random() < 0.3, "train": rng.random() < 0.5}
    c = _log(rng, 32, 4096)
    step = rng.choice((64, 64, 8, 1))
    c = max(step, c // step * step)
    groups = _log(rng, 1, 256)
    rows = max(1, min(_log(rng, 1, 16384), (1 << 27) // (c * groups)))
    return {"op": op, "groups": groups, "rows": rows, "c": c, "dtype": rng.choice(("f32", "f16", "bf16")),
            "gate": rng.choice(("none", "tokens", "groups", "channels")), "act": rng.choice(("none", "sigmoid", "silu", "tanh")),
            "next": rng.random() < 0.7, "train": rng.random() < 0.7}


# ------------------------------------------------------------------ inputs


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, dtype, *shape, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def _heads(g, dtype, b, h, t, d, scale=1.0):
    """[b, h, t, d] as a projection leaves it: the heads of a token side by side."""
    return _randn(g, dtype, b, t, h, d, scale=scale).transpose(1, 2)


def _frequencies(case):
    """Radians per position of each pair, in 64 bits on the host."""
    n, base = case["rot"], 10000.0
    kind, factor, length = case["scaling"], 8.0, 8192
    if kind == "base" and n > 2:
        base *= factor ** (n / (n - 2))
    f = torch.tensor(base, dtype=torch.float64) ** (-torch.arange(0, n, 2, dtype=torch.float64) / n)
    if kind == "linear":
        f = f / factor
    if kind == "by_parts":
        turns = length * f / TAU
        keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0, 1)
        f = f * keep + f / factor * (1 - keep)
    return f, 0.1 * math.log(factor) + 1 if kind == "by_parts" else 1.0


def prepare(case, seed):
    g, s = _gen(seed), {"case": case}
    dt, op, train = DTYPES[case["dtype"]], case["op"], bool(case.get("train"))
    leaves = []
    if op in ("decay", "step"):
        b, h, dk, dv = case["b"], case["h"], case["dk"], case["dv"]
        # Time constants between 16 and 4096 tokens over the heads.
        s["log_decay"] = -torch.exp(torch.linspace(math.log(1 / 16), math.log(1 / 4096), h, device="cuda"))
        state = torch.randn(b, h, dk, dv, generator=g, device="cuda") * 4
    if op == "decay":
        t = case["t"]
        s["q"], s["k"], s["v"] = (_heads(g, dt, b, h, t, d) for d in (dk, dk, dv))
        s["state"] = state if case["state"] else None
        s["lengths"] = torch.randint(0, t + 1, (b,), generator=g, device="cuda") if case["ragged"] else None
        leaves = ["q", "k", "v"] + (["state"] if case["state"] else [])
        if train:
            s["do"] = _heads(g, dt, b, h, t, dv)
            s["dstate"] = torch.randn(b, h, dk, dv, generator=g, device="cuda") if case["state"] else None
    elif op == "step":
        s["q"], s["k"], s["v"], s["state"] = _randn(g, dt, b, h, dk), _randn(g, dt, b, h, dk), _randn(g, dt, b, h, dv), state
    elif op == "rotary":
        b, t = case["b"], case["t"]
        s["q"], s["k"] = _heads(g, dt, b, case["h"], t, case["d"]), _heads(g, dt, b, case["hk"], t, case["d"])
        first = torch.randint(0, 1 << 20 if case["far"] else 4096, (b, 1), generator=g, device="cuda")
        s["positions"] = first + torch.arange(t, device="cuda")
        s["freq"], s["mag"] = _frequencies(case)
        s["freq_gpu"] = s["freq"].cuda()
        leaves = ["q", "k"]
        if train:
            s["dq"], s["dk"] = _heads(g, dt, b, case["h"], t, case["d"]), _heads(g, dt, b, case["hk"], t, case["d"])
    else:
        n, r, c = case["groups"], case["rows"], case["c"]
        s["x"], s["r"] = _randn(g, dt, n, r, c, scale=0.5), _randn(g, dt, n, r, c)
        s["w"], s["wn"] = ((1.0 + 0.1 * torch.randn(c, generator=g, device="cuda")).to(dt) for _ in range(2))
        shape = {"none": None, "tokens": (n, r, c), "groups": (n, 1, c), "channels": (c,)}[case["gate"]]
        s["gate"] = _randn(g, dt, *shape) if shape else None
        if not case["next"]:
            s["wn"] = None
        leaves = ["x", "r", "w"] + (["gate"] if shape else []) + (["wn"] if case["next"] else [])
        if train:
            s["ds"] = _randn(g, dt, n, r, c)
            s["dy"] = _randn(g, dt, n, r, c) if case["next"] else None
    if train:
        s["leaves"] = leaves
        for k in leaves:
            s[k].requires_grad_()
    return s


ALPHA = 0.7071  # residual scale of the sandwich cases


# ------------------------------------------------------------------ the framework's operators


def _run_own(s):
    from laplacianformer_b200 import ops

    case = s["case"]
    op = case["op"]
    if op == "step":
        return {"o": ops.decay_attention_step(s["q"], s["k"], s["v"], s["log_decay"], s["state"]), "state": s["state"]}
    if op == "decay":
        out = ops.decay_attention(s["q"], s["k"], s["v"], s["log_decay"], state=s["state"], lengths=s["lengths"],
                                  return_state=case["state"])
        out = dict(zip(("o", "state"), out)) if case["state"] else {"o": out}
        into = {"o": s.get("do"), "state": s.get("dstate")}
    elif op == "rotary":
        out = dict(zip(("q", "k"), ops.rotary(s["q"], s["k"], s["freq"], positions=s["positions"],
                                              interleaved=case["pairs"] == "neighbours", magnitude=s["mag"])))
        into = {"q": s.get("dq"), "k": s.get("dk")}
    else:
        out = ops.sandwich_norm(s["x"], s["w"], s["r"], gate=s["gate"], next_weight=s["wn"], gate_activation=case["act"], scale=ALPHA,
                                eps=EPS)
        out = dict(zip(("y", "s"), out)) if case["next"] else {"s": out}
        into = {"y": s.get("dy"), "s": s.get("ds")}
    if not case["train"]:
        return out
    grads = torch.autograd.grad([out[k] for k in out], [s[k] for k in s["leaves"]], [into[k] for k in out])
    return out | dict(zip(["grad_" + k for k in s["leaves"]], grads))


# ------------------------------------------------------------------ the plain form


def _f(t):
    return None if t is None else t.detach().float()


def _power(log_decay, n):
    """decay^n for a tensor n of exponents, [H, *n.shape], taken in 64 bits: n times the logarithm may be large."""
    return torch.exp(log_decay.double().view(-1, *[1] * n.dim()) * n.double()).float()


def _mix(a, b, c, log_decay):
    """sum over j <= i of decay^(i-j) (a_i . b_j) c_j, by chunks: products within one, and of a with the state before it."""
    B, H, T, da = a.shape
    n = -(-T // CHUNK)
    split = lambda x: torch.nn.functional.pad(x, (0, 0, 0, n * CHUNK - T)).reshape(B, H, n, CHUNK, x.shape[-1])  # noqa: E731
    a, b, c = split(a), split(b), split(c)
    i = torch.arange(CHUNK, device=a.device)
    d = i[:, None] - i[None, :]
    w = torch.where(d >= 0, _power(log_decay, d.clamp(min=0)), torch.zeros((), device=a.device))
    o = ((a @ b.mT) * w[:, None]) @ c
    if n > 1:
        kv = (b * _power(log_decay, CHUNK - 1 - i)[:, None, :, None]).mT @ c
        m = torch.arange(n, device=a.device)
        m = m[:, None] - m[None, :] - 1
        past = torch.where(m >= 0, _power(log_decay, m.clamp(min=0) * CHUNK), torch.zeros((), device=a.device))
        before = (past @ kv.flatten(3)).view(kv.shape)
        o = o + (a * _power(log_decay, i + 1)[:, None, :, None]) @ before
    return o.reshape(B, H, n * CHUNK, -1)[:, :, :T]


def _run_plain(s):
    case, dt = s["case"], DTYPES[s["case"]["dtype"]]
    op = case["op"]
    if op == "step":
        q, k, v = _f(s["q"]), _f(s["k"]), _f(s["v"])
        s["state"].mul_(torch.exp(s["log_decay"])[:, None, None]).add_(k[..., :, None] * v[..., None, :])
        return {"o": (case["dk"] ** -0.5 * (q[..., :, None] * s["state"]).sum(-2)).to(dt), "state": s["state"]}
    if op == "decay":
        q, k, v, st, g, T = _f(s["q"]), _f(s["k"]), _f(s["v"]), _f(s["state"]), s["log_decay"], case["t"]
        sigma, live = case["dk"] ** -0.5, None
        i = torch.arange(T, device=q.device)
        if case["ragged"]:
            live = i < s["lengths"][:, None]  # [B, T]
            q, k, v = (torch.where(live[:, None, :, None], x, torch.zeros((), device=q.device)) for x in (q, k, v))
        o = _mix(q, k, v, g)
        if st is not None:
            gone = _power(g, i + 1)[None, :, :, None]  # what is left of the first state at each token
            left = (s["lengths"] if live is not None else torch.full((case["b"],), T, device=q.device))[:, None] - 1 - i
            rest = _power(g, left.clamp(min=0)).transpose(0, 1)  # and of each token at the end, [B, H, T]
            end = _power(g, left[:, 0] + 1).transpose(0, 1)[..., None, None]
            rest = rest[..., None]
            o = o + gone * (q @ st)
        out = {"o": (sigma * o).to(dt)}
        if st is not None:
            out["state"] = end * st + (rest * k).mT @ v
        if case["train"]:
            do = sigma * _f(s["do"])
            if live is not None:
                do = torch.where(live[:, None, :, None], do, torch.zeros((), device=q.device))
            dq = _mix(do, v, k, g)
            dk, dv = _mix(v.flip(2), do.flip(2), q.flip(2), g).flip(2), _mix(k.flip(2), q.flip(2), do.flip(2), g).flip(2)
            if st is not None:
                ds = _f(s["dstate"])
                dq = dq + gone * (do @ st.mT)
                dk, dv = dk + rest * (v @ ds.mT), dv + rest * (k @ ds)
                out["grad_state"] = end * ds + (gone * q).mT @ do
            if live is not None:
                dq, dk, dv = (torch.where(live[:, None, :, None], x, torch.zeros((), device=q.device)) for x in (dq, dk, dv))
            out |= {"grad_q": dq.to(dt), "grad_k": dk.to(dt), "grad_v": dv.to(dt)}
        return out
    if op == "rotary":
        turns = s["positions"].double()[:, None, :, None] * (s["freq_gpu"] / TAU)
        angle = ((turns - turns.round()) * TAU).float()
        cos, sin = torch.cos(angle) * s["mag"], torch.sin(angle) * s["mag"]

        def turn(x, sin):
            r, x = case["rot"], x.detach().float()
            x, rest = x[..., :r], x[..., r:]
            if case["pairs"] == "halves":
                a, b = x[..., : r // 2], x[..., r // 2 :]
                x = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
            else:
                a, b = x[..., ::2], x[..., 1::2]
                x = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
            return torch.cat((x, rest), -1).to(dt)

        out = {"q": turn(s["q"], sin), "k": turn(s["k"], sin)}
        if case["train"]:
            out |= {"grad_q": turn(s["dq"], -sin), "grad_k": turn(s["dk"], -sin)}
        return out
    x, w, r, gate, wn = (_f(s[k]) for k in ("x", "w", "r", "gate", "wn"))
    rx = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)
    p = x * rx * w
    a, slope = _gate(gate, case["act"]) if gate is not None else (torch.ones((), device=x.device), None)
    t = r + ALPHA * a * p
    out = {"s": t.to(dt)}
    if wn is not None:
        rt = 1 / torch.sqrt((t * t).mean(-1, keepdim=True) + EPS)
        out["y"] = (t * rt * wn).to(dt)
    if case["train"]:
        dt_ = _f(s["ds"])
        if wn is not None:
            dy, th = _f(s["dy"]), t * rt
            u = dy * wn
            dt_ = dt_ + rt * (u - th * (u * th).mean(-1, keepdim=True))
            out["grad_wn"] = (dy * th).sum((0, 1)).to(dt)
        dp, xh = ALPHA * a * dt_, x * rx
        if gate is not None:
            dg = ALPHA * slope * p * dt_
            over = {"tokens": (), "groups": (1,), "channels": (0, 1)}[case["gate"]]
            out["grad_gate"] = (dg.sum(over, keepdim=case["gate"] == "groups") if over else dg).to(dt)
        u = dp * w
        out |= {"grad_r": dt_.to(dt), "grad_w": (dp * xh).sum((0, 1)).to(dt),
                "grad_x": (rx * (u - xh * (u * xh).mean(-1, keepdim=True))).to(dt)}
    return out


def _gate(g, act):
    """The gate's activation and its derivative."""
    if act == "none":
        return g, torch.ones_like(g)
    if act == "tanh":
        t = torch.tanh(g)
        return t, 1 - t * t
    p = 1 / (1 + torch.exp(-g))
    if act == "sigmoid":
        return p, p * (1 - p)
    return g * p, p * (1 + g * (1 - p))


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return _run_plain(state)


# ------------------------------------------------------------------ 64 bits


def _attend(q, k, v, decay, state, lengths, sigma, step=256):
    """The recurrence over pieces of `step` tokens, differentiable: S_t = decay S_(t-1) + k_t v_t^T, o_t = sigma q_t S_t."""
    B, H, T, _ = q.shape
    outs, at = [], torch.arange(T, device=q.device)
    for t0 in range(0, T, step):
        t1 = min(T, t0 + step)
        a, b, c, i = q[:, :, t0:t1], k[:, :, t0:t1], v[:, :, t0:t1], at[: t1 - t0].double()
        live = (at[t0:t1] < lengths[:, None])[:, None, :, None].double()
        b, c = b * live, c * live
        gap = i[:, None] - i[None, :]
        weight = torch.tril(decay.view(-1, 1, 1) ** gap.clamp(min=0))
        o = torch.einsum("bhij,bhjd->bhid", torch.einsum("bhid,bhjd->bhij", a, b) * weight, c)
        o = o + torch.einsum("bhid,bhde,hi->bhie", a, state, decay.view(-1, 1) ** (i + 1))
        outs.append(sigma * o * live)
        n = live.sum(2)[:, 0, 0]  # tokens of this piece per sequence
        left = (n.view(-1, 1, 1) - 1 - i).clamp(min=0)
        state = state * (decay ** n.view(-1, 1))[..., None, None] + torch.einsum("bhjd,bhje,bhj->bhde", b, c, decay.view(1, -1, 1) ** left)
    return torch.cat(outs, 2), state


def exact(case, seed):
    s = prepare(case, seed)
    op, train = case["op"], bool(case.get("train"))
    d = {k: v.detach().double().requires_grad_(train and k in s.get("leaves", ())) for k, v in s.items()
         if isinstance(v, torch.Tensor) and v.is_floating_point()}
    if op in ("decay", "step"):
        decay, sigma = torch.exp(d["log_decay"]), case["dk"] ** -0.5
        if op == "step":
            st = decay[:, None, None] * d["state"] + torch.einsum("bhd,bhe->bhde", d["k"], d["v"])
            return {"o": sigma * torch.einsum("bhd,bhde->bhe", d["q"], st), "state": st}
        B, H, T = case["b"], case["h"], case["t"]
        st = d["state"] if case["state"] else torch.zeros(B, H, case["dk"], case["dv"], dtype=torch.float64, device="cuda")
        lengths = s["lengths"] if case["ragged"] else torch.full((B,), T, device="cuda")
        if case["train"] and B * H * T * (case["dk"] + case["dv"] + 256) > 1 << 30:  # the saved scores: sequences in turn
            out = {k: [] for k in ("o", "state", "grad_q", "grad_k", "grad_v", "grad_state")}
            for b in range(B):
                leaf = [d[k][b : b + 1].detach().requires_grad_() for k in ("q", "k", "v")] + [st[b : b + 1].detach().requires_grad_()]
                o, e = _attend(*leaf[:3], decay, leaf[3], lengths[b : b + 1], sigma)
                total = (o * d["do"][b : b + 1]).sum() + ((e * d["dstate"][b : b + 1]).sum() if case["state"] else 0)
                for k, x in zip(out, (o, e, *torch.autograd.grad(total, leaf))):
                    out[k].append(x.detach())
            out = {k: torch.cat(x) for k, x in out.items()}
            return out if case["state"] else {k: x for k, x in out.items() if "state" not in k}
        o, e = _attend(d["q"], d["k"], d["v"], decay, st, lengths, sigma)
        out, total = {"o": o.detach()} | ({"state": e.detach()} if case["state"] else {}), None
        if train:
            total = (o * d["do"]).sum() + ((e * d["dstate"]).sum() if case["state"] else 0)
    elif op == "rotary":
        angle = s["positions"].double()[:, None, :, None] * _frequencies(case)[0].cuda()
        unit = torch.polar(torch.full_like(angle, s["mag"]), angle)
        r = case["rot"]

        def turn(x):
            z = x[..., :r]
            z = torch.complex(*(z.chunk(2, -1) if case["pairs"] == "halves" else (z[..., ::2], z[..., 1::2]))) * unit
            z = torch.cat((z.real, z.imag), -1) if case["pairs"] == "halves" else torch.view_as_real(z.resolve_conj()).flatten(-2)
            return torch.cat((z, x[..., r:]), -1)

        q, k = turn(d["q"]), turn(d["k"])
        out = {"q": q.detach(), "k": k.detach()}
        total = (q * d["dq"]).sum() + (k * d["dk"]).sum() if train else None
    else:
        act = {"none": lambda z: z, "sigmoid": torch.sigmoid, "silu": torch.nn.functional.silu, "tanh": torch.tanh}[case["act"]]
        p = torch.nn.functional.rms_norm(d["x"], (case["c"],), d["w"], EPS)
        t = d["r"] + ALPHA * (act(d["gate"]) * p if "gate" in d else p)
        out, total = {"s": t.detach()}, (t * d["ds"]).sum() if train else None
        if case["next"]:
            y = torch.nn.functional.rms_norm(t, (case["c"],), d["wn"], EPS)
            out["y"] = y.detach()
            total = total + (y * d["dy"]).sum() if train else None
    if train:
        out |= dict(zip(["grad_" + k for k in s["leaves"]], torch.autograd.grad(total, [d[k] for k in s["leaves"]])))
    return out


def work(case):
    e = {"f32": 4, "f16": 2, "bf16": 2}[case["dtype"]]
    op = case["op"]
    if op == "step":
        n, dk, dv = case["b"] * case["h"], case["dk"], case["dv"]
        return {"bytes": n * (8 * dk * dv + e * (2 * dk + 2 * dv)), "flops": 5 * n * dk * dv}
    if op == "decay":
        n, dk, dv, t = case["b"] * case["h"], case["dk"], case["dv"], case["t"]
        train = case["train"]
        # q, k, v in and o out; training: do in, dq, dk and dv out.  A state in and a state out, each with its gradient.
        rows = n * t * e * ((4 * dk + 4 * dv) if train else (2 * dk + 2 * dv))
        states = n * dk * dv * 4 * (4 if train else 2) if case["state"] else 0
        # The recurrence: state += k v, o = q state; backward the same two again for dq, three for the state's gradient, dk and dv.
        return {"bytes": rows + states, "flops": n * t * dk * dv * (14 if train else 4)}
    if op == "rotary":
        n = case["b"] * case["t"] * (case["h"] + case["hk"])
        return {"bytes": n * case["d"] * e * (4 if case["train"] else 2) + 8 * case["b"] * case["t"],
                "flops": n * case["rot"] * 3 * (2 if case["train"] else 1)}
    n, c, train = case["groups"] * case["rows"], case["c"], case["train"]
    gates = {"none": 0, "tokens": n, "groups": case["groups"], "channels": 1}[case["gate"]]
    nxt = 1 if case["next"] else 0
    # x, r in and s (y) out; training: ds (dy) in, dx, dr out; the gate and the weights, and their gradients.
    vecs = n * (3 + nxt) + gates + 1 + nxt
    if train:
        vecs += n * (3 + nxt) + gates + 1 + nxt
    return {"bytes": vecs * c * e, "flops": n * c * (40 if train else 14)}
