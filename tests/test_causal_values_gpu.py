"""The causal operators at small, large and far values: fp16 operands and gradients far from 1, decays that are NaN, wide gates,
far positions, more than 2^31 rows.

Tolerances as in test_causal_gpu.py: u half a step of the type, E of fp32, 1.25 u of the norm for an attention output."""
import ctypes
from fractions import Fraction

import pytest
import torch

from laplacianformer_b200 import capi, ops
from test_causal_gpu import BF16, E, F16, F32, TINY, U, attention64, decays, gen, heads, rand, rel, within

pytestmark = pytest.mark.gpu


def off(a, b, dtype):
    """Whether a is further from b than 1.25 u of its norm and half a smallest step per value, which its own rounding takes."""
    d = (a.detach().double() - b.detach().double()).norm()
    return not float(d) <= 1.25 * U[dtype] * float(b.norm()) + TINY[dtype] * b.numel() ** 0.5


# ------------------------------------------------------------------ attention in fp16 far from 1


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("t, d", [(100, 64), (700, 64), (5000, 32), (600, 128), (150, 50)])
@pytest.mark.parametrize("sizes", [
    # binary exponents of q, k, v and do
    (0, 6, 0, -20), (6, 0, 0, -22), (3, 3, 0, -16), (-18, 0, 9, 0), (0, -14, 6, -8), (-14, 0, 6, 4), (8, 8, -9, 0), (9, 9, -14, -10), (0, 0, 8, 8)])
def test_attention_far_from_one(t, d, sizes, dtype):
    """Small gradients (and small keys, queries and values) keep their digits beside large operands that bring the results into
    range; products of large ones do not overflow."""
    g, b, h = gen(t), 2, 3
    q, k, v, do = (heads(g, b, h, t, d, dtype, 2.0**s) for s in sizes)
    dec = torch.tensor([-0.05, -0.004, 0.0], device="cuda")
    state = rand(g, b, h, d, d, scale=2.0 ** (sizes[1] + sizes[2]))
    leaves = [x.requires_grad_() for x in (q, k, v, state)]
    o, end = ops.decay_attention(q, k, v, dec, state, return_state=True)
    dend = rand(g, b, h, d, d, scale=2.0 ** (sizes[0] + sizes[3]))
    got = torch.autograd.grad((o, end), leaves, (do, dend))
    l64 = [x.detach().double().requires_grad_() for x in leaves]
    o64, end64 = attention64(*l64[:3], dec, l64[3])
    want = torch.autograd.grad((o64, end64), l64, (do.double(), dend.double()))
    u = U[dtype]
    for j in range(h):
        for name, a, c in zip(("o", "dq", "dk", "dv"), (o, *got), (o64, *want)):
            a, c = a[:, j], c[:, j]
            if float(c.abs().max()) < 60000 or dtype == BF16:  # (else the result itself is out of fp16's range)
                assert not off(a, c, dtype), (name, j, rel(a, c) / u)
        # States: u^2 of each term's size in two parts, whose last bit in fp16 is 2^-25 of 2^15 / its largest (2^-22 = u^2 at 2^-14).
        assert rel(end[:, j], end64[:, j]) <= 1.5 * u * u + 60 * E, (j, rel(end[:, j], end64[:, j]))
        assert rel(got[3][:, j], want[3][:, j]) <= 1.5 * u * u + 60 * E, (j, rel(got[3][:, j], want[3][:, j]))


@pytest.mark.parametrize("t", [96, 1000])
def test_attention_rows_of_unlike_sizes_fp16(t):
    """Each token's outputs are as good as its own operands are, beside others a million times larger (queries, gradients), and
    sums of unlike terms are as good as their largest."""
    g, b, h, d = gen(t), 1, 3, 64
    q, k, v, do = heads(g, b, h, t, d, F32), heads(g, b, h, t, d, F16), heads(g, b, h, t, d, F16), heads(g, b, h, t, d, F32)
    size = torch.where(torch.arange(t, device="cuda") % 3 == 0, 1.0, 2.0**-20)[:, None]
    q, do, k = (q * size).to(F16), (do * size).to(F16), (k * 64).to(F16)
    dec = torch.tensor([-0.05, -0.004, 0.0], device="cuda")
    leaves = [x.requires_grad_() for x in (q, k, v)]
    o = ops.decay_attention(*leaves, dec)
    got = torch.autograd.grad(o, leaves, do)
    l64 = [x.detach().double().requires_grad_() for x in leaves]
    o64, _ = attention64(*l64, dec)
    want = torch.autograd.grad(o64, l64, do.double())
    big = size[:, 0] == 1
    for name, a, c in zip(("o", "dq"), (o, got[0]), (o64, want[0])):
        for j in range(h):
            for rows in (big, ~big):
                assert not off(a[0, j, rows], c[0, j, rows], F16), (name, j, rel(a[0, j, rows], c[0, j, rows]) / U[F16])
    for name, a, c in zip(("dk", "dv"), got[1:], want[1:]):
        for j in range(h):
            assert not off(a[0, j], c[0, j], F16), (name, j)


@pytest.mark.parametrize("t, at", [(128, 64), (300, 190)])
def test_attention_beside_outliers_fp16(t, at):
    """A token 2^27 times larger than the others costs those that do not see it (before it, or where it is forgotten) nothing."""
    g, b, h, d = gen(t), 2, 3, 64
    q, k, v, do = (heads(g, b, h, t, d, F16, s) for s in (1.0, 2.0**-12, 2.0**8, 2.0**-12))
    q, k, v, do = (x.clone() for x in (q, k, v, do))
    k[:, :, at, 3], do[:, :, at, 5] = 2.0**15, 2.0**15
    dec = torch.tensor([-1.5, -0.004, 0.0], device="cuda")
    leaves = [x.requires_grad_() for x in (q, k, v)]
    o, end = ops.decay_attention(*leaves, dec, return_state=True)
    got = torch.autograd.grad(o, leaves, do)
    l64 = [x.detach().double().requires_grad_() for x in leaves]
    o64, end64 = attention64(*l64, dec)
    want = torch.autograd.grad(o64, l64, do.double())
    for j in range(h):
        # o and dq look back, dk and dv ahead; after 30 tokens the first head has e^-45 of it left.
        before, after = slice(0, at), slice(at + 1, t)
        for name, a, c, rows in (("o", o, o64, before), ("dq", got[0], want[0], before), ("dk", got[1], want[1], after), ("dv", got[2], want[2], after)):
            assert not off(a[:, j, rows], c[:, j, rows], F16), (name, j, rel(a[:, j, rows], c[:, j, rows]) / U[F16])
        if j == 0:
            before, after = slice(0, at - 30), slice(at + 30, t)
            for name, a, c, rows in (("o", o, o64, after), ("dq", got[0], want[0], after), ("dk", got[1], want[1], before), ("dv", got[2], want[2], before)):
                assert not off(a[:, j, rows], c[:, j, rows], F16), (name, j, rel(a[:, j, rows], c[:, j, rows]) / U[F16])
            assert rel(end[:, j], end64[:, j]) <= 1.5 * U[F16] ** 2 + 60 * E


@pytest.mark.parametrize("b, t, d", [(2, 900, 64), (1, 900, 128), (60, 1100, 32), (100, 1100, 128), (20, 2000, 64), (10, 2000, 128)])
@pytest.mark.parametrize("with_state", [False, True])
def test_attention_of_chunks_of_unlike_sizes_fp16(b, t, d, with_state):
    """Keys, values and gradients that grow and shrink from one chunk to the next: a state goes on through all of them."""
    g, h = gen(t + d), 3
    size = torch.tensor([1.0, 2.0**-9, 2.0**6, 0.0, 2.0**-6, 2.0**7, 2.0**-12, 1.0, 2.0**3], device="cuda").repeat(2).repeat_interleave(128)[:t, None]
    q, k, v, do = (heads(g, b, h, t, d, F32) for _ in range(4))
    q, k, v, do = q.to(F16), (k * size).to(F16), (v * size.flip(0)).to(F16), (do * size * 2.0**-4).to(F16)
    dec = torch.tensor([-0.05, -0.004, 0.0], device="cuda")
    leaves = [x.requires_grad_() for x in (q, k, v)]
    out = ops.decay_attention(*leaves, dec, return_state=with_state)
    o, end = out if with_state else (out, None)
    got = torch.autograd.grad(o, leaves, do)
    l64 = [x.detach().double().requires_grad_() for x in leaves]
    o64, end64 = attention64(*l64, dec)
    want = torch.autograd.grad(o64, l64, do.double())
    for j in range(h):
        for name, a, c in zip(("o", "dq", "dk", "dv"), (o, *got), (o64, *want)):
            for n in range(0, t, 128):
                a_, c_ = a[:, j, n : n + 128], c[:, j, n : n + 128]
                if float(c_.abs().max()) < 60000:  # (else the result itself is out of fp16's range)
                    assert not off(a_, c_, F16), (name, j, n, rel(a_, c_) / U[F16])
        if with_state:
            assert rel(end[:, j], end64[:, j]) <= 1.5 * U[F16] ** 2 + 60 * E


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_attention_of_growing_heads(dtype):
    """log_decay a little above 0: weights above 1 go the same way."""
    g, b, t, d = gen(1), 2, 300, 64
    q, k, v, do = (heads(g, b, 2, t, d, dtype) for _ in range(4))
    dec = torch.tensor([0.01, 0.03], device="cuda")
    do = do * torch.exp(dec.view(1, 2, 1, 1) * (torch.arange(t, device="cuda").view(1, 1, t, 1) - t)).to(dtype)
    leaves = [x.requires_grad_() for x in (q, k, v)]
    o, end = ops.decay_attention(*leaves, dec, return_state=True)
    got = torch.autograd.grad(o, leaves, do)
    l64 = [x.detach().double().requires_grad_() for x in leaves]
    o64, end64 = attention64(*l64, dec)
    want = torch.autograd.grad(o64, l64, do.double())
    for j in range(2):
        for a, c in zip((o, *got), (o64, *want)):
            if float(c[:, j].abs().max()) < 60000 or dtype == BF16:  # (else the result itself is out of fp16's range)
                assert not off(a[:, j], c[:, j], dtype)
        assert rel(end[:, j], end64[:, j]) <= 1.5 * U[dtype] ** 2 + 60 * E


# ------------------------------------------------------------------ decays that are NaN


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("t, with_state", [(2, False), (100, False), (128, True), (300, False)])
def test_attention_nan_decay(t, with_state, dtype):
    """A head whose decay is NaN gives NaN (the first token has met no decay yet), and its gradients are NaN; no other head's are."""
    g, b, h, d = gen(t), 2, 3, 64
    q, k, v, do = (heads(g, b, h, t, d, dtype) for _ in range(4))
    state = rand(g, b, h, d, d) if with_state else None
    good, bad = torch.tensor([-0.1, -0.5, -0.01], device="cuda"), torch.tensor([-0.1, float("nan"), -0.01], device="cuda")
    out = []
    for dec in (good, bad):
        leaves = [x.detach().requires_grad_() for x in (q, k, v)]
        o, end = ops.decay_attention(*leaves, dec, state, return_state=True)
        out.append((o, *torch.autograd.grad(o, leaves, do), end))
    for a, c in zip(*out):
        assert torch.equal(a[:, ::2], c[:, ::2])
    o, dq, dk, dv, end = out[1]
    assert torch.isnan(end[:, 1]).all() and torch.isnan(o[:, 1, 1:]).all() and torch.isnan(dq[:, 1, 1:]).all()
    assert torch.isnan(dk[:, 1, :-1]).all() and torch.isnan(dv[:, 1, :-1]).all()


# ------------------------------------------------------------------ states in place


@pytest.mark.parametrize("b, h, t, d", [(2, 3, 100, 64), (1, 2, 5000, 64), (3, 1, 2000, 128), (7, 50, 1500, 32), (2, 2, 0, 16)])
def test_attention_states_in_place(b, h, t, d):
    """C callers may have the state, and its gradient, written over the one that is read."""
    g = gen(t)
    q, k, v, do = (heads(g, b, h, t, d, BF16) for _ in range(4))
    state, dec = rand(g, b, h, d, d).requires_grad_(), torch.tensor([-0.01, -0.5, -0.0001], device="cuda").repeat(20)[:h].clone()
    o, end = ops.decay_attention(q, k, v, dec, state, return_state=True)
    dend = rand(g, b, h, d, d)
    (want,) = torch.autograd.grad((o, end), state, (do, dend))
    ptr = lambda x: x.data_ptr() or None  # noqa: E731
    mine, out, grad, dv = state.detach().clone(), torch.empty(b, t, h, d, dtype=BF16, device="cuda"), dend.clone(), torch.empty(b, t, h, d, dtype=BF16, device="cuda")
    s = (ctypes.c_int64 * 3)(t * h * d, d, h * d)
    a = capi.DecayAttention(q=ptr(q), k=ptr(k), v=ptr(v), log_decay=ptr(dec), state=ptr(mine), state_out=ptr(mine), o=ptr(out), q_strides=s, k_strides=s, v_strides=s,
                            do_strides=s, b=b, h=h, t=t, key_size=d, value_size=d, scale=d**-0.5, dtype=capi.LF_BF16)
    L, stream = capi.lib(), torch.cuda.current_stream().cuda_stream

    def call(size, run):
        n = size(a)
        ws = torch.empty(n, dtype=torch.uint8, device="cuda")
        assert run(a, ptr(ws), n, stream) == capi.LF_OK, L.lf_last_error()

    call(L.lf_decay_attention_fwd_workspace_size, L.lf_decay_attention_fwd)
    assert torch.equal(mine, end) and torch.equal(out.transpose(1, 2), o)
    a.state, a.state_out, a.d_o, a.d_state_out, a.d_state, a.dv = ptr(state), None, ptr(do), ptr(grad), ptr(grad), ptr(dv)
    call(L.lf_decay_attention_bwd_workspace_size, L.lf_decay_attention_bwd)
    assert torch.equal(grad, want)


# ------------------------------------------------------------------ gates


def gate64(z, act):
    """(value, slope, the size of the slope's terms) in 64 bits without cancellation."""
    q, p = torch.sigmoid(z), torch.sigmoid(-z)
    if act == "sigmoid":
        return q, q * p, q * p
    if act == "silu":
        return z * q, q * (1 + z * p), q * (1 + z.abs() * p)
    return torch.tanh(z), 4 * torch.sigmoid(2 * z) * torch.sigmoid(-2 * z), 4 * torch.sigmoid(2 * z) * torch.sigmoid(-2 * z)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("act", ["sigmoid", "silu", "tanh"])
@pytest.mark.parametrize("rows, c, shared", [(40, 128, False), (30, 77, False), (20, 96, True), (2, 20001, False)])
def test_gates_far_from_zero(rows, c, shared, act, dtype):
    """Gates and their slopes are as good relative to themselves where they are saturated as elsewhere.  Roundings in units of E:
    rx 8 and its products 3, the exponential 4 (of 2 z for tanh: its argument is exact), a sum and a quotient 2, products 3, the
    scale 2: below 24; the slope takes two such quotients.  16-bit gates take the hardware's exponential, off by 2 + 1.173 |z| ulps
    of 2 E: 192 E at 80."""
    g, u, fast = gen(c), U[dtype], 192 * E * (dtype != F32)
    x, w, ds = rand(g, rows, c, dtype=dtype), rand(g, c, dtype=dtype), rand(g, rows, c, dtype=dtype)
    r = torch.zeros(rows, c, dtype=dtype, device="cuda")
    lim = 80.0 if act != "tanh" else 40.0
    z = (torch.rand(1 if shared else rows, c, generator=g, device="cuda") * 2 * lim - lim).to(dtype).requires_grad_()
    s = ops.sandwich_norm(x, w, r, z[0] if shared else z, None, act, 0.7)
    (dz,) = torch.autograd.grad(s, z, ds)
    x64, z64 = x.double(), z.detach().double()
    p = 0.7 * x64 / torch.sqrt((x64 * x64).mean(-1, keepdim=True) + 1e-6) * w.double()
    val, slope, size = gate64(z64, act)
    floor = {F32: 2.0**-126, BF16: 2.0**-126, F16: 2.0**-25}[dtype]
    within(s, p * val, (u + 24 * E + fast) * (p * val).abs() + floor, "s")
    want, most = ds.double() * p * slope, (ds.double() * p).abs() * size
    if shared:
        want, most = want.sum(0, keepdim=True), most.sum(0, keepdim=True)
    within(dz, want, u * want.abs() + (60 * E + 2 * fast) * most + floor, "dgate")


# ------------------------------------------------------------------ far positions

PI = Fraction(314159265358979323846264338327950288419716939937510582097494459230781640628620899862803482534211706798, 10**101)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("start", [0, 1000003, (1 << 31) - 3, (1 << 40) + 1, (1 << 47) + 12345, (1 << 53) - 8, -(1 << 52) - 1])
def test_rotary_far_positions(start, interleaved):
    """Angles at any position that 53 bits hold: the turns are formed here with 100 digits.  16 E of a pair's length, as for near ones."""
    g, b, h, t, d = gen(1), 1, 2, 4, 32
    q = heads(g, b, h, t, d, F32)
    f = torch.cat((ops.rotary_frequencies(d)[:8], torch.tensor([1.0, 3.0, 0.7, 100.0, 1e-3, 2.5, 1.0 / 3, 6.283185307179586], dtype=torch.float64)))
    at = [start + i for i in range(t)]
    turns = [[Fraction(p) * Fraction(float(x)) / (2 * PI) for x in f] for p in at]
    angle = torch.tensor([[float((y - round(y)) * 2 * PI) for y in row] for row in turns], dtype=torch.float64, device="cuda")
    z = q.double()
    z = torch.complex(z[..., ::2], z[..., 1::2]) if interleaved else torch.complex(z[..., : d // 2], z[..., d // 2 :])
    y = z * torch.polar(torch.ones_like(angle), angle)
    for got in (ops.rotary(q, None, f, torch.tensor(at, device="cuda"), interleaved=interleaved), ops.rotary(q, None, f, offset=start, interleaved=interleaved)):
        got = got.double()
        a = torch.complex(got[..., ::2], got[..., 1::2]) if interleaved else torch.complex(got[..., : d // 2], got[..., d // 2 :])
        assert ((a - y).abs() <= 16 * E * z.abs()).all(), float(((a - y).abs() / z.abs()).max() / E)


# ------------------------------------------------------------------ more rows than 32 bits count


@pytest.mark.parametrize("groups, shared, c", [(33846154, 65, 1), (1, (1 << 31) + 5, 1), (2, (1 << 31) + 5, 1), (4200000, 524, 4)])
def test_sandwich_rows_past_32_bits(groups, shared, c):
    """A gate row serves its own rows, past the 2^31st and the 2^32nd too."""
    rows = groups * shared
    if torch.cuda.mem_get_info()[0] < rows * c * 2 * 3 + (8 << 30):
        pytest.skip("needs %d GB" % (rows * c * 6 >> 30))
    g = gen(1)
    x = torch.empty(groups, shared, c, dtype=BF16, device="cuda").normal_(generator=g)
    gate, w = torch.empty(groups, 1, c, dtype=BF16, device="cuda").normal_(generator=g), rand(g, c, dtype=BF16)
    s = ops.sandwich_norm(x, w, x, gate, None, "none", 0.5).view(rows, c)
    at = torch.cat((torch.arange(0, rows, max(1, rows // 5000), device="cuda"), torch.arange(rows - 1000, rows, device="cuda")))
    y = x.view(rows, c)[at].double()
    want = y + 0.5 * gate.view(groups, c)[at // shared].double() * y / torch.sqrt((y * y).mean(-1, keepdim=True) + 1e-6) * w.double()
    within(s[at], want, U[BF16] * want.abs() + 24 * E * (y.abs() + (want - y).abs()), "s")
