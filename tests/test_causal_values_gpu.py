"""The causal operators at small, large and far values: fp16 operands and gradients far from 1, decays that are NaN, wide gates,
far positions, more than 2^31 rows.

Tolerances as in test_causal_gpu.py: u half a step of the type, E of fp32, 1.25 u of the norm for an attention output."""
from fractions import Fraction

import pytest
import torch

from laplacianformer_b200 import ops
from test_causal_gpu import BF16, E, F16, F32, U, decays, gen, heads, rand, within

pytestmark = pytest.mark.gpu


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
