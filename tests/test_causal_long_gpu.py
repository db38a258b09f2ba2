"""The decayed attention on sequences of many chunks: segments that sum their predecessors in several units, states and
outputs of heads that hardly forget, against a 64-bit recurrence over pieces of 512 tokens for some of the heads.

Tolerances as in test_causal_gpu.py: outputs and gradients 1.25 u of their norm per head.  States: u^2 of each term, and in
units of E of the state (fp32) what their sums and weights add, derived with each test."""
import pytest
import torch

from laplacianformer_b200 import ops
from test_causal_gpu import BF16, E, F16, TINY, U, attention64, gen, heads, rand, rel, within

pytestmark = pytest.mark.gpu


def pieces64(q, k, v, g, state, scale=None, absolute=False):
    """(o, state) of [B, H, T, .] by pieces, each the quadratic form."""
    parts = []
    for t in range(0, q.shape[2], 512):
        o, state = attention64(q[:, :, t : t + 512], k[:, :, t : t + 512], v[:, :, t : t + 512], g, state, None, scale, absolute)
        parts.append(o)
    return torch.cat(parts, 2), state


def fast_and_slow(h):
    """Heads that forget within a token, a chunk, a unit of chunks, a segment, and hardly at all."""
    return torch.tensor([-0.001, -0.3, -float("inf"), -0.02, -1e-5, -6.0, -0.0001, -0.1] * (h // 8 + 1), device="cuda")[:h]


# Segments of several units, the last one shorter, not joined and joined by a launch; more units than block slots; lengths that
# end inside a unit, at a segment's end and nowhere near; heads up to 64 and up to 128.
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("b, h, t, dk, dv, lengths, some", [
    (32, 2, 3136, 32, 32, None, [0, 31]), (32, 2, 3136, 32, 48, {0: 3136, 5: 2000, 31: 897, 9: 0}, [0, 5, 9, 31]), (3, 1, 41343, 64, 64, {1: 20001}, [0, 1]),
    (1, 8, 65536, 128, 128, None, [0]), (3, 8, 16384, 64, 40, {0: 5000, 2: 16000}, [0, 2]), (64, 1, 9000, 64, 64, {63: 2304, 1: 7000}, [1, 63]),
    (12, 1, 9000, 128, 96, {3: 8999}, [3, 4])])
def test_segments_of_several_units(b, h, t, dk, dv, lengths, some, dtype):
    g, u, dec = gen(t + dv), U[dtype], fast_and_slow(h)
    n = None
    if lengths is not None:
        n = torch.full((b,), t, device="cuda")
        for i, x in lengths.items():
            n[i] = x
    leaves = [heads(g, b, h, t, d, dtype).requires_grad_() for d in (dk, dk, dv)] + [rand(g, b, h, dk, dv, scale=3.0).requires_grad_()]
    o, end = ops.decay_attention(*leaves[:3], dec, leaves[3], n, return_state=True)
    do, dend = heads(g, b, h, t, dv, dtype), rand(g, b, h, dk, dv)
    got = torch.autograd.grad((o, end), leaves, (do, dend))
    for i in some:
        m = t if n is None else int(n[i])
        l64 = [x.detach()[i : i + 1].double() for x in leaves]
        l64[:3] = [x[:, :, :m] for x in l64[:3]]
        for x in l64:
            x.requires_grad_()
        if m == 0:
            assert torch.equal(end[i], leaves[3][i]) and not o[i].any() and not any(x[i].any() for x in got[:3])
            assert float((got[3][i] - dend[i]).abs().max()) <= 4 * E * float(dend[i].abs().max())
            continue
        o64, end64 = pieces64(*l64[:3], dec, l64[3])
        want = torch.autograd.grad((o64, end64), l64, (do[i : i + 1, :, :m].double(), dend[i : i + 1].double()))
        with torch.no_grad():
            size, end_size = pieces64(*l64[:3], dec, l64[3], absolute=True)
        scores = TINY[dtype] * (l64[2].detach().abs().sum(2, keepdim=True) + 1)
        within(o[i : i + 1, :, :m], o64, u * o64.abs() + (1.05 * u + 300 * E) * size + scores, "o")
        # Weights are at most 3 E off, and a sum of terms that remember 1e5 tokens has about 800 roundings, E each at most, in fp32.
        within(end[i : i + 1], end64, (1.1 * u * u + 800 * E) * end_size + TINY[dtype] * l64[2].detach().abs().sum(2)[..., None, :], "state")
        for j in range(h):
            assert rel(o[i, j, :m], o64[0, j]) <= 1.25 * u, ("o", i, j)
            assert rel(end[i, j], end64[0, j]) <= 1.5 * u * u + 144 * E, ("state", i, j, rel(end[i, j], end64[0, j]))
            for name, a, c in zip(("dq", "dk", "dv", "dstate"), got, want):
                a, c = a[i, j], c[0, j]
                if name != "dstate":
                    assert not a[m:].any()
                    a = a[:m]
                bound = 1.25 * u if name != "dstate" else 1.5 * u * u + 144 * E
                assert rel(a, c) <= bound or float(c.norm()) == 0 and not a.any(), (name, i, j, rel(a, c))


@pytest.mark.parametrize("b, t, d, memory", [(8, 1 << 20, 64, 10), (128, 16384, 64, 6), (8, 65536, 128, 6)])
def test_states_after_long_units(b, t, d, memory):
    """States that are outputs, of heads that remember 2^memory chunks, where segments sum 15 to 111 chunks of their predecessors at
    once.  In units of E of the state: a chunk's sum is cut off at most 8 times by 2 (16); weights l^n are off by 3 (two ulps, and E of
    the exponent, which is below 1 where the weight counts), at most twice for a term (6); and each chunk remembered is added with a
    rounding, up or down, that many times: sqrt(2^memory), five of them."""
    g, u = gen(b), U[F16]
    q, k, v, do = (heads(g, b, 1, t, d, F16).abs() for _ in range(4))  # (sums that grow: a cut that is always downwards shows)
    g0 = -(2.0 ** (-7 - memory))
    dec = torch.full((1,), g0, device="cuda")
    state = torch.zeros(b, 1, d, d, device="cuda").requires_grad_()
    o, end = ops.decay_attention(q, k, v, dec, state, scale=2.0**-12, return_state=True)
    (ds,) = torch.autograd.grad(o, state, do)
    i, bound = torch.arange(t, device="cuda").double(), u * u + (22 + 5 * 2.0 ** (memory / 2)) * E
    for j in (0, b - 1):
        want = (k[j, 0].double() * torch.exp(g0 * (t - 1 - i))[:, None]).mT @ v[j, 0].double()
        want_ds = (q[j, 0].double() * torch.exp(g0 * (i + 1))[:, None]).mT @ do[j, 0].double() * 2.0**-12
        assert rel(end[j, 0], want) <= bound and rel(ds[j, 0], want_ds) <= bound, (rel(end[j, 0], want) / E, rel(ds[j, 0], want_ds) / E)


@pytest.mark.parametrize("b, t, d", [(296, 65536, 32), (296, 12000, 64), (148, 30000, 128), (296, 8192, 64)])
def test_outputs_of_heads_that_forget_nothing(b, t, d):
    """Outputs from a state that grows over all chunks of one block.  Roundings to nearest leave the mean of o / o64 where it is; a sum
    that is cut off downwards does not.  A state of up to 64 chunks may be cut 16 times each by at most 2 E of it, 1 E on average, of
    a state that has grown half as far on average: 512 E.  Longer ones are added with rounded sums: 16 E for a chunk's own cuts, and
    roundings, which are as often up as down, of E at most: 16 + 64.  The roundings of n outputs, and of the d x d entries that each
    of the last 16 chunks meets (the state grows by more than a step from one to the next), scatter by u n^-1/2 or less (5 of them)."""
    if torch.cuda.mem_get_info()[0] < 30 << 30:
        pytest.skip("needs 30 GB")
    x = torch.empty(3, b, t, 1, d, dtype=F16, device="cuda").normal_(generator=gen(t)).abs_()
    q, k, v = x.transpose(2, 3)
    still, last, u = torch.zeros(1, device="cuda"), t // 512 * 512 - 2048, U[F16]
    o = ops.decay_attention(q, k, v, still, scale=2.0**-10)
    for j in (0, b - 1):
        state = torch.zeros(1, 1, d, d, dtype=torch.float64, device="cuda")
        for a in range(0, last, 4096):
            z = min(a + 4096, last)
            state += k[j : j + 1, :, a:z].double().mT @ v[j : j + 1, :, a:z].double()
        o64, _ = pieces64(*(y[j : j + 1, :, last:].double() for y in (q, k, v)), still, state, 2.0**-10)
        p = o[j : j + 1, :, last:].double()
        bias = float((p / o64 - 1).mean())
        assert abs(bias) <= (512 if t <= 8192 else 80) * E + 5 * u * (o64.numel() ** -0.5 + 0.25 / d), (bias / E, j)
        assert rel(p, o64) <= 1.25 * u
