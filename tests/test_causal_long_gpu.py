"""The decayed attention on sequences of many chunks, against a 64-bit recurrence over pieces of 512 tokens for some of the heads.

Tolerances as in test_causal_gpu.py: outputs and gradients 1.25 u of their norm per head."""
import pytest
import torch

from laplacianformer_b200 import ops
from test_causal_gpu import E, F16, U, attention64, gen, heads, rel

pytestmark = pytest.mark.gpu


def pieces64(q, k, v, g, state, scale=None, absolute=False):
    """(o, state) of [B, H, T, .] by pieces, each the quadratic form."""
    parts = []
    for t in range(0, q.shape[2], 512):
        o, state = attention64(q[:, :, t : t + 512], k[:, :, t : t + 512], v[:, :, t : t + 512], g, state, None, scale, absolute)
        parts.append(o)
    return torch.cat(parts, 2), state


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
