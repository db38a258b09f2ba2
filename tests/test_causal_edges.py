"""CPU-side checks of the causal operators' edges: row numbers past 32 bits, tensors that stay on the host, states in place."""
import ctypes
import os
import subprocess

import pytest
import torch

from laplacianformer_b200 import capi, ops
from laplacianformer_b200.block import DecayBlock

L = capi.lib()
P = 1 << 20  # stands for a device pointer: nothing here gets as far as using it
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

GROUPS = r"""
#include <stdio.h>
#include <stdlib.h>
#include "divisor.h"
int main(int argc, char** argv) {  // rows per group, then row numbers
    const lfb::LongDivisor g(atoll(argv[1]));
    for (int i = 2; i < argc; ++i) printf("%lld\n", (long long)g.of(atoll(argv[i])));
}
"""


@pytest.fixture(scope="module")
def groups(tmp_path_factory):
    """LongDivisor, which says which gate row serves a row, compiled for the host."""
    d = tmp_path_factory.mktemp("groups")
    (d / "groups.cpp").write_text(GROUPS)
    subprocess.run(["g++", "-O1", "-std=c++17", "-I", os.path.join(ROOT, "laplacianformer_b200", "csrc"), str(d / "groups.cpp"), "-o", str(d / "groups")],
                   check=True)

    def run(each, at):
        out = subprocess.run([str(d / "groups"), str(each), *map(str, at)], check=True, capture_output=True, text=True, timeout=20)
        return [int(x) for x in out.stdout.split()]

    return run


@pytest.mark.parametrize("rows, each", [(1, 1), (12, 1), (12, 5), (12, 12), ((1 << 31) - 1, 65), ((1 << 31) - 1, (1 << 31) - 1), ((1 << 31) - 1, 3), (1 << 31, 1 << 31),
                                        (2200000000, 65), (4000000100, 197), ((1 << 32) + 5, (1 << 32) + 5), (3 << 32, 1 << 32), (1 << 33, 7), (1 << 32, (1 << 31) + 1),
                                        (1 << 40, 3), (1 << 40, 1), (1 << 40, 2), (1 << 40, (1 << 39) + 1), (1 << 40, (1 << 40) - 1)])
def test_rows_of_a_shared_gate(groups, rows, each):
    at = sorted({r for base in (0, each, 2 * each, rows, 2200000000, 1 << 31, 1 << 32, rows // 2) for r in range(base - 2, base + 3) if 0 <= r < rows})
    assert groups(each, at) == [r // each for r in at]


def test_rows_that_no_memory_holds_are_refused():
    a = capi.SandwichNorm(x=1 << 20, weight=1 << 20, residual=1 << 20, s=1 << 20, gate=1 << 20, rows=1 << 40, cols=1, rows_per_gate=2, scale=1.0, eps=1e-6,
                          dtype=capi.LF_BF16)
    assert capi.lib().lf_sandwich_norm_fwd(a, None) == capi.LF_ERR_UNSUPPORTED


@pytest.mark.parametrize("scaling", ops.ROTARY_SCALINGS)
def test_frequencies_are_on_the_host(scaling):
    """Whatever the default device is: rotary() takes them from there."""
    want = ops.rotary_frequencies(16, scaling=scaling, factor=2.0, original_length=64)
    with torch.device("meta"):
        f = ops.rotary_frequencies(16, scaling=scaling, factor=2.0, original_length=64)
        block = DecayBlock(32, 2)
    assert f.device.type == "cpu" and torch.equal(f, want)
    assert block.frequencies.device.type == "cpu" and block.log_decay.device.type == "meta"


def attention(t, **kw):
    s = (ctypes.c_int64 * 3)(t * 2 * 64, 64, 2 * 64)
    return capi.DecayAttention(**{"q": P, "k": P, "v": P, "log_decay": P, "o": P, "b": 1, "h": 2, "t": t, "key_size": 64, "value_size": 64, "scale": 0.125,
                                  "dtype": capi.LF_BF16, "q_strides": s, "k_strides": s, "v_strides": s, "do_strides": s} | kw)


def test_states_in_place_are_read_from_a_copy():
    """Where a sequence is cut, several blocks read the state that one of them writes."""
    fwd, bwd, n = L.lf_decay_attention_fwd_workspace_size, L.lf_decay_attention_bwd_workspace_size, 2 * 64 * 64 * 4
    assert fwd(attention(100, state=P, state_out=P)) == 0  # one block reads and writes it
    assert fwd(attention(5000, state=P, state_out=P)) == fwd(attention(5000, state=P, state_out=2 * P)) + n
    back = {"d_o": P, "dv": P, "d_state_out": P}
    assert bwd(attention(5000, d_state=P, **back)) == bwd(attention(5000, d_state=2 * P, **back)) + n
    for near in (P + 4, P + n - 4, P - 4, P - n + 4):
        assert L.lf_decay_attention_fwd(attention(100, state=P, state_out=near), None, 0, None) == capi.LF_ERR_INVALID and b"overlap" in L.lf_last_error()
        assert L.lf_decay_attention_bwd(attention(100, d_state=near, **back), None, 0, None) == capi.LF_ERR_INVALID and b"overlap" in L.lf_last_error()
    assert fwd(attention(5000, state=P, state_out=P + n)) == fwd(attention(5000, state=P, state_out=2 * P))
