"""CPU-side checks of the block operators' edges: refusals that depend on empty sizes or on overlapping memory, workspace
bounds and the assignment of work units in shared launches."""
import ctypes
import os
import subprocess

import pytest

from laplacianformer_b200 import capi

L = capi.lib()
P = 1 << 20  # stands for a device pointer: nothing here gets as far as using it


# An empty sum needs no x and w, but all else that its epilogue reads.
@pytest.mark.parametrize("change", [{"residual": P, "ldr": 31}, {"ldx": -1}, {"ldw": -8}])
@pytest.mark.parametrize("x", [None, P])
def test_linear_refusals_of_empty_sums(change, x):
    a = capi.Linear(**{"x": x, "w": x, "y": P, "ldx": 0, "ldw": 0, "ldr": 32, "m": 100, "n": 32, "k": 0, "dtype": capi.LF_BF16} | change)
    assert L.lf_linear_fwd(a, None, 0, None) == capi.LF_ERR_INVALID
    a.x_scale = a.w_scale = P
    assert L.lf_linear_quant_fwd(a, None, 0, None) == capi.LF_ERR_INVALID


@pytest.mark.parametrize("x", [None, P])
@pytest.mark.parametrize("scales", [{"x_scale": P}, {"w_scale": P}, {}])
def test_linear_quant_needs_scales_of_empty_sums(x, scales):
    a = capi.Linear(x=x, w=x, y=P, m=100, n=32, k=0, dtype=capi.LF_BF16, **scales)
    assert L.lf_linear_quant_fwd(a, None, 0, None) == capi.LF_ERR_INVALID and b"scale" in L.lf_last_error()


def clip(grads, outs, sizes, dtypes):
    """lf_clip_grad_norm on (pretended) addresses; without a GPU what is not refused ends in LF_ERR_CUDA."""
    n = len(grads)
    t = lambda ty, v: (ty * n)(*v)  # noqa: E731
    return L.lf_clip_grad_norm(t(ctypes.c_void_p, grads), t(ctypes.c_void_p, outs), t(ctypes.c_int64, sizes), t(ctypes.c_int, dtypes), n, 1.0, P,
                               2 * P, 1 << 20, None)


# Tensors of 64 fp32 elements (256 bytes) at these offsets, as (grads, outs).
@pytest.mark.parametrize("grads, outs", [
    ((0, 0), (0, 0)),                        # one gradient twice, in place
    ((0, 0), (1024, 1024)),                  # one output twice
    ((0, 512), (0, 128)),                    # an output beside its own in-place neighbour's end
    ((0, 252), (0, 252)),                    # views that share an element, in place
    ((0, 512), (1024, 1276)),                # outputs that share an element
    ((0, 512), (4, 1024)),                   # an output that starts inside its gradient
    ((512, 0), (508, 1024)),                 # or ends inside it
    ((0, 512), (512, 1024)),                 # an output on another's gradient
    ((0, 512, 1024), (512, 0, 1024)),        # outputs exchanged
    ((0, 0, 512), (0, 1024, 512)),           # read again by the second gradient while the first is written
    ((4096, 0, 2048), (4096, 2052, 2048)),   # not in order of address
])
def test_clip_refuses_overlapping_tensors(grads, outs):
    base = 1 << 30
    n = len(grads)
    code = clip([base + v for v in grads], [base + v for v in outs], [64] * n, [capi.LF_F32] * n)
    assert code == capi.LF_ERR_INVALID and b"overlap" in L.lf_last_error()


def test_clip_refuses_a_view_beside_its_base():
    base = 1 << 30
    assert clip([base, base + 100], [base, base + 100], [1000, 10], [capi.LF_F16, capi.LF_BF16]) == capi.LF_ERR_INVALID
    assert clip([base + 100, base], [base + 100, base], [10, 1000], [capi.LF_F16, capi.LF_BF16]) == capi.LF_ERR_INVALID


# Rows of partial sums that the norm's backward can write: one per resident block, of at most 2048 threads an SM.  Widths
# from the narrowest row groups to rows that are read twice.
@pytest.mark.parametrize("cols, per_sm", [(64, 8), (256, 8), (512, 32), (768, 21), (1024, 16), (1536, 10), (2048, 8), (2049, 4), (8192, 4), (20000, 4)])
def test_norm_workspace_has_a_row_per_resident_block(cols, per_sm):
    sms = L.lf_rms_norm_bwd_workspace_size(1 << 20, 64) // (8 * 64 * 4)
    assert 100 <= sms <= 200
    assert L.lf_rms_norm_bwd_workspace_size(1 << 20, cols) == per_sm * sms * cols * 4
    assert L.lf_rms_norm_bwd_workspace_size(3, cols) == 3 * cols * 4


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    """The kernels' own assignment of work units, compiled for the host."""
    d = tmp_path_factory.mktemp("plan")
    (d / "plan.cpp").write_text('#include "unit_plan.h"\n'
                                'extern "C" int unit_at(int l, int e, int c, int p, int k) { return lfb::unit_at(l, e, c, p, k); }\n'
                                'extern "C" int extra_units(int l, int n, int p, double r) { return lfb::extra_units(l, n, p, r); }\n')
    csrc = os.path.join(os.path.dirname(capi.__file__), "csrc")
    subprocess.check_call(["g++", "-O1", "-shared", "-fPIC", "-I", csrc, str(d / "plan.cpp"), "-o", str(d / "plan.so")])
    lib = ctypes.CDLL(str(d / "plan.so"))
    lib.extra_units.argtypes = [ctypes.c_int, ctypes.c_int, ctypes.c_int, ctypes.c_double]
    return lib


def assigned(plan, longer, last, lanes, ratio):
    """Units of each CTA of a launch of `longer` units and `last` shorter ones on at most `lanes` CTAs."""
    total = longer + last
    P = min(lanes, total)
    extra, out = plan.extra_units(longer, last, P, ratio), []
    for c in range(P):
        mine, k = [], 0
        while (u := plan.unit_at(longer, extra, c, P, k)) < total:
            mine.append(u)
            k += 1
        out.append(mine)
    return out


@pytest.mark.parametrize("longer, last, lanes", [(1, 1, 148), (28, 36, 74), (32, 32, 74), (16, 48, 148), (64, 128, 148), (147, 1, 148), (148, 5, 148),
                                                 (149, 3, 148), (200, 400, 148), (74, 74, 74), (75, 75, 74), (1, 500, 74), (500, 1, 74), (0, 9, 74),
                                                 (30, 43, 74), (30, 45, 74), (1000, 1000, 148), (7, 0, 74)])
@pytest.mark.parametrize("ratio", [1.0, 1.4, 2.0, 3.7, 9.0])
def test_shared_launches_use_every_lane(plan, longer, last, lanes, ratio):
    """Each unit once, in rising order on a CTA, none idle while another has two, and loads within a long unit."""
    cta = assigned(plan, longer, last, lanes, ratio)
    assert sorted(u for mine in cta for u in mine) == list(range(longer + last))
    assert all(mine == sorted(mine) and mine for mine in cta)
    load = [sum(ratio if u < longer else 1 for u in mine) for mine in cta]
    assert max(load) - min(load) <= max(ratio, 1) + 1
    if longer + last <= lanes:
        assert all(len(mine) == 1 for mine in cta)
