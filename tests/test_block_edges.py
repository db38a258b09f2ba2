"""CPU-side checks of the block operators' edges: refusals that depend on empty sizes or on overlapping memory, workspace
bounds and the assignment of work units in shared launches."""
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
