"""CPU-side checks of the causal operators: what the C ABI and the extension refuse before any device work, workspace sizes, and
that nothing falls back to the CPU."""
import ctypes

import pytest
import torch

from laplacianformer_b200 import capi, ops

L = capi.lib()
BF16, F16, F32, F64 = capi.LF_BF16, capi.LF_F16, capi.LF_F32, capi.LF_F64
P = 1 << 20  # stands for a device pointer: nothing here gets as far as using it


def strides(h, t, d):
    return (ctypes.c_int64 * 3)(t * h * d, d, h * d)


def attention(**kw):
    b, h, t, dk, dv = 2, 3, 100, 64, 32
    s = {"q_strides": strides(h, t, dk), "k_strides": strides(h, t, dk), "v_strides": strides(h, t, dv), "do_strides": strides(h, t, dv)}
    return capi.DecayAttention(**{"q": P, "k": P, "v": P, "log_decay": P, "o": P, "b": b, "h": h, "t": t, "key_size": dk, "value_size": dv,
                                  "scale": 0.125, "dtype": BF16} | s | kw)


@pytest.mark.parametrize("change, code", [
    ({"dtype": F32}, "LF_ERR_DTYPE"), ({"dtype": F64}, "LF_ERR_DTYPE"), ({"dtype": 9}, "LF_ERR_DTYPE"), ({"b": -1}, "LF_ERR_INVALID"),
    ({"t": -1}, "LF_ERR_INVALID"), ({"key_size": 0}, "LF_ERR_INVALID"), ({"value_size": 0}, "LF_ERR_INVALID"), ({"key_size": 129}, "LF_ERR_UNSUPPORTED"),
    ({"value_size": 256}, "LF_ERR_UNSUPPORTED"), ({"scale": 0.0}, "LF_ERR_INVALID"), ({"scale": -1.0}, "LF_ERR_INVALID"), ({"scale": float("nan")}, "LF_ERR_INVALID"),
    ({"scale": float("inf")}, "LF_ERR_INVALID"), ({"q": None}, "LF_ERR_INVALID"), ({"k": None}, "LF_ERR_INVALID"), ({"v": None}, "LF_ERR_INVALID"),
    ({"o": None}, "LF_ERR_INVALID"), ({"log_decay": None}, "LF_ERR_INVALID"), ({"q": P + 1}, "LF_ERR_INVALID"), ({"o": P + 1}, "LF_ERR_INVALID"),
    ({"state": P + 2}, "LF_ERR_INVALID"), ({"lengths": P + 4}, "LF_ERR_INVALID"), ({"t": 1 << 31}, "LF_ERR_UNSUPPORTED"),
    ({"b": 1 << 24, "h": 1 << 10}, "LF_ERR_UNSUPPORTED")])
def test_attention_refusals(change, code):
    assert L.lf_decay_attention_fwd(attention(**change), None, 0, None) == getattr(capi, code)
    assert L.lf_last_error()
    assert L.lf_decay_attention_fwd_workspace_size(attention(**change)) == 0


def test_attention_workspaces():
    assert L.lf_decay_attention_fwd(None, None, 0, None) == capi.LF_ERR_INVALID
    assert L.lf_decay_attention_fwd(attention(b=0), None, 0, None) == capi.LF_OK
    assert L.lf_decay_attention_fwd_workspace_size(attention()) == 0  # one chunk per sequence, operands as they are
    odd = attention(value_size=37, v_strides=strides(3, 100, 37))
    assert L.lf_decay_attention_fwd_workspace_size(odd) == (2 * 100 * 3 * 40 * 2 + 255) // 256 * 256
    assert L.lf_decay_attention_fwd(odd, None, 0, None) == capi.LF_ERR_INVALID and b"workspace" in L.lf_last_error()
    assert L.lf_decay_attention_fwd(odd, P + 16, 1 << 30, None) == capi.LF_ERR_INVALID
    long = attention(t=5000, **{n + "_strides": strides(3, 5000, d) for n, d in (("q", 64), ("k", 64), ("v", 32))})
    need = L.lf_decay_attention_sums_size(long)  # of the segments that a sequence is cut into, 64x64 floats each
    assert need > 0 and need % (64 * 64 * 4) == 0 and L.lf_decay_attention_fwd_workspace_size(long) == need
    long.sums = P
    assert L.lf_decay_attention_fwd_workspace_size(long) == 0
    assert L.lf_decay_attention_fwd(attention(sums=P + 16), None, 0, None) == capi.LF_ERR_INVALID and b"sums" in L.lf_last_error()
    assert L.lf_decay_attention_sums_size(attention()) == 0 and L.lf_decay_attention_sums_size(None) == 0
    assert L.lf_decay_attention_bwd(attention(), None, 0, None) == capi.LF_ERR_INVALID  # no d_o
    assert L.lf_decay_attention_bwd(attention(d_o=P, d_state=P), None, 0, None) == capi.LF_ERR_INVALID  # the state's gradient without dv


def step(**kw):
    s = (ctypes.c_int64 * 2)(192, 64)
    return capi.DecayStep(**{"q": P, "k": P, "v": P, "log_decay": P, "state": P, "o": P, "b": 2, "h": 3, "key_size": 64, "value_size": 64, "scale": 0.125,
                             "dtype": F32, "q_strides": s, "k_strides": s, "v_strides": s} | kw)


@pytest.mark.parametrize("change, code", [
    ({"dtype": F64}, "LF_ERR_DTYPE"), ({"key_size": 129}, "LF_ERR_UNSUPPORTED"), ({"value_size": 0}, "LF_ERR_INVALID"), ({"scale": 0.0}, "LF_ERR_INVALID"),
    ({"state": None}, "LF_ERR_INVALID"), ({"state": P + 2}, "LF_ERR_INVALID"), ({"q": P + 2}, "LF_ERR_INVALID"), ({"o": None}, "LF_ERR_INVALID"), ({"b": -1}, "LF_ERR_INVALID")])
def test_step_refusals(change, code):
    assert L.lf_decay_attention_step(step(**change), None) == getattr(capi, code)
    assert L.lf_decay_attention_step(step(b=0), None) == capi.LF_OK


def rotary(**kw):
    s = ((ctypes.c_int64 * 3) * 2)((ctypes.c_int64 * 3)(6400, 64, 64), (ctypes.c_int64 * 3)(6400, 64, 64))
    return capi.Rotary(**{"x": (ctypes.c_void_p * 2)(P, P), "y": (ctypes.c_void_p * 2)(P, P), "strides": s, "heads": (ctypes.c_int64 * 2)(1, 1),
                          "frequencies": (ctypes.c_double * 64)(), "b": 1, "t": 100, "size": 64, "pairs": 32, "magnitude": 1.0, "dtype": BF16} | kw)


@pytest.mark.parametrize("change, code", [
    ({"dtype": F64}, "LF_ERR_DTYPE"), ({"pairs": 33}, "LF_ERR_INVALID"), ({"pairs": -1}, "LF_ERR_INVALID"), ({"size": 400, "pairs": 129}, "LF_ERR_UNSUPPORTED"),
    ({"t": 1 << 31}, "LF_ERR_UNSUPPORTED"), ({"b": 1 << 20, "t": 1 << 12}, "LF_ERR_UNSUPPORTED"), ({"frequencies": None}, "LF_ERR_INVALID"),
    ({"x": (ctypes.c_void_p * 2)(P, None)}, "LF_ERR_INVALID"), ({"y": (ctypes.c_void_p * 2)(P + 1, P)}, "LF_ERR_INVALID"), ({"positions": P + 4}, "LF_ERR_INVALID"),
    ({"t": -1}, "LF_ERR_INVALID"), ({"heads": (ctypes.c_int64 * 2)(-1, 1)}, "LF_ERR_INVALID")])
def test_rotary_refusals(change, code):
    assert L.lf_rotary(rotary(**change), None) == getattr(capi, code)
    assert L.lf_rotary(rotary(t=0), None) == capi.LF_OK and L.lf_rotary(rotary(heads=(ctypes.c_int64 * 2)(0, 0)), None) == capi.LF_OK


def sandwich(**kw):
    return capi.SandwichNorm(**{"x": P, "weight": P, "residual": P, "s": P, "rows": 12, "cols": 64, "rows_per_gate": 1, "scale": 1.0, "eps": 1e-6, "dtype": F32} | kw)


@pytest.mark.parametrize("change, code", [
    ({"dtype": F64}, "LF_ERR_DTYPE"), ({"x": None}, "LF_ERR_INVALID"), ({"weight": None}, "LF_ERR_INVALID"), ({"residual": None}, "LF_ERR_INVALID"),
    ({"s": None}, "LF_ERR_INVALID"), ({"y": P}, "LF_ERR_INVALID"), ({"next_weight": P}, "LF_ERR_INVALID"), ({"gate": P, "rows_per_gate": 5}, "LF_ERR_INVALID"),
    ({"gate": P, "rows_per_gate": 0}, "LF_ERR_INVALID"), ({"activation": 4}, "LF_ERR_INVALID"), ({"activation": -1}, "LF_ERR_INVALID"), ({"x": P + 2}, "LF_ERR_INVALID"),
    ({"rows": -1}, "LF_ERR_INVALID"), ({"cols": 1 << 31}, "LF_ERR_INVALID")])
def test_sandwich_refusals(change, code):
    assert L.lf_sandwich_norm_fwd(sandwich(**change), None) == getattr(capi, code)


def test_sandwich_sizes():
    assert L.lf_sandwich_norm_fwd(None, None) == capi.LF_ERR_INVALID
    assert L.lf_sandwich_norm_fwd(sandwich(rows=0), None) == capi.LF_OK and L.lf_sandwich_norm_fwd(sandwich(cols=0), None) == capi.LF_OK
    need = L.lf_sandwich_norm_bwd_workspace_size
    assert need(sandwich(rstd=P, ds=P, dx=P)) == 0 and need(sandwich(rstd=P, ds=P, d_weight=P)) >= 64 * 4
    bwd = L.lf_sandwich_norm_bwd
    assert bwd(sandwich(rstd=P, ds=P, d_weight=P), None, 0, None) == capi.LF_ERR_INVALID and b"workspace" in L.lf_last_error()
    assert bwd(sandwich(rstd=P, dx=P), None, 0, None) == capi.LF_ERR_INVALID  # neither ds nor dy
    assert bwd(sandwich(rstd=P, ds=P, d_gate=P), P, 1 << 20, None) == capi.LF_ERR_INVALID  # no gate
    assert bwd(sandwich(rstd=P, ds=P, d_next_weight=P, next_weight=P), P, 1 << 20, None) == capi.LF_ERR_INVALID  # no dy


def test_no_cpu_fallback():
    z = lambda *s, dt=torch.bfloat16: torch.zeros(*s, dtype=dt)  # noqa: E731
    g = torch.zeros(2)
    for call in (lambda: ops.decay_attention(z(1, 2, 3, 8), z(1, 2, 3, 8), z(1, 2, 3, 8), g),
                 lambda: ops.decay_attention_step(z(1, 2, 8), z(1, 2, 8), z(1, 2, 8), g, z(1, 2, 8, 8, dt=torch.float32)),
                 lambda: ops.rotary(z(1, 2, 3, 8), None, ops.rotary_frequencies(8)), lambda: ops.sandwich_norm(z(2, 8), z(8), z(2, 8))):
        with pytest.raises(RuntimeError, match="GPU"):
            call()


def test_names():
    with pytest.raises(ValueError, match="one of none"):
        ops.sandwich_norm(torch.zeros(1, 1), torch.zeros(1), torch.zeros(1, 1), gate_activation="relu")
    with pytest.raises(ValueError, match="one of none"):
        ops.rotary_frequencies(8, scaling="cubic")
    for bad in ({"dim": 7}, {"dim": -2}, {"dim": 8, "base": 0.0}, {"dim": 8, "factor": -1.0}, {"dim": 8, "scaling": "by_parts"},
                {"dim": 8, "scaling": "by_parts", "original_length": 100, "low": 4.0, "high": 4.0}):
        with pytest.raises(ValueError):
            ops.rotary_frequencies(**bad)
    assert ops.rotary_frequencies(0).numel() == 0
