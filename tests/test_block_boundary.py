"""CPU-side checks of the block operators: what the C ABI and the extension refuse before any device work, workspace
sizes, the struct layouts, and that nothing falls back to the CPU."""
import ctypes

import pytest
import torch

from laplacianformer_b200 import capi, ops

L = capi.lib()
BF16, F16, F32, F64 = capi.LF_BF16, capi.LF_F16, capi.LF_F32, capi.LF_F64
P = 1 << 20  # stands for a device pointer: nothing here gets as far as using it


def linear(**kw):
    return capi.Linear(**{"x": P, "w": P, "y": P, "ldx": 64, "ldw": 64, "ldr": 32, "m": 100, "n": 32, "k": 64, "dtype": BF16} | kw)


def ffn(**kw):
    return capi.GatedFfn(**{"x": P, "w_in": P, "w_out": P, "y": P, "ldx": 64, "ldr": 64, "m": 100, "c": 64, "f": 96, "dtype": F16} | kw)


@pytest.mark.parametrize("change, code", [
    ({"dtype": F32}, "LF_ERR_DTYPE"), ({"dtype": F64}, "LF_ERR_DTYPE"), ({"dtype": 9}, "LF_ERR_DTYPE"),
    ({"activation": 5}, "LF_ERR_INVALID"), ({"activation": -1}, "LF_ERR_INVALID"), ({"m": -1}, "LF_ERR_INVALID"),
    ({"x": None}, "LF_ERR_INVALID"), ({"w": None}, "LF_ERR_INVALID"), ({"y": None}, "LF_ERR_INVALID"),
    ({"ldx": 63}, "LF_ERR_INVALID"), ({"ldw": 63}, "LF_ERR_INVALID"), ({"residual": P, "ldr": 31}, "LF_ERR_INVALID"),
    ({"x": P + 1}, "LF_ERR_INVALID"), ({"bias": P + 1}, "LF_ERR_INVALID"), ({"y": P + 1}, "LF_ERR_INVALID"),
    ({"m": 1 << 31}, "LF_ERR_UNSUPPORTED"), ({"n": 1 << 31, "ldr": 1 << 31}, "LF_ERR_UNSUPPORTED")])
def test_linear_refusals(change, code):
    assert L.lf_linear_fwd(linear(**change), None, 0, None) == getattr(capi, code)
    assert L.lf_last_error()


def test_linear_sizes():
    assert L.lf_linear_fwd(None, None, 0, None) == capi.LF_ERR_INVALID
    for empty in ({"m": 0}, {"n": 0}):
        assert L.lf_linear_fwd_workspace_size(linear(**empty)) == 0
        assert L.lf_linear_fwd(linear(**empty), None, 0, None) == capi.LF_OK
    assert L.lf_linear_fwd_workspace_size(linear()) == 0
    # operands that TMA cannot address are packed into the workspace: here 100 rows of 72 and 32 of 72
    odd = linear(k=65, ldx=65, ldw=65)
    assert L.lf_linear_fwd_workspace_size(odd) == (100 * 72 * 2 + 255) // 256 * 256 + (32 * 72 * 2 + 255) // 256 * 256
    assert L.lf_linear_fwd(odd, None, 0, None) == capi.LF_ERR_INVALID and b"workspace" in L.lf_last_error()
    assert L.lf_linear_fwd(odd, P + 16, 1 << 20, None) == capi.LF_ERR_INVALID
    assert L.lf_linear_bwd(linear(dx=P), None, 0, None) == capi.LF_ERR_INVALID  # no dy
    assert L.lf_linear_bwd(linear(dx=P, dy=P, lddy=31), None, 0, None) == capi.LF_ERR_INVALID
    # the recomputed dz of an activation takes workspace, the plain product's does not
    assert L.lf_linear_bwd_workspace_size(linear(dx=P, dy=P, lddy=32, activation=4)) >= 100 * 32 * 2
    assert L.lf_linear_bwd_workspace_size(linear(dx=P, dy=P, lddy=32)) == 0
    assert L.lf_linear_quant_fwd(linear(), None, 0, None) == capi.LF_ERR_INVALID  # no scales
    assert L.lf_linear_quant_fwd(linear(x_scale=P + 2, w_scale=P), None, 0, None) == capi.LF_ERR_INVALID


@pytest.mark.parametrize("change, code", [
    ({"dtype": F32}, "LF_ERR_DTYPE"), ({"activation": 7}, "LF_ERR_INVALID"), ({"f": -1}, "LF_ERR_INVALID"),
    ({"w_in": None}, "LF_ERR_INVALID"), ({"w_out": None}, "LF_ERR_INVALID"), ({"ldx": 10}, "LF_ERR_INVALID"),
    ({"residual": P, "ldr": 10}, "LF_ERR_INVALID"), ({"w_in": P + 1}, "LF_ERR_INVALID"), ({"f": 1 << 30}, "LF_ERR_UNSUPPORTED")])
def test_gated_ffn_refusals(change, code):
    assert L.lf_gated_ffn_fwd(ffn(**change), P, 1 << 30, None) == getattr(capi, code)


def test_gated_ffn_sizes():
    wide = {"c": 128, "ldx": 128, "ldr": 128}
    assert L.lf_gated_ffn_fwd_workspace_size(ffn(**wide)) >= 100 * 96 * 2  # h of 100 x 96
    assert L.lf_gated_ffn_fwd_workspace_size(ffn()) == 0  # up to 64 channels h stays in shared memory
    assert L.lf_gated_ffn_bwd_workspace_size(ffn(dy=P, lddy=128, dx=P, **wide)) >= 3 * 100 * 96 * 2  # dg, du and h
    assert L.lf_gated_ffn_bwd_workspace_size(ffn(dy=P, lddy=64, dx=P)) == 0  # these too stay there
    assert L.lf_gated_ffn_bwd_workspace_size(ffn(dy=P, lddy=64, dw_out=P)) >= 64 * 96 * 4  # its partial sums
    assert L.lf_gated_ffn_fwd(ffn(**wide), None, 0, None) == capi.LF_ERR_INVALID and b"workspace" in L.lf_last_error()
    assert L.lf_gated_ffn_bwd(ffn(dx=P), P, 1 << 30, None) == capi.LF_ERR_INVALID  # no dy
    assert L.lf_gated_ffn_fwd(ffn(m=0), None, 0, None) == capi.LF_OK


def test_norm_refusals():
    ok = dict(rows=4, cols=8)
    fwd = lambda x=P, r=None, w=P, y=P, s=None, rows=4, cols=8, dt=F32: L.lf_rms_norm_fwd(x, r, w, y, s, None, rows, cols, dt, 1e-6, None)  # noqa: E731
    assert fwd(dt=F64) == capi.LF_ERR_DTYPE and fwd(dt=7) == capi.LF_ERR_DTYPE
    assert fwd(x=None) == fwd(w=None) == fwd(y=None) == fwd(rows=-1) == fwd(cols=-1) == capi.LF_ERR_INVALID
    assert fwd(r=P) == fwd(s=P) == capi.LF_ERR_INVALID  # residual and sum go together
    assert fwd(x=P + 2) == capi.LF_ERR_INVALID and fwd(cols=1 << 31) == capi.LF_ERR_INVALID
    assert fwd(rows=0) == capi.LF_OK and fwd(cols=0) == capi.LF_OK
    need = L.lf_rms_norm_bwd_workspace_size(ok["rows"], ok["cols"])
    assert need >= ok["cols"] * 4
    assert L.lf_rms_norm_bwd(P, None, P, P, P, P, P, 4, 8, F32, None, 0, None) == capi.LF_ERR_INVALID  # dw without workspace
    assert L.lf_rms_norm_bwd(P, None, P, P, P, None, None, 4, 8, F32, None, 0, None) == capi.LF_OK  # nothing asked for
    assert L.lf_rms_norm_quant_fwd(P, None, P, None, P, None, 4, 8, F32, 1e-6, None) == capi.LF_ERR_INVALID
    assert L.lf_quantize_rows(P, P, None, 4, 8, F16, None) == capi.LF_ERR_INVALID


def test_clip_refusals():
    def clip(ptrs, outs, sizes, dts, max_norm=1.0, norm=P, ws=P, n=1 << 20):
        c = len(ptrs)
        t = lambda ty, v: (ty * max(1, c))(*v)  # noqa: E731
        return L.lf_clip_grad_norm(t(ctypes.c_void_p, ptrs), t(ctypes.c_void_p, outs), t(ctypes.c_int64, sizes), t(ctypes.c_int, dts), c,
                                   max_norm, norm, ws, n, None)

    assert clip([P], [P], [10], [F64]) == capi.LF_ERR_DTYPE
    for bad in (clip([P], [None], [10], [F32]), clip([P], [P], [-1], [F32]), clip([P + 2], [P], [10], [F32]), clip([P], [P], [10], [F32], -1.0),
                clip([P], [P], [10], [F32], float("nan")), clip([P], [P], [10], [F32], norm=None), clip([P], [P], [10], [F32], ws=None),
                clip([P], [P], [1 << 30], [F32], n=8)):
        assert bad == capi.LF_ERR_INVALID
    assert L.lf_clip_grad_norm_workspace_size((ctypes.c_int64 * 2)(1 << 20, 5), 2) > 0


def test_no_cpu_fallback():
    z = lambda *s, dt=torch.bfloat16: torch.zeros(*s, dtype=dt)  # noqa: E731
    for call in (lambda: ops.rms_norm(z(2, 8), z(8)), lambda: ops.rms_norm_quant(z(2, 8), z(8)), lambda: ops.quantize_rows(z(2, 8)),
                 lambda: ops.linear(z(2, 8), z(4, 8)), lambda: ops.gated_feed_forward(z(2, 8), z(6, 8), z(8, 3)),
                 lambda: ops.clip_grad_norm([z(3)], 1.0),
                 lambda: ops.linear_quant(z(2, 8).to(torch.float8_e4m3fn), torch.ones(2), z(4, 8).to(torch.float8_e4m3fn), torch.ones(4))):
        with pytest.raises(RuntimeError, match="GPU"):
            call()


def test_activation_names():
    assert set(ops.ACTIVATIONS) == {"none", "relu", "gelu", "gelu_tanh", "silu"}
    with pytest.raises(ValueError, match="one of none"):
        ops.linear(torch.zeros(1, 1), torch.zeros(1, 1), activation="tanh")
    with pytest.raises(TypeError, match="float16 or bfloat16"):
        ops.linear_quant(torch.zeros(1, 1), None, None, None, dtype=torch.float32)
