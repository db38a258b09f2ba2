"""PyTorch autograd front end for the B200 operators.

The reference ships the two operators as raw out-parameter functions with no
``autograd.Function`` (it only exposes ``Laplace_subtraction_cuda``); the
paper's attention module calls forward and the two backward ops itself.
These wrappers give that composition:

* :func:`laplace_subtraction` — ``S = LaplaceSub(Q, K^T)``; backward runs the
  fused one-pass kernel for dQ and dK^T.
* :func:`newton_inverse` — Newton–Schulz inverse; backward is the reference's
  analytic ``-V^T G V^T`` (src/NewtonInverse_cuda_kernel.cu:466-573).

The rest of a transformer block (the reference has none of it): :func:`rms_norm`,
:func:`linear` and :func:`gated_feed_forward` with their backward passes (autograd
nodes of the extension),
:func:`rms_norm_quant`, :func:`quantize_rows` and :func:`linear_quant` for
serving with 8-bit operands, and :func:`clip_grad_norm`.

What a block that reads its tokens in order needs (none of it in the reference):
:func:`decay_attention`, its form for single tokens :func:`decay_attention_step`,
:func:`rotary`, and :func:`sandwich_norm`, the norms around a sublayer.

Every call goes to the ``Laplace_subtraction_cuda`` extension; there is no CPU
fallback and a missing extension raises ImportError.
"""
from __future__ import annotations

import math

import torch

_EXT = None


def ext():
    """The compiled Laplace_subtraction_cuda module (raises if it is missing)."""
    global _EXT
    if _EXT is None:
        try:
            import Laplace_subtraction_cuda as m  # noqa: N813
        except ImportError as e:  # pragma: no cover - depends on the build
            raise ImportError(
                "Laplace_subtraction_cuda is not built; run `python setup.py build_ext --inplace` "
                "(there is no CPU fallback for these operators)"
            ) from e
        _EXT = m
    return _EXT


INIT_REFERENCE, INIT_SCALED_TRANSPOSE = 0, 1
PREC_SPLIT3, PREC_MIXED, PREC_FP32_SIMT = 0, 1, 2


class LaplaceSubtractionFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, query, key):
        query = query.contiguous()
        key = key.contiguous()
        out = query.new_empty(query.shape[0], query.shape[1], query.shape[2], key.shape[3])
        ext().LaplaceSubtraction_forward(query, key, out)
        ctx.save_for_backward(query, key)
        return out

    @staticmethod
    def backward(ctx, grad):
        query, key = ctx.saved_tensors
        need_q, need_k = ctx.needs_input_grad[0], ctx.needs_input_grad[1]
        dq = torch.empty_like(query) if need_q else None
        dk = torch.empty_like(key) if need_k else None
        if need_q or need_k:
            ext().LaplaceSubtraction_backward(grad.contiguous(), query, key, dq, dk)
        return dq, dk


def laplace_subtraction(query: torch.Tensor, key: torch.Tensor) -> torch.Tensor:
    """S[b,h,n,m] = sum_d |query[b,h,n,d] - key[b,h,d,m]| with key given as [B,H,D,M]."""
    return LaplaceSubtractionFn.apply(query, key)


class LaplaceKernelFn(torch.autograd.Function):
    """Kmat = exp(scale * LaplaceSub(Q, K^T)), forward fused into one kernel;
    backward in one kernel too: dS = scale * Kmat * dKmat is formed while the
    fused LaplaceSub backward stages its gradient tile (LaplaceKernel_backward)."""

    @staticmethod
    def forward(ctx, query, key, scale):
        query = query.contiguous()
        key = key.contiguous()
        out = query.new_empty(query.shape[0], query.shape[1], query.shape[2], key.shape[3])
        ext().LaplaceKernel_forward(query, key, out, float(scale))
        ctx.save_for_backward(query, key, out)
        ctx.scale = float(scale)
        return out

    @staticmethod
    def backward(ctx, grad):
        query, key, out = ctx.saved_tensors
        need_q, need_k = ctx.needs_input_grad[0], ctx.needs_input_grad[1]
        dq = torch.empty_like(query) if need_q else None
        dk = torch.empty_like(key) if need_k else None
        if need_q or need_k:
            ext().LaplaceKernel_backward(grad.contiguous(), out, ctx.scale, query, key, dq, dk)
        return dq, dk, None


def laplace_kernel(query: torch.Tensor, key: torch.Tensor, scale: float) -> torch.Tensor:
    """exp(scale * sum_d |query - key|) with key given as [B,H,D,M]; S is never materialised."""
    return LaplaceKernelFn.apply(query, key, scale)


class NewtonInverseFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, mat, iters, init_mode, reg, precision):
        mat = mat.contiguous()
        out = torch.empty_like(mat)
        ext().NewtonInverse_forward_ex(mat, out, int(iters), int(init_mode), float(reg), int(precision))
        ctx.save_for_backward(out)
        return out

    @staticmethod
    def backward(ctx, grad):
        (inv,) = ctx.saved_tensors
        dmat = torch.empty_like(inv)
        ext().NewtonInverse_backward(grad.contiguous(), inv, dmat)
        return dmat, None, None, None, None


def newton_inverse(mat: torch.Tensor, iters: int, init_mode: int = INIT_REFERENCE, reg: float | None = None,
                   precision: int = PREC_SPLIT3) -> torch.Tensor:
    """Newton–Schulz inverse of [B,H,N,N] matrices (reference semantics by default)."""
    if reg is None:
        reg = 0.01 if init_mode == INIT_REFERENCE else 0.0
    return NewtonInverseFn.apply(mat, iters, init_mode, reg, precision)


class LandmarkInverseFn(torch.autograd.Function):
    """X = NewtonInverse(exp(scale * LaplaceSub(L, L^T))) with A built inside
    the inverse kernel (lf_laplace_newton_inverse_fwd).  Backward:
    dA = -X^T G X^T (the inverse's analytic backward), dS = scale * A * dA with
    A recomputed by the fused exp forward, then the LaplaceKernel backward
    (dS formed inside it) with L as both query and key: dL = dQ + (dK^T)^T."""

    @staticmethod
    def forward(ctx, lmk, scale, iters, init_mode, reg, precision):
        from . import capi

        lmk = lmk.contiguous()
        x = capi.laplace_newton_inverse_fwd(lmk, scale, iters, init_mode=init_mode, reg=reg, precision=precision)
        ctx.save_for_backward(lmk, x)
        ctx.scale = float(scale)
        return x

    @staticmethod
    def backward(ctx, grad):
        lmk, x = ctx.saved_tensors
        da = torch.empty_like(x)
        ext().NewtonInverse_backward(grad.contiguous(), x, da)
        lT = lmk.transpose(-1, -2).contiguous()
        a = torch.empty_like(x)
        ext().LaplaceKernel_forward(lmk, lT, a, ctx.scale)
        dq = torch.empty_like(lmk)
        dkT = torch.empty_like(lT)
        ext().LaplaceKernel_backward(da, a, ctx.scale, lmk, lT, dq, dkT)  # dS = scale * A * dA in the kernel
        return dq + dkT.transpose(-1, -2), None, None, None, None, None


def landmark_inverse(lmk: torch.Tensor, scale: float, iters: int, init_mode: int = INIT_REFERENCE,
                     reg: float | None = None, precision: int = PREC_SPLIT3) -> torch.Tensor:
    """Inverse of the landmark kernel matrix exp(scale * cdist_1(L, L)) for fp32 L [B,H,M,D], M <= 128,
    D <= 128, in one kernel (the matrix is never stored)."""
    if reg is None:
        reg = 0.01 if init_mode == INIT_REFERENCE else 0.0
    return LandmarkInverseFn.apply(lmk, scale, iters, init_mode, reg, precision)


def newton_residual(mat: torch.Tensor, inv: torch.Tensor, reg: float = 0.0) -> torch.Tensor:
    """||(A + reg I) X - I||_F per matrix, shape [B,H]."""
    res = torch.empty(mat.shape[0], mat.shape[1], device=mat.device,
                      dtype=torch.float64 if mat.dtype == torch.float64 else torch.float32)
    ext().NewtonInverse_residual(mat.contiguous(), inv.contiguous(), res, float(reg))
    return res


ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}


def _act(name: str) -> int:
    try:
        return ACTIVATIONS[name]
    except KeyError:
        raise ValueError(f"unknown activation {name!r}: one of {', '.join(ACTIVATIONS)}") from None


def rms_norm(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None, eps: float = 1e-6):
    """y = s / sqrt(mean(s^2) + eps) * weight over the last dimension, s = x + residual.

    Returns y, or (y, s) when a residual is given (s continues the residual
    stream).  fp32, fp16 and bf16; statistics in fp32.  Strided rows are copied first."""
    y, s = ext().RmsNorm(x, weight, residual, eps)
    return y if residual is None else (y, s)


def rms_norm_quant(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None, eps: float = 1e-6):
    """:func:`rms_norm` with its output in 8 bits, for :func:`linear_quant`: (q, scale), or (q, scale, s) with a
    residual; y is about q * scale, q float8_e4m3fn, one fp32 scale per row (max|y| / 448).  No gradient."""
    q, scale, s = ext().RmsNorm_quant_forward(x, weight, residual, eps)
    return (q, scale) if residual is None else (q, scale, s)


def quantize_rows(x: torch.Tensor):
    """(q, scale) with x about q * scale, q float8_e4m3fn and one fp32 scale per row (weights for :func:`linear_quant`)."""
    return ext().Quantize_rows(x)


def linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, activation: str = "none",
           residual: torch.Tensor | None = None) -> torch.Tensor:
    """activation(x @ weight.T + bias) + residual, finished in the product's kernel, for fp16 and bf16.

    x [..., K] (rows may be strided), weight [N, K] as torch.nn.Linear keeps it,
    bias [N], residual [..., N], all of one dtype (autocast is not followed).
    activation: none, relu, gelu, gelu_tanh or silu; the backward recomputes the
    pre-activation instead of keeping it.  Operands whose rows do not start on
    16-byte boundaries are packed in a launch before, and a product with few
    output tiles is split along K and joined in a launch after.  First order,
    reverse mode only."""
    return ext().Linear(x, weight, bias, residual, _act(activation))


def linear_quant(q: torch.Tensor, scale: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor,
                 bias: torch.Tensor | None = None, activation: str = "none", residual: torch.Tensor | None = None,
                 dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """:func:`linear` on 8-bit operands: q [..., K] and weight [N, K] float8_e4m3fn with one fp32 scale per row
    (:func:`rms_norm_quant`, :func:`quantize_rows`); bias, residual and output fp16 or bf16.  No gradient."""
    if dtype not in (torch.float16, torch.bfloat16):
        raise TypeError(f"unsupported dtype {dtype}: float16 or bfloat16")
    return ext().Linear_quant_forward(q, scale, weight, weight_scale, bias, residual, _act(activation),
                                      dtype == torch.bfloat16)


def gated_feed_forward(x: torch.Tensor, w_in: torch.Tensor, w_out: torch.Tensor, b_in: torch.Tensor | None = None,
                       b_out: torch.Tensor | None = None, activation: str = "silu",
                       residual: torch.Tensor | None = None) -> torch.Tensor:
    """(activation(g) * u) @ w_out.T + b_out + residual with [g | u] = x @ w_in.T + b_in, for fp16 and bf16.

    x [..., C], w_in [2F, C] (gate rows, then up rows), w_out [C, F], all of one
    dtype.  Gate and up projection, the activation and their product run in one
    kernel and the down projection in another; with up to 64 channels all of it
    is one kernel (except for few tokens of many hidden columns).  Between the
    passes only x is kept, the backward recomputes the projections.  In fp16 the
    hidden values and their gradients become infinite beyond 65504."""
    return ext().GatedFeedForward(x, w_in, w_out, b_in, b_out, residual, _act(activation))


def clip_grad_norm(grads, max_norm: float, out=None):
    """Global 2-norm of all tensors in `grads` and their copies scaled by min(1, max_norm / (norm + 1e-6)).

    Returns (norm, out): norm a float32 device scalar (nothing is read back to
    the host), out the clipped tensors.  `out` may be given, `grads` itself
    included (in place); written tensors may not overlap others.  fp32, fp16 and
    bf16 tensors may be mixed.  A NaN norm gives NaN, an infinite one zeros."""
    grads = list(grads)
    out = [torch.empty_like(g) for g in grads] if out is None else list(out)
    return ext().ClipGradNorm(grads, out, float(max_norm)), out


def decay_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor, state: torch.Tensor | None = None,
                    lengths: torch.Tensor | None = None, scale: float | None = None, return_state: bool = False):
    """Causal linear attention with a decay per head: S_t = exp(log_decay) S_(t-1) + k_t v_t^T, o_t = scale q_t S_t.

    q, k [B, H, N, Dk] and v [B, H, N, Dv], fp16 or bf16, sizes up to 128, with any strides (views of a joint projection
    are read in place); log_decay float32 [H], meant to be at most 0 (no gradient).  state: float32 [B, H, Dk, Dv] before
    the first token (zeros if None).  lengths: int64 [B] on the GPU, for sequences padded at their end: tokens past the
    length enter no result, and their outputs and gradients are 0.  scale defaults to Dk^-0.5.

    Returns o [B, H, N, Dv] (in memory [B, N, H, Dv], so that o.transpose(1, 2).reshape(B, N, H * Dv) copies nothing), or
    (o, state after the last token) with return_state, for the next piece of a prompt or :func:`decay_attention_step`.
    Work is linear in N, by chunks of 128 tokens on the tensor cores; a value that is not finite reaches its whole chunk.
    fp16 operands are scaled inside, so that small gradients keep their digits.  First order, reverse mode only."""
    o, s = ext().DecayAttention(q, k, v, log_decay, state, lengths, q.shape[-1] ** -0.5 if scale is None else scale, return_state)
    return (o, s) if return_state else o


def decay_attention_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor, state: torch.Tensor,
                         scale: float | None = None) -> torch.Tensor:
    """:func:`decay_attention` of one token per sequence: q, k [B, H, Dk], v [B, H, Dv] (fp32, fp16 or bf16); the state,
    contiguous float32 [B, H, Dk, Dv], is updated in place.  Returns o [B, H, Dv].  No gradient."""
    return ext().DecayAttention_step(q, k, v, log_decay, state, q.shape[-1] ** -0.5 if scale is None else scale)


ROTARY_SCALINGS = ("none", "linear", "base", "by_parts")


def rotary_frequencies(dim: int, base: float = 10000.0, scaling: str = "none", factor: float = 1.0, original_length: float | None = None,
                       low: float = 1.0, high: float = 32.0) -> torch.Tensor:
    """Radians per position of the dim / 2 pairs of :func:`rotary`, base^(-2i / dim), float64 on the host.

    For contexts `factor` times longer than the trained ones: "linear" divides all frequencies by factor (positions are
    interpolated), "base" raises the base by factor^(dim / (dim - 2)) (the last pair is interpolated, the first kept), and
    "by_parts" keeps pairs that turn over `high` times within original_length, interpolates those below `low` turns, and
    blends in between."""
    if dim < 0 or dim % 2:
        raise ValueError("dim must be even")
    if scaling not in ROTARY_SCALINGS:
        raise ValueError(f"unknown scaling {scaling!r}: one of {', '.join(ROTARY_SCALINGS)}")
    if not factor > 0 or not base > 0:
        raise ValueError("base and factor must be positive")
    if scaling == "base" and dim > 2:
        base = base * factor ** (dim / (dim - 2))
    host = {"dtype": torch.float64, "device": "cpu"}  # (whatever the default device is)
    f = torch.pow(torch.tensor(base, **host), torch.arange(0, dim, 2, **host) / -max(dim, 1))
    if scaling == "linear":
        f = f / factor
    elif scaling == "by_parts":
        if original_length is None or not high > low:
            raise ValueError("by_parts needs original_length, and high above low")
        keep = ((original_length * f / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
        f = f * (keep + (1 - keep) / factor)
    return f


def rotary(q: torch.Tensor, k: torch.Tensor | None, frequencies: torch.Tensor, positions: torch.Tensor | None = None, offset: int = 0,
           interleaved: bool = False, magnitude: float = 1.0):
    """Rotary positions: pair i of each head turns by position * frequencies[i] and is scaled by magnitude.

    q [B, H, N, D] and k [B, Hk, N, D] (or None), fp32, fp16 or bf16, with any strides; frequencies from
    :func:`rotary_frequencies` (at most 128 pairs; channels past the pairs are copied).  Pairs are channels (i, i + pairs),
    or (2i, 2i + 1) if interleaved.  positions: int64 [N] or [B, N] on the GPU, or None: offset, offset + 1 and so on.
    Angles are exact to fp32 at positions up to 2^53.

    Returns (q, k) turned, or q alone without k, in memory [B, N, H, D].  First order, reverse mode only."""
    y, z = ext().Rotary(q, k, frequencies, positions, offset, interleaved, magnitude)
    return y if k is None else (y, z)


GATE_ACTIVATIONS = {"none": 0, "sigmoid": 1, "silu": 2, "tanh": 3}


def sandwich_norm(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor, gate: torch.Tensor | None = None,
                  next_weight: torch.Tensor | None = None, gate_activation: str = "none", scale: float = 1.0, eps: float = 1e-6):
    """What lies between two sublayers: the norm after one, its gate, the residual scale, the addition, the next one's norm.

        s = residual + scale * gate_activation(gate) * rms_norm(x, weight)
        y = rms_norm(s, next_weight)

    Returns (y, s), or s alone without next_weight.  fp32, fp16 and bf16, all of one dtype; statistics in fp32, y from the
    unrounded s.  gate: x's shape (per token), [..., 1, C] (shared by the tokens of a sequence) or [C]; in general ones in
    the place of x's last dimensions before the channels.  Strided operands are copied first.  First order, reverse mode
    only."""
    try:
        act = GATE_ACTIVATIONS[gate_activation]
    except KeyError:
        raise ValueError(f"unknown gate activation {gate_activation!r}: one of {', '.join(GATE_ACTIVATIONS)}") from None
    s, y = ext().SandwichNorm(x, weight, residual, gate, next_weight, act, scale, eps)
    return s if next_weight is None else (y, s)
