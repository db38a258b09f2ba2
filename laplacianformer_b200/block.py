"""A pre-norm transformer block around the Laplacian attention, made of the block operators of
:mod:`laplacianformer_b200.ops` (the reference ships no block):

    n      = rms_norm(x)
    a      = laplacian_attention(linear(n, W_qkv, b_qkv))
    m, s   = rms_norm(linear(a, W_proj, b_proj), residual=x)      s = x + projection
    out    = gated_feed_forward(m, W_in, W_out, residual=s)

fp16 or bf16.  For serving, :meth:`LaplacianBlock.quantize_` lays the query-key-value weights out in 8 bits; the
norm then writes 8-bit activations for them (no gradient).  The 16-bit weights stay the parameter: the 8-bit ones are
made anew after they have changed, and are not part of the module's state.
"""
from __future__ import annotations

import torch

from . import ops
from .attention import laplacian_attention, pool_landmarks


class LaplacianBlock(torch.nn.Module):
    """x [B, grid^2, dim] -> [B, grid^2, dim]; hidden defaults to 8/3 of dim, rounded up to a multiple of 64."""

    def __init__(self, dim: int, heads: int, grid: int, pool: int = 2, hidden: int | None = None, iters: int = 8,
                 activation: str = "silu", sigma: float | None = None, dtype: torch.dtype = torch.bfloat16, device=None):
        super().__init__()
        if dim % heads:
            raise ValueError("dim must be a multiple of heads")
        hidden = (8 * dim // 3 + 63) // 64 * 64 if hidden is None else hidden
        self.heads, self.grid, self.pool, self.iters = heads, grid, pool, iters
        self.activation, self.sigma = activation, sigma
        kw = {"dtype": dtype, "device": device}

        def weight(n, k):
            return torch.nn.Parameter(torch.randn(n, k, device=device).mul_(k**-0.5).to(dtype))

        self.norm1 = torch.nn.Parameter(torch.ones(dim, **kw))
        self.norm2 = torch.nn.Parameter(torch.ones(dim, **kw))
        self.w_qkv, self.b_qkv = weight(3 * dim, dim), torch.nn.Parameter(torch.zeros(3 * dim, **kw))
        self.w_proj, self.b_proj = weight(dim, dim), torch.nn.Parameter(torch.zeros(dim, **kw))
        self.w_in, self.w_out = weight(2 * hidden, dim), weight(dim, hidden)
        self.quantized = False
        self.q8 = self._q8_of = None

    def quantize_(self) -> "LaplacianBlock":
        """Keeps the query-key-value weights in 8 bits too; forward passes without gradients use them from now on.

        They are laid out again when w_qkv has been written, replaced or moved since, when the module changes between
        train() and eval(), and within every captured graph.  The only write that this cannot see is one through
        w_qkv.data in between, which leaves no trace: call quantize_() after it."""
        self.quantized = True
        self._lay_out()
        return self

    def _lay_out(self):
        """w_qkv in 8 bits, with what shows that it has changed since: the parameter itself, its storage (held, so that
        its address is not given to another) and its version."""
        w = self.w_qkv.detach()
        pair = ops.quantize_rows(w)
        if w.is_cuda and torch.cuda.is_current_stream_capturing():
            return pair  # belongs to the graph, whose replays shall follow the weights
        self.q8, self._q8_of = pair, (self.w_qkv, w, None if w.is_inference() else w._version)
        return pair

    def _weights8(self):
        if self._q8_of is not None and not (self.w_qkv.is_cuda and torch.cuda.is_current_stream_capturing()):
            of, w, version = self._q8_of
            if of is self.w_qkv and w.data_ptr() == of.data_ptr() and version is not None and of._version == version:
                return self.q8
        return self._lay_out()

    def _drop8(self):
        self.q8 = self._q8_of = None

    def train(self, mode: bool = True) -> "LaplacianBlock":
        self._drop8()
        return super().train(mode)

    def _apply(self, *args, **kwargs):  # to(), cuda(), half() and the like
        self._drop8()
        return super()._apply(*args, **kwargs)

    def _qkv(self, x: torch.Tensor) -> torch.Tensor:
        if self.quantized and not torch.is_grad_enabled():
            q, scale = ops.rms_norm_quant(x, self.norm1)
            return ops.linear_quant(q, scale, *self._weights8(), self.b_qkv, dtype=x.dtype)
        return ops.linear(ops.rms_norm(x, self.norm1), self.w_qkv, self.b_qkv)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        B, N, C = x.shape
        q, k, v = self._qkv(x).view(B, N, 3, self.heads, C // self.heads).permute(2, 0, 3, 1, 4).contiguous().unbind(0)
        landmarks = pool_landmarks(k, self.grid, self.pool).contiguous()
        a = laplacian_attention(q, k, v, landmarks, self.iters, self.sigma).transpose(1, 2).reshape(B, N, C)
        m, s = ops.rms_norm(ops.linear(a, self.w_proj, self.b_proj), self.norm2, residual=x)
        return ops.gated_feed_forward(m, self.w_in, self.w_out, activation=self.activation, residual=s)
