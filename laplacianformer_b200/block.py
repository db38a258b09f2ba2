"""Transformer blocks made of the operators of :mod:`laplacianformer_b200.ops` (the reference ships no block).

:class:`LaplacianBlock`, pre-norm, around the Laplacian attention (every token sees all others of its image):

    n      = rms_norm(x)
    a      = laplacian_attention(linear(n, W_qkv, b_qkv))
    m, s   = rms_norm(linear(a, W_proj, b_proj), residual=x)      s = x + projection
    out    = gated_feed_forward(m, W_in, W_out, residual=s)

fp16 or bf16.  For serving, :meth:`LaplacianBlock.quantize_` lays the query-key-value weights out in 8 bits; the
norm then writes 8-bit activations for them (no gradient).  The 16-bit weights stay the parameter: the 8-bit ones are
made anew after they have changed, and are not part of the module's state.

:class:`DecayBlock`, around the causal linear attention with a decay per head, for sequences that grow (a token sees
those before it), with norms before and after each sublayer:

    n      = rms_norm(x)
    q, k, v = linear(n, W_qkv, b_qkv);  q, k = rotary(q, k)
    a      = decay_attention(q, k, v)
    m, s   = sandwich_norm(linear(a, W_proj, b_proj), residual=x, gate=linear(n, W_gate, b_gate))
    out    = sandwich_norm(gated_feed_forward(m, W_in, W_out), residual=s, gate=channels)

Its memory of a sequence is one matrix per head, whatever the length: a prompt leaves it behind and single tokens
update it in place.  fp16 or bf16.
"""
from __future__ import annotations

import math

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
        self._q8 = None

    @property
    def q8(self):
        """The 8-bit query-key-value weights and their scales, where they are laid out."""
        return None if self._q8 is None else self._q8[0]

    def quantize_(self) -> "LaplacianBlock":
        """Keeps the query-key-value weights in 8 bits too; forward passes without gradients use them from now on.

        They are laid out again when w_qkv has been written, replaced or moved since, when the module changes between
        train() and eval(), and within every captured graph.  The only write that this cannot see is one through
        w_qkv.data in between, which leaves no trace: call quantize_() after it."""
        self.quantized = True
        self._lay_out()
        return self

    def _lay_out(self):
        """w_qkv in 8 bits, kept with what shows that it has changed since (the parameter itself, its storage, which is
        held so that its address is not given to another, and its version) and with the stream that made it."""
        w = self.w_qkv.detach()
        pair = ops.quantize_rows(w)
        if torch.cuda.is_current_stream_capturing():
            return pair  # belongs to the graph, whose replays shall follow the weights
        stream = torch.cuda.current_stream(w.device)
        self._q8 = pair, self.w_qkv, w, None if w.is_inference() else w._version, stream, stream.record_event()
        return pair

    def _weights8(self):
        kept = self._q8  # read once: another thread may lay out at the same time
        if kept is None or torch.cuda.is_current_stream_capturing():
            return self._lay_out()
        pair, of, w, version, stream, made = kept
        if of is not self.w_qkv or w.data_ptr() != of.data_ptr() or version is None or of._version != version:
            return self._lay_out()
        here = torch.cuda.current_stream(w.device)
        if here != stream:
            here.wait_event(made)
            for t in pair:
                t.record_stream(here)
        return pair

    def __getstate__(self):  # copies and pickles lay out their own
        return {**self.__dict__, "_q8": None}

    def train(self, mode: bool = True) -> "LaplacianBlock":
        self._q8 = None
        return super().train(mode)

    def _apply(self, *args, **kwargs):  # to(), cuda(), half() and the like
        self._q8 = None
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


class DecayBlock(torch.nn.Module):
    """x [B, N, dim] -> [B, N, dim], causal; hidden defaults to 8/3 of dim, rounded up to a multiple of 64.

    decays: the factors per token by which the heads forget, log-spaced from 1 - 1/8 to 1 - 1/512 if None; they are kept
    as float32 logarithms, whatever the module is converted to.  rotary_dim: channels of each head that turn (all).
    residual_scale multiplies what the sublayers add, for deep stacks."""

    def __init__(self, dim: int, heads: int, hidden: int | None = None, decays=None, rotary_dim: int | None = None, base: float = 10000.0,
                 activation: str = "silu", residual_scale: float = 1.0, dtype: torch.dtype = torch.bfloat16, device=None):
        super().__init__()
        if dim % heads:
            raise ValueError("dim must be a multiple of heads")
        hidden = (8 * dim // 3 + 63) // 64 * 64 if hidden is None else hidden
        rotary_dim = dim // heads // 2 * 2 if rotary_dim is None else rotary_dim
        if not 0 <= rotary_dim <= dim // heads:
            raise ValueError("rotary_dim must be between 0 and the head size")
        if decays is None:
            decays = [1 - 2.0 ** -(3 + 6 * h / max(heads - 1, 1)) for h in range(heads)]
        if len(decays) != heads or not all(0 < d <= 1 for d in decays):
            raise ValueError("decays must be one factor in (0, 1] per head")
        self.heads, self.activation, self.residual_scale = heads, activation, residual_scale
        kw = {"dtype": dtype, "device": device}

        def weight(n, k):
            return torch.nn.Parameter(torch.randn(n, k, device=device).mul_(k**-0.5).to(dtype))

        def const(value, n):
            return torch.nn.Parameter(torch.full((n,), value, **kw))

        self.norm1, self.norm1_out, self.norm2, self.norm2_out = (const(1.0, dim) for _ in range(4))
        self.w_qkv, self.b_qkv = weight(3 * dim, dim), const(0.0, 3 * dim)
        self.w_gate, self.b_gate = weight(dim, dim), const(0.0, dim)
        self.w_proj, self.b_proj = weight(dim, dim), const(0.0, dim)
        self.w_in, self.w_out = weight(2 * hidden, dim), weight(dim, hidden)
        self.channels = const(1.0, dim)
        self.frequencies = ops.rotary_frequencies(rotary_dim, base)  # host
        self.register_buffer("log_decay", torch.tensor([math.log(d) for d in decays], dtype=torch.float32, device=device))

    def _apply(self, *args, **kwargs):  # to(), half() and the like leave the logarithms' type alone
        kept = self.log_decay
        super()._apply(*args, **kwargs)
        if self.log_decay.dtype != kept.dtype:
            self.log_decay = kept.to(self.log_decay.device)
        return self

    def new_state(self, batch: int) -> torch.Tensor:
        """The memory of `batch` sequences before their first token."""
        d = self.norm1.numel() // self.heads
        return torch.zeros(batch, self.heads, d, d, dtype=torch.float32, device=self.norm1.device)

    def _rest(self, a: torch.Tensor, n: torch.Tensor, x: torch.Tensor) -> torch.Tensor:
        gate = ops.linear(n, self.w_gate, self.b_gate)
        m, s = ops.sandwich_norm(ops.linear(a, self.w_proj, self.b_proj), self.norm1_out, x, gate, self.norm2, "sigmoid", self.residual_scale)
        f = ops.gated_feed_forward(m, self.w_in, self.w_out, activation=self.activation)
        return ops.sandwich_norm(f, self.norm2_out, s, self.channels, scale=self.residual_scale)

    def forward(self, x: torch.Tensor, state: torch.Tensor | None = None, lengths: torch.Tensor | None = None, offset: int = 0,
                positions: torch.Tensor | None = None, return_state: bool = False):
        """Whole sequences, or their next piece: `state` is the memory before it (nothing if None), offset the place of
        its first token (or positions, int64 [B, N] on the GPU, where sequences differ), lengths the tokens of each
        sequence in a padded batch.  Returns the outputs, or (outputs, memory after the last token)."""
        B, N, C = x.shape
        n = ops.rms_norm(x, self.norm1)
        q, k, v = ops.linear(n, self.w_qkv, self.b_qkv).view(B, N, 3, self.heads, C // self.heads).permute(2, 0, 3, 1, 4).unbind(0)
        q, k = ops.rotary(q, k, self.frequencies, positions, offset)
        a = ops.decay_attention(q, k, v, self.log_decay, state, lengths, return_state=return_state)
        a, after = a if return_state else (a, None)
        out = self._rest(a.transpose(1, 2).reshape(B, N, C), n, x)
        return (out, after) if return_state else out

    @torch.no_grad()
    def step(self, x: torch.Tensor, state: torch.Tensor, positions: torch.Tensor) -> torch.Tensor:
        """One token of each sequence, x [B, dim] at positions (int64 [B] on the GPU); the state is updated in place."""
        B, C = x.shape
        n = ops.rms_norm(x, self.norm1)
        q, k, v = ops.linear(n, self.w_qkv, self.b_qkv).view(B, 3, self.heads, 1, C // self.heads).unbind(1)
        q, k = ops.rotary(q, k, self.frequencies, positions.unsqueeze(1))
        a = ops.decay_attention_step(q.squeeze(2), k.squeeze(2), v.squeeze(2), self.log_decay, state)
        return self._rest(a.reshape(B, C), n, x)
