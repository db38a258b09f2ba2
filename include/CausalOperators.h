// Causal operators of the Laplace_subtraction_cuda extension on PyTorch tensors
// (implemented in laplacianformer_b200/csrc/torch_causal_ops.cpp on top of the C
// ABI in laplacian_b200.h).  The reference has no counterpart.  They return
// their outputs, which come from the caching allocator on the current stream.
// Undefined tensors stand for absent operands; gradients that are not asked for
// come back undefined.  Heads are [batch, heads, tokens, size] with any strides
// (the last dimension contiguous, else copied); outputs lie in memory as
// [batch, tokens, heads, size].
#pragma once
#include <torch/types.h>

#include <tuple>

namespace laplace {

// (o, state after the last token, or undefined).  sums: filled for the backward, which then sums less (may stay undefined).
std::tuple<at::Tensor, at::Tensor> DecayAttention_forward(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                                          const at::Tensor& log_decay, const at::Tensor& state, const at::Tensor& lengths,
                                                          double scale, bool want_state, at::Tensor* sums = nullptr);
// (dq, dk, dv, d_state) from d_o and the gradient d_state of the last state (may be undefined).
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> DecayAttention_backward(
    const at::Tensor& d_o, const at::Tensor& d_state, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
    const at::Tensor& log_decay, const at::Tensor& state, const at::Tensor& lengths, double scale, bool need_q, bool need_k, bool need_v,
    bool need_state, const at::Tensor& sums = {});
// One token: heads are [batch, heads, size]; `state` is updated in place.
at::Tensor DecayAttention_step(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& log_decay,
                               const at::Tensor& state, double scale);

// The same as autograd nodes; without a tensor that requires a gradient they are the _forward functions.
std::tuple<at::Tensor, at::Tensor> DecayAttention(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& log_decay,
                                                  const at::Tensor& state, const at::Tensor& lengths, double scale, bool want_state);

// Queries and keys (k may be undefined) turned by their positions ([tokens] or [batch, tokens] int64, or undefined:
// offset on); frequencies is a float64 vector on the host.  `inverse` turns back, which is the backward pass.
std::tuple<at::Tensor, at::Tensor> Rotary_forward(const at::Tensor& q, const at::Tensor& k, const at::Tensor& frequencies,
                                                  const at::Tensor& positions, int64_t offset, bool interleaved, double magnitude, bool inverse);
std::tuple<at::Tensor, at::Tensor> Rotary(const at::Tensor& q, const at::Tensor& k, const at::Tensor& frequencies, const at::Tensor& positions,
                                          int64_t offset, bool interleaved, double magnitude);

// (s, y, rstd); y is undefined without a next weight, rstd without `keep`.
std::tuple<at::Tensor, at::Tensor, at::Tensor> SandwichNorm_forward(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& residual,
                                                                    const at::Tensor& gate, const at::Tensor& next, int64_t activation,
                                                                    double scale, double eps, bool keep);
// (dx, dw, dr, dg, dn) from the gradients ds and dy (one of them may be undefined).
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor> SandwichNorm_backward(
    const at::Tensor& ds, const at::Tensor& dy, const at::Tensor& x, const at::Tensor& s, const at::Tensor& rstd, const at::Tensor& weight,
    const at::Tensor& gate, const at::Tensor& next, int64_t activation, double scale, double eps, bool need_x, bool need_w, bool need_r,
    bool need_g, bool need_n);
// (s, y).
std::tuple<at::Tensor, at::Tensor> SandwichNorm(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& residual, const at::Tensor& gate,
                                                const at::Tensor& next, int64_t activation, double scale, double eps);

}  // namespace laplace
