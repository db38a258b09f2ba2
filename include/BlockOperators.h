// Block operators of the Laplace_subtraction_cuda extension: norm, matrix
// product, gated feed-forward block and gradient clipping on PyTorch tensors
// (implemented in laplacianformer_b200/csrc/torch_block_ops.cpp on top of the
// C ABI in laplacian_b200.h).  The reference has no counterpart.  Unlike its
// out-parameter operators these return their outputs, which come from the
// caching allocator on the current stream.  Undefined tensors stand for absent
// operands; gradients that are not asked for come back undefined.
#pragma once
#include <torch/types.h>

#include <tuple>
#include <vector>

namespace laplace {

// (y, s, rstd); s and rstd are undefined without a residual and without `keep`.
std::tuple<at::Tensor, at::Tensor, at::Tensor> RmsNorm_forward(const at::Tensor& x, const at::Tensor& weight,
                                                               const at::Tensor& residual, double eps, bool keep);
// (dx, dw) from dy and the gradient ds of s (may be undefined).
std::tuple<at::Tensor, at::Tensor> RmsNorm_backward(const at::Tensor& dy, const at::Tensor& ds, const at::Tensor& s,
                                                    const at::Tensor& rstd, const at::Tensor& weight, bool need_x,
                                                    bool need_w);
// (q, scale, s).
std::tuple<at::Tensor, at::Tensor, at::Tensor> RmsNorm_quant_forward(const at::Tensor& x, const at::Tensor& weight,
                                                                     const at::Tensor& residual, double eps);
// (q, scale).
std::tuple<at::Tensor, at::Tensor> Quantize_rows(const at::Tensor& x);

at::Tensor Linear_forward(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& bias,
                          const at::Tensor& residual, int64_t activation);
at::Tensor Linear_quant_forward(const at::Tensor& q, const at::Tensor& scale, const at::Tensor& weight,
                                const at::Tensor& weight_scale, const at::Tensor& bias, const at::Tensor& residual,
                                int64_t activation, at::ScalarType dtype);
// (dx, dw, db).
std::tuple<at::Tensor, at::Tensor, at::Tensor> Linear_backward(const at::Tensor& dy, const at::Tensor& x,
                                                               const at::Tensor& weight, const at::Tensor& bias,
                                                               int64_t activation, bool need_x, bool need_w,
                                                               bool need_b);

at::Tensor GatedFeedForward_forward(const at::Tensor& x, const at::Tensor& w_in, const at::Tensor& w_out,
                                    const at::Tensor& b_in, const at::Tensor& b_out, const at::Tensor& residual,
                                    int64_t activation);
// (dx, dw_in, dw_out, db_in, db_out).
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor> GatedFeedForward_backward(
    const at::Tensor& dy, const at::Tensor& x, const at::Tensor& w_in, const at::Tensor& w_out, const at::Tensor& b_in,
    int64_t activation, bool need_x, bool need_w_in, bool need_w_out, bool need_b_in, bool need_b_out);

// Writes the clipped gradients to `outs` (which may be `grads`) and returns the norm (a float32 scalar).
at::Tensor ClipGradNorm(const std::vector<const at::Tensor*>& grads, const std::vector<const at::Tensor*>& outs, double max_norm);

// The same operators as autograd nodes; without a tensor that requires a
// gradient they are the _forward functions.  RmsNorm returns (y, s).
std::tuple<at::Tensor, at::Tensor> RmsNorm(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& residual, double eps);
at::Tensor Linear(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& bias, const at::Tensor& residual,
                  int64_t activation);
at::Tensor GatedFeedForward(const at::Tensor& x, const at::Tensor& w_in, const at::Tensor& w_out, const at::Tensor& b_in,
                            const at::Tensor& b_out, const at::Tensor& residual, int64_t activation);

}  // namespace laplace
