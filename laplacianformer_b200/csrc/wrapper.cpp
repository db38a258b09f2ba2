// pybind11 module Laplace_subtraction_cuda: the reference's operator names
// and signatures (src/wrapper.cpp:73-98) plus the extended B200 operators.
#include <torch/extension.h>

#include <string>

#include "BlockOperators.h"
#include "CausalOperators.h"
#include "LaplaceSubtraction.h"
#include "NewtonInverse.h"
#include "laplacian_b200.h"

namespace laplace {

// "CUDA <major>.<minor>[.<patch>]" of the runtime the library was built with
// (reference src/wrapper.cpp:14-38).
std::string get_cuda_version() {
    int v = lf_cudart_version();
    std::string s = "CUDA " + std::to_string(v / 1000) + "." + std::to_string(v / 10 % 100);
    if (v % 10 != 0) s += "." + std::to_string(v % 10);
    return s;
}

bool has_cuda() { return true; }

// Host compiler of this extension (reference src/wrapper.cpp:42-69).  Built
// with std::to_string: std::ostringstream in this extension crashes at call
// time under torch 2.11 / pybind11 3 (the reference's helpers do too).
std::string get_compiler_version() {
#if defined(__clang_major__)
    return "clang " + std::to_string(__clang_major__) + "." + std::to_string(__clang_minor__) + "." +
           std::to_string(__clang_patchlevel__);
#elif defined(__GNUC__)
    return "GCC " + std::to_string(__GNUC__) + "." + std::to_string(__GNUC_MINOR__);
#else
    return "unknown";
#endif
}

}  // namespace laplace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    using namespace laplace;
    m.def("get_compiler_version", &get_compiler_version, "get_compiler_version");
    m.def("get_cuda_version", &get_cuda_version, "get_cuda_version");
    m.def("has_cuda", &has_cuda, "has_cuda");

    m.def("LaplaceSubtraction_forward", &LaplaceSubtraction_forward, "LaplaceSubtraction_forward");
    m.def("LaplaceSubtraction_backward_query", &LaplaceSubtraction_backward_query, "LaplaceSubtraction_backward_query");
    m.def("LaplaceSubtraction_backward_key", &LaplaceSubtraction_backward_key, "LaplaceSubtraction_backward_key");
    m.def("LaplaceSubtraction_reduce_forward", &LaplaceSubtraction_reduce_forward, "LaplaceSubtraction_reduce_forward");
    m.def("NewtonInverse_forward", &NewtonInverse_forward, "NewtonInverse_forward (mat, output, iter)");
    m.def("NewtonInverse_backward", &NewtonInverse_backward, "NewtonInverse_backward (grad_output, inverse, grad_mat)");
    m.def("NewtonInverse_is_supported", &NewtonInverse_is_supported, "NewtonInverse_is_supported (N)");

    // Extended operators (no counterpart in the reference module).
    m.def("LaplaceSubtraction_backward",
          [](const at::Tensor& g, const at::Tensor& q, const at::Tensor& k, c10::optional<at::Tensor> dq,
             c10::optional<at::Tensor> dk) {
              LaplaceSubtraction_backward(g, q, k, dq.has_value() ? *dq : at::Tensor(), dk.has_value() ? *dk : at::Tensor());
          },
          "LaplaceSubtraction_backward (gradOutput, query, key, gradQuery, gradKey): both gradients in one pass; "
          "pass an undefined tensor (None) to skip one",
          py::arg("gradOutput"), py::arg("query"), py::arg("key"), py::arg("gradQuery"), py::arg("gradKey"));
    m.def("LaplaceKernel_forward", &LaplaceKernel_forward,
          "LaplaceKernel_forward (query, key, output, scale): output = exp(scale * LaplaceSub(query, key)), fused",
          py::arg("query"), py::arg("key"), py::arg("output"), py::arg("scale"));
    m.def("LaplaceKernel_backward",
          [](const at::Tensor& g, const at::Tensor& out, double scale, const at::Tensor& q, const at::Tensor& k,
             c10::optional<at::Tensor> dq, c10::optional<at::Tensor> dk) {
              LaplaceKernel_backward(g, out, scale, q, k, dq.has_value() ? *dq : at::Tensor(),
                                     dk.has_value() ? *dk : at::Tensor());
          },
          "LaplaceKernel_backward (gradOutput, output, scale, query, key, gradQuery, gradKey): gradients of "
          "output = exp(scale * LaplaceSub(query, key)); dS = scale * output * gradOutput is formed in the kernel",
          py::arg("gradOutput"), py::arg("output"), py::arg("scale"), py::arg("query"), py::arg("key"),
          py::arg("gradQuery"), py::arg("gradKey"));
    m.def("NewtonInverse_forward_ex", &NewtonInverse_forward_ex,
          "NewtonInverse_forward_ex (mat, output, iter, init_mode, reg, precision)", py::arg("mat"), py::arg("output"),
          py::arg("iter"), py::arg("init_mode") = 0, py::arg("reg") = 0.01, py::arg("precision") = 0);
    m.def("NewtonInverse_residual", &NewtonInverse_residual,
          "NewtonInverse_residual (mat, inverse, residual, reg): ||(A + reg I) X - I||_F per matrix");

    // Block operators (no counterpart in the reference module).
    using T = c10::optional<at::Tensor>;
    auto t = [](const T& v) { return v.has_value() ? *v : at::Tensor(); };
    auto o = [](const at::Tensor& v) { return v.defined() ? T(v) : T(); };
    m.def("RmsNorm_forward",
          [=](const at::Tensor& x, const at::Tensor& w, const T& r, double eps, bool keep) {
              auto [y, s, rstd] = RmsNorm_forward(x, w, t(r), eps, keep);
              return std::make_tuple(y, o(s), o(rstd));
          },
          "RmsNorm_forward (x, weight, residual, eps, keep) -> (y, s, rstd)");
    m.def("RmsNorm_backward",
          [=](const at::Tensor& dy, const T& ds, const at::Tensor& s, const at::Tensor& rstd, const at::Tensor& w,
              bool need_x, bool need_w) {
              auto [dx, dw] = RmsNorm_backward(dy, t(ds), s, rstd, w, need_x, need_w);
              return std::make_tuple(o(dx), o(dw));
          },
          "RmsNorm_backward (dy, ds, s, rstd, weight, need_x, need_w) -> (dx, dw)");
    m.def("RmsNorm_quant_forward",
          [=](const at::Tensor& x, const at::Tensor& w, const T& r, double eps) {
              auto [q, scale, s] = RmsNorm_quant_forward(x, w, t(r), eps);
              return std::make_tuple(q, scale, o(s));
          },
          "RmsNorm_quant_forward (x, weight, residual, eps) -> (q, scale, s)");
    m.def("Quantize_rows", &Quantize_rows, "Quantize_rows (x) -> (q, scale)");
    m.def("Linear_forward",
          [=](const at::Tensor& x, const at::Tensor& w, const T& b, const T& r, int64_t act) {
              return Linear_forward(x, w, t(b), t(r), act);
          },
          "Linear_forward (x, weight, bias, residual, activation) -> y");
    m.def("Linear_quant_forward",
          [=](const at::Tensor& q, const at::Tensor& scale, const at::Tensor& w, const at::Tensor& wscale, const T& b,
              const T& r, int64_t act, bool bf16) {
              return Linear_quant_forward(q, scale, w, wscale, t(b), t(r), act, bf16 ? at::kBFloat16 : at::kHalf);
          },
          "Linear_quant_forward (q, scale, weight, weight_scale, bias, residual, activation, bf16) -> y");
    m.def("Linear_backward",
          [=](const at::Tensor& dy, const at::Tensor& x, const at::Tensor& w, const T& b, int64_t act, bool need_x,
              bool need_w, bool need_b) {
              auto [dx, dw, db] = Linear_backward(dy, x, w, t(b), act, need_x, need_w, need_b);
              return std::make_tuple(o(dx), o(dw), o(db));
          },
          "Linear_backward (dy, x, weight, bias, activation, need_x, need_w, need_b) -> (dx, dw, db)");
    m.def("GatedFeedForward_forward",
          [=](const at::Tensor& x, const at::Tensor& wi, const at::Tensor& wo, const T& bi, const T& bo, const T& r,
              int64_t act) { return GatedFeedForward_forward(x, wi, wo, t(bi), t(bo), t(r), act); },
          "GatedFeedForward_forward (x, w_in, w_out, b_in, b_out, residual, activation) -> y");
    m.def("GatedFeedForward_backward",
          [=](const at::Tensor& dy, const at::Tensor& x, const at::Tensor& wi, const at::Tensor& wo, const T& bi,
              int64_t act, bool nx, bool nwi, bool nwo, bool nbi, bool nbo) {
              auto [dx, dwi, dwo, dbi, dbo] = GatedFeedForward_backward(dy, x, wi, wo, t(bi), act, nx, nwi, nwo, nbi, nbo);
              return std::make_tuple(o(dx), o(dwi), o(dwo), o(dbi), o(dbo));
          },
          "GatedFeedForward_backward (dy, x, w_in, w_out, b_in, activation, need_x, need_w_in, need_w_out, need_b_in, "
          "need_b_out) -> (dx, dw_in, dw_out, db_in, db_out)");
    m.def("RmsNorm",
          [=](const at::Tensor& x, const at::Tensor& w, const T& r, double eps) {
              auto [y, s] = RmsNorm(x, w, t(r), eps);
              return std::make_tuple(y, o(s));
          },
          "RmsNorm (x, weight, residual, eps) -> (y, s), with autograd");
    m.def("Linear",
          [=](const at::Tensor& x, const at::Tensor& w, const T& b, const T& r, int64_t act) { return Linear(x, w, t(b), t(r), act); },
          "Linear (x, weight, bias, residual, activation) -> y, with autograd");
    m.def("GatedFeedForward",
          [=](const at::Tensor& x, const at::Tensor& wi, const at::Tensor& wo, const T& bi, const T& bo, const T& r,
              int64_t act) { return GatedFeedForward(x, wi, wo, t(bi), t(bo), t(r), act); },
          "GatedFeedForward (x, w_in, w_out, b_in, b_out, residual, activation) -> y, with autograd");
    // Causal operators (no counterpart in the reference module).
    m.def("DecayAttention_forward",
          [=](const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& g, const T& s, const T& n, double scale, bool want) {
              auto [y, e] = DecayAttention_forward(q, k, v, g, t(s), t(n), scale, want);
              return std::make_tuple(y, o(e));
          },
          "DecayAttention_forward (q, k, v, log_decay, state, lengths, scale, want_state) -> (o, state)");
    m.def("DecayAttention_backward",
          [=](const at::Tensor& d, const T& ds, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& g, const T& s,
              const T& n, double scale, bool nq, bool nk, bool nv, bool ns) {
              auto [a, b, c, e] = DecayAttention_backward(d, t(ds), q, k, v, g, t(s), t(n), scale, nq, nk, nv, ns);
              return std::make_tuple(o(a), o(b), o(c), o(e));
          },
          "DecayAttention_backward (d_o, d_state, q, k, v, log_decay, state, lengths, scale, need_q, need_k, need_v, need_state) -> "
          "(dq, dk, dv, d_state)");
    m.def("DecayAttention_step", &DecayAttention_step,
          "DecayAttention_step (q, k, v, log_decay, state, scale) -> o; state is updated in place");
    m.def("DecayAttention",
          [=](const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& g, const T& s, const T& n, double scale, bool want) {
              auto [y, e] = DecayAttention(q, k, v, g, t(s), t(n), scale, want);
              return std::make_tuple(y, o(e));
          },
          "DecayAttention (q, k, v, log_decay, state, lengths, scale, want_state) -> (o, state), with autograd");
    m.def("Rotary_forward",
          [=](const at::Tensor& q, const T& k, const at::Tensor& f, const T& pos, int64_t offset, bool interleaved, double magnitude, bool inverse) {
              auto [a, b] = Rotary_forward(q, t(k), f, t(pos), offset, interleaved, magnitude, inverse);
              return std::make_tuple(a, o(b));
          },
          "Rotary_forward (q, k, frequencies, positions, offset, interleaved, magnitude, inverse) -> (q, k)");
    m.def("Rotary",
          [=](const at::Tensor& q, const T& k, const at::Tensor& f, const T& pos, int64_t offset, bool interleaved, double magnitude) {
              auto [a, b] = Rotary(q, t(k), f, t(pos), offset, interleaved, magnitude);
              return std::make_tuple(a, o(b));
          },
          "Rotary (q, k, frequencies, positions, offset, interleaved, magnitude) -> (q, k), with autograd");
    m.def("SandwichNorm_forward",
          [=](const at::Tensor& x, const at::Tensor& w, const at::Tensor& r, const T& g, const T& n, int64_t act, double scale, double eps, bool keep) {
              auto [s, y, rstd] = SandwichNorm_forward(x, w, r, t(g), t(n), act, scale, eps, keep);
              return std::make_tuple(s, o(y), o(rstd));
          },
          "SandwichNorm_forward (x, weight, residual, gate, next_weight, gate_activation, scale, eps, keep) -> (s, y, rstd)");
    m.def("SandwichNorm_backward",
          [=](const T& ds, const T& dy, const at::Tensor& x, const at::Tensor& s, const at::Tensor& rstd, const at::Tensor& w, const T& g, const T& n,
              int64_t act, double scale, double eps, bool nx, bool nw, bool nr, bool ng, bool nn) {
              auto [a, b, c, d, e] = SandwichNorm_backward(t(ds), t(dy), x, s, rstd, w, t(g), t(n), act, scale, eps, nx, nw, nr, ng, nn);
              return std::make_tuple(o(a), o(b), o(c), o(d), o(e));
          },
          "SandwichNorm_backward (ds, dy, x, s, rstd, weight, gate, next_weight, gate_activation, scale, eps, need_x, need_w, need_r, need_g, "
          "need_n) -> (dx, dw, dr, dg, dn)");
    m.def("SandwichNorm",
          [=](const at::Tensor& x, const at::Tensor& w, const at::Tensor& r, const T& g, const T& n, int64_t act, double scale, double eps) {
              auto [s, y] = SandwichNorm(x, w, r, t(g), t(n), act, scale, eps);
              return std::make_tuple(s, o(y));
          },
          "SandwichNorm (x, weight, residual, gate, next_weight, gate_activation, scale, eps) -> (s, y), with autograd");
    // Lists are read in place: a copied Tensor per gradient would cost more than the kernels on a small model.
    auto tensors = [](const py::list& list) {
        std::vector<const at::Tensor*> v(list.size());
        for (size_t i = 0; i < v.size(); ++i) {
            PyObject* p = PyList_GET_ITEM(list.ptr(), (Py_ssize_t)i);
            TORCH_CHECK(THPVariable_Check(p), "tensors expected");
            v[i] = &THPVariable_Unpack(p);
        }
        return v;
    };
    m.def("ClipGradNorm",
          [=](const py::list& grads, const py::list& outs, double max_norm) {
              return ClipGradNorm(tensors(grads), tensors(outs), max_norm);
          },
          "ClipGradNorm (grads, outs, max_norm) -> norm");
}
