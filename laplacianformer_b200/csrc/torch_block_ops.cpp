// PyTorch-tensor front end of the block operators: argument checks, output and
// workspace allocation on the current stream, then one call into the C ABI.
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include "BlockOperators.h"
#include "laplacian_b200.h"

namespace laplace {
namespace {

// Messages are assembled with std::to_string (see torch_ops.cpp).
std::string num(int64_t v) { return std::to_string(v); }

int dtype_code(const at::Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return LF_F32;
        case at::kDouble: return LF_F64;
        case at::kHalf: return LF_F16;
        case at::kBFloat16: return LF_BF16;
        default: TORCH_CHECK(false, std::string("unsupported dtype ") + c10::toString(t.scalar_type()));
    }
    return -1;
}

lf_stream_t stream_of(const at::Tensor& t) {
    return reinterpret_cast<lf_stream_t>(at::cuda::getCurrentCUDAStream(t.device().index()).stream());
}

void raise_on(int rc, const char* op) {
    TORCH_CHECK(rc == LF_OK, std::string(op) + " failed (code " + num(rc) + "): " + lf_last_error());
}

void need_cuda(const at::Tensor& t, const char* name) {
    TORCH_CHECK(t.is_cuda(), std::string(name) + " must be on GPU: not implemented on the CPU");
}

// An operand beside `like`: same device and dtype.
void check_operand(const at::Tensor& t, const at::Tensor& like, const char* name) {
    need_cuda(t, name);
    TORCH_CHECK(t.device() == like.device(), std::string(name) + " must be on the input's device");
    TORCH_CHECK(t.scalar_type() == like.scalar_type(), std::string(name) + " must have the input's dtype");
}

void check_shape(const at::Tensor& t, at::IntArrayRef sizes, const char* name) {
    TORCH_CHECK(t.sizes() == sizes, std::string(name) + " has a wrong shape");
}

void check_vector(const at::Tensor& t, const at::Tensor& like, int64_t n, const char* name) {
    check_operand(t, like, name);
    TORCH_CHECK(t.dim() == 1 && t.size(0) == n, std::string(name) + " must have " + num(n) + " elements");
}

void check_matrix(const at::Tensor& t, const at::Tensor& like, int64_t rows, int64_t cols, const char* name) {
    check_operand(t, like, name);
    TORCH_CHECK(t.dim() == 2 && t.size(0) == rows && t.size(1) == cols,
                std::string(name) + " must be [" + num(rows) + ", " + num(cols) + "]");
}

int64_t rows_of(const at::Tensor& t) {
    int64_t r = 1;
    for (int64_t i = 0; i + 1 < t.dim(); ++i) r *= t.size(i);
    return r;
}

const void* ptr(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// A tensor as rows of contiguous elements: itself where its leading
// dimensions merge into one stride, else a contiguous copy.
struct Rows {
    at::Tensor t;
    int64_t ld = 0;
};
Rows as_rows(const at::Tensor& t) {
    if (!t.defined()) return {};
    const int64_t cols = t.size(-1);
    if (t.is_contiguous()) return {t, cols};
    if (t.numel() && (cols == 1 || t.stride(-1) == 1)) {
        int64_t ld = cols, span = 1;  // rows so far are ld apart, span of them
        bool merges = true;
        for (int64_t i = t.dim() - 2; i >= 0 && merges; --i) {
            if (t.size(i) == 1) continue;
            if (span == 1) ld = t.stride(i);
            else merges = t.stride(i) == ld * span;
            span *= t.size(i);
        }
        if (merges && ld >= cols) return {t, ld};  // (expanded rows have a stride of zero)
    }
    return {t.contiguous(), cols};
}

// A contiguous tensor of the caching allocator on like's device (without the
// dispatcher, which would take longer than a small operator's launch).
at::Tensor fresh(at::IntArrayRef sizes, at::ScalarType dtype, const at::Tensor& like) {
    return at::detail::empty_cuda(sizes, dtype, like.device(), c10::nullopt);
}
at::Tensor fresh(at::IntArrayRef sizes, const at::Tensor& like) { return fresh(sizes, like.scalar_type(), like); }

at::Tensor workspace(size_t bytes, const at::Tensor& like) {
    return bytes ? fresh({(int64_t)bytes}, at::kByte, like) : at::Tensor();
}

at::Tensor maybe(bool want, at::IntArrayRef sizes, const at::Tensor& like) { return want ? fresh(sizes, like) : at::Tensor(); }
void* mut(at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

at::Tensor dense(const at::Tensor& t) { return t.defined() ? t.contiguous() : t; }

std::vector<int64_t> with_last(const at::Tensor& t, int64_t n) {
    std::vector<int64_t> s = t.sizes().vec();
    s.back() = n;
    return s;
}

void check_norm(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& residual) {
    need_cuda(x, "x");
    TORCH_CHECK(x.dim() >= 1, "x must have at least one dimension");
    check_vector(weight, x, x.size(-1), "weight");
    if (residual.defined()) {
        check_operand(residual, x, "residual");
        check_shape(residual, x.sizes(), "residual");
    }
}

}  // namespace

std::tuple<at::Tensor, at::Tensor, at::Tensor> RmsNorm_forward(const at::Tensor& x_, const at::Tensor& weight_,
                                                               const at::Tensor& residual_, double eps, bool keep) {
    check_norm(x_, weight_, residual_);
    c10::cuda::CUDAGuard guard(x_.device());
    const at::Tensor x = dense(x_), weight = dense(weight_), residual = dense(residual_);
    at::Tensor y = fresh(x.sizes(), x), s, rstd;
    if (residual.defined()) s = fresh(x.sizes(), x);
    if (keep) rstd = fresh({rows_of(x)}, at::kFloat, x);
    raise_on(lf_rms_norm_fwd(ptr(x), ptr(residual), ptr(weight), mut(y), mut(s), (float*)mut(rstd), rows_of(x), x.size(-1),
                             dtype_code(x), eps, stream_of(x)),
             "RmsNorm_forward");
    return {y, s, rstd};
}

std::tuple<at::Tensor, at::Tensor> RmsNorm_backward(const at::Tensor& dy_, const at::Tensor& ds_, const at::Tensor& s_,
                                                    const at::Tensor& rstd, const at::Tensor& weight_, bool need_x,
                                                    bool need_w) {
    check_norm(s_, weight_, ds_);
    check_operand(dy_, s_, "dy");
    check_shape(dy_, s_.sizes(), "dy");
    need_cuda(rstd, "rstd");
    TORCH_CHECK(rstd.scalar_type() == at::kFloat && rstd.is_contiguous() && rstd.numel() == rows_of(s_),
                "rstd must be float32 with one value per row");
    c10::cuda::CUDAGuard guard(s_.device());
    const at::Tensor dy = dense(dy_), ds = dense(ds_), s = dense(s_), weight = dense(weight_);
    at::Tensor dx = maybe(need_x, s.sizes(), s), dw = maybe(need_w, weight.sizes(), weight);
    const int64_t rows = rows_of(s), cols = s.size(-1);
    const size_t need = need_w ? lf_rms_norm_bwd_workspace_size(rows, cols) : 0;
    at::Tensor ws = workspace(need, s);
    raise_on(lf_rms_norm_bwd(ptr(dy), ptr(ds), ptr(s), (const float*)rstd.data_ptr(), ptr(weight), mut(dx), mut(dw), rows,
                             cols, dtype_code(s), mut(ws), need, stream_of(s)),
             "RmsNorm_backward");
    return {dx, dw};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> RmsNorm_quant_forward(const at::Tensor& x_, const at::Tensor& weight_,
                                                                     const at::Tensor& residual_, double eps) {
    check_norm(x_, weight_, residual_);
    c10::cuda::CUDAGuard guard(x_.device());
    const at::Tensor x = dense(x_), weight = dense(weight_), residual = dense(residual_);
    at::Tensor q = fresh(x.sizes(), at::kFloat8_e4m3fn, x), s;
    at::Tensor scale = fresh(x.sizes().slice(0, x.dim() - 1), at::kFloat, x);
    if (residual.defined()) s = fresh(x.sizes(), x);
    raise_on(lf_rms_norm_quant_fwd(ptr(x), ptr(residual), ptr(weight), mut(q), (float*)mut(scale), mut(s), rows_of(x),
                                   x.size(-1), dtype_code(x), eps, stream_of(x)),
             "RmsNorm_quant_forward");
    return {q, scale, s};
}

std::tuple<at::Tensor, at::Tensor> Quantize_rows(const at::Tensor& x_) {
    need_cuda(x_, "x");
    TORCH_CHECK(x_.dim() >= 1, "x must have at least one dimension");
    c10::cuda::CUDAGuard guard(x_.device());
    const at::Tensor x = dense(x_);
    at::Tensor q = fresh(x.sizes(), at::kFloat8_e4m3fn, x);
    at::Tensor scale = fresh(x.sizes().slice(0, x.dim() - 1), at::kFloat, x);
    raise_on(lf_quantize_rows(ptr(x), mut(q), (float*)mut(scale), rows_of(x), x.size(-1), dtype_code(x), stream_of(x)),
             "Quantize_rows");
    return {q, scale};
}

namespace {

// Checks shared by the products; fills sizes, strides and the forward operands.
struct LinearCall {
    lf_linear_t a{};
    Rows x, w, r;
    at::Tensor bias;
};
LinearCall linear_call(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& bias, const at::Tensor& residual,
                       int64_t activation, const at::Tensor& like) {
    need_cuda(x, "x");
    TORCH_CHECK(x.dim() >= 1, "x must have at least one dimension");
    TORCH_CHECK(weight.dim() == 2, "weight must be [out features, in features]");
    check_matrix(weight, x, weight.size(0), x.size(-1), "weight");
    const int64_t n = weight.size(0);
    if (bias.defined()) check_vector(bias, like, n, "bias");
    if (residual.defined()) {
        check_operand(residual, like, "residual");
        check_shape(residual, with_last(x, n), "residual");
    }
    LinearCall c;
    c.x = as_rows(x), c.w = as_rows(weight), c.r = as_rows(residual);
    c.bias = dense(bias);
    c.a.x = ptr(c.x.t), c.a.w = ptr(c.w.t), c.a.bias = ptr(c.bias), c.a.residual = ptr(c.r.t);
    c.a.ldx = c.x.ld, c.a.ldw = c.w.ld, c.a.ldr = c.r.ld;
    c.a.m = rows_of(x), c.a.n = n, c.a.k = x.size(-1);
    c.a.activation = (int32_t)activation;
    return c;
}

}  // namespace

at::Tensor Linear_forward(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& bias, const at::Tensor& residual,
                          int64_t activation) {
    LinearCall c = linear_call(x, weight, bias, residual, activation, x);
    c10::cuda::CUDAGuard guard(x.device());
    at::Tensor y = fresh(with_last(x, c.a.n), x);
    c.a.y = y.data_ptr();
    c.a.dtype = dtype_code(x);
    const size_t need = lf_linear_fwd_workspace_size(&c.a);
    at::Tensor ws = workspace(need, x);
    raise_on(lf_linear_fwd(&c.a, mut(ws), need, stream_of(x)), "Linear_forward");
    return y;
}

at::Tensor Linear_quant_forward(const at::Tensor& q, const at::Tensor& scale, const at::Tensor& weight,
                                const at::Tensor& weight_scale, const at::Tensor& bias, const at::Tensor& residual,
                                int64_t activation, at::ScalarType dtype) {
    TORCH_CHECK(q.scalar_type() == at::kFloat8_e4m3fn, "q must be float8_e4m3fn");
    TORCH_CHECK(dtype == at::kHalf || dtype == at::kBFloat16, "dtype must be float16 or bfloat16");
    need_cuda(q, "q");
    c10::cuda::CUDAGuard guard(q.device());
    at::Tensor like = fresh({0}, dtype, q);
    LinearCall c = linear_call(q, weight, bias, residual, activation, like);
    for (const auto* s : {&scale, &weight_scale}) {
        need_cuda(*s, "scale");
        TORCH_CHECK(s->scalar_type() == at::kFloat && s->device() == q.device(), "scales must be float32 on the input's device");
    }
    TORCH_CHECK(scale.numel() == c.a.m && weight_scale.numel() == c.a.n, "scales must have one value per row");
    const at::Tensor sx = dense(scale), sw = dense(weight_scale);
    at::Tensor y = fresh(with_last(q, c.a.n), like);
    c.a.y = y.data_ptr();
    c.a.x_scale = (const float*)sx.data_ptr(), c.a.w_scale = (const float*)sw.data_ptr();
    c.a.dtype = dtype_code(like);
    const size_t need = lf_linear_quant_fwd_workspace_size(&c.a);
    at::Tensor ws = workspace(need, q);
    raise_on(lf_linear_quant_fwd(&c.a, mut(ws), need, stream_of(q)), "Linear_quant_forward");
    return y;
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> Linear_backward(const at::Tensor& dy, const at::Tensor& x,
                                                               const at::Tensor& weight, const at::Tensor& bias,
                                                               int64_t activation, bool need_x, bool need_w,
                                                               bool need_b) {
    LinearCall c = linear_call(x, weight, bias, at::Tensor(), activation, x);
    check_operand(dy, x, "dy");
    check_shape(dy, with_last(x, c.a.n), "dy");
    c10::cuda::CUDAGuard guard(x.device());
    const Rows g = as_rows(dy);
    at::Tensor dx = maybe(need_x, x.sizes(), x), dw = maybe(need_w, weight.sizes(), weight), db = maybe(need_b, {c.a.n}, x);
    c.a.dy = ptr(g.t), c.a.lddy = g.ld;
    c.a.dx = mut(dx), c.a.dw = mut(dw), c.a.db = mut(db);
    c.a.dtype = dtype_code(x);
    const size_t need = lf_linear_bwd_workspace_size(&c.a);
    at::Tensor ws = workspace(need, x);
    raise_on(lf_linear_bwd(&c.a, mut(ws), need, stream_of(x)), "Linear_backward");
    return {dx, dw, db};
}

namespace {

struct FfnCall {
    lf_gated_ffn_t a{};
    Rows x, r;
    at::Tensor w_in, w_out, b_in, b_out;
};
FfnCall ffn_call(const at::Tensor& x, const at::Tensor& w_in, const at::Tensor& w_out, const at::Tensor& b_in,
                 const at::Tensor& b_out, const at::Tensor& residual, int64_t activation) {
    need_cuda(x, "x");
    TORCH_CHECK(x.dim() >= 1, "x must have at least one dimension");
    TORCH_CHECK(w_out.dim() == 2, "w_out must be [channels, hidden]");
    const int64_t c = x.size(-1), f = w_out.size(1);
    check_matrix(w_in, x, 2 * f, c, "w_in");
    check_matrix(w_out, x, c, f, "w_out");
    if (b_in.defined()) check_vector(b_in, x, 2 * f, "b_in");
    if (b_out.defined()) check_vector(b_out, x, c, "b_out");
    if (residual.defined()) {
        check_operand(residual, x, "residual");
        check_shape(residual, x.sizes(), "residual");
    }
    FfnCall k;
    k.x = as_rows(x), k.r = as_rows(residual);
    k.w_in = dense(w_in), k.w_out = dense(w_out), k.b_in = dense(b_in), k.b_out = dense(b_out);
    k.a.x = ptr(k.x.t), k.a.w_in = ptr(k.w_in), k.a.w_out = ptr(k.w_out), k.a.b_in = ptr(k.b_in), k.a.b_out = ptr(k.b_out);
    k.a.residual = ptr(k.r.t), k.a.ldx = k.x.ld, k.a.ldr = k.r.ld;
    k.a.m = rows_of(x), k.a.c = c, k.a.f = f;
    k.a.activation = (int32_t)activation, k.a.dtype = dtype_code(x);
    return k;
}

}  // namespace

at::Tensor GatedFeedForward_forward(const at::Tensor& x, const at::Tensor& w_in, const at::Tensor& w_out,
                                    const at::Tensor& b_in, const at::Tensor& b_out, const at::Tensor& residual,
                                    int64_t activation) {
    FfnCall k = ffn_call(x, w_in, w_out, b_in, b_out, residual, activation);
    c10::cuda::CUDAGuard guard(x.device());
    at::Tensor y = fresh(x.sizes(), x);
    k.a.y = y.data_ptr();
    const size_t need = lf_gated_ffn_fwd_workspace_size(&k.a);
    at::Tensor ws = workspace(need, x);
    raise_on(lf_gated_ffn_fwd(&k.a, mut(ws), need, stream_of(x)), "GatedFeedForward_forward");
    return y;
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor> GatedFeedForward_backward(
    const at::Tensor& dy, const at::Tensor& x, const at::Tensor& w_in, const at::Tensor& w_out, const at::Tensor& b_in,
    int64_t activation, bool need_x, bool need_w_in, bool need_w_out, bool need_b_in, bool need_b_out) {
    FfnCall k = ffn_call(x, w_in, w_out, b_in, at::Tensor(), at::Tensor(), activation);
    check_operand(dy, x, "dy");
    check_shape(dy, x.sizes(), "dy");
    c10::cuda::CUDAGuard guard(x.device());
    const Rows g = as_rows(dy);
    at::Tensor dx = maybe(need_x, x.sizes(), x), dwi = maybe(need_w_in, w_in.sizes(), x), dwo = maybe(need_w_out, w_out.sizes(), x);
    at::Tensor dbi = maybe(need_b_in, {2 * k.a.f}, x), dbo = maybe(need_b_out, {k.a.c}, x);
    k.a.dy = ptr(g.t), k.a.lddy = g.ld;
    k.a.dx = mut(dx), k.a.dw_in = mut(dwi), k.a.dw_out = mut(dwo), k.a.db_in = mut(dbi), k.a.db_out = mut(dbo);
    const size_t need = lf_gated_ffn_bwd_workspace_size(&k.a);
    at::Tensor ws = workspace(need, x);
    raise_on(lf_gated_ffn_bwd(&k.a, mut(ws), need, stream_of(x)), "GatedFeedForward_backward");
    return {dx, dwi, dwo, dbi, dbo};
}

at::Tensor ClipGradNorm(const std::vector<const at::Tensor*>& grads, const std::vector<const at::Tensor*>& outs, double max_norm) {
    TORCH_CHECK(!grads.empty(), "clip_grad_norm needs at least one gradient");
    TORCH_CHECK(grads.size() == outs.size(), "one output per gradient expected");
    const size_t n = grads.size();
    std::vector<const void*> in(n);
    std::vector<void*> out(n);
    std::vector<int64_t> sizes(n);
    std::vector<int> dtypes(n);
    const at::Device device = grads[0]->device();
    for (size_t i = 0; i < n; ++i) {
        const at::Tensor &g = *grads[i], &o = *outs[i];
        need_cuda(g, "gradient");
        TORCH_CHECK(g.device() == device, "all gradients must be on one device");
        check_operand(o, g, "output");
        TORCH_CHECK(o.sizes() == g.sizes(), "an output must have its gradient's shape and strides");
        if (!g.is_contiguous() || !o.is_contiguous()) {
            TORCH_CHECK(g.is_non_overlapping_and_dense(), "gradients must be dense");
            TORCH_CHECK(o.strides() == g.strides(), "an output must have its gradient's shape and strides");
        }
        in[i] = g.data_ptr();
        out[i] = o.data_ptr();
        sizes[i] = g.numel();
        dtypes[i] = dtype_code(g);
    }
    c10::cuda::CUDAGuard guard(device);
    at::Tensor norm = fresh({}, at::kFloat, *grads[0]);
    const size_t need = lf_clip_grad_norm_workspace_size(sizes.data(), (int64_t)n);
    at::Tensor ws = workspace(need, *grads[0]);
    raise_on(lf_clip_grad_norm(in.data(), out.data(), sizes.data(), dtypes.data(), (int64_t)n, max_norm,
                               (float*)norm.data_ptr(), mut(ws), need, stream_of(*grads[0])),
             "ClipGradNorm");
    // The outputs were written behind autograd's back: tell it, so that a
    // backward pass that saved one of them is refused.
    for (const at::Tensor* o : outs)
        if (!o->is_inference()) o->unsafeGetTensorImpl()->bump_version();
    return norm;
}

// ---------------------------------------------------------------------------
// Autograd nodes.  They live here rather than in Python because a small
// training step spends more time in Python nodes than in the kernels.
// ---------------------------------------------------------------------------
namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

at::Tensor opt(const c10::optional<at::Tensor>& t) { return t.has_value() ? *t : at::Tensor(); }
c10::optional<at::Tensor> as_opt(const at::Tensor& t) { return t.defined() ? c10::optional<at::Tensor>(t) : c10::nullopt; }

void first_order(const char* op) {
    TORCH_CHECK(!at::GradMode::is_enabled(), std::string(op) + " has no second derivative (create_graph is not supported)");
}

struct RmsNormNode : torch::autograd::Function<RmsNormNode> {
    static variable_list forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& weight,
                                 const c10::optional<at::Tensor>& residual, double eps) {
        at::AutoDispatchBelowADInplaceOrView below;
        auto [y, s, rstd] = RmsNorm_forward(x, weight, opt(residual), eps, true);
        ctx->save_for_backward({s.defined() ? s : x, rstd, weight});
        ctx->saved_data["residual"] = s.defined();
        ctx->set_materialize_grads(false);
        if (s.defined()) return {y, s};
        return {y};
    }
    static variable_list backward(AutogradContext* ctx, variable_list g) {
        first_order("rms_norm");
        const auto saved = ctx->get_saved_variables();
        const bool residual = ctx->saved_data["residual"].toBool();
        const at::Tensor ds = residual ? g[1] : at::Tensor();
        // Inputs of the node: x, weight and, where given, the residual.
        const bool nx = ctx->needs_input_grad(0), nw = ctx->needs_input_grad(1), nr = residual && ctx->needs_input_grad(2);
        at::Tensor dx, dw;
        if (!g[0].defined()) dx = ds;  // only the sum was used: its gradient passes through
        else std::tie(dx, dw) = RmsNorm_backward(g[0], ds, saved[0], saved[1], saved[2], nx || nr, nw);
        return {nx ? dx : at::Tensor(), dw, nr ? dx : at::Tensor(), at::Tensor()};
    }
};

struct LinearNode : torch::autograd::Function<LinearNode> {
    static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& weight,
                              const c10::optional<at::Tensor>& bias, const c10::optional<at::Tensor>& residual, int64_t act) {
        at::AutoDispatchBelowADInplaceOrView below;
        ctx->save_for_backward({x, weight, opt(bias)});
        ctx->saved_data["act"] = act;
        ctx->saved_data["residual"] = residual.has_value();
        return Linear_forward(x, weight, opt(bias), opt(residual), act);
    }
    static variable_list backward(AutogradContext* ctx, variable_list g) {
        first_order("linear");
        const auto saved = ctx->get_saved_variables();
        const bool bias = saved[2].defined(), residual = ctx->saved_data["residual"].toBool();
        const bool nx = ctx->needs_input_grad(0), nw = ctx->needs_input_grad(1), nb = bias && ctx->needs_input_grad(2);
        const bool nr = residual && ctx->needs_input_grad(2 + bias);
        at::Tensor dx, dw, db;
        if (nx || nw || nb)
            std::tie(dx, dw, db) = Linear_backward(g[0], saved[0], saved[1], saved[2], ctx->saved_data["act"].toInt(), nx, nw, nb);
        return {dx, dw, db, nr ? g[0] : at::Tensor(), at::Tensor()};
    }
};

struct GatedFeedForwardNode : torch::autograd::Function<GatedFeedForwardNode> {
    static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& w_in, const at::Tensor& w_out,
                              const c10::optional<at::Tensor>& b_in, const c10::optional<at::Tensor>& b_out,
                              const c10::optional<at::Tensor>& residual, int64_t act) {
        at::AutoDispatchBelowADInplaceOrView below;
        ctx->save_for_backward({x, w_in, w_out, opt(b_in)});
        ctx->saved_data["act"] = act;
        ctx->saved_data["b_out"] = b_out.has_value();
        ctx->saved_data["residual"] = residual.has_value();
        return GatedFeedForward_forward(x, w_in, w_out, opt(b_in), opt(b_out), opt(residual), act);
    }
    static variable_list backward(AutogradContext* ctx, variable_list g) {
        first_order("gated_feed_forward");
        const auto saved = ctx->get_saved_variables();
        const bool bi = saved[3].defined(), bo = ctx->saved_data["b_out"].toBool(), r = ctx->saved_data["residual"].toBool();
        const bool n0 = ctx->needs_input_grad(0), n1 = ctx->needs_input_grad(1), n2 = ctx->needs_input_grad(2);
        const bool n3 = bi && ctx->needs_input_grad(3), n4 = bo && ctx->needs_input_grad(3 + bi);
        const bool n5 = r && ctx->needs_input_grad(3 + bi + bo);
        at::Tensor dx, dwi, dwo, dbi, dbo;
        if (n0 || n1 || n2 || n3 || n4)
            std::tie(dx, dwi, dwo, dbi, dbo) = GatedFeedForward_backward(g[0], saved[0], saved[1], saved[2], saved[3],
                                                                        ctx->saved_data["act"].toInt(), n0, n1, n2, n3, n4);
        return {dx, dwi, dwo, dbi, dbo, n5 ? g[0] : at::Tensor(), at::Tensor()};
    }
};

// Whether a backward pass can be asked for.  There is no forward-mode
// derivative: a tangent that the plain call would drop is refused.
bool tracked(const char* op, std::initializer_list<const at::Tensor*> ts) {
    bool any = false;
    for (const at::Tensor* t : ts) {
        if (!t->defined()) continue;
        TORCH_CHECK(!t->_fw_grad(/*level=*/0).defined(), std::string(op) + " has no forward-mode derivative");
        any = any || t->requires_grad();
    }
    return any && at::GradMode::is_enabled();
}

}  // namespace

std::tuple<at::Tensor, at::Tensor> RmsNorm(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& residual, double eps) {
    if (tracked("rms_norm", {&x, &weight, &residual})) {
        variable_list out = RmsNormNode::apply(x, weight, as_opt(residual), eps);
        return {out[0], out.size() > 1 ? out[1] : at::Tensor()};
    }
    auto [y, s, rstd] = RmsNorm_forward(x, weight, residual, eps, false);
    return {y, s};
}

at::Tensor Linear(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& bias, const at::Tensor& residual, int64_t act) {
    if (tracked("linear", {&x, &weight, &bias, &residual})) return LinearNode::apply(x, weight, as_opt(bias), as_opt(residual), act);
    return Linear_forward(x, weight, bias, residual, act);
}

at::Tensor GatedFeedForward(const at::Tensor& x, const at::Tensor& w_in, const at::Tensor& w_out, const at::Tensor& b_in,
                            const at::Tensor& b_out, const at::Tensor& residual, int64_t act) {
    if (tracked("gated_feed_forward", {&x, &w_in, &w_out, &b_in, &b_out, &residual}))
        return GatedFeedForwardNode::apply(x, w_in, w_out, as_opt(b_in), as_opt(b_out), as_opt(residual), act);
    return GatedFeedForward_forward(x, w_in, w_out, b_in, b_out, residual, act);
}

}  // namespace laplace
