// What the tensor front ends of the block and the causal operators share:
// argument checks, allocation on the current stream, and autograd's conditions.
#pragma once

#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

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

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

at::Tensor opt(const c10::optional<at::Tensor>& t) { return t.has_value() ? *t : at::Tensor(); }
c10::optional<at::Tensor> as_opt(const at::Tensor& t) { return t.defined() ? c10::optional<at::Tensor>(t) : c10::nullopt; }

void first_order(const char* op) {
    TORCH_CHECK(!at::GradMode::is_enabled(), std::string(op) + " has no second derivative (create_graph is not supported)");
}

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
}  // namespace laplace
