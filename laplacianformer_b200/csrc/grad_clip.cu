// Global gradient norm over many tensors, and clipping:
//   n = sqrt(sum over all tensors of g^2),  c = min(1, max_norm / (n + 1e-6)),  out = c g
//
// Two kernels over equal chunks of the tensors (their table travels in the
// launch parameters, so nothing is copied to the device beforehand; it is sized
// by the tensors, 29 bytes each: 15 KB for 512 cost the host 4 us more per launch
// than 2.8 KB for 96).  The first writes one fp64 partial sum of squares per
// chunk; in the second every block adds the partials in the same order, so each
// has the same coefficient without another launch, and scales its chunks, last
// chunk first: what the first kernel read last is still in L2.  No atomics: the
// norm does not depend on timing.  A chunk's squares are added in fp32 by 256
// threads (at most 256 each), the rest in fp64; a chunk whose fp32 sum is not
// finite is read again and added in fp64, so that the norm is finite where it
// can be.  A NaN norm gives NaN everywhere; an infinite one a coefficient of
// zero, and NaN at infinite elements.
//
// Bound by memory: 302 M bf16 gradients (0.6 GB) 105 us for the sums (5.8
// TB/s) and 200 us for the scaling (6.0 TB/s), of 6.5 measured for a copy.
#include <algorithm>
#include <new>
#include <vector>

#include "lf_common.cuh"

namespace lfb {
namespace {

constexpr int kFewTensors = 96, kSomeTensors = 256, kMaxTensors = 512;  // per launch
constexpr int kThreads = 256;

template <int N>
struct Table {
    const void* in[N];
    void* out[N];
    int64_t n[N];
    int first[N + 1];  // first chunk of each tensor within this launch
    uint8_t dtype[N];
    int count, chunk;  // tensors; elements per chunk
    int base, total;   // first chunk of this launch among all; chunks of all launches
};

template <typename T>
__device__ __forceinline__ float sum_sq(const T* p, int64_t n) {
    constexpr int V = 16 / sizeof(T);
    const int t = threadIdx.x;
    // Elements before the first 16-byte boundary, whole vectors, the rest.
    int64_t head = ((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / sizeof(T);
    head = head < n ? head : n;
    const int64_t nv = (n - head) / V;
    float a = 0.f;
    for (int64_t i = t; i < head; i += kThreads) {
        const float v = Elem<T>::load(p[i]);
        a = __fmaf_rn(v, v, a);
    }
    const uint4* q = reinterpret_cast<const uint4*>(p + head);
    float b[4] = {0.f, 0.f, 0.f, 0.f};
    int64_t i = t;
    auto add = [&](const uint4& u, float& s) {
        const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float v = Elem<T>::load(e[j]);
            s = __fmaf_rn(v, v, s);
        }
    };
    for (; i + 3 * kThreads < nv; i += 4 * kThreads) {
        uint4 u[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) u[k] = q[i + k * kThreads];
#pragma unroll
        for (int k = 0; k < 4; ++k) add(u[k], b[k]);
    }
    for (; i < nv; i += kThreads) add(q[i], b[0]);
    for (int64_t j = head + nv * V + t; j < n; j += kThreads) {
        const float v = Elem<T>::load(p[j]);
        a = __fmaf_rn(v, v, a);
    }
    return a + ((b[0] + b[1]) + (b[2] + b[3]));
}

// The same sum in fp64, for a chunk whose squares pass the largest fp32 number
// (any element above 1.8e19) although its norm does not.
template <typename T>
__device__ __noinline__ double sum_sq_wide(const T* p, int64_t n) {
    double a = 0.;
    for (int64_t i = threadIdx.x; i < n; i += kThreads) {
        const double v = Elem<T>::load(p[i]);
        a = __fma_rn(v, v, a);
    }
    return a;
}

template <typename T>
__device__ __forceinline__ void scale_to(const T* p, T* o, int64_t n, float c) {
    constexpr int V = 16 / sizeof(T);
    const int t = threadIdx.x;
    const uintptr_t pa = reinterpret_cast<uintptr_t>(p) & 15, oa = reinterpret_cast<uintptr_t>(o) & 15;
    if (pa != oa) {  // input and output never reach a 16-byte boundary together
        for (int64_t i = t; i < n; i += kThreads) o[i] = Elem<T>::store(Elem<T>::load(p[i]) * c);
        return;
    }
    int64_t head = ((16 - pa) & 15) / sizeof(T);
    head = head < n ? head : n;
    const int64_t nv = (n - head) / V;
    for (int64_t i = t; i < head; i += kThreads) o[i] = Elem<T>::store(Elem<T>::load(p[i]) * c);
    const uint4* q = reinterpret_cast<const uint4*>(p + head);
    uint4* w = reinterpret_cast<uint4*>(o + head);
    auto mul = [&](uint4 u) {
        T* e = reinterpret_cast<T*>(&u);
#pragma unroll
        for (int j = 0; j < V; ++j) e[j] = Elem<T>::store(Elem<T>::load(e[j]) * c);
        return u;
    };
    int64_t i = t;
    for (; i + 3 * kThreads < nv; i += 4 * kThreads) {
        uint4 u[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) u[k] = q[i + k * kThreads];
#pragma unroll
        for (int k = 0; k < 4; ++k) w[i + k * kThreads] = mul(u[k]);
    }
    for (; i < nv; i += kThreads) w[i] = mul(q[i]);
    for (int64_t j = head + nv * V + t; j < n; j += kThreads) o[j] = Elem<T>::store(Elem<T>::load(p[j]) * c);
}

// Tensor that holds chunk k: the last one whose first chunk is <= k (tensors
// without elements have no chunk and are passed over).
template <int N>
__device__ __forceinline__ int tensor_of(const Table<N>& t, int k) {
    int lo = 0, hi = t.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (t.first[mid] <= k) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

template <typename V>
__device__ __forceinline__ V block_sum(V v, V* sh) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
    __syncthreads();
    v = sh[0];
#pragma unroll
    for (int i = 1; i < kThreads / 32; ++i) v += sh[i];
    return v;
}

template <int N>
__global__ void __launch_bounds__(kThreads) grad_sq_kernel(const __grid_constant__ Table<N> t, double* part) {
    __shared__ double sh[kThreads / 32];
    grid_release();
    grid_wait();
    const int chunks = t.first[t.count];
    for (int k = blockIdx.x; k < chunks; k += gridDim.x) {
        const int i = tensor_of(t, k);
        const int64_t at = (int64_t)(k - t.first[i]) * t.chunk;
        const int64_t n = t.n[i] - at < t.chunk ? t.n[i] - at : t.chunk;
        float v;
        if (t.dtype[i] == LF_F32) v = sum_sq((const float*)t.in[i] + at, n);
        else if (t.dtype[i] == LF_F16) v = sum_sq((const __half*)t.in[i] + at, n);
        else v = sum_sq((const __nv_bfloat16*)t.in[i] + at, n);
        double s = block_sum<double>((double)v, sh);  // at most chunk/256 squares are added in fp32
        if (!isfinite(s)) {  // for all threads of the block
            double d;
            if (t.dtype[i] == LF_F32) d = sum_sq_wide((const float*)t.in[i] + at, n);
            else if (t.dtype[i] == LF_F16) d = sum_sq_wide((const __half*)t.in[i] + at, n);
            else d = sum_sq_wide((const __nv_bfloat16*)t.in[i] + at, n);
            s = block_sum<double>(d, sh);
        }
        if (threadIdx.x == 0) part[t.base + k] = s;
    }
}

template <int N>
__global__ void __launch_bounds__(kThreads) grad_scale_kernel(const __grid_constant__ Table<N> t, const double* part,
                                                              float max_norm, float* norm) {
    __shared__ double sh[kThreads / 32];
    grid_release();
    grid_wait();
    double s = 0.;
    for (int k = threadIdx.x; k < t.total; k += kThreads) s += part[k];
    const float n = (float)sqrt(block_sum<double>(s, sh));
    if (blockIdx.x == 0 && threadIdx.x == 0) *norm = n;
    const float r = max_norm / (n + 1e-6f);
    const float c = r > 1.f ? 1.f : r;  // a NaN norm gives a NaN coefficient
    const int chunks = t.first[t.count];
    for (int k = chunks - 1 - blockIdx.x; k >= 0; k -= gridDim.x) {
        const int i = tensor_of(t, k);
        const int64_t at = (int64_t)(k - t.first[i]) * t.chunk;
        const int64_t m = t.n[i] - at < t.chunk ? t.n[i] - at : t.chunk;
        if (c == 1.f && t.in[i] == t.out[i]) continue;  // in place and nothing to change
        if (t.dtype[i] == LF_F32) scale_to((const float*)t.in[i] + at, (float*)t.out[i] + at, m, c);
        else if (t.dtype[i] == LF_F16) scale_to((const __half*)t.in[i] + at, (__half*)t.out[i] + at, m, c);
        else scale_to((const __nv_bfloat16*)t.in[i] + at, (__nv_bfloat16*)t.out[i] + at, m, c);
    }
}

// Elements per chunk: enough chunks to fill the SMs several times, at most
// 64 K elements so that a thread adds few squares in fp32.
int chunk_of(const int64_t* sizes, int64_t count) {
    int64_t total = 0;
    for (int64_t i = 0; i < count; ++i) total += sizes[i];
    int chunk = 2048;
    while (chunk < 65536 && total / chunk > 8 * (int64_t)num_sms()) chunk *= 2;
    return chunk;
}

int64_t chunks_of(const int64_t* sizes, int64_t count, int chunk) {
    int64_t k = 0;
    for (int64_t i = 0; i < count; ++i) k += (sizes[i] + chunk - 1) / chunk;
    return k;
}

// Whether a tensor that is written shares memory with another one (an output
// with any other output, or with any gradient but its own in place): its
// elements would be read before or after the write by chance.  Gradients that
// are only read may overlap.  Of a call of 11 us for 80 tensors this takes 0.3 us
// in order of address (views of one buffer) and 0.8 in any order; 5 of 55 for 700.
bool overlapping(const void* const* grads, void* const* outs, const int64_t* sizes, const int* dtypes, int64_t count) {
    struct Span {
        uintptr_t at, end;
    };
    std::vector<Span> written, read;
    written.reserve(count);
    for (int64_t i = 0; i < count; ++i) {
        const size_t bytes = (size_t)sizes[i] * dtype_size(dtypes[i]);
        if (bytes == 0) continue;
        const uintptr_t g = (uintptr_t)grads[i], o = (uintptr_t)outs[i];
        written.push_back({o, o + bytes});
        if (g != o) read.push_back({g, g + bytes});
    }
    const auto before = [](const Span& a, const Span& b) { return a.at < b.at; };
    for (auto* v : {&written, &read})
        if (!std::is_sorted(v->begin(), v->end(), before)) std::sort(v->begin(), v->end(), before);
    uintptr_t written_to = 0, read_to = 0;  // ends of the tensors that start before
    auto r = read.begin();
    for (const Span& w : written) {
        for (; r != read.end() && r->at < w.at; ++r) {
            if (r->at < written_to) return true;
            read_to = std::max(read_to, r->end);
        }
        if (w.at < written_to || w.at < read_to) return true;
        written_to = w.end;
    }
    return r != read.end() && r->at < written_to;
}

template <int N>
int run_clip(const void* const* grads, void* const* outs, const int64_t* sizes, const int* dtypes, int64_t count, int chunk,
             int total, float max_norm, float* norm, double* part, cudaStream_t st) {
    // All sums before the first scaling: a launch scales what it summed last.
    for (int pass = 0; pass < 2; ++pass) {
        int64_t i = 0;
        int base = 0;
        do {
            static thread_local Table<N> t;
            t.chunk = chunk;
            t.base = base;
            t.total = total;
            t.count = 0;
            t.first[0] = 0;
            for (; i < count && t.count < N; ++i) {
                if (sizes[i] == 0) continue;
                const int j = t.count++;
                t.in[j] = grads[i];
                t.out[j] = outs[i];
                t.n[j] = sizes[i];
                t.dtype[j] = (uint8_t)dtypes[i];
                t.first[j + 1] = t.first[j] + (int)((sizes[i] + chunk - 1) / chunk);
            }
            const int chunks = t.first[t.count];
            base += chunks;
            const int slots = 8 * num_sms();
            const unsigned grid = (unsigned)(chunks < 1 ? 1 : chunks < slots ? chunks : slots);
            if (pass == 0) launch_early(grad_sq_kernel<N>, grid, kThreads, 0, 1, st, t, part);
            else launch_early(grad_scale_kernel<N>, grid, kThreads, 0, 1, st, t, (const double*)part, max_norm, norm);
            if (int rc = check_launch("lf_clip_grad_norm")) return rc;
        } while (i < count);
    }
    return LF_OK;
}

}  // namespace
}  // namespace lfb

using namespace lfb;

extern "C" size_t lf_clip_grad_norm_workspace_size(const int64_t* sizes, int64_t count) {
    if (!sizes || count <= 0) return 16;
    for (int64_t i = 0; i < count; ++i)
        if (sizes[i] < 0) return 0;
    return (size_t)(chunks_of(sizes, count, chunk_of(sizes, count)) + 2) * sizeof(double);
}

extern "C" int lf_clip_grad_norm(const void* const* grads, void* const* outs, const int64_t* sizes, const int* dtypes,
                                 int64_t count, double max_norm, float* norm, void* workspace, size_t workspace_bytes,
                                 lf_stream_t stream) {
    clear_error();
    cudaStream_t st = (cudaStream_t)stream;
    if (count < 0 || !norm || (count > 0 && (!grads || !outs || !sizes || !dtypes)) || !(max_norm >= 0)) {
        set_error("lf_clip_grad_norm: bad arguments (count=%lld, max_norm=%g)", (long long)count, max_norm);
        return LF_ERR_INVALID;
    }
    for (int64_t i = 0; i < count; ++i) {
        if (dtypes[i] != LF_F32 && dtypes[i] != LF_F16 && dtypes[i] != LF_BF16) {
            set_error("lf_clip_grad_norm: unsupported dtype code %d of tensor %lld", dtypes[i], (long long)i);
            return LF_ERR_DTYPE;
        }
        if (sizes[i] < 0 || (sizes[i] > 0 && (!grads[i] || !outs[i])) ||
            !aligned(grads[i], dtype_size(dtypes[i])) || !aligned(outs[i], dtype_size(dtypes[i]))) {
            set_error("lf_clip_grad_norm: bad size or pointer of tensor %lld", (long long)i);
            return LF_ERR_INVALID;
        }
    }
    try {
        if (overlapping(grads, outs, sizes, dtypes, count)) {
            set_error("lf_clip_grad_norm: tensors overlap (an output may share memory with its own gradient alone)");
            return LF_ERR_INVALID;
        }
    } catch (const std::bad_alloc&) {
        set_error("lf_clip_grad_norm: out of host memory for %lld tensors", (long long)count);
        return LF_ERR_UNSUPPORTED;
    }
    if (!workspace || !aligned(workspace, 8) || workspace_bytes < lf_clip_grad_norm_workspace_size(sizes, count)) {
        set_error("lf_clip_grad_norm: needs %zu bytes of workspace", lf_clip_grad_norm_workspace_size(sizes, count));
        return LF_ERR_INVALID;
    }
    const int chunk = chunk_of(sizes, count);
    const int64_t total = chunks_of(sizes, count, chunk);
    if (total > INT32_MAX) {
        set_error("lf_clip_grad_norm: too many elements");
        return LF_ERR_UNSUPPORTED;
    }
    auto run = count <= kFewTensors ? run_clip<kFewTensors> : count <= kSomeTensors ? run_clip<kSomeTensors> : run_clip<kMaxTensors>;
    return run(grads, outs, sizes, dtypes, count, chunk, (int)total, (float)max_norm, norm, (double*)workspace, st);
}
