// Root-mean-square norm with the residual's addition, its backward pass, its
// output in 8 bits (e4m3, one scale per row) and the row quantiser alone.
//
//   s = x + r,  rstd = 1/sqrt(mean(s^2) + eps),  y = s rstd w
//   a = dy w,  xhat = s rstd
//   dx = dr = rstd (a - xhat mean(a xhat)) + ds,   dw = sum_rows dy xhat
//   8 bits: scale = max|y| / 448 (1 for a row of zeros), q = e4m3(y / scale)
//
// Every tensor is read once and written once, so the passes are bound by
// memory.  A row belongs to a group of G threads that keeps it in registers
// between the statistics and the output; w stays in registers over all rows
// of a group.  Statistics and sums are fp32 (row sums by shuffles in a fixed
// order); dw is summed per thread, then per block, then over the blocks'
// partials in block order, so results do not depend on timing.
//
// Measured (bf16, 131072 rows of 1024): forward with residual 161 us (6.6
// TB/s), backward 183 us (5.9 TB/s), of 6.5 measured for a copy; fp32, 6304
// rows of 771 (scalar accesses, in L2): 15 and 17 us.
#include <initializer_list>
#include <mutex>

#include "lf_common.cuh"

namespace lfb {
namespace {

constexpr float kE4m3Max = 448.f;

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Pack {
    T v[VEC];
};

template <typename T, int VEC>
__device__ __forceinline__ Pack<T, VEC> load_pack(const T* p) {
    return *reinterpret_cast<const Pack<T, VEC>*>(p);
}

// Maximum that keeps a NaN (fmaxf drops it), so that a row with a NaN gets a NaN scale.
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// Reduction over a group of G threads; every thread gets the result.  G <= 32:
// the group is part of a warp; otherwise the group is the whole block.
template <int G, bool MAX>
__device__ __forceinline__ float group_reduce(float v, float* red) {
    constexpr int W = G < 32 ? G : 32;
#pragma unroll
    for (int o = W / 2; o > 0; o >>= 1) {
        const float u = __shfl_xor_sync(0xffffffffu, v, o);
        v = MAX ? max_nan(v, u) : v + u;
    }
    if constexpr (G > 32) {
        const int warp = threadIdx.x >> 5;
        __syncthreads();  // the previous use of red
        if ((threadIdx.x & 31) == 0) red[warp] = v;
        __syncthreads();
        v = red[0];
#pragma unroll
        for (int i = 1; i < G / 32; ++i) v = MAX ? max_nan(v, red[i]) : v + red[i];
    }
    return v;
}

// The scale of a row whose largest size is m.  The quotient is what may not be
// zero: it underflows for m below 3e-43 (fp32 rows), where zeros would become NaN.
__device__ __forceinline__ float row_scale(float m) {
    const float scale = m / kE4m3Max;
    return scale == 0.f ? 1.f : scale;
}

__device__ __forceinline__ uint16_t e4m3x2(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}

template <int VEC>
__device__ __forceinline__ void store_e4m3(uint8_t* p, const float* v) {
    if constexpr (VEC == 1) {
        *p = (uint8_t)(e4m3x2(v[0], 0.f) & 0xff);
    } else {
        uint32_t w[VEC / 4];
#pragma unroll
        for (int i = 0; i < VEC / 4; ++i)
            w[i] = (uint32_t)e4m3x2(v[4 * i], v[4 * i + 1]) | ((uint32_t)e4m3x2(v[4 * i + 2], v[4 * i + 3]) << 16);
        if constexpr (VEC == 8) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
        else *reinterpret_cast<uint32_t*>(p) = w[0];
    }
}

struct NormArgs {
    const void *x, *res, *w;
    void *y, *s;
    uint8_t* q;
    float *scale, *rstd;
    int64_t rows, cols;
    float eps;
    bool normalise;  // false: the row quantiser alone
};

template <int G>
constexpr int block_of() {
    return G <= 32 ? 256 : G;
}

// Blocks per SM that the forward is compiled for.  Rows of two vectors per
// thread run best with 16 (one warp per row) or 24 warps per SM resident:
// bf16, width 1024, 131072 rows: 167 us at 24 warps, 201 at 32, where values
// spill (171 without a bound); width 512: 96 us at 16, 115 at 24 (130 without).
template <int NV, int G>
constexpr int fwd_blocks() {
    return NV != 2 ? 1 : G <= 32 ? 2 : G >= 512 ? 1 : 24 * 32 / G;
}

// Element j of vector i of thread g is column (i*G + g)*VEC + j.
template <typename T, int VEC, int NV, int G, bool QUANT>
__global__ void __launch_bounds__(block_of<G>(), fwd_blocks<NV, G>()) rms_fwd_kernel(const NormArgs p) {
    constexpr int RPB = block_of<G>() / G;  // rows in flight per block
    __shared__ float red[32];
    grid_release();
    grid_wait();
    const int g = threadIdx.x % G, sub = threadIdx.x / G;
    const int cols = (int)p.cols;
    Pack<T, VEC> w[NV];
    if (p.w) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if ((i * G + g) * VEC < cols) w[i] = load_pack<T, VEC>((const T*)p.w + (i * G + g) * VEC);
    }
    const float inv_cols = 1.f / (float)cols;
    // The row index is clamped, not skipped, so that every lane takes part in the shuffles.
    for (int64_t base = (int64_t)blockIdx.x * RPB; base < p.rows; base += (int64_t)gridDim.x * RPB) {
        const bool live = base + sub < p.rows;
        const int64_t off = (live ? base + sub : p.rows - 1) * p.cols;
        float v[NV * VEC];
        Pack<T, VEC> xa[NV], ra[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * G + g) * VEC;
            if (c < cols) {
                xa[i] = load_pack<T, VEC>((const T*)p.x + off + c);
                if (p.res) ra[i] = load_pack<T, VEC>((const T*)p.res + off + c);
            }
        }
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const bool in = (i * G + g) * VEC < cols;
            Pack<T, VEC> sv;
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                float t = 0.f;
                if (in) {
                    t = Elem<T>::load(xa[i].v[j]);
                    if (p.res) t += Elem<T>::load(ra[i].v[j]);
                }
                sv.v[j] = Elem<T>::store(t);
                v[i * VEC + j] = t;
                ss = __fmaf_rn(t, t, ss);
            }
            if (in && live && p.s) *reinterpret_cast<Pack<T, VEC>*>((T*)p.s + off + (i * G + g) * VEC) = sv;
        }
        if (p.normalise) {
            ss = group_reduce<G, false>(ss, red);
            const float rstd = 1.f / sqrtf(ss * inv_cols + p.eps);
            if (p.rstd && live && g == 0) p.rstd[base + sub] = rstd;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const bool in = (i * G + g) * VEC < cols;
                Pack<T, VEC> o;
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    float& t = v[i * VEC + j];
                    t = in ? t * rstd * Elem<T>::load(w[i].v[j]) : 0.f;
                    o.v[j] = Elem<T>::store(t);
                }
                if (!QUANT && in && live) *reinterpret_cast<Pack<T, VEC>*>((T*)p.y + off + (i * G + g) * VEC) = o;
            }
        }
        if constexpr (QUANT) {
            float m = 0.f;
#pragma unroll
            for (int i = 0; i < NV * VEC; ++i) m = max_nan(m, fabsf(v[i]));
            m = group_reduce<G, true>(m, red);
            const float scale = row_scale(m);
            if (live && g == 0) p.scale[base + sub] = scale;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c = (i * G + g) * VEC;
                if (c < cols && live) {
#pragma unroll
                    for (int j = 0; j < VEC; ++j) v[i * VEC + j] = v[i * VEC + j] / scale;
                    store_e4m3<VEC>(p.q + off + c, v + i * VEC);
                }
            }
        }
    }
}

// Rows too long for registers: one block per row, which reads the row again
// for the output (it is in L1 or L2 by then).
template <typename T, bool QUANT>
__global__ void __launch_bounds__(512) rms_fwd_long_kernel(const NormArgs p) {
    __shared__ float red[32];
    grid_release();
    grid_wait();
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const T* x = (const T*)p.x + row * p.cols;
        const T* r = p.res ? (const T*)p.res + row * p.cols : nullptr;
        float ss = 0.f;
        for (int64_t c = threadIdx.x; c < p.cols; c += 512) {
            float t = Elem<T>::load(x[c]);
            if (r) t += Elem<T>::load(r[c]);
            ss = __fmaf_rn(t, t, ss);
        }
        float rstd = 1.f, m = 0.f;
        if (p.normalise) {
            rstd = 1.f / sqrtf(group_reduce<512, false>(ss, red) / (float)p.cols + p.eps);
            if (p.rstd && threadIdx.x == 0) p.rstd[row] = rstd;
        }
        for (int pass = QUANT ? 0 : 1; pass < 2; ++pass) {
            const float scale = QUANT && pass ? row_scale(m) : 1.f;
            if (QUANT && pass && threadIdx.x == 0) p.scale[row] = scale;
            for (int64_t c = threadIdx.x; c < p.cols; c += 512) {
                float t = Elem<T>::load(x[c]);
                if (r) t += Elem<T>::load(r[c]);
                if (pass && p.s) ((T*)p.s)[row * p.cols + c] = Elem<T>::store(t);
                if (p.normalise) t = t * rstd * Elem<T>::load(((const T*)p.w)[c]);
                if (!pass) m = max_nan(m, fabsf(t));
                else if (QUANT) {
                    const float u = t / scale;
                    store_e4m3<1>(p.q + row * p.cols + c, &u);
                } else ((T*)p.y)[row * p.cols + c] = Elem<T>::store(t);
            }
            if (!pass) m = group_reduce<512, true>(m, red);
        }
    }
}

// The backward takes xhat from the sum that the forward stored (or from x where
// there is no residual): its rounding is the only one besides the outputs', and
// leaves dw with about sqrt(2) of one rounding's error.  Reading x and r again
// instead would cost a quarter more traffic and keep both alive.
struct NormBwdArgs {
    const void *dy, *ds, *s, *w;
    const float* rstd;
    void* dx;
    float* part;  // [gridDim.x][cols] sums of dy xhat, or null
    int64_t rows, cols;
};

template <typename T, int VEC, int NV, int G>
__global__ void __launch_bounds__(block_of<G>()) rms_bwd_kernel(const NormBwdArgs p) {
    constexpr int RPB = block_of<G>() / G;
    extern __shared__ float dwsum[];  // [warps][cols] when G <= 32
    __shared__ float red[32];
    grid_release();
    grid_wait();
    const int g = threadIdx.x % G, sub = threadIdx.x / G;
    const int cols = (int)p.cols;
    Pack<T, VEC> w[NV];
    float dw[NV * VEC];
#pragma unroll
    for (int i = 0; i < NV; ++i)
        if ((i * G + g) * VEC < cols) w[i] = load_pack<T, VEC>((const T*)p.w + (i * G + g) * VEC);
#pragma unroll
    for (int i = 0; i < NV * VEC; ++i) dw[i] = 0.f;
    const float inv_cols = 1.f / (float)cols;
    for (int64_t base = (int64_t)blockIdx.x * RPB; base < p.rows; base += (int64_t)gridDim.x * RPB) {
        const bool live = base + sub < p.rows;
        const int64_t row = live ? base + sub : p.rows - 1, off = row * p.cols;
        Pack<T, VEC> dy[NV], s[NV], ds[NV];
        const float rstd = p.rstd[row];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * G + g) * VEC;
            if (c < cols) {
                dy[i] = load_pack<T, VEC>((const T*)p.dy + off + c);
                s[i] = load_pack<T, VEC>((const T*)p.s + off + c);
                if (p.ds) ds[i] = load_pack<T, VEC>((const T*)p.ds + off + c);
            }
        }
        float dot = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if ((i * G + g) * VEC < cols) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const float d = Elem<T>::load(dy[i].v[j]), xh = Elem<T>::load(s[i].v[j]) * rstd;
                    const float t = d * xh;
                    dot = __fmaf_rn(t, Elem<T>::load(w[i].v[j]), dot);
                    if (live) dw[i * VEC + j] += t;
                }
            }
        const float mean = group_reduce<G, false>(dot, red) * inv_cols;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * G + g) * VEC;
            if (c < cols && live && p.dx) {
                Pack<T, VEC> o;
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const float a = Elem<T>::load(dy[i].v[j]) * Elem<T>::load(w[i].v[j]);
                    const float xh = Elem<T>::load(s[i].v[j]) * rstd;
                    float t = rstd * __fmaf_rn(-xh, mean, a);
                    if (p.ds) t += Elem<T>::load(ds[i].v[j]);
                    o.v[j] = Elem<T>::store(t);
                }
                *reinterpret_cast<Pack<T, VEC>*>((T*)p.dx + off + c) = o;
            }
        }
    }
    if (!p.part) return;
    if constexpr (G <= 32) {
        // Groups of one warp by shuffles, then the warps in order.
#pragma unroll
        for (int i = 0; i < NV * VEC; ++i)
#pragma unroll
            for (int o = G; o < 32; o <<= 1) dw[i] += __shfl_xor_sync(0xffffffffu, dw[i], o);
        const int warp = threadIdx.x >> 5;
        if ((threadIdx.x & 31) < G) {
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if ((i * G + g) * VEC < cols) {
#pragma unroll
                    for (int j = 0; j < VEC; ++j) dwsum[warp * cols + (i * G + g) * VEC + j] = dw[i * VEC + j];
                }
        }
        __syncthreads();
        for (int c = threadIdx.x; c < cols; c += 256) {
            float t = 0.f;
#pragma unroll
            for (int k = 0; k < 8; ++k) t += dwsum[k * cols + c];
            p.part[(int64_t)blockIdx.x * p.cols + c] = t;
        }
    } else {
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if ((i * G + g) * VEC < cols) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) p.part[(int64_t)blockIdx.x * p.cols + (i * G + g) * VEC + j] = dw[i * VEC + j];
            }
    }
}

// Long rows: the row is read twice; dw partials live in global memory, a
// column always handled by the same thread of the same block.
template <typename T>
__global__ void __launch_bounds__(512) rms_bwd_long_kernel(const NormBwdArgs p) {
    __shared__ float red[32];
    grid_release();
    grid_wait();
    float* part = p.part ? p.part + (int64_t)blockIdx.x * p.cols : nullptr;
    if (part)
        for (int64_t c = threadIdx.x; c < p.cols; c += 512) part[c] = 0.f;
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const int64_t off = row * p.cols;
        const T *dy = (const T*)p.dy + off, *s = (const T*)p.s + off, *w = (const T*)p.w;
        const float rstd = p.rstd[row];
        float dot = 0.f;
        for (int64_t c = threadIdx.x; c < p.cols; c += 512) {
            const float t = Elem<T>::load(dy[c]) * (Elem<T>::load(s[c]) * rstd);
            dot = __fmaf_rn(t, Elem<T>::load(w[c]), dot);
            if (part) part[c] += t;
        }
        const float mean = group_reduce<512, false>(dot, red) / (float)p.cols;
        if (p.dx)
            for (int64_t c = threadIdx.x; c < p.cols; c += 512) {
                const float a = Elem<T>::load(dy[c]) * Elem<T>::load(w[c]), xh = Elem<T>::load(s[c]) * rstd;
                float t = rstd * __fmaf_rn(-xh, mean, a);
                if (p.ds) t += Elem<T>::load(((const T*)p.ds)[off + c]);
                ((T*)p.dx)[off + c] = Elem<T>::store(t);
            }
    }
}

// dw[c] = sum over blocks of part[block][c]: 32 columns per block, 32 strided
// partial sums per column joined in order.
template <typename T>
__global__ void __launch_bounds__(1024) rms_dw_kernel(const float* part, T* dw, int blocks, int64_t cols) {
    __shared__ float sh[32][33];
    grid_release();
    grid_wait();
    const int lane = threadIdx.x & 31, k = threadIdx.x >> 5;
    const int64_t c = (int64_t)blockIdx.x * 32 + lane;
    float t = 0.f;
    if (c < cols)
#pragma unroll 4
        for (int b = k; b < blocks; b += 32) t += part[(int64_t)b * cols + c];
    sh[k][lane] = t;
    __syncthreads();
    if (k == 0 && c < cols) {
#pragma unroll
        for (int i = 1; i < 32; ++i) t += sh[i][lane];
        dw[c] = Elem<T>::store(t);
    }
}

// Vectors per thread (NV) and threads per row (G).  Rows that divide into
// 16-byte vectors: one or two vectors per thread in the forward and one in
// the backward, whose running dw takes the registers of another; more
// registers per thread cost more occupancy than the wider row groups' block
// reductions (bf16 width 1024: forward (2,64) 167 us, (1,128) 209, (4,32) 277;
// backward (1,128) 181, (2,64) 183, (4,32) 391; width 512 forward (2,32) 96,
// (1,64) 103).  Widths between powers of two get row groups of three warps or
// six, so that few threads idle (width 1536, 65536 rows: forward (2,96) 128,
// (2,128) 144; backward (1,192) 141, (1,256) 162).  Other rows use scalar (still coalesced) accesses, four or
// eight per thread.
#define LFB_NORM_FWD(T, V, cols, vec, CALL)             \
    if (vec) {                                          \
        if (cols <= 8 * V) { CALL(T, V, 1, 8); }        \
        else if (cols <= 16 * V) { CALL(T, V, 1, 16); } \
        else if (cols <= 32 * V) { CALL(T, V, 1, 32); } \
        else if (cols <= 64 * V) { CALL(T, V, 2, 32); } \
        else if (cols <= 128 * V) { CALL(T, V, 2, 64); } \
        else if (cols <= 192 * V) { CALL(T, V, 2, 96); } \
        else if (cols <= 256 * V) { CALL(T, V, 2, 128); } \
        else if (cols <= 384 * V) { CALL(T, V, 2, 192); } \
        else if (cols <= 512 * V) { CALL(T, V, 2, 256); } \
        else if (cols <= 1024 * V) { CALL(T, V, 2, 512); } \
        else if (cols <= 2048 * V) { CALL(T, V, 4, 512); } \
        else long_rows = true;                          \
    } else LFB_NORM_SCALAR(T, cols, CALL)
#define LFB_NORM_BWD(T, V, cols, vec, CALL)             \
    if (vec) {                                          \
        if (cols <= 8 * V) { CALL(T, V, 1, 8); }        \
        else if (cols <= 16 * V) { CALL(T, V, 1, 16); } \
        else if (cols <= 32 * V) { CALL(T, V, 1, 32); } \
        else if (cols <= 64 * V) { CALL(T, V, 1, 64); } \
        else if (cols <= 96 * V) { CALL(T, V, 1, 96); } \
        else if (cols <= 128 * V) { CALL(T, V, 1, 128); } \
        else if (cols <= 192 * V) { CALL(T, V, 1, 192); } \
        else if (cols <= 256 * V) { CALL(T, V, 1, 256); } \
        else if (cols <= 512 * V) { CALL(T, V, 1, 512); } \
        else if (cols <= 1024 * V) { CALL(T, V, 2, 512); } \
        else if (cols <= 2048 * V) { CALL(T, V, 4, 512); } \
        else long_rows = true;                          \
    } else LFB_NORM_SCALAR(T, cols, CALL)
#define LFB_NORM_SCALAR(T, cols, CALL)              \
    {                                               \
        if (cols <= 128) { CALL(T, 1, 4, 32); }     \
        else if (cols <= 512) { CALL(T, 1, 4, 128); } \
        else if (cols <= 1024) { CALL(T, 1, 4, 256); } \
        else if (cols <= 2048) { CALL(T, 1, 4, 512); } \
        else if (cols <= 4096) { CALL(T, 1, 8, 512); } \
        else long_rows = true;                      \
    }

// Blocks that are resident at once: the kernels walk the rows in strides of
// the grid, and one resident wave measured best (two: 1 % slower, one block
// per row group: 6 %).
template <auto Kernel>
int resident_blocks(int block, size_t smem) {
    static std::once_flag once[64];
    static int per_sm[64];
    int dev = 0;
    cudaGetDevice(&dev);
    dev &= 63;
    std::call_once(once[dev], [&] {
        int v = 0;
        if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&v, Kernel, block, smem) != cudaSuccess || v < 1) v = 1;
        per_sm[dev] = v;
    });
    return per_sm[dev] * num_sms();
}

unsigned row_blocks(int64_t rows, int per_block, int slots) {
    const int64_t want = (rows + per_block - 1) / per_block;
    return (unsigned)(want < slots ? want : slots);
}

// Blocks per SM of the backward, at most 2048 threads' worth: by the smallest
// block that any type and alignment takes for a row of this width (the tables
// above; up to 256 columns eight, which is as many as a warp per row gives).
int64_t bwd_blocks_per_sm(int64_t cols) {
    return cols <= 256 ? 8 : 2048 / (cols <= 512 ? 64 : cols <= 768 ? 96 : cols <= 1024 ? 128 : cols <= 1536 ? 192 : cols <= 2048 ? 256 : 512);
}

// Rows of partial sums in the backward's workspace: never fewer than its blocks.
int64_t bwd_part_rows(int64_t rows, int64_t cols) {
    const int64_t most = (int64_t)num_sms() * bwd_blocks_per_sm(cols);
    return rows < most ? rows : most;
}

template <typename T, bool QUANT>
void launch_fwd(const NormArgs& a, bool vec, cudaStream_t st) {
    constexpr int V = 16 / sizeof(T);
    bool long_rows = false;
#define LFB_CALL(TT, VV, NV, G)                                                                                        \
    launch_early(rms_fwd_kernel<TT, VV, NV, G, QUANT>,                                                                 \
                 row_blocks(a.rows, block_of<G>() / G, resident_blocks<rms_fwd_kernel<TT, VV, NV, G, QUANT>>(block_of<G>(), 0)), \
                 block_of<G>(), 0, 1, st, a)
    LFB_NORM_FWD(T, V, a.cols, vec, LFB_CALL)
#undef LFB_CALL
    if (long_rows)
        launch_early(rms_fwd_long_kernel<T, QUANT>, row_blocks(a.rows, 1, resident_blocks<rms_fwd_long_kernel<T, QUANT>>(512, 0)), 512, 0, 1, st, a);
}

template <typename T>
void launch_bwd(const NormBwdArgs& a, void* dw, bool vec, cudaStream_t st) {
    constexpr int V = 16 / sizeof(T);
    bool long_rows = false;
    unsigned blocks = 1;
    const int64_t most = bwd_part_rows(a.rows, a.cols);
    auto grid = [&](int per_block, int slots) {
        return blocks = row_blocks(a.rows, per_block, (int)(slots < most ? slots : most));
    };
    // Shared memory of the largest width that a warp-per-row group takes, so that residency does not depend on cols.
#define LFB_CALL(TT, VV, NV, G)                                                                                   \
    launch_early(rms_bwd_kernel<TT, VV, NV, G>,                                                                   \
                 grid(block_of<G>() / G, resident_blocks<rms_bwd_kernel<TT, VV, NV, G>>(block_of<G>(), G <= 32 ? G * NV * VV * 32 : 0)), \
                 block_of<G>(), G <= 32 ? G * NV * VV * 32 : 0, 1, st, a)
    LFB_NORM_BWD(T, V, a.cols, vec, LFB_CALL)
#undef LFB_CALL
    if (long_rows) launch_early(rms_bwd_long_kernel<T>, grid(1, resident_blocks<rms_bwd_long_kernel<T>>(512, 0)), 512, 0, 1, st, a);
    if (dw) launch_early(rms_dw_kernel<T>, (unsigned)((a.cols + 31) / 32), 1024, 0, 1, st, a.part, (T*)dw, (int)blocks, a.cols);
}

int check_rows(const char* what, int64_t rows, int64_t cols, int dtype, std::initializer_list<const void*> ptrs,
               std::initializer_list<const void*> floats) {
    if (dtype != LF_F32 && dtype != LF_F16 && dtype != LF_BF16) {
        set_error("%s: unsupported dtype code %d (fp32, fp16 and bf16)", what, dtype);
        return LF_ERR_DTYPE;
    }
    if (rows < 0 || cols < 0 || cols > INT32_MAX) {
        set_error("%s: bad sizes rows=%lld cols=%lld", what, (long long)rows, (long long)cols);
        return LF_ERR_INVALID;
    }
    bool ok = true;  // a misaligned access would fault
    for (const void* p : ptrs) ok = ok && aligned(p, dtype_size(dtype));
    for (const void* p : floats) ok = ok && aligned(p, 4);
    if (!ok) {
        set_error("%s: a pointer is not aligned to its elements", what);
        return LF_ERR_INVALID;
    }
    return LF_OK;
}

bool vector_rows(int64_t cols, int dtype, std::initializer_list<const void*> ptrs) {
    if (cols * dtype_size(dtype) % 16) return false;
    for (const void* p : ptrs)
        if (p && !aligned(p, 16)) return false;
    return true;
}

int run_fwd(const char* what, const NormArgs& a, bool quant, int dtype, cudaStream_t st) {
    const bool vec = vector_rows(a.cols, dtype, {a.x, a.res, a.w, a.y, a.s}) && (!a.q || aligned(a.q, 8));
    if (dtype == LF_F32) {
        if (quant) launch_fwd<float, true>(a, vec, st);
        else launch_fwd<float, false>(a, vec, st);
    } else if (dtype == LF_F16) {
        if (quant) launch_fwd<__half, true>(a, vec, st);
        else launch_fwd<__half, false>(a, vec, st);
    } else {
        if (quant) launch_fwd<__nv_bfloat16, true>(a, vec, st);
        else launch_fwd<__nv_bfloat16, false>(a, vec, st);
    }
    return check_launch(what);
}

}  // namespace
}  // namespace lfb

using namespace lfb;

extern "C" int lf_rms_norm_fwd(const void* x, const void* residual, const void* weight, void* y, void* s, float* rstd,
                               int64_t rows, int64_t cols, int dtype, double eps, lf_stream_t stream) {
    clear_error();
    if (int rc = check_rows("lf_rms_norm_fwd", rows, cols, dtype, {x, residual, weight, y, s}, {rstd})) return rc;
    if (rows == 0 || cols == 0) return LF_OK;
    if (!x || !weight || !y || (residual != nullptr) != (s != nullptr)) {
        set_error("lf_rms_norm_fwd: x, weight and y are required, residual and s go together");
        return LF_ERR_INVALID;
    }
    NormArgs a{x, residual, weight, y, s, nullptr, nullptr, rstd, rows, cols, (float)eps, true};
    return run_fwd("lf_rms_norm_fwd", a, false, dtype, (cudaStream_t)stream);
}

extern "C" int lf_rms_norm_quant_fwd(const void* x, const void* residual, const void* weight, void* q, float* scale,
                                     void* s, int64_t rows, int64_t cols, int dtype, double eps, lf_stream_t stream) {
    clear_error();
    if (int rc = check_rows("lf_rms_norm_quant_fwd", rows, cols, dtype, {x, residual, weight, s}, {scale})) return rc;
    if (rows == 0) return LF_OK;
    // Rows without values have a scale as well: the kernel reads and writes nothing else of them.
    if (!scale || (cols > 0 && (!x || !weight || !q || (residual != nullptr) != (s != nullptr)))) {
        set_error("lf_rms_norm_quant_fwd: x, weight, q and scale are required, residual and s go together");
        return LF_ERR_INVALID;
    }
    NormArgs a{x, residual, weight, nullptr, s, (uint8_t*)q, scale, nullptr, rows, cols, (float)eps, true};
    return run_fwd("lf_rms_norm_quant_fwd", a, true, dtype, (cudaStream_t)stream);
}

extern "C" int lf_quantize_rows(const void* x, void* q, float* scale, int64_t rows, int64_t cols, int dtype,
                                lf_stream_t stream) {
    clear_error();
    if (int rc = check_rows("lf_quantize_rows", rows, cols, dtype, {x}, {scale})) return rc;
    if (rows == 0) return LF_OK;
    if (!scale || (cols > 0 && (!x || !q))) {
        set_error("lf_quantize_rows: x, q and scale are required");
        return LF_ERR_INVALID;
    }
    NormArgs a{x, nullptr, nullptr, nullptr, nullptr, (uint8_t*)q, scale, nullptr, rows, cols, 0.f, false};
    return run_fwd("lf_quantize_rows", a, true, dtype, (cudaStream_t)stream);
}

extern "C" size_t lf_rms_norm_bwd_workspace_size(int64_t rows, int64_t cols) {
    if (rows <= 0 || cols <= 0) return 0;
    return (size_t)bwd_part_rows(rows, cols) * cols * sizeof(float);
}

extern "C" int lf_rms_norm_bwd(const void* dy, const void* ds, const void* s, const float* rstd, const void* weight,
                               void* dx, void* dw, int64_t rows, int64_t cols, int dtype, void* workspace,
                               size_t workspace_bytes, lf_stream_t stream) {
    clear_error();
    if (int rc = check_rows("lf_rms_norm_bwd", rows, cols, dtype, {dy, ds, s, weight, dx, dw}, {rstd})) return rc;
    if (cols == 0 || (!dx && !dw)) return LF_OK;
    cudaStream_t st = (cudaStream_t)stream;
    if (rows == 0) {
        if (dw && cudaMemsetAsync(dw, 0, cols * dtype_size(dtype), st) != cudaSuccess) return check_launch("lf_rms_norm_bwd");
        return LF_OK;
    }
    if (!dy || !s || !rstd || !weight) {
        set_error("lf_rms_norm_bwd: dy, s, rstd and weight are required");
        return LF_ERR_INVALID;
    }
    if (dw && (!workspace || !aligned(workspace, 16) || workspace_bytes < lf_rms_norm_bwd_workspace_size(rows, cols))) {
        set_error("lf_rms_norm_bwd: dw needs %zu bytes of 16-byte aligned workspace, got %zu",
                  lf_rms_norm_bwd_workspace_size(rows, cols), workspace ? workspace_bytes : (size_t)0);
        return LF_ERR_INVALID;
    }
    NormBwdArgs a{dy, ds, s, weight, rstd, dx, dw ? (float*)workspace : nullptr, rows, cols};
    const bool vec = vector_rows(cols, dtype, {dy, ds, s, weight, dx});
    if (dtype == LF_F32) launch_bwd<float>(a, dw, vec, st);
    else if (dtype == LF_F16) launch_bwd<__half>(a, dw, vec, st);
    else launch_bwd<__nv_bfloat16>(a, dw, vec, st);
    return check_launch("lf_rms_norm_bwd");
}
