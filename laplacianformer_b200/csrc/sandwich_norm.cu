// The norms before and after a sublayer in one pass over its output x: norm,
// gate, residual scale, the residual's addition and the next sublayer's norm.
//
//   xh = x rx,  rx = 1/sqrt(mean(x^2) + eps),  p = xh w
//   s  = r + alpha act(g) p
//   th = s rt,  rt = 1/sqrt(mean(s^2) + eps),  y = th wn
// Backward, from dy and the gradient ds of s:
//   u = dy wn,   dr = rt (u - th mean(u th)) + ds,   dwn = sum dy th
//   dp = alpha act(g) dr,   dg = alpha act'(g) p dr,   dw = sum dp xh
//   e = dp w,    dx = rx (e - xh mean(e xh))
//
// Memory bound: every tensor is read once and written once.  A row belongs to a
// group of threads that keeps it in registers through both norms; weights and
// their gradients' sums stay in registers over all rows of a group.  Sums are
// fp32 in a fixed order.  A gate row may serve several rows: then a block takes
// rows of one gate row at a time and keeps the gate's gradient in registers too;
// partial sums of the blocks join in block order in a second launch.  The
// backward takes th from the stored s, whose rounding is the only one besides
// the outputs'.
#include <algorithm>

#include "norm_rows.cuh"

namespace lfb {
namespace {

struct SandwichArgs {
    const void *x, *w, *r, *gate, *wn;
    void *s, *y;
    float* rstd;             // [2][rows], or null
    const void *dy, *ds;
    void *dx, *dr, *dgate;
    float *part_w, *part_wn; // [gridDim.x][cols]
    float* part_g;           // [groups][parts][cols] where several blocks share a gate row, else null
    int64_t rows, cols, shared;   // rows per gate row
    LongDivisor per_gate;
    int64_t groups, parts, per_part;  // the backward's units: `parts` runs of at most per_part rows in each group of rows
    float alpha, eps;
    int act;
};

// The sigmoids q of z and p of -z: neither is a difference, so that both keep their digits however far z is from 0.  (Where e^-z
// overflows, below -88, q is 0 and p only has to be finite.)
// (expf is good to 2 units in the last place, the hardware's reciprocal to 1.  The hardware's exponential is off by 2 + 1.17 |z|
// of them, 1.1e-5 at 80, below a 30th of a 16-bit rounding and hence good enough for 16-bit gates: 131072x1024 training 604-615
// us, 653 with expf of -|z|.)
template <typename T>
__device__ __forceinline__ void sigmoids(float z, float& q, float& p) {
    const float e = sizeof(T) == 2 ? __expf(-z) : expf(-z);
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(q) : "f"(1.f + e));
    p = fminf(e, 3e38f) * q;
}

// Rows on their way.  A row's two reductions follow one another, so a group
// that waited for its row to arrive first would leave the memory idle.  Each
// thread copies its packs of the next rows (K operands) to places of its own in
// shared memory, asynchronously: that takes no registers and no barriers (bf16,
// 131072x1024, a gate per token: forward 414 -> 212 us, backward 739 -> 380).
// Rows without 16-byte packs (fp32 6304x771: 29 us so, 25 without) and rows of
// very wide groups, which do not fit, are loaded when their turn comes.
template <typename T, int VEC, int NV, int K, int BLOCK>
struct RowStream {
    static constexpr int kPack = (int)sizeof(Pack<T, VEC>), kStage = K * NV * BLOCK * kPack;
    static constexpr int kFit = (96 << 10) / kStage, kStages = kPack < 16 || kFit < 2 ? 0 : kFit < 4 ? kFit : 4;
    static constexpr int kBytes = kStages * kStage;

    uint8_t* base;  // of this thread
    __device__ __forceinline__ explicit RowStream(uint8_t* smem) : base(smem + threadIdx.x * kPack) {}
    __device__ __forceinline__ uint8_t* at(int stage, int k, int i) const { return base + ((stage * K + k) * NV + i) * (BLOCK * kPack); }
    __device__ __forceinline__ void copy(int stage, int k, int i, const T* src) const {
        const uint32_t dst = static_cast<uint32_t>(__cvta_generic_to_shared(at(stage, k, i)));
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
    }
    __device__ __forceinline__ Pack<T, VEC> get(int stage, int k, int i) const { return *reinterpret_cast<const Pack<T, VEC>*>(at(stage, k, i)); }
};
__device__ __forceinline__ void copies_committed() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_but() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// act(g), and with SLOPE its derivative in d: q(z) q(-z) for the sigmoid q, q(z) (1 + z q(-z)), and 4 q(2z) q(-2z) for tanh.
template <typename T, bool SLOPE, int N>
__device__ __forceinline__ void gate_values(float (&v)[N], float (&d)[N], int act) {
    float q, p;
    if (act == LF_GATE_SIGMOID) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            sigmoids<T>(v[j], q, p);
            if (SLOPE) d[j] = q * p;
            v[j] = q;
        }
    } else if (act == LF_GATE_SILU) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            sigmoids<T>(v[j], q, p);
            if (SLOPE) d[j] = q * __fmaf_rn(v[j], p, 1.f);
            v[j] *= q;
        }
    } else if (act == LF_GATE_TANH) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            if (SLOPE) sigmoids<T>(2.f * v[j], q, p), d[j] = 4.f * q * p;
            v[j] = tanhf(v[j]);
        }
    } else if (SLOPE) {
#pragma unroll
        for (int j = 0; j < N; ++j) d[j] = 1.f;
    }
}

template <typename T, int VEC, int NV, int G>
__global__ void __launch_bounds__(block_of<G>()) sandwich_fwd_kernel(const SandwichArgs p) {
    constexpr int RPB = block_of<G>() / G;
    using Stream = RowStream<T, VEC, NV, 3, block_of<G>()>;
    constexpr int S = Stream::kStages;
    extern __shared__ __align__(16) uint8_t staged[];
    __shared__ float red[32];
    grid_release();
    grid_wait();
    const Stream stream(staged);
    const int g = threadIdx.x % G, sub = threadIdx.x / G, cols = (int)p.cols;
    Pack<T, VEC> w[NV], wn[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i)
        if ((i * G + g) * VEC < cols) {
            w[i] = load_pack<T, VEC>((const T*)p.w + (i * G + g) * VEC);
            if (p.wn) wn[i] = load_pack<T, VEC>((const T*)p.wn + (i * G + g) * VEC);
        }
    const float inv_cols = 1.f / (float)cols;
    // The row index is clamped, not skipped, so that every lane takes part in the shuffles.
    const int64_t step = (int64_t)gridDim.x * RPB, first = (int64_t)blockIdx.x * RPB;
    auto row_of = [&](int64_t base) { return min(base + sub, p.rows - 1); };
    auto gate_of = [&](int64_t row) { return (p.shared == 1 ? row : p.per_gate.of(row)) * p.cols; };
    auto fetch = [&](int64_t base, int stage) {
        if (base < p.rows) {
            const int64_t row = row_of(base), off = row * p.cols, goff = p.gate ? gate_of(row) : 0;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c = (i * G + g) * VEC;
                if (c < cols) {
                    stream.copy(stage, 0, i, (const T*)p.x + off + c);
                    stream.copy(stage, 1, i, (const T*)p.r + off + c);
                    if (p.gate) stream.copy(stage, 2, i, (const T*)p.gate + goff + c);
                }
            }
        }
        copies_committed();
    };
    if constexpr (S > 0) {
#pragma unroll
        for (int k = 0; k + 1 < S; ++k) fetch(first + k * step, k);
    }
    int stage = 0;
    for (int64_t base = first; base < p.rows; base += step) {
        const bool live = base + sub < p.rows;
        const int64_t row = row_of(base), off = row * p.cols;
        Pack<T, VEC> x[NV], r[NV], ga[NV];
        float ss = 0.f, t[NV * VEC];
        if constexpr (S > 0) {
            copies_but<(S > 1 ? S - 2 : 0)>();
#pragma unroll
            for (int i = 0; i < NV; ++i) x[i] = stream.get(stage, 0, i), r[i] = stream.get(stage, 1, i), ga[i] = stream.get(stage, 2, i);
            fetch(base + (S - 1) * step, stage == 0 ? S - 1 : stage - 1);
            stage = stage + 1 == S ? 0 : stage + 1;
        } else {
            const int64_t goff = p.gate ? gate_of(row) : 0;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c = (i * G + g) * VEC;
                if (c < cols) {
                    x[i] = load_pack<T, VEC>((const T*)p.x + off + c);
                    r[i] = load_pack<T, VEC>((const T*)p.r + off + c);
                    if (p.gate) ga[i] = load_pack<T, VEC>((const T*)p.gate + goff + c);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if ((i * G + g) * VEC < cols) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const float v = Elem<T>::load(x[i].v[j]);
                    ss = __fmaf_rn(v, v, ss);
                }
            }
        const float rx = 1.f / sqrtf(group_reduce<G, false>(ss, red) * inv_cols + p.eps);
        ss = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * G + g) * VEC;
            if (c < cols) {
                float a[VEC], none[VEC];
                Pack<T, VEC> o;
                if (p.gate) {
#pragma unroll
                    for (int j = 0; j < VEC; ++j) a[j] = Elem<T>::load(ga[i].v[j]);
                    gate_values<T, false>(a, none, p.act);
                }
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    float v = Elem<T>::load(x[i].v[j]) * rx * Elem<T>::load(w[i].v[j]);
                    if (p.gate) v *= a[j];
                    v = __fmaf_rn(p.alpha, v, Elem<T>::load(r[i].v[j]));
                    t[i * VEC + j] = v;
                    ss = __fmaf_rn(v, v, ss);
                    o.v[j] = Elem<T>::store(v);
                }
                if (live) *reinterpret_cast<Pack<T, VEC>*>((T*)p.s + off + c) = o;
            }
        }
        if (p.rstd && live && g == 0) p.rstd[row] = rx;
        if (p.wn) {
            const float rt = 1.f / sqrtf(group_reduce<G, false>(ss, red) * inv_cols + p.eps);
            if (p.rstd && live && g == 0) p.rstd[p.rows + row] = rt;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c = (i * G + g) * VEC;
                if (c < cols && live) {
                    Pack<T, VEC> o;
#pragma unroll
                    for (int j = 0; j < VEC; ++j) o.v[j] = Elem<T>::store(t[i * VEC + j] * rt * Elem<T>::load(wn[i].v[j]));
                    *reinterpret_cast<Pack<T, VEC>*>((T*)p.y + off + c) = o;
                }
            }
        }
    }
}

// Rows too long for registers: one block per row, which reads it again for each step (from L1 or L2).
template <typename T>
__device__ __forceinline__ float gate_at(const SandwichArgs& p, int64_t at, float& slope) {
    float v[1] = {1.f}, d[1] = {0.f};
    if (p.gate) v[0] = Elem<T>::load(((const T*)p.gate)[at]), gate_values<T, true>(v, d, p.act);
    slope = d[0];
    return v[0];
}
template <typename T>
__global__ void __launch_bounds__(512) sandwich_fwd_long_kernel(const SandwichArgs p) {
    __shared__ float red[32];
    grid_release();
    grid_wait();
    const float inv_cols = 1.f / (float)p.cols;
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const int64_t off = row * p.cols, goff = row / p.shared * p.cols;
        const T *x = (const T*)p.x + off, *r = (const T*)p.r + off;
        float ss = 0.f, slope;
        for (int64_t c = threadIdx.x; c < p.cols; c += 512) {
            const float v = Elem<T>::load(x[c]);
            ss = __fmaf_rn(v, v, ss);
        }
        const float rx = 1.f / sqrtf(group_reduce<512, false>(ss, red) * inv_cols + p.eps);
        auto sum = [&](int64_t c) {
            return __fmaf_rn(p.alpha, Elem<T>::load(x[c]) * rx * Elem<T>::load(((const T*)p.w)[c]) * gate_at<T>(p, goff + c, slope), Elem<T>::load(r[c]));
        };
        ss = 0.f;
        for (int64_t c = threadIdx.x; c < p.cols; c += 512) {
            const float t = sum(c);
            ss = __fmaf_rn(t, t, ss);
            if (!p.wn) ((T*)p.s)[off + c] = Elem<T>::store(t);
        }
        if (p.rstd && threadIdx.x == 0) p.rstd[row] = rx;
        if (!p.wn) continue;
        const float rt = 1.f / sqrtf(group_reduce<512, false>(ss, red) * inv_cols + p.eps);
        if (p.rstd && threadIdx.x == 0) p.rstd[p.rows + row] = rt;
        for (int64_t c = threadIdx.x; c < p.cols; c += 512) {
            const float t = sum(c);
            ((T*)p.s)[off + c] = Elem<T>::store(t);
            ((T*)p.y)[off + c] = Elem<T>::store(t * rt * Elem<T>::load(((const T*)p.wn)[c]));
        }
    }
}

// Sums over the groups of a block (G <= 32), or a group that is the block, to dst[cols].
template <typename D, int VEC, int NV, int G>
__device__ __forceinline__ void put_sums(float (&v)[NV * VEC], D* dst, int cols, float* sh) {
    const int g = threadIdx.x % G;
    if constexpr (G <= 32) {
        // Groups of one warp by shuffles, then the warps in order.
#pragma unroll
        for (int i = 0; i < NV * VEC; ++i)
#pragma unroll
            for (int o = G; o < 32; o <<= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
        __syncthreads();  // the last use of sh
        if ((threadIdx.x & 31) < G) {
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if ((i * G + g) * VEC < cols) {
#pragma unroll
                    for (int j = 0; j < VEC; ++j) sh[(threadIdx.x >> 5) * cols + (i * G + g) * VEC + j] = v[i * VEC + j];
                }
        }
        __syncthreads();
        for (int c = threadIdx.x; c < cols; c += 256) {
            float t = 0.f;
#pragma unroll
            for (int k = 0; k < 8; ++k) t += sh[k * cols + c];
            dst[c] = Elem<D>::store(t);
        }
    } else {
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if ((i * G + g) * VEC < cols) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) dst[(i * G + g) * VEC + j] = Elem<D>::store(v[i * VEC + j]);
            }
    }
}

template <typename T, int VEC, int NV, int G>
__global__ void __launch_bounds__(block_of<G>()) sandwich_bwd_kernel(const SandwichArgs p) {
    constexpr int RPB = block_of<G>() / G;
    using Stream = RowStream<T, VEC, NV, 5, block_of<G>()>;
    constexpr int S = Stream::kStages;
    extern __shared__ __align__(16) uint8_t staged[];
    float* const sums = reinterpret_cast<float*>(staged + Stream::kBytes);  // [warps][cols] when G <= 32
    __shared__ float red[32];
    grid_release();
    grid_wait();
    const Stream stream(staged);
    const int g = threadIdx.x % G, sub = threadIdx.x / G, cols = (int)p.cols;
    const bool own_gate = p.gate && p.shared == 1, kept_gate = p.gate && p.shared > 1 && (p.dgate || p.part_g);
    Pack<T, VEC> w[NV], wn[NV];
    float dw[NV * VEC], dwn[NV * VEC], dg[NV * VEC];
#pragma unroll
    for (int i = 0; i < NV; ++i)
        if ((i * G + g) * VEC < cols) {
            w[i] = load_pack<T, VEC>((const T*)p.w + (i * G + g) * VEC);
            if (p.wn) wn[i] = load_pack<T, VEC>((const T*)p.wn + (i * G + g) * VEC);
        }
#pragma unroll
    for (int i = 0; i < NV * VEC; ++i) dw[i] = dwn[i] = dg[i] = 0.f;
    const float inv_cols = 1.f / (float)cols;
    const int64_t group_rows = p.rows / p.groups;
    for (int64_t unit = blockIdx.x; unit < p.groups * p.parts; unit += gridDim.x) {
        const int64_t group = unit / p.parts, part = unit - group * p.parts;
        const int64_t first = group * group_rows + min(group_rows, part * p.per_part);
        const int64_t last = group * group_rows + min(group_rows, (part + 1) * p.per_part);
        auto row_of = [&](int64_t base) { return min(base + sub, last - 1); };
        auto fetch = [&](int64_t base, int stage) {
            if (base < last) {
                const int64_t row = row_of(base), off = row * p.cols, goff = p.shared == 1 ? off : group * p.cols;
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    const int c = (i * G + g) * VEC;
                    if (c < cols) {
                        stream.copy(stage, 0, i, (const T*)p.x + off + c);
                        if (p.dy) stream.copy(stage, 1, i, (const T*)p.s + off + c), stream.copy(stage, 2, i, (const T*)p.dy + off + c);
                        if (p.ds) stream.copy(stage, 3, i, (const T*)p.ds + off + c);
                        if (p.gate) stream.copy(stage, 4, i, (const T*)p.gate + goff + c);
                    }
                }
            }
            copies_committed();
        };
        if constexpr (S > 0) {
#pragma unroll
            for (int k = 0; k + 1 < S; ++k) fetch(first + k * RPB, k);
        }
        int stage = 0;
        float rx_next = 0.f, rt_next = 0.f;
        if (first < last) rx_next = p.rstd[row_of(first)], rt_next = p.wn ? p.rstd[p.rows + row_of(first)] : 0.f;
        for (int64_t base = first; base < last; base += RPB) {
            const bool live = base + sub < last;
            const int64_t row = row_of(base), off = row * p.cols;
            const float rx = rx_next, rt = rt_next;
            const int64_t after = row_of(base + RPB);
            rx_next = p.rstd[after], rt_next = p.wn ? p.rstd[p.rows + after] : 0.f;
            Pack<T, VEC> x[NV], s[NV], dy[NV], ds[NV], ga[NV];
            if constexpr (S > 0) {
                copies_but<(S > 1 ? S - 2 : 0)>();
#pragma unroll
                for (int i = 0; i < NV; ++i)
                    x[i] = stream.get(stage, 0, i), s[i] = stream.get(stage, 1, i), dy[i] = stream.get(stage, 2, i), ds[i] = stream.get(stage, 3, i),
                    ga[i] = stream.get(stage, 4, i);
                fetch(base + (S - 1) * RPB, stage == 0 ? S - 1 : stage - 1);
                stage = stage + 1 == S ? 0 : stage + 1;
            } else {
                const int64_t goff = p.shared == 1 ? off : group * p.cols;
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    const int c = (i * G + g) * VEC;
                    if (c < cols) {
                        x[i] = load_pack<T, VEC>((const T*)p.x + off + c);
                        if (p.dy) s[i] = load_pack<T, VEC>((const T*)p.s + off + c), dy[i] = load_pack<T, VEC>((const T*)p.dy + off + c);
                        if (p.ds) ds[i] = load_pack<T, VEC>((const T*)p.ds + off + c);
                        if (p.gate) ga[i] = load_pack<T, VEC>((const T*)p.gate + goff + c);
                    }
                }
            }
            float dot = 0.f, mean = 0.f;
            if (p.dy) {
#pragma unroll
                for (int i = 0; i < NV; ++i)
                    if ((i * G + g) * VEC < cols) {
#pragma unroll
                        for (int j = 0; j < VEC; ++j) {
                            const float t = Elem<T>::load(dy[i].v[j]) * (Elem<T>::load(s[i].v[j]) * rt);
                            dot = __fmaf_rn(t, Elem<T>::load(wn[i].v[j]), dot);
                            if (live) dwn[i * VEC + j] += t;
                        }
                    }
                mean = group_reduce<G, false>(dot, red) * inv_cols;
            }
            dot = 0.f;
            float e[NV * VEC];  // dp w
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c = (i * G + g) * VEC;
                if (c < cols) {
                    float a[VEC], slope[VEC];
                    Pack<T, VEC> o, og;
                    if (p.gate) {
#pragma unroll
                        for (int j = 0; j < VEC; ++j) a[j] = Elem<T>::load(ga[i].v[j]);
                        gate_values<T, true>(a, slope, p.act);
                    }
#pragma unroll
                    for (int j = 0; j < VEC; ++j) {
                        float d = 0.f;
                        if (p.dy) d = rt * __fmaf_rn(-(Elem<T>::load(s[i].v[j]) * rt), mean, Elem<T>::load(dy[i].v[j]) * Elem<T>::load(wn[i].v[j]));
                        if (p.ds) d += Elem<T>::load(ds[i].v[j]);
                        o.v[j] = Elem<T>::store(d);
                        d *= p.alpha;
                        const float xh = Elem<T>::load(x[i].v[j]) * rx, wv = Elem<T>::load(w[i].v[j]);
                        float dp = d;
                        if (p.gate) {
                            const float v = d * (xh * wv) * slope[j];
                            og.v[j] = Elem<T>::store(v);
                            if (live) dg[i * VEC + j] += v;
                            dp = d * a[j];
                        }
                        if (live) dw[i * VEC + j] = __fmaf_rn(dp, xh, dw[i * VEC + j]);
                        e[i * VEC + j] = dp * wv;
                        dot = __fmaf_rn(e[i * VEC + j], xh, dot);
                    }
                    if (live && p.dr) *reinterpret_cast<Pack<T, VEC>*>((T*)p.dr + off + c) = o;
                    if (live && own_gate && p.dgate) *reinterpret_cast<Pack<T, VEC>*>((T*)p.dgate + off + c) = og;
                }
            }
            if (p.dx) {
                mean = group_reduce<G, false>(dot, red) * inv_cols;
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    const int c = (i * G + g) * VEC;
                    if (c < cols && live) {
                        Pack<T, VEC> o;
#pragma unroll
                        for (int j = 0; j < VEC; ++j)
                            o.v[j] = Elem<T>::store(rx * __fmaf_rn(-(Elem<T>::load(x[i].v[j]) * rx), mean, e[i * VEC + j]));
                        *reinterpret_cast<Pack<T, VEC>*>((T*)p.dx + off + c) = o;
                    }
                }
            }
        }
        if constexpr (S > 0) copies_but<0>();  // (rows past the unit's end were not copied: the groups that are left are empty)
        if (kept_gate) {
            if (p.part_g) put_sums<float, VEC, NV, G>(dg, p.part_g + unit * p.cols, cols, sums);
            else put_sums<T, VEC, NV, G>(dg, (T*)p.dgate + group * p.cols, cols, sums);
#pragma unroll
            for (int i = 0; i < NV * VEC; ++i) dg[i] = 0.f;
        }
    }
    if (p.part_w) put_sums<float, VEC, NV, G>(dw, p.part_w + (int64_t)blockIdx.x * p.cols, cols, sums);
    if (p.part_wn) put_sums<float, VEC, NV, G>(dwn, p.part_wn + (int64_t)blockIdx.x * p.cols, cols, sums);
}

// Long rows: sums live in global memory, a column always handled by the same thread of the same block.
template <typename T>
__global__ void __launch_bounds__(512) sandwich_bwd_long_kernel(const SandwichArgs p) {
    __shared__ float red[32];
    grid_release();
    grid_wait();
    const float inv_cols = 1.f / (float)p.cols;
    float* const pw = p.part_w ? p.part_w + (int64_t)blockIdx.x * p.cols : nullptr;
    float* const pn = p.part_wn ? p.part_wn + (int64_t)blockIdx.x * p.cols : nullptr;
    for (int64_t c = threadIdx.x; c < p.cols; c += 512) {
        if (pw) pw[c] = 0.f;
        if (pn) pn[c] = 0.f;
    }
    const int64_t group_rows = p.rows / p.groups;
    for (int64_t unit = blockIdx.x; unit < p.groups * p.parts; unit += gridDim.x) {
        const int64_t group = unit / p.parts, part = unit - group * p.parts;
        const int64_t first = group * group_rows + min(group_rows, part * p.per_part);
        const int64_t last = group * group_rows + min(group_rows, (part + 1) * p.per_part);
        float* const pg = p.part_g ? p.part_g + unit * p.cols : nullptr;
        if (pg)
            for (int64_t c = threadIdx.x; c < p.cols; c += 512) pg[c] = 0.f;
        for (int64_t row = first; row < last; ++row) {
            const int64_t off = row * p.cols, goff = row / p.shared * p.cols;
            const float rx = p.rstd[row], rt = p.wn ? p.rstd[p.rows + row] : 0.f;
            const T *x = (const T*)p.x + off, *s = (const T*)p.s + off, *dy = p.dy ? (const T*)p.dy + off : nullptr;
            float dot = 0.f, mean = 0.f, slope;
            if (dy) {
                for (int64_t c = threadIdx.x; c < p.cols; c += 512) {
                    const float t = Elem<T>::load(dy[c]) * (Elem<T>::load(s[c]) * rt);
                    dot = __fmaf_rn(t, Elem<T>::load(((const T*)p.wn)[c]), dot);
                    if (pn) pn[c] += t;
                }
                mean = group_reduce<512, false>(dot, red) * inv_cols;
            }
            auto grad_s = [&](int64_t c) {
                float d = 0.f;
                if (dy) d = rt * __fmaf_rn(-(Elem<T>::load(s[c]) * rt), mean, Elem<T>::load(dy[c]) * Elem<T>::load(((const T*)p.wn)[c]));
                if (p.ds) d += Elem<T>::load(((const T*)p.ds)[off + c]);
                return d;
            };
            dot = 0.f;
            for (int64_t c = threadIdx.x; c < p.cols; c += 512) {
                const float ds = grad_s(c), d = ds * p.alpha, xh = Elem<T>::load(x[c]) * rx, wv = Elem<T>::load(((const T*)p.w)[c]);
                const float dp = d * gate_at<T>(p, goff + c, slope), v = d * (xh * wv) * slope;
                if (p.dr) ((T*)p.dr)[off + c] = Elem<T>::store(ds);
                if (p.gate && p.shared == 1 && p.dgate) ((T*)p.dgate)[off + c] = Elem<T>::store(v);
                if (pg) pg[c] += v;
                if (pw) pw[c] = __fmaf_rn(dp, xh, pw[c]);
                dot = __fmaf_rn(dp * wv, xh, dot);
            }
            if (!p.dx) continue;
            const float mx = group_reduce<512, false>(dot, red) * inv_cols;
            for (int64_t c = threadIdx.x; c < p.cols; c += 512) {
                const float dp = grad_s(c) * p.alpha * gate_at<T>(p, goff + c, slope);
                ((T*)p.dx)[off + c] = Elem<T>::store(rx * __fmaf_rn(-(Elem<T>::load(x[c]) * rx), mx, dp * Elem<T>::load(((const T*)p.w)[c])));
            }
        }
    }
}

// Rows of sums from their partial rows, joined in order, 32 columns per block: dw and dwn by all 32 warps, and four of
// the gate's rows at a time by 8 warps each (their partial rows are few; there may be more of them than a grid is high).
struct JoinArgs {
    const float* part[3];
    void* out[3];
    int64_t cols, parts[3], gates;
};
constexpr int kGateWarps = 8;
template <typename T>
__global__ void __launch_bounds__(1024) sandwich_join_kernel(const JoinArgs p) {
    __shared__ float sh[32][33];
    grid_release();
    grid_wait();
    const int lane = threadIdx.x & 31, k = threadIdx.x >> 5;
    const int job = min(2, (int)blockIdx.y), warps = job == 2 ? kGateWarps : 32;
    if (!p.out[job]) return;
    const int64_t c = (int64_t)blockIdx.x * 32 + lane, n = p.parts[job], rows = job == 2 ? p.gates : 1;
    const int per = 32 / warps, stride = ((int)gridDim.y - 2) * per;
    for (int64_t row0 = job == 2 ? ((int)blockIdx.y - 2) * per : 0; row0 < rows; row0 += stride) {
        const int64_t row = row0 + k / warps;
        const bool in = c < p.cols && row < rows;
        const float* part = p.part[job] + row * n * p.cols;
        float t = 0.f;
        if (in)
#pragma unroll 8
            for (int64_t b = k % warps; b < n; b += warps) t += part[b * p.cols + c];
        sh[k][lane] = t;
        __syncthreads();
        if (in && k % warps == 0) {
            for (int i = 1; i < warps; ++i) t += sh[k + i][lane];
            ((T*)p.out[job])[row * p.cols + c] = Elem<T>::store(t);
        }
        if (job != 2) return;
        __syncthreads();
    }
}

// resident_blocks() of a kernel that may take more than 48 KB of shared memory.
template <auto Kernel>
int resident_with(int block, int smem) {
    static std::once_flag once[64];
    int dev = 0;
    cudaGetDevice(&dev);
    std::call_once(once[dev & 63], [&] { cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem); });
    return resident_blocks<Kernel>(block, smem);
}

template <typename T>
void launch_sandwich_fwd(const SandwichArgs& a, bool vec, cudaStream_t st) {
    constexpr int V = 16 / sizeof(T);
    bool long_rows = false;
#define LFB_CALL(TT, VV, NV, G)                                                                                   \
    {                                                                                                             \
        constexpr int smem = RowStream<TT, VV, NV, 3, block_of<G>()>::kBytes;                                     \
        const int slots = resident_with<sandwich_fwd_kernel<TT, VV, NV, G>>(block_of<G>(), smem);                 \
        launch_early(sandwich_fwd_kernel<TT, VV, NV, G>, row_blocks(a.rows, block_of<G>() / G, slots), block_of<G>(), smem, 1, st, a); \
    }
    LFB_NORM_FWD(T, V, a.cols, vec, LFB_CALL)
#undef LFB_CALL
    if (long_rows)
        launch_early(sandwich_fwd_long_kernel<T>, row_blocks(a.rows, 1, resident_blocks<sandwich_fwd_long_kernel<T>>(512, 0)), 512, 0, 1, st, a);
}

// How the backward's rows are dealt out: groups of rows that share a gate row
// (all rows in one group where each has its own), each in so many parts that
// the blocks which can be resident have one.
struct Units {
    int64_t groups, parts, per_part;
    bool gate_parts;  // partial gate rows join afterwards
};
Units units_of(int64_t rows, int64_t cols, int64_t shared, bool gate, bool long_rows) {
    const int64_t most = bwd_part_rows(rows, cols);
    Units u{gate && shared > 1 ? rows / shared : 1, 1, 0, false};
    const int64_t group_rows = rows / u.groups;
    u.parts = std::max<int64_t>(1, std::min(group_rows, (most + u.groups - 1) / u.groups));
    u.per_part = (group_rows + u.parts - 1) / u.parts;
    u.parts = (group_rows + u.per_part - 1) / u.per_part;
    u.gate_parts = gate && shared > 1 && (u.parts > 1 || long_rows);
    return u;
}

template <typename T>
void launch_sandwich_bwd(const SandwichArgs& a, bool vec, int64_t most, int* blocks, cudaStream_t st) {
    constexpr int V = 16 / sizeof(T);
    bool long_rows = false;
    auto grid = [&](int slots) {
        *blocks = (int)std::min<int64_t>({most, slots, a.groups * a.parts});
        return (unsigned)*blocks;
    };
    // Shared memory of the largest width that a warp-per-row group takes, so that residency does not depend on cols.
#define LFB_CALL(TT, VV, NV, G)                                                                                   \
    {                                                                                                             \
        constexpr int smem = RowStream<TT, VV, NV, 5, block_of<G>()>::kBytes + (G <= 32 ? G * NV * VV * 32 : 0);  \
        const int slots = resident_with<sandwich_bwd_kernel<TT, VV, NV, G>>(block_of<G>(), smem);                 \
        launch_early(sandwich_bwd_kernel<TT, VV, NV, G>, grid(slots), block_of<G>(), smem, 1, st, a);             \
    }
    LFB_NORM_BWD(T, V, a.cols, vec, LFB_CALL)
#undef LFB_CALL
    if (long_rows) launch_early(sandwich_bwd_long_kernel<T>, grid(resident_blocks<sandwich_bwd_long_kernel<T>>(512, 0)), 512, 0, 1, st, a);
}

// Whether the tables above leave rows of this width to the kernels for long rows.
bool is_long(int64_t cols, int dtype, bool vec) { return vec ? cols > 2048 * 16 / (int64_t)dtype_size(dtype) : cols > 4096; }

int check_sandwich(const char* what, const lf_sandwich_norm_t* a) {
    if (!a) {
        set_error("%s: no arguments", what);
        return LF_ERR_INVALID;
    }
    if (int rc = check_rows(what, a->rows, a->cols, a->dtype,
                            {a->x, a->weight, a->residual, a->gate, a->next_weight, a->s, a->y, a->dy, a->ds, a->dx, a->d_residual, a->d_gate,
                             a->d_weight, a->d_next_weight},
                            {a->rstd}))
        return rc;
    if (a->activation < LF_GATE_NONE || a->activation > LF_GATE_TANH) {
        set_error("%s: unknown gate activation %d", what, a->activation);
        return LF_ERR_INVALID;
    }
    if (a->gate && a->rows > 0 && (a->rows_per_gate < 1 || a->rows % a->rows_per_gate)) {
        set_error("%s: rows must be a multiple of rows_per_gate", what);
        return LF_ERR_INVALID;
    }
    if (a->gate && a->rows_per_gate > 1 && a->rows >= (int64_t)1 << 40) {
        set_error("%s: a gate row for several rows is supported for less than 2^40 rows", what);
        return LF_ERR_UNSUPPORTED;
    }
    return LF_OK;
}

SandwichArgs sandwich_args(const lf_sandwich_norm_t* a) {
    SandwichArgs p{};
    p.x = a->x, p.w = a->weight, p.r = a->residual, p.gate = a->gate, p.wn = a->next_weight, p.s = a->s, p.y = a->y, p.rstd = a->rstd;
    p.dy = a->dy, p.ds = a->ds, p.dx = a->dx, p.dr = a->d_residual, p.dgate = a->d_gate;
    p.rows = a->rows, p.cols = a->cols, p.shared = a->gate ? a->rows_per_gate : 1;
    p.per_gate = LongDivisor(p.shared);
    p.alpha = (float)a->scale, p.eps = (float)a->eps, p.act = a->activation;
    return p;
}

bool sandwich_vec(const lf_sandwich_norm_t* a) {
    return vector_rows(a->cols, a->dtype, {a->x, a->weight, a->residual, a->gate, a->next_weight, a->s, a->y, a->dy, a->ds, a->dx, a->d_residual, a->d_gate});
}

}  // namespace
}  // namespace lfb

using namespace lfb;

extern "C" int lf_sandwich_norm_fwd(const lf_sandwich_norm_t* a, lf_stream_t stream) {
    clear_error();
    const char* what = "lf_sandwich_norm_fwd";
    if (int rc = check_sandwich(what, a)) return rc;
    if (a->rows == 0 || a->cols == 0) return LF_OK;
    if (!a->x || !a->weight || !a->residual || !a->s || (a->next_weight != nullptr) != (a->y != nullptr)) {
        set_error("%s: x, weight, residual and s are required, next_weight and y go together", what);
        return LF_ERR_INVALID;
    }
    const SandwichArgs p = sandwich_args(a);
    const bool vec = sandwich_vec(a);
    cudaStream_t st = (cudaStream_t)stream;
    if (a->dtype == LF_F32) launch_sandwich_fwd<float>(p, vec, st);
    else if (a->dtype == LF_F16) launch_sandwich_fwd<__half>(p, vec, st);
    else launch_sandwich_fwd<__nv_bfloat16>(p, vec, st);
    return check_launch(what);
}

extern "C" size_t lf_sandwich_norm_bwd_workspace_size(const lf_sandwich_norm_t* a) {
    if (!a || a->rows <= 0 || a->cols <= 0 || (a->gate && (a->rows_per_gate < 1 || a->rows % a->rows_per_gate)) || !dtype_size(a->dtype)) return 0;
    const bool kept = a->gate && a->rows_per_gate > 1 && a->d_gate;
    const Units u = units_of(a->rows, a->cols, a->gate ? a->rows_per_gate : 1, a->gate != nullptr, is_long(a->cols, a->dtype, sandwich_vec(a)));
    const int64_t most = bwd_part_rows(a->rows, a->cols);
    return (size_t)((a->d_weight ? most : 0) + (a->d_next_weight ? most : 0) + (kept && u.gate_parts ? u.groups * u.parts : 0)) * a->cols * sizeof(float);
}

extern "C" int lf_sandwich_norm_bwd(const lf_sandwich_norm_t* a, void* workspace, size_t workspace_bytes, lf_stream_t stream) {
    clear_error();
    const char* what = "lf_sandwich_norm_bwd";
    if (int rc = check_sandwich(what, a)) return rc;
    if (a->cols == 0) return LF_OK;
    cudaStream_t st = (cudaStream_t)stream;
    const size_t es = dtype_size(a->dtype);
    if (a->rows == 0) {  // (without rows there is a gate row only where one serves all of them, and its number is the caller's)
        for (void* d : {a->d_weight, a->d_next_weight})
            if (d && cudaMemsetAsync(d, 0, a->cols * es, st) != cudaSuccess) return check_launch(what);
        return LF_OK;
    }
    if (!a->x || !a->weight || !a->rstd || (a->dy && (!a->next_weight || !a->s)) || (!a->dy && !a->ds)) {
        set_error("%s: x, weight, rstd and dy or ds are required, dy with s and next_weight", what);
        return LF_ERR_INVALID;
    }
    if ((a->d_gate && !a->gate) || (a->d_next_weight && !a->dy)) {
        set_error("%s: a gradient is asked for of an operand that is not given", what);
        return LF_ERR_INVALID;
    }
    const size_t need = lf_sandwich_norm_bwd_workspace_size(a);
    if (need && (!workspace || !aligned(workspace, 16) || workspace_bytes < need)) {
        set_error("%s: needs %zu bytes of 16-byte aligned workspace, got %zu", what, need, workspace ? workspace_bytes : (size_t)0);
        return LF_ERR_INVALID;
    }
    SandwichArgs p = sandwich_args(a);
    const bool vec = sandwich_vec(a), kept = a->gate && p.shared > 1 && a->d_gate;
    const Units u = units_of(p.rows, p.cols, p.shared, a->gate != nullptr, is_long(p.cols, a->dtype, vec));
    const int64_t most = bwd_part_rows(p.rows, p.cols);
    p.groups = u.groups, p.parts = u.parts, p.per_part = u.per_part;
    float* at = (float*)workspace;
    if (a->d_weight) p.part_w = at, at += most * p.cols;
    if (a->d_next_weight) p.part_wn = at, at += most * p.cols;
    if (kept && u.gate_parts) p.part_g = at;
    if (a->gate && p.shared > 1 && !a->d_gate) p.dgate = nullptr;
    int blocks = 1;
    if (a->dtype == LF_F32) launch_sandwich_bwd<float>(p, vec, most, &blocks, st);
    else if (a->dtype == LF_F16) launch_sandwich_bwd<__half>(p, vec, most, &blocks, st);
    else launch_sandwich_bwd<__nv_bfloat16>(p, vec, most, &blocks, st);
    if (p.part_w || p.part_wn || p.part_g) {
        JoinArgs j{{p.part_w, p.part_wn, p.part_g}, {a->d_weight, a->d_next_weight, p.part_g ? a->d_gate : nullptr}, p.cols, {blocks, blocks, u.parts}, u.groups};
        const dim3 grid((unsigned)((p.cols + 31) / 32), (unsigned)(p.part_g ? 2 + std::min<int64_t>((u.groups * kGateWarps + 31) / 32, 65000) : 2));
        if (a->dtype == LF_F32) launch_early(sandwich_join_kernel<float>, grid, 1024, 0, 1, st, j);
        else if (a->dtype == LF_F16) launch_early(sandwich_join_kernel<__half>, grid, 1024, 0, 1, st, j);
        else launch_early(sandwich_join_kernel<__nv_bfloat16>, grid, 1024, 0, 1, st, j);
    }
    return check_launch(what);
}
