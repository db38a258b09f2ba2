// Matrix products with fused epilogues on the tcgen05 tensor cores, and the
// operators made of them:
//
//   linear      z = x W^T + b,  y = act(z) + r
//               dz = dy act'(z), dx = dz W, dW = dz^T x, db = sum dz
//   8-bit form  z = sx sw (q qw^T) + b on e4m3 operands
//   gated FFN   [g|u] = x Win^T + bin,  h = act(g) u,  y = h Wout^T + bout + r
//               dh = dy Wout,  dg = dh u act'(g),  du = dh act(g)
//               dx = [dg|du] Win,  dWin = [dg|du]^T x,  dWout = dy^T h
//
// One persistent kernel (tc_gemm_kernel) runs every product (narrow_ffn_kernel
// the whole forward of a block of at most 64 channels, narrow_ffn_bwd_kernel its
// backward with at most 256 hidden columns): operands come
// through TMA into a ring of 128-byte-swizzled stages, one warp issues the
// tcgen05 products into accumulators in tensor memory, and sixteen warps turn
// finished accumulators into outputs while the next tile's products run.
// Either operand may be stored K-major or transposed (MN-major), so no
// product needs a transposed copy.  The backward passes recompute z, g, u and
// h from x in 32 bits instead of reading rounded copies of them back: a
// feed-forward block keeps nothing but its input between the passes, and its
// gradients have one 16-bit rounding less, for 2 of 11 units of arithmetic.
//
// Roundings to 16 bits besides the outputs': h, dg, du and dz, as operands of
// the products that follow (the tensor cores take 16-bit operands; a second
// part of each would double those products).  The bias gradients of the
// activation and of the gate are sums of these rounded values, and in fp16 all
// four become infinite beyond 65504.
//
// Measured on a B200 (131072 tokens, 1024 channels, 4096 hidden, bf16): gated
// forward 1.4-1.7 ms (1.3-1.5 PFLOP/s, tensor pipe 95 % active), gated backward
// 2.75-2.86 ms (1.2), down projection 0.81-0.85 ms (1.3), the three gradients'
// products 3.84-4.03 ms (1.4), against cuBLAS's 1.38 PFLOP/s under the same power cap.
#include <algorithm>
#include <mutex>
#include <type_traits>

#include "tc_ptx.cuh"
#include "tma_map.h"
#include "unit_plan.h"

namespace lfb {

// Set by a kernel whose bounded wait expired (merged into lf_device_status).
__device__ int g_gemm_status = 0;

int gemm_status(bool clear) {
    int v = 0;
    if (cudaMemcpyFromSymbol(&v, g_gemm_status, sizeof(int)) != cudaSuccess) return LF_ERR_CUDA;
    if (clear) {
        int z = 0;
        if (cudaMemcpyToSymbol(g_gemm_status, &z, sizeof(int)) != cudaSuccess) return LF_ERR_CUDA;
    }
    return v;
}

namespace {

// ---------------------------------------------------------------------------
// Activations
// ---------------------------------------------------------------------------
// The epilogues are bound by instruction issue where K is short, so the
// activations are written on the hardware's exponential and reciprocal (about
// 2 units in the last place each, against results of 11 or 8 bits).
__device__ __forceinline__ float exp2_fast(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float rcp_fast(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float sigmoid(float z) { return rcp_fast(1.f + exp2_fast(-1.44269504f * z)); }

// Phi(z) and phi(z) of the normal distribution.  Phi(-x) = t P(t) e^(-x^2/2)
// with t = 1/(1 + 0.37295830 x/sqrt(2)), a form in which the relative error stays
// small however far out x is (an approximation of erf to an absolute error
// loses the tail's digits: at z = -4 gelu(z) is 1.3e-4).  P is this file's own
// minimax fit of e^(y^2) erfc(y) / (2 t) over 0 <= y <= 9.4, relative error 5.2e-7; the
// exponential is the density's, and its rounded argument costs z^2 2^-23 more.
__device__ __forceinline__ float normal_cdf(float z, float& density) {
    const float t = rcp_fast(__fmaf_rn(0.26372134f, fabsf(z), 1.f));
    const float e = exp2_fast(-0.72134752f * z * z);
    float q = __fmaf_rn(t, -0.069681955f, 0.20568058f);
    q = __fmaf_rn(t, q, -0.079053195f);
    q = __fmaf_rn(t, q, 0.150431945f);
    q = __fmaf_rn(t, q, 0.07974451f);
    q = __fmaf_rn(t, q, 0.10782365f);
    q = __fmaf_rn(t, q, 0.10505422f) * (t * e);  // Phi(-|z|)
    density = e * 0.39894228f;
    return z >= 0.f ? 1.f - q : q;
}
// (1 + tanh(k (z + c z^3))) / 2
__device__ __forceinline__ float tanh_gate(float z) {
    return sigmoid(1.59576912f * z * __fmaf_rn(0.044715f * z, z, 1.f));
}

template <int ACT>
__device__ __forceinline__ float act_value(float z) {
    float d;
    if constexpr (ACT == LF_ACT_RELU) return z < 0.f ? 0.f : z;  // keeps NaN
    if constexpr (ACT == LF_ACT_SILU) return z * sigmoid(z);
    if constexpr (ACT == LF_ACT_GELU) return z * normal_cdf(z, d);
    if constexpr (ACT == LF_ACT_GELU_TANH) return z * tanh_gate(z);
    return z;
}

// The activation's value and derivative.
template <int ACT>
__device__ __forceinline__ void act_both(float z, float& a, float& slope) {
    if constexpr (ACT == LF_ACT_RELU) {
        a = z < 0.f ? 0.f : z;
        slope = z > 0.f ? 1.f : 0.f;
    } else if constexpr (ACT == LF_ACT_SILU) {
        const float p = sigmoid(z);
        a = z * p;
        slope = __fmaf_rn(a, 1.f - p, p);
    } else if constexpr (ACT == LF_ACT_GELU) {
        float d;
        const float p = normal_cdf(z, d);
        a = z * p;
        slope = __fmaf_rn(z, d, p);
    } else if constexpr (ACT == LF_ACT_GELU_TANH) {
        const float p = tanh_gate(z);
        a = z * p;
        const float d = fminf(__fmaf_rn(0.21406445f * z, z, 1.59576912f), 1e30f);  // of the gate's argument: k (1 + 3 c z^2),
        slope = __fmaf_rn(a * (1.f - p), d, p);                                   // finite where p is 0 or 1
    } else {
        a = z;
        slope = 1.f;
    }
}

template <class F>
__device__ __forceinline__ void with_act(int act, F&& f) {
    switch (act) {
        case LF_ACT_RELU: f(std::integral_constant<int, LF_ACT_RELU>()); break;
        case LF_ACT_GELU: f(std::integral_constant<int, LF_ACT_GELU>()); break;
        case LF_ACT_GELU_TANH: f(std::integral_constant<int, LF_ACT_GELU_TANH>()); break;
        case LF_ACT_SILU: f(std::integral_constant<int, LF_ACT_SILU>()); break;
        default: f(std::integral_constant<int, LF_ACT_NONE>()); break;
    }
}

// Four consecutive elements of a row of n at p (column c); beyond the row: 0.
template <typename T>
__device__ __forceinline__ uint2 load4(const T* p, int c, int n, bool vec) {
    if (vec && c + 4 <= n) return *reinterpret_cast<const uint2*>(p + c);
    uint2 u = make_uint2(0u, 0u);
    T* e = reinterpret_cast<T*>(&u);
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (c + j < n) e[j] = p[c + j];
    return u;
}
template <typename T>
__device__ __forceinline__ float4 widen4(uint2 u) {
    const float2 a = unpack2<T>(u.x), b = unpack2<T>(u.y);
    return make_float4(a.x, a.y, b.x, b.y);
}
template <typename T>
__device__ __forceinline__ void store4(T* p, int c, int n, bool vec, float4 v) {
    const uint2 u = make_uint2(pack2<T>(v.x, v.y), pack2<T>(v.z, v.w));
    if (vec && c + 4 <= n) {
        *reinterpret_cast<uint2*>(p + c) = u;
        return;
    }
    const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (c + j < n) p[c + j] = e[j];
}

// What follows the product of one output: bias, activation, residual; or,
// for the backward, the activation's derivative times the upstream gradient.
struct Epilogue {
    void* out;
    const void *bias, *res;  // res: the residual, or dy when act_bwd
    const float *sa, *sb;    // row and column scales of the 8-bit form
    int64_t ldo, ldr;
    int act;
    bool act_bwd, vec_out, vec_res;
    bool tma, pairs;         // the output's rows can be written by TMA; their elements in pairs
};

template <int ACT>
__device__ __forceinline__ float4 finish4(float4 z, float4 bias, float4 r, bool act_bwd) {
    z.x += bias.x, z.y += bias.y, z.z += bias.z, z.w += bias.w;
    if (act_bwd) {
        float a, s;
        act_both<ACT>(z.x, a, s), z.x = r.x * s;
        act_both<ACT>(z.y, a, s), z.y = r.y * s;
        act_both<ACT>(z.z, a, s), z.z = r.z * s;
        act_both<ACT>(z.w, a, s), z.w = r.w * s;
        return z;
    }
    return make_float4(act_value<ACT>(z.x) + r.x, act_value<ACT>(z.y) + r.y, act_value<ACT>(z.z) + r.z,
                       act_value<ACT>(z.w) + r.w);
}

// ---------------------------------------------------------------------------
// The product kernel
// ---------------------------------------------------------------------------
enum Mode { kLinear, kGated, kGatedBwd };

constexpr int kBM = 128;                  // rows of a tile per CTA
constexpr int kRowBytes = 128;            // a stage holds 128 bytes of K: 64 16-bit or 128 8-bit elements
// Sixteen warps hide the epilogue's latencies (eight: 225 against 197 us for
// 100352 x 64 x 256, forward and backward) at 96 registers each, which the
// epilogues keep to by 16 columns at a time: the stages leave hardly any L1,
// so spilled registers cost an L2 round trip (59 against 38 us for the 8-bit
// 25088 x 512 -> 1536).
constexpr int kEpiWarps = 16;             // four per 32-lane quarter of the tensor memory
constexpr int kControlWarps = 3;          // copies of A, products, copies of B
constexpr int kGemmThreads = 32 * (kControlWarps + kEpiWarps);
constexpr int kStageOut = 2048;           // output staging per epilogue warp: 32 rows of 64 bytes
// and the values of 32 columns: two 16-bit biases, or a scale and a bias in fp32
template <bool FP8>
constexpr int column_bytes() { return FP8 ? 256 : 128; }
constexpr int kEpiCols = kEpiWarps / 4 * 32;  // columns that the epilogue warps read at a time
constexpr int kMaxStages = 8;
constexpr int kTmemAll = 512;
constexpr int kBarrierBytes = 256;
constexpr int kSmemLimit = 227 * 1024;
constexpr int kGroupRows = 2048;          // rows that are walked together, so that their operands stay in L2

// One product out of up to N that a launch runs.
struct alignas(64) Problem {
    CUtensorMap a, b, a2, b2, out;  // a2, b2: dy and Wout of the gated backward
    Epilogue e;
    float* part;               // split K: raw sums [split][rows][ldp]
    int64_t ldp;
    int m, n;                  // rows of one row segment; output columns (hidden columns of the gated modes)
    int msegs, tiles_m, tiles_n, splits;
    Divisor per_split, per_group, per_seg, group_rows, last_rows;  // tiles; row tiles of a whole and of the last group
    int iters, split_iters, seg_iters;  // K steps in all, per split, per K segment
    int bn;                    // columns of a tile's (first) product
    uint32_t idesc, idesc2;
    bool a_mn, b_mn;
};

template <int N>
struct GemmArgs {
    Problem p[N];
    int first[N + 1];          // first work unit of each problem; first[N] units in all
    int longer, extra;         // units of the problems before the last; see unit_plan.h
    int stages, stage_bytes;
};

// The k-th unit of CTA (or pair) c of P; first[N] or more: none left.
template <int N>
__device__ __forceinline__ int unit_of(const GemmArgs<N>& a, int c, int P, int k) {
    if constexpr (N == 1) return c + k * P;
    else return unit_at(a.longer, a.extra, c, P, k);
}
template <int N>
__device__ __forceinline__ int problem_of(const GemmArgs<N>& a, int& unit) {
    int i = 0;
    if constexpr (N > 1) {
#pragma unroll
        for (int j = 1; j < N; ++j) i += unit >= a.first[j] ? 1 : 0;
        unit -= a.first[i];
    }
    return i;
}

__device__ __forceinline__ uint32_t leader_addr(const void* p) {  // the same shared memory in CTA 0 of the cluster
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(smem_u32(p)));
    return r;
}
// Copies into this CTA's shared memory.  A pair's copies all count on the
// barrier of its first CTA, which issues the products.
template <int CTAS>
__device__ __forceinline__ void tma_load(void* dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z) {
    if constexpr (CTAS == 2)
        asm volatile(
            "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%3, %4, "
            "%5}], [%2];" ::"r"(smem_u32(dst)),
            "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z)
            : "memory");
    else
        asm volatile(
            "cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
                smem_u32(dst)),
            "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z)
            : "memory");
}
__device__ __forceinline__ void tma_store(const CUtensorMap* map, const void* src, int x, int y, int z) {
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(map), "r"(smem_u32(src)),
                 "r"(x), "r"(y), "r"(z)
                 : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
__device__ __forceinline__ void mbar_expect(uint64_t* bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
// Tells the leader that this warp has read its accumulators (the tensor-memory
// loads are done; nothing else is ordered, so stores in flight do not hold the
// next products back).
template <int CTAS>
__device__ __forceinline__ void arrive_leader(uint64_t* bar) {
    if constexpr (CTAS == 2)
        asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(leader_addr(bar)) : "memory");
    else
        asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
#define LFB_MMA(CG, KIND)                                                                              \
    asm volatile(                                                                                      \
        "{\n\t.reg .pred p, q;\n\t"                                                                    \
        "setp.ne.b32 p, %4, 0;\n\t"                                                                    \
        "setp.ne.b32 q, %5, 0;\n\t"                                                                    \
        "@q tcgen05.mma.cta_group::" CG ".kind::" KIND " [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d_tmem),   \
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(go)                                   \
        : "memory")
// D[tmem] (+)= A[smem] B[smem]; the whole warp executes it, the lane with go != 0 issues it.
template <int CTAS, bool FP8>
__device__ __forceinline__ void mma(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate,
                                    uint32_t go) {
    if constexpr (CTAS == 2 && FP8) LFB_MMA("2", "f8f6f4");
    else if constexpr (CTAS == 2) LFB_MMA("2", "f16");
    else if constexpr (FP8) LFB_MMA("1", "f8f6f4");
    else LFB_MMA("1", "f16");
}
#undef LFB_MMA
// Arrives on the barrier (of both CTAs of a pair) when the products issued so far are done.
template <int CTAS>
__device__ __forceinline__ void commit(uint64_t* bar) {
    if constexpr (CTAS == 2)
        asm volatile(
            "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
                smem_u32(bar)),
            "h"((uint16_t)3)
            : "memory");
    else mma_commit(bar);
}
template <int CTAS>
__device__ __forceinline__ void tmem_take(uint32_t* dst) {
    if constexpr (CTAS == 2) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(dst)), "r"(kTmemAll) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else tmem_alloc(dst, kTmemAll);
}
template <int CTAS>
__device__ __forceinline__ void tmem_free(uint32_t taddr) {
    if constexpr (CTAS == 2)
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(kTmemAll) : "memory");
    else tmem_dealloc(taddr, kTmemAll);
}
template <int CTAS>
__device__ __forceinline__ void sync_all() {
    if constexpr (CTAS == 2)
        asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    else __syncthreads();
}
struct Tile {
    int seg, m0, n0, split, it0, it1;
};
// Work units: for each split of K, row tiles in groups of kGroupRows, within a
// group all row tiles of one column tile before the next column tile.
template <int CTAS>
__device__ __forceinline__ Tile tile_of(const Problem& p, int unit, int bn_out, int rank) {
    Tile t;
    t.split = p.per_split.of(unit);
    int r = unit - t.split * (int)p.per_split.d;
    const int group = p.per_group.of(r);
    r -= group * (int)p.per_group.d;
    const bool whole = (group + 1) * (int)p.group_rows.d <= p.msegs * p.tiles_m;
    const int ni = whole ? p.group_rows.of(r) : p.last_rows.of(r);
    const int mi = group * (int)p.group_rows.d + r - ni * (int)(whole ? p.group_rows.d : p.last_rows.d);
    t.n0 = ni * bn_out;
    t.seg = p.per_seg.of(mi);
    t.m0 = ((mi - t.seg * p.tiles_m) * CTAS + rank) * kBM;
    t.it0 = t.split * p.split_iters;
    t.it1 = min(p.iters, t.it0 + p.split_iters);
    return t;
}

// Staging of one warp: 32 rows of 64 bytes in shared memory whose 16-byte
// chunks are swizzled as TMA's 64-byte swizzle does, so that neither a lane per
// row nor four lanes per row meet bank conflicts.
__device__ __forceinline__ uint8_t* stage_at(uint8_t* st, int row, int chunk) {
    return st + row * 64 + ((chunk ^ ((row >> 1) & 3)) << 4);
}
// Columns 16 half .. of the calling lane's row, as 16-bit values.
template <typename T>
__device__ __forceinline__ uint4 pack8(const float* v) {
    return make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
}
template <typename T>
__device__ __forceinline__ void pack16(uint4 (&u)[2], const float (&v)[16]) {
    u[0] = pack8<T>(v), u[1] = pack8<T>(v + 8);
}
__device__ __forceinline__ void stage16(uint8_t* st, int lane, int half, const uint4 (&u)[2]) {
#pragma unroll
    for (int c = 0; c < 2; ++c) *reinterpret_cast<uint4*>(stage_at(st, lane, half * 2 + c)) = u[c];
}
// Adds 16 column values to a row's.
template <typename T>
__device__ __forceinline__ void add_columns(float (&v)[16], const T* p) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        const uint4 u = reinterpret_cast<const uint4*>(p)[c];
        const uint32_t* w = reinterpret_cast<const uint32_t*>(&u);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float2 x = unpack2<T>(w[k]);
            v[8 * c + 2 * k] += x.x, v[8 * c + 2 * k + 1] += x.y;
        }
    }
}

// Writes staged outputs to rows that TMA cannot address: 64-byte row segments by
// 4-byte stores (pairs: rows and columns even) or 2-byte ones.
template <typename T>
__device__ __forceinline__ void put_rows(uint8_t* st, int lane, T* out, int64_t ld, int rows, int cols, bool pairs) {
    __syncwarp();
    if (pairs) {
        const int c = (lane & 15) * 2, r0 = lane >> 4;
        T* o = out + r0 * ld + c;
#pragma unroll 4
        for (int r = r0; r < 32; r += 2, o += 2 * ld)
            if (r < rows && c < cols)
                *reinterpret_cast<uint32_t*>(o) = *reinterpret_cast<const uint32_t*>(stage_at(st, r, c >> 3) + (c & 7) * 2);
    } else {
        T* o = out + lane;
#pragma unroll 4
        for (int r = 0; r < 32; ++r, o += ld)
            if (r < rows && lane < cols) *o = *reinterpret_cast<const T*>(stage_at(st, r, lane >> 3) + (lane & 7) * 2);
    }
}

template <typename T>
__device__ __forceinline__ T column_value(const T* p, int col, int n) {
    return p && col < n ? p[col] : Elem<T>::store(0.f);
}

// A CTA (CTAS = 1) or a pair of CTAs on two SMs (CTAS = 2) walks tiles of
// 128 CTAS rows.  In a pair every CTA holds its own rows of A, half of B's
// columns and the accumulators of its own rows; its first CTA issues the
// products of both.  A 256-column pair tile fetches 64 bytes per cycle and SM
// where a single CTA's fetches 96, more than L2 delivers (131072 x 1024 x 4096:
// 10.1 against 14.7 ms, forward and backward).
//
// kLinear: out = epilogue(A B^T), two accumulator buffers.
// kGated: B's tile is bn/2 gate and bn/2 up rows of Win, the accumulator's
// halves are g and u of the same hidden columns.
// kGatedBwd: a tile is 2 bh hidden columns: [g|u] = x Win^T of one half
// (accumulators from 0 on), dh = dy Wout of both (from 256 on, so that dy is
// read once for them), then [g|u] of the other half.  All of the tensor memory
// is in use, so the products of a half wait until the epilogue has taken the
// last half's g and u into registers, which it does first; dh is overwritten a
// whole product later.
template <typename T, int MODE, bool FP8, int CTAS, int N>
__global__ void __launch_bounds__(kGemmThreads, 1) tc_gemm_kernel(const __grid_constant__ GemmArgs<N> args) {
    extern __shared__ __align__(1024) uint8_t smem[];  // stages, output staging, barriers
    uint8_t* out_stage = smem + args.stages * args.stage_bytes;
    uint64_t* full = reinterpret_cast<uint64_t*>(out_stage + kEpiWarps * (kStageOut + column_bytes<FP8>()));
    uint64_t *empty = full + kMaxStages, *tfull = empty + kMaxStages, *tempty = tfull + 2, *dempty = tempty + 2, *drain = dempty + 1;
    uint32_t* tmem_ptr = reinterpret_cast<uint32_t*>(drain + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = CTAS == 2 ? (int)(blockIdx.x & 1) : 0;
    constexpr int BK = FP8 ? 128 : 64;
    constexpr int kABytes = kBM * kRowBytes;
    constexpr int kDh = 256;                                   // tensor memory columns of dh

    grid_release();
    if (threadIdx.x == 0) {
        for (int i = 0; i < args.stages; ++i) mbar_init(&full[i], 2), mbar_init(&empty[i], 1);
        for (int i = 0; i < 2; ++i)
            mbar_init(&tfull[i], 1), mbar_init(&tempty[i], kEpiWarps * CTAS);
        mbar_init(dempty, kEpiWarps * CTAS);
        mbar_init(drain, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) tmem_take<CTAS>(tmem_ptr);
    tc_fence_before();
    __syncthreads();
    sync_all<CTAS>();
    tc_fence_after();
    grid_wait();
    const uint32_t tmem = *tmem_ptr;
    const int cta = blockIdx.x / CTAS, ctas = gridDim.x / CTAS;
    // One work unit after another, in the same order in every role.
#define LFB_EACH_UNIT(OK)                                                                                        \
    for (int turn = 0, unit; OK && (unit = unit_of(args, cta, ctas, turn)) < args.first[N]; ++turn)
#define LFB_PROBLEM(RANK)                                                                                        \
    const Problem& p = args.p[problem_of(args, unit)];                                                           \
    const int bh = p.bn / 2; /* hidden columns of a gated tile */                                                \
    const Tile t = tile_of<CTAS>(p, unit, MODE == kGated ? bh : p.bn, RANK);                                     \
    const int subs = MODE == kGatedBwd && t.n0 + bh < p.n ? 2 : 1 /* halves of a kGatedBwd tile */
    bool ok = true;

    if (warp == 0 || warp == 2) {
        // One warp copies A, the other B: a copy takes its issuer a few
        // hundred cycles, and one warp for both could not feed the products.
        const bool is_a = warp == 0;
        if (elect_one()) {
            int s = 0, issued = 0;
            uint32_t ph = 0;
            const uint32_t bars = CTAS == 2 ? leader_addr(full) : smem_u32(full);
            LFB_EACH_UNIT(ok) {
                LFB_PROBLEM(rank);
                const int bw = p.bn / CTAS;                    // B rows that this CTA holds
                const int n = t.it1 - t.it0;
                int ks = t.it0 / p.seg_iters, in_seg = t.it0 - ks * p.seg_iters;  // gated modes: product and step of K
                for (int left = MODE == kGatedBwd ? n * (1 + subs) : n; left > 0; --left) {
                    if (!(ok = mbar_wait(&empty[s], ph ^ 1))) break;
                    const bool dh = MODE == kGatedBwd && ks == 1;
                    const int k0 = in_seg * BK, n0 = MODE == kGatedBwd && ks == 2 ? t.n0 + bh : t.n0;
                    uint8_t* dst = smem + s * args.stage_bytes + (is_a ? 0 : kABytes);
                    const uint32_t bar = bars + 8 * s;
                    if (rank == 0) mbar_expect(&full[s], (is_a ? kABytes : bw * kRowBytes) * CTAS);
                    if (is_a) {
                        if (dh) tma_load<CTAS>(dst, &p.a2, bar, k0, t.m0, 0);
                        else if (!p.a_mn) tma_load<CTAS>(dst, &p.a, bar, k0, t.m0, MODE == kLinear ? ks : 0);
                        else
                            for (int j = 0; j < kBM / 64; ++j) tma_load<CTAS>(dst + j * 8192, &p.a, bar, t.m0 + 64 * j, k0, t.seg);
                    } else if (dh) {
                        for (int j = 0; j < bw / 64; ++j) tma_load<CTAS>(dst + j * 8192, &p.b2, bar, t.n0 + rank * bw + 64 * j, k0, 0);
                    } else if (MODE != kLinear) {
                        if (CTAS == 2) tma_load<CTAS>(dst, &p.b, bar, k0, n0, rank);  // one CTA the gate rows, the other the up rows
                        else
                            for (int j = 0; j < 2; ++j) tma_load<CTAS>(dst + j * bh * kRowBytes, &p.b, bar, k0, n0, j);
                    } else if (!p.b_mn) {
                        tma_load<CTAS>(dst, &p.b, bar, k0, t.n0 + rank * bw, ks);
                    } else {
                        for (int j = 0; j < bw / 64; ++j) tma_load<CTAS>(dst + j * 8192, &p.b, bar, t.n0 + rank * bw + 64 * j, k0, ks);
                    }
                    ++issued;
                    if (++in_seg == p.seg_iters) in_seg = 0, ++ks;
                    if (++s == args.stages) s = 0, ph ^= 1;
                }
            }
            // A wait ran out: let the copies in flight land before the block
            // ends (the leader's barriers count both CTAs' copies).
            if (!ok && rank == 0)
                for (int k = max(0, issued - args.stages); k < issued; ++k)
                    mbar_wait(&full[k % args.stages], (k / args.stages) & 1, 100000000ull);
        }
        __syncwarp();
    } else if (warp == 1) {
        if (rank == 0) {
            const uint32_t go = elect_one() ? 1u : 0u;
            int s = 0, buf = 0;
            uint32_t ph = 0, bph = 0, dph = 0;
            LFB_EACH_UNIT(ok) {
                LFB_PROBLEM(0);
                const uint32_t a_lbo = p.a_mn ? 8192 : 16, b_lbo = p.b_mn ? 8192 : 16, idesc = p.idesc;
                const uint64_t a_step = p.a_mn ? 128 : 2, b_step = p.b_mn ? 128 : 2;
                const int n = t.it1 - t.it0, products = MODE == kGatedBwd ? 1 + subs : 1;
                for (int product = 0; ok && product < products; ++product) {
                    const bool dh = MODE == kGatedBwd && product == 1;
                    // The accumulators' last reader: the half before (g and u), the tile before (dh), two tiles ago (others).
                    if (dh) ok = mbar_wait(dempty, dph ^ 1);
                    else ok = mbar_wait(&tempty[buf], bph ^ 1);
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t acc = tmem + (dh ? kDh : buf * 256);
                    for (int i = 0; i < n; ++i) {
                        if (!(ok = mbar_wait(&full[s], ph))) break;
                        tc_fence_after();
                        const uint32_t sa = smem_u32(smem + s * args.stage_bytes), sb = sa + kABytes;
                        const uint64_t da = make_desc(sa, dh ? 16 : a_lbo, 1024), db = make_desc(sb, dh ? 8192 : b_lbo, 1024);
                        const uint64_t as = dh ? 2 : a_step, bs = dh ? 128 : b_step;
                        const uint32_t id = dh ? p.idesc2 : idesc;
#pragma unroll
                        for (int k = 0; k < 4; ++k) mma<CTAS, FP8>(acc, da + k * as, db + k * bs, id, i > 0 || k > 0 ? 1u : 0u, go);
                        if (go) commit<CTAS>(&empty[s]);
                        if (++s == args.stages) s = 0, ph ^= 1;
                    }
                    if (!ok || (MODE == kGatedBwd && product == 0)) continue;
                    if (go) commit<CTAS>(&tfull[buf]);
                    if (MODE != kGatedBwd) buf ^= 1;
                    if (buf == 0) bph ^= 1;
                }
                dph ^= 1;
            }
            if (!ok) {  // products in flight end before the tensor memory is freed
                if (go) commit<CTAS>(drain);
                mbar_wait(drain, 0, 100000000ull);
            }
        }
    } else {
        const int ew = warp - kControlWarps, quad = warp & 3, cg = ew >> 2;  // lanes of the tensor memory, columns of a tile
        uint8_t* st = out_stage + ew * kStageOut;
        T* cv = reinterpret_cast<T*>(out_stage + kEpiWarps * kStageOut + ew * column_bytes<FP8>());
        float* cs = reinterpret_cast<float*>(cv);  // 8-bit form: 32 scales, then 32 biases
        // Writes the staged 32x32 outputs by TMA, and waits until they may be overwritten.
        auto put = [&](const CUtensorMap* out, int col, int row, int plane, bool some) {
            fence_async_smem();
            __syncwarp();
            if (lane == 0 && some) tma_store(out, st, col, row, plane);
        };
        auto reuse = [&] {
            if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
            __syncwarp();
        };
        int buf = 0;
        uint32_t bph = 0;
        LFB_EACH_UNIT(ok) {
            LFB_PROBLEM(rank);
            const Epilogue& e = p.e;
            const uint32_t lanes = (uint32_t)(quad * 32) << 16;
            const int rows = p.m - t.m0 - quad * 32;                           // rows that exist from the warp's first on
            const int64_t row0 = (int64_t)t.seg * p.m + t.m0 + quad * 32;      // in the output
            for (int sub = 0; sub < subs; ++sub) {
                const int n0 = t.n0 + sub * bh, cend = min(MODE == kLinear ? p.bn : bh, p.n - n0);
                uint64_t* tf = &tfull[buf];
                const int last = cg * 32 + (cend - cg * 32 - 1) / kEpiCols * kEpiCols;  // this warp's last 32 columns (if it has any)
                auto release = [&](uint64_t* bar) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) arrive_leader<CTAS>(bar);
                };
                if (cg * 32 >= cend) {                                           // none: wait for the tile all the same
                    if (!(ok = mbar_wait(tf, bph))) break;
                    tc_fence_after();
                    release(&tempty[buf]);
                    if (MODE == kGatedBwd && sub == subs - 1) release(dempty);
                } else
                if constexpr (MODE == kLinear) {
                    const uint32_t acc = tmem + buf * 256 + lanes;
                    const float sa = FP8 && lane < rows && !p.part ? e.sa[row0 + lane] : 1.f;
                    const int first = cg * 32;
                    if (!p.part) {
                        // Finished in the accumulator's layout (a lane owns a
                        // row); the column values and the residual of the next
                        // columns are fetched ahead.
                        T bias;
                        float sb = 1.f;
                        uint4 r[4];
                        auto fetch = [&](int c0) {
                            const int col = t.n0 + c0 + lane, col8 = t.n0 + c0 + (lane & 3) * 8;
                            bias = column_value((const T*)e.bias, col, p.n);
                            if (FP8) sb = col < p.n ? e.sb[col] : 1.f;
                            if (!e.res) return;
                            if (!e.vec_res) {  // a column per lane, two rows per register
                                const T* q = (const T*)e.res + row0 * e.ldr + col;
                                uint32_t* w = reinterpret_cast<uint32_t*>(r);
#pragma unroll
                                for (int i = 0; i < 16; ++i, q += 2 * e.ldr) {
                                    const T a = 2 * i < rows && col < p.n ? q[0] : Elem<T>::store(0.f);
                                    const T b = 2 * i + 1 < rows && col < p.n ? q[e.ldr] : Elem<T>::store(0.f);
                                    w[i] = (uint32_t)*reinterpret_cast<const uint16_t*>(&a) | (uint32_t)*reinterpret_cast<const uint16_t*>(&b) << 16;
                                }
                                return;
                            }
                            const T* q = (const T*)e.res + (row0 + (lane >> 2)) * e.ldr + col8;
#pragma unroll
                            for (int i = 0; i < 4; ++i, q += 8 * e.ldr)
                                r[i] = i * 8 + (lane >> 2) < rows && col8 < p.n ? *reinterpret_cast<const uint4*>(q) : make_uint4(0u, 0u, 0u, 0u);
                        };
                        fetch(first);
                        if (!(ok = mbar_wait(tf, bph))) break;
                        tc_fence_after();
                        for (int c0 = first; c0 < cend; c0 += kEpiCols) {
                            reuse();
                            if (FP8) cs[lane] = sb, cs[32 + lane] = Elem<T>::load(bias);
                            else if (e.bias) cv[lane] = bias;
                            if (e.res && e.vec_res) {  // to the lane that owns the row
#pragma unroll
                                for (int i = 0; i < 4; ++i) *reinterpret_cast<uint4*>(stage_at(st, i * 8 + (lane >> 2), lane & 3)) = r[i];
                            } else if (e.res) {
                                const uint32_t* w = reinterpret_cast<const uint32_t*>(r);
#pragma unroll
                                for (int i = 0; i < 16; ++i) {
                                    *reinterpret_cast<uint16_t*>(stage_at(st, 2 * i, lane >> 3) + (lane & 7) * 2) = (uint16_t)w[i];
                                    *reinterpret_cast<uint16_t*>(stage_at(st, 2 * i + 1, lane >> 3) + (lane & 7) * 2) = (uint16_t)(w[i] >> 16);
                                }
                            }
                            fetch(c0 + kEpiCols);
                            __syncwarp();
                            uint4 o[2][2];
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                float v[16];
                                tmem_ld16(acc + c0 + h * 16, v);
                                tmem_wait_ld();
                                reg_fence(v);
                                if (h == 1 && c0 == last) release(&tempty[buf]);
                                if (FP8) {  // (v sw) sx + b in pairs
                                    const uint64_t sx = pk2(sa, sa);
#pragma unroll
                                    for (int j = 0; j < 16; j += 2) {
                                        const uint64_t w = *reinterpret_cast<const uint64_t*>(cs + h * 16 + j);
                                        const uint64_t b = *reinterpret_cast<const uint64_t*>(cs + 32 + h * 16 + j);
                                        upk2(fma2(mul2(pk2(v[j], v[j + 1]), w), sx, b), v[j], v[j + 1]);
                                    }
                                } else if (e.bias) add_columns(v, cv + h * 16);
                                if (e.act != LF_ACT_NONE)
                                    with_act(e.act, [&](auto act) {
#pragma unroll
                                        for (int j = 0; j < 16; ++j) {
                                            float a, slope;
                                            if (e.act_bwd) act_both<decltype(act)::value>(v[j], a, slope);
                                            else slope = act_value<decltype(act)::value>(v[j]);
                                            v[j] = slope;
                                        }
                                    });
                                if (e.res) {  // added to the activation, or dy times its derivative
#pragma unroll
                                    for (int c = 0; c < 2; ++c) {
                                        const uint4 u = *reinterpret_cast<const uint4*>(stage_at(st, lane, 2 * h + c));
                                        const uint32_t* w = reinterpret_cast<const uint32_t*>(&u);
#pragma unroll
                                        for (int k = 0; k < 4; ++k) {
                                            const float2 x = unpack2<T>(w[k]);
                                            float &y0 = v[8 * c + 2 * k], &y1 = v[8 * c + 2 * k + 1];
                                            y0 = e.act_bwd ? y0 * x.x : y0 + x.x;
                                            y1 = e.act_bwd ? y1 * x.y : y1 + x.y;
                                        }
                                    }
                                }
                                pack16<T>(o[h], v);
                            }
                            __syncwarp();
                            stage16(st, lane, 0, o[0]);
                            stage16(st, lane, 1, o[1]);
                            if (e.tma) put(&p.out, t.n0 + c0, t.m0 + quad * 32, t.seg, rows > 0);
                            else put_rows<T>(st, lane, (T*)e.out + row0 * e.ldo + t.n0 + c0, e.ldo, rows, cend - c0, e.pairs);
                        }
                    } else {
                        // Split-K partials: raw sums through shared memory, 16
                        // columns at a time, as row segments.
                        if (!(ok = mbar_wait(tf, bph))) break;
                        tc_fence_after();
                        reuse();  // the last tile may have been another problem's
                        for (int c0 = first; c0 < cend; c0 += kEpiCols) {
#pragma unroll 1
                            for (int h = 0; h < 2; ++h) {
                                const int col = t.n0 + c0 + h * 16 + (lane & 3) * 4, row = lane >> 2;
                                float v[16];
                                tmem_ld16(acc + c0 + h * 16, v);
                                tmem_wait_ld();
                                reg_fence(v);
                                if (c0 == last && h == 1) release(&tempty[buf]);
                                __syncwarp();
#pragma unroll
                                for (int c = 0; c < 4; ++c)
                                    *reinterpret_cast<float4*>(stage_at(st, lane, c)) = make_float4(v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]);
                                __syncwarp();
                                float* q = p.part + ((int64_t)t.split * p.msegs * p.m + row0 + row) * p.ldp + col;
#pragma unroll
                                for (int i = 0; i < 4; ++i, q += 8 * p.ldp)
                                    if (i * 8 + row < rows && col < p.ldp)
                                        *reinterpret_cast<float4*>(q) = *reinterpret_cast<const float4*>(stage_at(st, i * 8 + row, lane & 3));
                            }
                        }
                    }
                } else {
                    const T* bias = (const T*)e.bias;
                    const uint32_t acc = tmem + buf * 256 + lanes;
                    const int c0 = cg * 32;                                        // the warp's only columns
                    const T bg = column_value(bias, n0 + c0 + lane, p.n);
                    const T bu = column_value(bias ? bias + p.n : bias, n0 + c0 + lane, p.n);
                    if (!(ok = mbar_wait(tf, bph))) break;
                    tc_fence_after();
                    if (MODE == kGated) reuse();
                    if (bias) {
                        cv[lane] = bg, cv[32 + lane] = bu;
                        __syncwarp();
                    }
                    // 16 columns at a time; outputs wait as 16-bit pairs.
                    uint4 og[2][2], ou[2][2];
                    if constexpr (MODE == kGated) {
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            float g[16], u[16];
                            tmem_ld16(acc + c0 + h * 16, g);
                            tmem_ld16(acc + bh + c0 + h * 16, u);
                            tmem_wait_ld();
                            reg_fence(g);
                            reg_fence(u);
                            if (h == 1) release(&tempty[buf]);
                            if (bias) add_columns(g, cv + h * 16), add_columns(u, cv + 32 + h * 16);
                            with_act(e.act, [&](auto act) {
#pragma unroll
                                for (int j = 0; j < 16; ++j) u[j] *= act_value<decltype(act)::value>(g[j]);
                            });
                            pack16<T>(ou[h], u);
                        }
                    } else {
                        float g[2][16], u[2][16];
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            tmem_ld16(acc + c0 + h * 16, g[h]);
                            tmem_ld16(acc + bh + c0 + h * 16, u[h]);
                        }
                        tmem_wait_ld();
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            reg_fence(g[h]);
                            reg_fence(u[h]);
                        }
                        release(tempty);
                        reuse();
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            if (bias) add_columns(g[h], cv + h * 16), add_columns(u[h], cv + 32 + h * 16);
                            uint4 oh[2];
#pragma unroll
                            for (int c = 0; c < 2; ++c) {  // eight columns of dh at a time: registers are full
                                float d[8];
                                tmem_ld8(tmem + kDh + sub * bh + lanes + c0 + h * 16 + c * 8, d);
                                tmem_wait_ld();
                                reg_fence(d);
                                if (h == 1 && c == 1 && sub == subs - 1) release(dempty);
                                // h = act(g) u, du = dh act(g), dg = dh u act'(g), in d, g and u
                                with_act(e.act, [&](auto act) {
#pragma unroll
                                    for (int j = 0; j < 8; ++j) {
                                        float a, slope;
                                        float &gj = g[h][c * 8 + j], &uj = u[h][c * 8 + j];
                                        act_both<decltype(act)::value>(gj, a, slope);
                                        const float dh = d[j];
                                        d[j] = a * uj;
                                        gj = a * dh;
                                        uj *= slope * dh;
                                    }
                                });
                                oh[c] = pack8<T>(d);
                                og[h][c] = pack8<T>(&g[h][c * 8]);
                                ou[h][c] = pack8<T>(&u[h][c * 8]);
                            }
                            stage16(st, lane, h, oh);
                        }
                    }
                    const int row = t.m0 + quad * 32;
                    if constexpr (MODE == kGatedBwd) {  // planes dg, du, h
                        put(&p.out, n0 + c0, row, 2, rows > 0);
                        reuse();
                        stage16(st, lane, 0, og[0]);
                        stage16(st, lane, 1, og[1]);
                        put(&p.out, n0 + c0, row, 1, rows > 0);
                        reuse();
                    }
                    stage16(st, lane, 0, ou[0]);
                    stage16(st, lane, 1, ou[1]);
                    put(&p.out, n0 + c0, row, 0, rows > 0);
                }
                if (MODE != kGatedBwd) buf ^= 1;
                if (buf == 0) bph ^= 1;
            }
        }
        if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");  // outputs written, staging read
    }
    if (!ok && lane == 0) atomicExch(&g_gemm_status, (int)LF_ERR_TIMEOUT);
    tc_fence_before();
    __syncthreads();
    sync_all<CTAS>();  // no CTA of a pair leaves while the other's products read its operands
    tc_fence_after();
    if (warp == 1) tmem_free<CTAS>(tmem);
#undef LFB_EACH_UNIT
#undef LFB_PROBLEM
}

// ---------------------------------------------------------------------------
// The feed-forward block's forward for at most 64 channels, in one kernel
// ---------------------------------------------------------------------------
// With so few channels the products are short and h is most of the traffic (at
// 64 channels and 256 hidden columns 102 of 140 MB per 100,000 tokens), so h
// never leaves the SM: a CTA owns 128 tokens and walks the hidden columns in
// blocks of 64,
//   [g|u] = x [Wg|Wu]^T      (two accumulator buffers)
//   h = act(g) u             to shared memory as the next product's A operand
//   y += h Wout^T            (accumulators of two tiles in turn)
// Each product has a warp that issues it, so that the first ones run ahead of
// the second ones; two groups of eight epilogue warps take the blocks in turn,
// and a tile's y goes to the group of its last block, after that group's next
// block.  Up to five blocks of weights (320 hidden columns) are copied once and
// stay; more go through a ring.
constexpr int kHB = 64;                   // hidden columns of a block
constexpr int kNarrow = 64;               // channels

struct alignas(64) NarrowArgs {
    CUtensorMap x, win, wout, out;
    Epilogue e;                // out, output bias, residual, activation of the gate
    const void* b_in;
    int m, c, f, tiles, blocks, stages;
    uint32_t idesc1, idesc2;
};

template <typename T>
__global__ void __launch_bounds__(kGemmThreads, 1) narrow_ffn_kernel(const __grid_constant__ NarrowArgs p) {
    extern __shared__ __align__(1024) uint8_t smem[];  // x (two tiles), h (two blocks), weight stages, staging, barriers
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    constexpr int x_bytes = kBM * kRowBytes, w_bytes = 3 * kHB * kRowBytes;
    constexpr int kHBytes = kBM * kRowBytes;
    uint8_t* const hs = smem + 2 * x_bytes;
    uint8_t* const ring = hs + 2 * kHBytes;
    uint8_t* const out_stage = ring + p.stages * w_bytes;
    uint64_t* const bars = reinterpret_cast<uint64_t*>(out_stage + kEpiWarps * (kStageOut + column_bytes<false>()));
    uint64_t *wfull = bars, *wempty = bars + 6, *xfull = bars + 12, *xempty = bars + 14, *gfull = bars + 16, *gempty = bars + 18,
             *hfull = bars + 20, *hempty = bars + 22, *yfull = bars + 24, *yempty = bars + 26, *drain = bars + 28;
    uint32_t* tmem_ptr = reinterpret_cast<uint32_t*>(bars + 30);
    constexpr int kY = 256;                                    // tensor memory columns of y
    grid_release();
    if (threadIdx.x == 0) {
        for (int i = 0; i < p.stages; ++i) mbar_init(&wfull[i], 1), mbar_init(&wempty[i], 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&xfull[i], 1), mbar_init(&xempty[i], 1), mbar_init(&gfull[i], 1), mbar_init(&gempty[i], 8);
            mbar_init(&hfull[i], 8), mbar_init(&hempty[i], 1), mbar_init(&yfull[i], 1), mbar_init(&yempty[i], 8);
        }
        mbar_init(&drain[0], 1), mbar_init(&drain[1], 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) tmem_take<1>(tmem_ptr);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    grid_wait();
    const uint32_t tmem = *tmem_ptr;
    const int mine = (p.tiles - (int)blockIdx.x + (int)gridDim.x - 1) / (int)gridDim.x;  // this CTA's tiles
    const int total = mine * p.blocks;                                                  // and their blocks
    const bool resident = p.blocks <= p.stages;                                         // all weights stay in shared memory
    const int ring_len = resident ? p.blocks : p.stages;
    bool ok = true;

    if (warp == 2) {  // copies: x tiles; per block 64 gate and 64 up rows of Win and Wout's columns
        if (elect_one()) {
            int s = 0, j = 0, t = 0, issued = 0;
            uint32_t ph = 0;
            for (int g = 0; g < total; ++g) {
                if (j == 0) {
                    const int b = t & 1;
                    if (!(ok = mbar_wait(&xempty[b], (t >> 1 & 1) ^ 1))) break;
                    mbar_expect(&xfull[b], x_bytes);
                    tma_load<1>(smem + b * x_bytes, &p.x, smem_u32(&xfull[b]), 0, (int)(blockIdx.x + t * gridDim.x) * kBM, 0);
                    ++t;
                }
                if (!resident || g < p.blocks) {
                    if (!(ok = mbar_wait(&wempty[s], ph ^ 1))) break;
                    uint8_t* dst = ring + s * w_bytes;
                    const uint32_t bar = smem_u32(&wfull[s]);
                    mbar_expect(&wfull[s], w_bytes);
                    tma_load<1>(dst, &p.win, bar, 0, j * kHB, 0);  // both planes: gate, then up rows
                    tma_load<1>(dst + 2 * kHB * kRowBytes, &p.wout, bar, j * kHB, 0, 0);
                    ++issued;
                    if (++s == p.stages) s = 0, ph ^= 1;
                }
                if (++j == p.blocks) j = 0;
            }
            if (!ok) {  // a wait ran out: let the copies in flight land
                for (int k = max(0, t - 2); k < t; ++k) mbar_wait(&xfull[k & 1], k >> 1 & 1, 100000000ull);
                for (int k = max(0, issued - p.stages); k < issued; ++k)
                    mbar_wait(&wfull[k % p.stages], (k / p.stages) & 1, 100000000ull);
            }
        }
        __syncwarp();
    } else if (warp == 1) {  // [g|u] = x [Wg|Wu]^T
        const uint32_t go = elect_one() ? 1u : 0u;
        int s = 0, j = 0, t = 0;
        uint32_t ph = 0;
        for (int g = 0; g < total; ++g) {
            const int b = g & 1;
            if (j == 0) ok = mbar_wait(&xfull[t & 1], t >> 1 & 1);
            ok = ok && mbar_wait(&wfull[s], resident ? 0 : ph) && mbar_wait(&gempty[b], (g >> 1 & 1) ^ 1);
            if (!ok) break;
            tc_fence_after();
            const uint64_t da = make_desc(smem_u32(smem + (t & 1) * x_bytes), 16, 1024);
            const uint64_t db = make_desc(smem_u32(ring + s * w_bytes), 16, 1024);
#pragma unroll
            for (int i = 0; i < 4; ++i) mma<1, false>(tmem + b * 128, da + i * 2, db + i * 2, p.idesc1, i > 0 ? 1u : 0u, go);
            if (go) commit<1>(&gfull[b]);
            if (++j == p.blocks) {
                if (go) commit<1>(&xempty[t & 1]);
                j = 0, ++t;
            }
            if (++s == ring_len) s = 0, ph ^= 1;
        }
        if (!ok) {  // products in flight end before the tensor memory is freed
            if (go) commit<1>(&drain[0]);
            mbar_wait(&drain[0], 0, 100000000ull);
        }
    } else if (warp == 0) {  // y += h Wout^T
        const uint32_t go = elect_one() ? 1u : 0u;
        int s = 0, j = 0, t = 0;
        uint32_t ph = 0;
        for (int g = 0; g < total; ++g) {
            const int b = g & 1;
            if (j == 0) ok = mbar_wait(&yempty[t & 1], (t >> 1 & 1) ^ 1);
            ok = ok && mbar_wait(&wfull[s], resident ? 0 : ph) && mbar_wait(&hfull[b], g >> 1 & 1);
            if (!ok) break;
            tc_fence_after();
            const uint64_t da = make_desc(smem_u32(hs + b * kHBytes), 16, 1024);
            const uint64_t db = make_desc(smem_u32(ring + s * w_bytes) + 2 * kHB * kRowBytes, 16, 1024);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                mma<1, false>(tmem + kY + (t & 1) * 128, da + i * 2, db + i * 2, p.idesc2, j > 0 || i > 0 ? 1u : 0u, go);
            if (go) commit<1>(&hempty[b]);
            if (go && !resident) commit<1>(&wempty[s]);  // h was made of the first product, so that one has read its weights too
            if (++j == p.blocks) {
                if (go) commit<1>(&yfull[t & 1]);
                j = 0, ++t;
            }
            if (++s == ring_len) s = 0, ph ^= 1;
        }
        if (!ok) {
            if (go) commit<1>(&drain[1]);
            mbar_wait(&drain[1], 0, 100000000ull);
        }
    } else {
        const int ew = warp - kControlWarps, quad = warp & 3, half = ew >> 2 & 1, group = ew >> 3;
        uint8_t* st = out_stage + ew * kStageOut;
        T* cv = reinterpret_cast<T*>(out_stage + kEpiWarps * kStageOut + ew * column_bytes<false>());
        const uint32_t lanes = (uint32_t)(quad * 32) << 16;
        const Epilogue& e = p.e;
        auto arrive = [&](uint64_t* bar) {
            __syncwarp();
            if (lane == 0) arrive_leader<1>(bar);
        };
        // A warp writes 32 rows and 32 columns of a tile's y.
        const int c0 = half * 32;
        auto first_row = [&](int t) { return (int)(blockIdx.x + t * gridDim.x) * kBM + quad * 32; };
        uint4 r[4];  // its residual, where that comes in 16-byte chunks
        auto fetch = [&](int t) {
            if (!e.res || !e.vec_res) return;
            const int m0 = first_row(t), col8 = c0 + (lane & 3) * 8;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int row = m0 + i * 8 + (lane >> 2);
                r[i] = make_uint4(0u, 0u, 0u, 0u);
                if (row < p.m && col8 < p.c) r[i] = *reinterpret_cast<const uint4*>((const T*)e.res + (int64_t)row * e.ldr + col8);
            }
        };
        // y of tile t: accumulators, output bias, residual.
        auto finish = [&](int t) {
            const int m0 = first_row(t), rows = p.m - m0;
            if (!(ok = mbar_wait(&yfull[t & 1], t >> 1 & 1))) return;
            tc_fence_after();
            if (c0 < p.c) {
                if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                __syncwarp();
                if (e.bias) cv[lane] = column_value((const T*)e.bias, c0 + lane, p.c);
                if (e.res && e.vec_res) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) *reinterpret_cast<uint4*>(stage_at(st, i * 8 + (lane >> 2), lane & 3)) = r[i];
                } else if (e.res) {
#pragma unroll 8
                    for (int r = 0; r < 32; ++r)
                        *reinterpret_cast<T*>(stage_at(st, r, lane >> 3) + (lane & 7) * 2) =
                            r < rows && c0 + lane < p.c ? ((const T*)e.res)[(int64_t)(m0 + r) * e.ldr + c0 + lane] : Elem<T>::store(0.f);
                }
                __syncwarp();
                uint4 o[2][2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float v[16];
                    tmem_ld16(tmem + kY + (t & 1) * 128 + lanes + c0 + h * 16, v);
                    tmem_wait_ld();
                    reg_fence(v);
                    if (e.bias) add_columns(v, cv + h * 16);
                    if (e.res) {
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            const uint4 u = *reinterpret_cast<const uint4*>(stage_at(st, lane, 2 * h + c));
                            const uint32_t* w = reinterpret_cast<const uint32_t*>(&u);
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                const float2 x = unpack2<T>(w[k]);
                                v[8 * c + 2 * k] += x.x, v[8 * c + 2 * k + 1] += x.y;
                            }
                        }
                    }
                    pack16<T>(o[h], v);
                }
                tc_fence_before();
                arrive(&yempty[t & 1]);
                stage16(st, lane, 0, o[0]);
                stage16(st, lane, 1, o[1]);
                if (e.tma) {
                    fence_async_smem();
                    __syncwarp();
                    if (lane == 0 && rows > 0) tma_store(&p.out, st, c0, m0, 0);
                } else {
                    put_rows<T>(st, lane, (T*)e.out + (int64_t)m0 * e.ldo + c0, e.ldo, rows, p.c - c0, e.pairs);
                }
            } else arrive(&yempty[t & 1]);
        };
        int owed = -1;  // a tile whose y this group still has to write
        int t = group / p.blocks, j = group - t * p.blocks;     // this block's tile and place in it
        for (int g = group; ok && g < total; g += 2) {
            const int n0 = j * kHB + half * 32;
            const T bg = column_value((const T*)p.b_in, n0 + lane, p.f);
            const T bu = column_value(p.b_in ? (const T*)p.b_in + p.f : nullptr, n0 + lane, p.f);
            if (!(ok = mbar_wait(&gfull[group], g >> 1 & 1))) break;
            tc_fence_after();
            if (p.b_in) {
                cv[lane] = bg, cv[32 + lane] = bu;
                __syncwarp();
            }
            uint4 o[2][2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float gt[16], u[16];
                const uint32_t acc = tmem + group * 128 + lanes + half * 32 + h * 16;
                tmem_ld16(acc, gt);
                tmem_ld16(acc + kHB, u);
                tmem_wait_ld();
                reg_fence(gt);
                reg_fence(u);
                if (h == 1) {
                    tc_fence_before();
                    arrive(&gempty[group]);
                }
                if (p.b_in) add_columns(gt, cv + h * 16), add_columns(u, cv + 32 + h * 16);
                with_act(e.act, [&](auto act) {
#pragma unroll
                    for (int k = 0; k < 16; ++k) u[k] *= act_value<decltype(act)::value>(gt[k]);
                });
                const int left = p.f - (n0 + h * 16);
                if (left < 16) {  // columns past the last: zeros even where x is infinite
#pragma unroll
                    for (int k = 0; k < 16; ++k)
                        if (k >= left) u[k] = 0.f;
                }
                pack16<T>(o[h], u);
            }
            if (!(ok = mbar_wait(&hempty[group], (g >> 1 & 1) ^ 1))) break;
            const int row = quad * 32 + lane;
            uint8_t* hr = hs + group * kHBytes + row * kRowBytes;
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int c = 0; c < 2; ++c) *reinterpret_cast<uint4*>(hr + (((half * 4 + h * 2 + c) ^ (row & 7)) << 4)) = o[h][c];
            fence_async_smem();
            arrive(&hfull[group]);
            if (owed >= 0) {
                finish(owed);
                owed = -1;
            }
            if (j == p.blocks - 1) fetch(owed = t);
            for (j += 2; j >= p.blocks; j -= p.blocks) ++t;
        }
        if (ok && owed >= 0) finish(owed);
        if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }
    if (!ok && lane == 0) atomicExch(&g_gemm_status, (int)LF_ERR_TIMEOUT);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 1) tmem_free<1>(tmem);
}

// ---------------------------------------------------------------------------
// The feed-forward block's backward for at most 64 channels and 256 hidden
// columns, in one kernel
// ---------------------------------------------------------------------------
// Here too the hidden tensors (h, dg, du: 154 MB written and 256 read again for
// 100,000 tokens of 64 channels and 256 hidden columns, where x, dy and dx have
// 38) stay in the SM.  A CTA owns 128 hidden columns, whose weights stay in
// shared memory, and every slots-th tile of 128 tokens; it takes them in two
// blocks of 64 columns:
//   [g|u] = x [Wg|Wu]^T,  dh = dy Wout
//   dg = dh u act'(g),  du = dh act(g),  h = act(g) u     to shared memory
//   dx += dg Wg + du Wu
// and once a tile
//   dWg += dg^T x,  dWu += du^T x,  dWout^T += h^T dy,
//   db_in += [dg|du]^T 1,  db_out += dy^T 1
// whose sums stay in tensor memory until the last tile; the partial sums of the
// slots are joined by another launch.  The tiles in shared memory serve as K-major
// operands for dx and as transposed ones for the weights.  More than 128 hidden
// columns take a cluster of two CTAs, one for each half, on the same tokens: each
// sends the other half of the rows of its dx through distributed shared memory
// and writes the sum for its own; four warps do that, so that the epilogue warps
// need not wait for the other CTA (100352 x 64 x 256: 52 against 73 us).
//
// At that size the kernel reads x and dy once from memory (26 MB) and is bound
// by the latency of a block's round from products to shared memory (3400
// cycles, of which the matrix pipe is busy for a quarter and the issue slots for
// a third): beside the sums, the tensor memory has no room for a second block's g, u
// and dh.  Blocks of 32 columns in two groups of warps measured 56 us.
constexpr int kBwdHidden = 128;           // hidden columns of a CTA
constexpr int kBwdThreads = kGemmThreads + 128;  // and four warps that write dx

struct alignas(64) NarrowBwdArgs {
    CUtensorMap x, dy, win, wout;
    const void* b_in;
    void* dx;
    float *part_in, *part_out;            // [slots][2f][ld_in], [slots][c][ld_out]; null: not asked for
    float *part_bi, *part_bo;             // [slots][ld_bi], [slots][ld_bo]: the biases'
    int ld_in, ld_out, ld_bi, ld_bo;
    int m, c, f, tiles, blocks, act;
    bool vec_dx;
    uint32_t id_gu, id_n, id_w, id_b;
};

__device__ __forceinline__ uint32_t peer_addr(const void* p, uint32_t rank) {  // the same shared memory in another CTA of the cluster
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
    return r;
}
__device__ __forceinline__ void peer_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool peer_wait(uint64_t* bar, uint32_t parity) {
    const bool done = mbar_wait(bar, parity);
    asm volatile("fence.acq_rel.cluster;" ::: "memory");
    return done;
}

template <typename T, int CTAS>
__global__ void __launch_bounds__(kBwdThreads, 1) narrow_ffn_bwd_kernel(const __grid_constant__ NarrowBwdArgs p) {
    extern __shared__ __align__(1024) uint8_t smem[];
    constexpr int tile_bytes = kBM * kRowBytes, w_bytes = 3 * kHB * kRowBytes;
    uint8_t* const weights = smem + 4 * tile_bytes;            // after two of x | dy
    uint8_t* const dg_s = weights + 2 * w_bytes;               // dg, du, h: two blocks each
    uint8_t *const du_s = dg_s + 2 * tile_bytes, *const h_s = du_s + 2 * tile_bytes;
    uint8_t* const inbox = h_s + 2 * tile_bytes;               // dx rows from the other CTA
    uint8_t* const ones = inbox + 16384;                       // B operand of the bias gradients
    T* const bias = reinterpret_cast<T*>(ones + 2048);
    uint64_t* const bars = reinterpret_cast<uint64_t*>(bias + 2 * kBwdHidden);
    uint64_t *wfull = bars, *xfull = bars + 1, *xempty = bars + 3, *gfull = bars + 5, *gempty = bars + 6, *hfull = bars + 7,
             *hempty = bars + 9, *dxfull = bars + 10, *dxempty = bars + 11, *infull = bars + 12, *inempty = bars + 13,
             *done = bars + 14, *drain = bars + 15;
    uint32_t* tmem_ptr = reinterpret_cast<uint32_t*>(bars + 17);
    constexpr int kDh = 128, kDx = 192, kDw = 256, kDb = 448;  // tensor memory columns; g and u from 0 on
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = CTAS == 2 ? (int)(blockIdx.x & 1) : 0, slot = (int)blockIdx.x / CTAS, slots = (int)gridDim.x / CTAS;
    grid_release();
    if (threadIdx.x == 0) {
        mbar_init(wfull, 1), mbar_init(gfull, 1), mbar_init(gempty, kEpiWarps), mbar_init(hempty, 1);
        mbar_init(dxfull, 1), mbar_init(dxempty, 4), mbar_init(infull, 2), mbar_init(inempty, 2), mbar_init(done, 1);
        for (int i = 0; i < 2; ++i)
            mbar_init(&xfull[i], 1), mbar_init(&xempty[i], 1), mbar_init(&hfull[i], kEpiWarps), mbar_init(&drain[i], 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    for (int i = threadIdx.x; i < 512; i += kBwdThreads) reinterpret_cast<uint32_t*>(ones)[i] = pack2<T>(1.f, 1.f);
    fence_async_smem();
    grid_wait();
    if (threadIdx.x < 2 * kBwdHidden) {
        const int up = threadIdx.x >= kBwdHidden, col = rank * kBwdHidden + (threadIdx.x & (kBwdHidden - 1));
        bias[threadIdx.x] = column_value(p.b_in ? (const T*)p.b_in + (up ? p.f : 0) : nullptr, col, p.f);
    }
    if (warp == 1) tmem_take<1>(tmem_ptr);
    tc_fence_before();
    __syncthreads();
    sync_all<CTAS>();
    tc_fence_after();
    const uint32_t tmem = *tmem_ptr;
    const int mine = (p.tiles - slot + slots - 1) / slots;
    const int n_first = rank * kBwdHidden;
    bool ok = true;

    if (warp == 2) {  // copies: the weights once, then x and dy of a tile
        if (elect_one()) {
            mbar_expect(wfull, p.blocks * w_bytes);
            for (int j = 0; j < p.blocks; ++j) {
                uint8_t* dst = weights + j * w_bytes;
                tma_load<1>(dst, &p.win, smem_u32(wfull), 0, n_first + j * kHB, 0);  // both planes: gate, then up rows
                tma_load<1>(dst + 2 * kHB * kRowBytes, &p.wout, smem_u32(wfull), n_first + j * kHB, 0, 0);
            }
            int t = 0;
            for (; t < mine; ++t) {
                const int b = t & 1;
                if (!(ok = mbar_wait(&xempty[b], (t >> 1 & 1) ^ 1))) break;
                mbar_expect(&xfull[b], 2 * tile_bytes);
                uint8_t* dst = smem + b * 2 * tile_bytes;
                tma_load<1>(dst, &p.x, smem_u32(&xfull[b]), 0, (slot + t * slots) * kBM, 0);
                tma_load<1>(dst + tile_bytes, &p.dy, smem_u32(&xfull[b]), 0, (slot + t * slots) * kBM, 0);
            }
            if (!ok) {  // a wait ran out: let the copies in flight land
                mbar_wait(wfull, 0, 100000000ull);
                for (int k = max(0, t - 2); k < t; ++k) mbar_wait(&xfull[k & 1], k >> 1 & 1, 100000000ull);
            }
        }
        __syncwarp();
    } else if (warp == 1) {  // [g|u] = x [Wg|Wu]^T, dh = dy Wout
        const uint32_t go = elect_one() ? 1u : 0u;
        ok = mbar_wait(wfull, 0);
        for (int t = 0, g = 0; ok && t < mine; ++t) {
            if (!(ok = mbar_wait(&xfull[t & 1], t >> 1 & 1))) break;
            const uint64_t dx = make_desc(smem_u32(smem + (t & 1) * 2 * tile_bytes), 16, 1024);
            const uint64_t ddy = make_desc(smem_u32(smem + (t & 1) * 2 * tile_bytes) + tile_bytes, 16, 1024);
            for (int j = 0; j < p.blocks; ++j, ++g) {
                if (!(ok = mbar_wait(gempty, (g & 1) ^ 1))) break;
                tc_fence_after();
                const uint32_t w = smem_u32(weights + j * w_bytes);
                const uint64_t dw = make_desc(w, 16, 1024), dwo = make_desc(w + 2 * kHB * kRowBytes, 8192, 1024);
#pragma unroll
                for (int i = 0; i < 4; ++i) mma<1, false>(tmem, dx + i * 2, dw + i * 2, p.id_gu, i > 0 ? 1u : 0u, go);
#pragma unroll
                for (int i = 0; i < 4; ++i) mma<1, false>(tmem + kDh, ddy + i * 2, dwo + i * 128, p.id_n, i > 0 ? 1u : 0u, go);
                if (go) commit<1>(gfull);
            }
        }
        if (!ok) {  // products in flight end before the tensor memory is freed
            if (go) commit<1>(&drain[0]);
            mbar_wait(&drain[0], 0, 100000000ull);
        }
    } else if (warp == 0) {  // dx of a tile and the weights' sums
        const uint32_t go = elect_one() ? 1u : 0u;
        ok = mbar_wait(wfull, 0);
        for (int t = 0; ok && t < mine; ++t) {
            ok = mbar_wait(&xfull[t & 1], t >> 1 & 1) && (!p.dx || mbar_wait(dxempty, (t & 1) ^ 1));
            for (int j = 0; ok && j < p.blocks; ++j) {
                if (!(ok = mbar_wait(&hfull[j], t & 1))) break;
                tc_fence_after();
                if (!p.dx) continue;
                const uint64_t dwg = make_desc(smem_u32(weights + j * w_bytes), 8192, 1024);
                const uint64_t dwu = make_desc(smem_u32(weights + j * w_bytes) + kHB * kRowBytes, 8192, 1024);
                const uint64_t dg = make_desc(smem_u32(dg_s + j * tile_bytes), 16, 1024);
                const uint64_t du = make_desc(smem_u32(du_s + j * tile_bytes), 16, 1024);
#pragma unroll
                for (int i = 0; i < 4; ++i) mma<1, false>(tmem + kDx, dg + i * 2, dwg + i * 128, p.id_n, j > 0 || i > 0 ? 1u : 0u, go);
#pragma unroll
                for (int i = 0; i < 4; ++i) mma<1, false>(tmem + kDx, du + i * 2, dwu + i * 128, p.id_n, 1u, go);
            }
            if (!ok) break;
            if (go && p.dx) commit<1>(dxfull);
            // the tiles again, transposed: 128 hidden columns by 128 tokens
            const uint64_t dg = make_desc(smem_u32(dg_s), tile_bytes, 1024), du = make_desc(smem_u32(du_s), tile_bytes, 1024);
            const uint64_t h = make_desc(smem_u32(h_s), tile_bytes, 1024), one = make_desc(smem_u32(ones), 16, 1024);
            const uint64_t x = make_desc(smem_u32(smem + (t & 1) * 2 * tile_bytes), 8192, 1024);
            const uint64_t dy = make_desc(smem_u32(smem + (t & 1) * 2 * tile_bytes) + tile_bytes, 8192, 1024);
            const uint64_t x_dy = make_desc(smem_u32(smem + (t & 1) * 2 * tile_bytes), tile_bytes, 1024);  // rows 64 on are dy's
#pragma unroll 1
            for (int i = 0; i < kBM / 16; ++i) {
                const uint32_t more = t > 0 || i > 0 ? 1u : 0u;
                if (p.part_in) {
                    mma<1, false>(tmem + kDw, dg + i * 128, x + i * 128, p.id_w, more, go);
                    mma<1, false>(tmem + kDw + 64, du + i * 128, x + i * 128, p.id_w, more, go);
                }
                if (p.part_out) mma<1, false>(tmem + kDw + 128, h + i * 128, dy + i * 128, p.id_w, more, go);
                if (p.part_bo && rank == 0)
                    mma<1, false>(tmem + kDb + 32, x_dy + i * 128, one, p.id_b, more, go);
                if (p.part_bi) {
                    mma<1, false>(tmem + kDb, dg + i * 128, one, p.id_b, more, go);
                    mma<1, false>(tmem + kDb + 16, du + i * 128, one, p.id_b, more, go);
                }
            }
            if (go) commit<1>(hempty), commit<1>(&xempty[t & 1]);
        }
        if (ok && go) commit<1>(done);
        if (!ok) {
            if (go) commit<1>(&drain[1]);
            mbar_wait(&drain[1], 0, 100000000ull);
        }
    } else if (warp >= kControlWarps + kEpiWarps) {  // dx: a warp has 32 of a tile's rows
        const int quad = warp & 3, row = quad * 32 + lane;
        const uint32_t acc = tmem + ((uint32_t)(quad * 32) << 16) + kDx;
        const bool owner = CTAS == 1 || quad >> 1 == rank;  // whether this CTA writes them
        uint8_t* const box = inbox + (quad & 1) * 8192 + lane * 16;
        for (int t = 0; p.dx && t < mine; ++t) {
            ok = mbar_wait(dxfull, t & 1);
            if (CTAS == 2) ok = ok && (owner ? peer_wait(infull, t & 1) : peer_wait(inempty, (t & 1) ^ 1));
            if (!ok) break;
            tc_fence_after();
            const int r = (slot + t * slots) * kBM + row;
#pragma unroll
            for (int c0 = 0; c0 < 64; c0 += 16) {
                float v[16];
                tmem_ld16(acc + c0, v);
                tmem_wait_ld();
                reg_fence(v);
                if (c0 == 48) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) arrive_leader<1>(dxempty);
                }
                if (CTAS == 2 && !owner) {
                    const uint32_t dst = peer_addr(box + c0 * 128, rank ^ 1);
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(dst + k * 512), "f"(v[4 * k]),
                                     "f"(v[4 * k + 1]), "f"(v[4 * k + 2]), "f"(v[4 * k + 3])
                                     : "memory");
                    continue;
                }
                if (CTAS == 2) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const float4 u = *reinterpret_cast<const float4*>(box + c0 * 128 + k * 512);
                        v[4 * k] += u.x, v[4 * k + 1] += u.y, v[4 * k + 2] += u.z, v[4 * k + 3] += u.w;
                    }
                }
                if (r < p.m) {
                    uint4 u[2];
                    pack16<T>(u, v);
                    T* o = (T*)p.dx + (int64_t)r * p.c + c0;
                    if (p.vec_dx) {
                        if (c0 < p.c) reinterpret_cast<uint4*>(o)[0] = u[0];
                        if (c0 + 8 < p.c) reinterpret_cast<uint4*>(o)[1] = u[1];
                    } else {
#pragma unroll
                        for (int k = 0; k < 16; ++k)
                            if (c0 + k < p.c) o[k] = Elem<T>::store(v[k]);
                    }
                }
                __syncwarp();
            }
            if (CTAS == 2) {
                __syncwarp();
                if (lane == 0) peer_arrive(peer_addr(owner ? inempty : infull, rank ^ 1));
            }
        }
    } else {
        const int ew = warp - kControlWarps, quad = warp & 3, c0 = (ew >> 2) * 16;  // 32 rows and 16 columns of everything
        const uint32_t acc = tmem + ((uint32_t)(quad * 32) << 16) + c0;
        const int row = quad * 32 + lane;
        auto arrive = [&](uint64_t* bar) {
            __syncwarp();
            if (lane == 0) arrive_leader<1>(bar);
        };
        for (int t = 0, g = 0; ok && t < mine; ++t) {
            for (int j = 0; j < p.blocks; ++j, ++g) {
                if (!(ok = mbar_wait(gfull, g & 1))) break;
                tc_fence_after();
                float gt[16], u[16], d[16];
                tmem_ld16(acc, gt);
                tmem_ld16(acc + kHB, u);
                tmem_ld16(acc + kDh, d);
                tmem_wait_ld();
                reg_fence(gt);
                reg_fence(u);
                reg_fence(d);
                tc_fence_before();
                arrive(gempty);
                if (p.b_in) add_columns(gt, bias + j * kHB + c0), add_columns(u, bias + kBwdHidden + j * kHB + c0);
                with_act(p.act, [&](auto act) {
#pragma unroll
                    for (int k = 0; k < 16; ++k) {
                        float a, slope;
                        act_both<decltype(act)::value>(gt[k], a, slope);
                        gt[k] = d[k] * u[k] * slope;
                        u[k] *= a;
                        d[k] *= a;
                    }
                });
                const int left = p.f - (n_first + j * kHB + c0);
                if (left < 16) {  // columns past the last: zeros even where x or dy is infinite
#pragma unroll
                    for (int k = 0; k < 16; ++k)
                        if (k >= left) gt[k] = u[k] = d[k] = 0.f;
                }
                uint4 o[3][2];
                pack16<T>(o[0], gt);
                pack16<T>(o[1], d);
                pack16<T>(o[2], u);
                if (!(ok = mbar_wait(hempty, (t & 1) ^ 1))) break;
                uint8_t* const at = dg_s + j * tile_bytes + row * kRowBytes;
#pragma unroll
                for (int k = 0; k < 3; ++k)
#pragma unroll
                    for (int c = 0; c < 2; ++c)
                        *reinterpret_cast<uint4*>(at + k * 2 * tile_bytes + (((c0 / 8 + c) ^ (row & 7)) << 4)) = o[k][c];
                fence_async_smem();
                arrive(&hfull[j]);
            }
        }
        if (ok && (ok = mbar_wait(done, 0))) {  // the slot's partial sums
            tc_fence_after();
            const int n = n_first + row;
            float v[16];
            if (p.part_in) {
                for (int plane = 0; plane < 2; ++plane) {
                    tmem_ld16(acc + kDw + plane * 64, v);
                    tmem_wait_ld();
                    reg_fence(v);
                    float* o = p.part_in + ((int64_t)slot * 2 * p.f + plane * p.f + n) * p.ld_in + c0;
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        if (n < p.f && c0 + 4 * k < p.ld_in)
                            reinterpret_cast<float4*>(o)[k] = make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
                }
            }
            if (p.part_out) {
                tmem_ld16(acc + kDw + 128, v);
                tmem_wait_ld();
                reg_fence(v);
#pragma unroll
                for (int k = 0; k < 16; ++k)
                    if (n < p.f && c0 + k < p.c) p.part_out[((int64_t)slot * p.c + c0 + k) * p.ld_out + n] = v[k];
            }
            if (p.part_bo && rank == 0 && c0 == 0) {
                tmem_ld16(acc + kDb + 32, v);
                tmem_wait_ld();
                reg_fence(v);
                if (row >= 64 && row - 64 < p.c) p.part_bo[(int64_t)slot * p.ld_bo + row - 64] = v[0];
                __syncwarp();
            }
            if (p.part_bi && c0 < 32) {  // 16 equal columns each for gate and up
                tmem_ld16(acc + kDb, v);
                tmem_wait_ld();
                reg_fence(v);
                if (n < p.f) p.part_bi[(int64_t)slot * p.ld_bi + (c0 ? p.f : 0) + n] = v[0];
            }
        }
    }
    if (!ok && lane == 0) atomicExch(&g_gemm_status, (int)LF_ERR_TIMEOUT);
    tc_fence_before();
    __syncthreads();
    sync_all<CTAS>();  // the other CTA may still write to this one's shared memory
    tc_fence_after();
    if (warp == 1) tmem_free<1>(tmem);
}

// Joins the splits of K and applies the epilogue, for up to four products
// (blockIdx.y).  `walkers` threads share four columns, each adds every
// walkers-th split, and their sums join in order: a thread for all splits of a
// small output would wait for one load after another.
struct JoinJob {
    const float* part;
    int64_t rows, ldp;
    int splits, n, walkers;
    Epilogue e;
};
struct JoinJobs {
    JoinJob job[4];
};
template <typename T>
__global__ void __launch_bounds__(256) split_join_kernel(const __grid_constant__ JoinJobs jobs) {
    __shared__ float4 sh[256];
    grid_release();
    grid_wait();
    const JoinJob& j = jobs.job[blockIdx.y];
    const Epilogue& e = j.e;
    const int each = 256 / j.walkers, w = threadIdx.x / each, o = threadIdx.x - w * each;
    const int64_t groups = j.ldp / 4, total = j.rows * groups;
    for (int64_t base = (int64_t)blockIdx.x * each; base < total; base += (int64_t)gridDim.x * each) {
        const int64_t i = base + o, row = i / groups;
        const int col = (int)(i - row * groups) * 4;
        float4 z = make_float4(0.f, 0.f, 0.f, 0.f);
        if (i < total)
#pragma unroll 4
            for (int s = w; s < j.splits; s += j.walkers) {
                const float4 v = *reinterpret_cast<const float4*>(j.part + ((int64_t)s * j.rows + row) * j.ldp + col);
                z.x += v.x, z.y += v.y, z.z += v.z, z.w += v.w;
            }
        if (j.walkers > 1) {
            __syncthreads();
            sh[threadIdx.x] = z;
            __syncthreads();
            for (int k = 1; w == 0 && k < j.walkers; ++k) {
                const float4 v = sh[k * each + o];
                z.x += v.x, z.y += v.y, z.z += v.z, z.w += v.w;
            }
        }
        if (w || i >= total) continue;
        if (e.sa) {
            const float s = e.sa[row];
            float* q = reinterpret_cast<float*>(&z);
#pragma unroll
            for (int k = 0; k < 4; ++k) q[k] *= s * (col + k < j.n ? e.sb[col + k] : 0.f);
        }
        float4 b = make_float4(0.f, 0.f, 0.f, 0.f), x = b;
        if (e.bias) b = widen4<T>(load4((const T*)e.bias, col, j.n, false));
        if (e.res) x = widen4<T>(load4((const T*)e.res + row * e.ldr, col, j.n, e.vec_res));
        with_act(e.act, [&](auto act) {
            store4((T*)e.out + row * e.ldo, col, j.n, e.vec_out, finish4<decltype(act)::value>(z, b, x, e.act_bwd));
        });
    }
}

// Copies a matrix whose rows TMA cannot address (row pitch or base not a
// multiple of 16 bytes) to rows of ldo elements: 16 bytes of output per lane
// (whose scalar loads share cache lines).
template <typename U>
__global__ void __launch_bounds__(256) pack_rows_kernel(const U* in, int64_t ldi, U* out, int64_t ldo, int64_t rows, int64_t cols) {
    constexpr int V = 16 / sizeof(U);
    grid_release();
    grid_wait();
    const int lane = threadIdx.x & 31;
    const int64_t per_row = (ldo + 32 * V - 1) / (32 * V), total = rows * per_row;  // warps' work: a row's next 512 bytes
    for (int64_t i = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); i < total; i += (int64_t)gridDim.x * 8) {
        const int64_t r = i / per_row, c = ((i - r * per_row) * 32 + lane) * V;
        if (c >= ldo) continue;
        U v[V];
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = c + j < cols ? in[r * ldi + c + j] : U(0);
        *reinterpret_cast<uint4*>(out + r * ldo + c) = *reinterpret_cast<const uint4*>(v);
    }
}

// Column sums of up to three matrices in one launch (blockIdx.z).  First step:
// part[slice][c] over the rows of a slice.  A thread adds V neighbouring
// columns; tx threads cover a row and 256/tx rows go side by side, whose sums
// join in order.
struct ColsumJob {
    const void* in;
    void* out;
    float* part;
    int64_t ld, cols;
};
struct ColsumJobs {
    ColsumJob job[3];
    int64_t rows, slice;
    int slices, tx;
};
template <typename T, int V>
__global__ void __launch_bounds__(256) colsum_kernel(const ColsumJobs p) {
    __shared__ float sh[256 * V];
    grid_release();
    grid_wait();
    const ColsumJob j = p.job[blockIdx.z];
    const int walkers = 256 / p.tx, w = threadIdx.x / p.tx, width = p.tx * V, at = (threadIdx.x - w * p.tx) * V;
    const int64_t c0 = (int64_t)blockIdx.x * width;
    if (c0 >= j.cols) return;
    const int64_t r0 = (int64_t)blockIdx.y * p.slice + w, r1 = min(p.rows, (int64_t)(blockIdx.y + 1) * p.slice);
    float a[V];
#pragma unroll
    for (int k = 0; k < V; ++k) a[k] = 0.f;
    if (c0 + at < j.cols) {
        const T* q = (const T*)j.in + c0 + at;
#pragma unroll 4
        for (int64_t r = r0; r < r1; r += walkers) {
            if constexpr (V == 1) a[0] += Elem<T>::load(q[r * j.ld]);
            else {
                const uint4 u = *reinterpret_cast<const uint4*>(q + r * j.ld);
                const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
                for (int k = 0; k < V; ++k) a[k] += Elem<T>::load(e[k]);
            }
        }
    }
#pragma unroll
    for (int k = 0; k < V; ++k) sh[w * width + at + k] = a[k];
    __syncthreads();
    for (int i = threadIdx.x; i < width; i += 256)
        if (c0 + i < j.cols) {
            float t = 0.f;
            for (int k = 0; k < walkers; ++k) t += sh[k * width + i];
            j.part[(int64_t)blockIdx.y * j.cols + c0 + i] = t;
        }
}
template <typename T>
__global__ void __launch_bounds__(1024) colsum_join_kernel(const ColsumJobs p) {
    __shared__ float sh[32][33];
    grid_release();
    grid_wait();
    const ColsumJob j = p.job[blockIdx.z];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int64_t c = (int64_t)blockIdx.x * 32 + lane;
    float t = 0.f;
    if (c < j.cols)
#pragma unroll 4
        for (int s = w; s < p.slices; s += 32) t += j.part[(int64_t)s * j.cols + c];
    sh[w][lane] = t;
    __syncthreads();
    if (w == 0 && c < j.cols) {
#pragma unroll
        for (int i = 1; i < 32; ++i) t += sh[i][lane];
        ((T*)j.out)[c] = Elem<T>::store(t);
    }
}

// Products of a few rows (MT at most): bound by reading the weights once.
// One to eight warps share a weight row, each lane has four 16-byte loads in
// flight, the sums meet by shuffles and shared memory in a fixed order.
// (Reading the second product's weights of a feed-forward block while the first
// still runs made the pair slower, 11.5 us against 9.8: both are bound by the
// same reads.)
template <typename T, bool GATED, int MT, bool VEC>
__global__ void __launch_bounds__(256) few_rows_kernel(const T* x, int64_t ldx, const T* w, int64_t ldw, int m, int n, int k,
                                                       int wpr, const Epilogue e) {
    __shared__ float sh[8][GATED ? 2 : 1][MT];
    grid_release();
    grid_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int part = warp % wpr, col = blockIdx.x * (8 / wpr) + warp / wpr;
    float a[GATED ? 2 : 1][MT];
#pragma unroll
    for (int q = 0; q < (GATED ? 2 : 1); ++q)
#pragma unroll
        for (int i = 0; i < MT; ++i) a[q][i] = 0.f;
    if (col < n) {
        const T* wr[2] = {w + (int64_t)col * ldw, GATED ? w + (int64_t)(n + col) * ldw : nullptr};
        if constexpr (VEC) {
            const int nv = k / 8, step = wpr * 32;
            for (int v0 = part * 32 + lane; v0 < nv; v0 += 4 * step) {
                uint4 u[GATED ? 2 : 1][4];
#pragma unroll
                for (int q = 0; q < (GATED ? 2 : 1); ++q)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (v0 + j * step < nv) u[q][j] = *(reinterpret_cast<const uint4*>(wr[q]) + v0 + j * step);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int v = v0 + j * step;
                    if (v >= nv) break;
#pragma unroll
                    for (int i = 0; i < MT; ++i) {
                        if (i >= m) break;
                        const uint4 xv = *(reinterpret_cast<const uint4*>(x + i * ldx) + v);
                        const uint32_t* xe = reinterpret_cast<const uint32_t*>(&xv);
#pragma unroll
                        for (int q = 0; q < (GATED ? 2 : 1); ++q) {
                            const uint32_t* we = reinterpret_cast<const uint32_t*>(&u[q][j]);
#pragma unroll
                            for (int h = 0; h < 4; ++h) {
                                const float2 xf = unpack2<T>(xe[h]), wf = unpack2<T>(we[h]);
                                a[q][i] = __fmaf_rn(xf.x, wf.x, a[q][i]);
                                a[q][i] = __fmaf_rn(xf.y, wf.y, a[q][i]);
                            }
                        }
                    }
                }
            }
        } else {
            for (int v = part * 32 + lane; v < k; v += wpr * 32) {
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    if (i >= m) break;
                    const float xf = Elem<T>::load(x[i * ldx + v]);
#pragma unroll
                    for (int q = 0; q < (GATED ? 2 : 1); ++q) a[q][i] = __fmaf_rn(xf, Elem<T>::load(wr[q][v]), a[q][i]);
                }
            }
        }
    }
#pragma unroll
    for (int q = 0; q < (GATED ? 2 : 1); ++q)
#pragma unroll
        for (int i = 0; i < MT; ++i) {
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) a[q][i] += __shfl_xor_sync(0xffffffffu, a[q][i], o);
            if (lane == 0) sh[warp][q][i] = a[q][i];
        }
    __syncthreads();
    if (part == 0 && col < n && lane < m) {
        float z[2] = {0.f, 0.f};
#pragma unroll
        for (int q = 0; q < (GATED ? 2 : 1); ++q) {
            for (int i = 0; i < wpr; ++i) z[q] += sh[warp + i][q][lane];
            if (e.bias) z[q] += Elem<T>::load(((const T*)e.bias)[q * n + col]);
        }
        float y = 0.f;
        with_act(e.act, [&](auto act) { y = act_value<decltype(act)::value>(z[0]); });
        if (GATED) y *= z[1];
        if (e.res) y += Elem<T>::load(((const T*)e.res)[lane * e.ldr + col]);
        ((T*)e.out)[lane * e.ldo + col] = Elem<T>::store(y);
    }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
// A matrix in device memory as TMA sees it: `rows` rows of `inner` contiguous
// elements, ld elements apart, in `planes` planes `plane` elements apart.
struct Mat {
    const void* p = nullptr;
    int64_t inner = 0, rows = 0, ld = 0, planes = 1, plane = 0;
};

bool encode(CUtensorMap* map, const Mat& a, int dtype, int box_inner, int box_rows,
            CUtensorMapSwizzle swizzle = CU_TENSOR_MAP_SWIZZLE_128B, int box_planes = 1) {
    const int es = dtype == LF_F8E4M3 ? 1 : 2;
    const CUtensorMapDataType ty = dtype == LF_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                   : dtype == LF_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_UINT8;
    const cuuint64_t dims[3] = {(cuuint64_t)a.inner, (cuuint64_t)a.rows, (cuuint64_t)a.planes};
    const cuuint64_t strides[2] = {(cuuint64_t)(a.ld * es), (cuuint64_t)((a.planes > 1 ? a.plane : a.rows * a.ld) * es)};
    const cuuint32_t box[3] = {(cuuint32_t)box_inner, (cuuint32_t)box_rows, (cuuint32_t)box_planes};
    return encode_tiled(map, ty, 3, a.p, dims, strides, box, swizzle);
}

bool encode_out(CUtensorMap* map, const Mat& a, int dtype) { return encode(map, a, dtype, 32, 32, CU_TENSOR_MAP_SWIZZLE_64B); }

// Whether TMA can address rows of ld elements of es bytes at p.
bool tma_ok(const void* p, int64_t ld, int es) { return aligned(p, 16) && ld * es % 16 == 0; }

int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

// Bump allocator over the caller's workspace; with base 0 it only counts.
struct Arena {
    uintptr_t base;
    size_t used = 0;
    void* take(size_t bytes) {
        const size_t at = used;
        used += up((int64_t)bytes, 256);
        return base ? reinterpret_cast<void*>(base + at) : nullptr;
    }
};

// One product out[m, n] = A B^T (+ epilogue), A and B in either major.
struct Product {
    Mat a, b;
    bool a_mn = false, b_mn = false;
    int64_t m = 0, n = 0, k = 0;   // rows of one row segment, columns, K of one K segment
    int msegs = 1, ksegs = 1;
    Epilogue e{};
    int dtype = 0, op_dtype = 0;   // output type; operand type
};

// Tile of a launch: CTAs per tile, columns, splits of K.
struct Shape {
    int ctas, bn, splits;
};

// SM cycles of one K step of a tile: the tensor pipe's (two per column), or
// fetching the CTA's operands through L2 at about 60 bytes per cycle.
double step_cycles(int ctas, int cols, int b_rows) { return std::max(2.0 * cols, (kBM + b_rows / ctas) * kRowBytes / 60.0); }

// Tile shape and splits of K by an estimate in SM cycles: the epilogue of a
// tile overlaps the next tile's products, a pair takes 1000 cycles longer to
// start and end, and a split costs writing and reading the partial sums once
// more and another launch.  Over 56 shapes (16 to 12000 rows, 64 to 4096
// columns and K) the choice measured 1.03 times the best one's time, 1.2 at
// worst.
Shape choose(const Product& q, double* cycles = nullptr) {
    const int bk = q.op_dtype == LF_F8E4M3 ? 128 : 64;
    const int64_t iters = (q.k + bk - 1) / bk * q.ksegs, sms = num_sms();
    Shape best{1, 256, 1};
    double least = 1e30;
    for (int ctas : {2, 1})
        for (int bn : {256, 128, 64}) {
            if (ctas == 2 && bn == 64) continue;
            const int64_t tiles = (q.m + kBM * ctas - 1) / (kBM * ctas) * q.msegs * ((q.n + bn - 1) / bn);
            for (int s = 1; s <= 64; s *= 2) {
                if (s > 1 && iters / s < 4) break;
                const int64_t per = (iters + s - 1) / s, units = tiles * ((iters + per - 1) / per);
                const int64_t waves = (units * ctas + sms - 1) / sms;
                const double main = per * step_cycles(ctas, bn, bn), epi = 500 + bn * 10.0;
                double t = waves * std::max(main, epi) + std::min(main, epi) + (ctas == 2 ? 1000 : 0);
                if (s > 1) t += 6500 + (double)s * q.m * q.msegs * q.n * 8 / 3400.0;
                if (t < least) least = t, best = {ctas, bn, s};
            }
        }
    if (cycles) *cycles = least;
    return best;
}

// The same for several products that share a launch (one CTA count): for each
// the widest tile that costs least work, and splits where a unit would be
// longer than a share of the whole launch (several shares are tried).
double choose_together(const Product* q, int count, int ctas, Shape* out) {
    const double lanes = (double)num_sms() / ctas;
    double total = 0, least = 1e30;
    int bn_of[3];
    auto unit = [&](int i, int bn, int s) {
        const int64_t iters = (q[i].k + 63) / 64 * q[i].ksegs;
        return std::max(((iters + s - 1) / s) * step_cycles(ctas, bn, bn), 500 + bn * 10.0);
    };
    auto tiles = [&](int i, int bn) {
        return (double)((q[i].m + kBM * ctas - 1) / (kBM * ctas) * q[i].msegs * ((q[i].n + bn - 1) / bn));
    };
    for (int i = 0; i < count; ++i) {
        double best = 1e30;
        for (int bn : {256, 128, 64}) {
            if (ctas == 2 && bn == 64) continue;
            const double w = tiles(i, bn) * unit(i, bn, 1);
            if (w < 0.99 * best) best = w, bn_of[i] = bn;
        }
        total += best;
    }
    for (double share : {0.12, 0.25, 0.5, 1.0, 2.0}) {
        const double limit = std::max(share * total / lanes, 2000.0);
        double work = 0, longest = 0, shortest = 1e30, filler = 0, join = 0;
        Shape s[3];
        for (int i = 0; i < count; ++i) {
            const int64_t iters = (q[i].k + 63) / 64 * q[i].ksegs;
            int n = 1;
            while (unit(i, bn_of[i], n) > limit && n < 64 && iters / (2 * n) >= 4) n *= 2;
            const double u = unit(i, bn_of[i], n);
            work += tiles(i, bn_of[i]) * n * u;
            longest = std::max(longest, u);
            if (u < shortest) shortest = u, filler = tiles(i, bn_of[i]) * n * u / lanes;
            if (n > 1) join += (double)n * q[i].m * q[i].msegs * q[i].n * 8 / 3400.0;
            s[i] = {ctas, bn_of[i], n};
        }
        // Short units even out what the long ones leave, where there are enough of them.
        const double uneven = 0.5 * (filler >= longest ? shortest : longest);
        const double t = std::max(longest, work / lanes + uneven) + (join > 0 ? 6500 + join : 0) + (ctas == 2 ? 1000 : 0);
        if (t < least) {
            least = t;
            for (int i = 0; i < count; ++i) out[i] = s[i];
        }
    }
    return least;
}

size_t part_bytes(const Product& q, const Shape& s) {
    return s.splits > 1 ? (size_t)s.splits * q.m * q.msegs * up(q.n, 4) * 4 : 0;
}

uint32_t idesc_of(int dtype, bool a_mn, bool b_mn, int ctas, int n) {
    const uint32_t f = dtype == LF_BF16 ? 1u : 0u;  // kind::f16: 0 fp16, 1 bf16; kind::f8f6f4: 0 e4m3
    return (1u << 4) | (f << 7) | (f << 10) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) |
           ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kBM * ctas >> 4) << 24);
}

int64_t units_of(const Problem& p) { return (int64_t)p.splits * p.msegs * p.tiles_m * p.tiles_n; }

void set_divisors(Problem& g, int ctas) {
    const int row_tiles = g.msegs * g.tiles_m, group = std::min(row_tiles, kGroupRows / (kBM * ctas));
    g.per_split = Divisor(row_tiles * g.tiles_n);
    g.per_group = Divisor(group * g.tiles_n);
    g.per_seg = Divisor(g.tiles_m);
    g.group_rows = Divisor(group);
    g.last_rows = Divisor(row_tiles % group ? row_tiles % group : group);
}

template <auto Kernel, bool FP8, int N>
int launch_gemm(GemmArgs<N>& g, int ctas, cudaStream_t st) {
    constexpr int rest = kEpiWarps * (kStageOut + column_bytes<FP8>()) + kBarrierBytes;
    g.stages = std::min(kMaxStages, (kSmemLimit - rest) / g.stage_bytes);
    static std::once_flag once[64];  // per kernel and device
    int dev = 0;
    cudaGetDevice(&dev);
    std::call_once(once[dev & 63], [] { cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemLimit); });
    const unsigned grid = (unsigned)(std::min(g.first[N], num_sms() / ctas) * ctas);
    launch_early(Kernel, grid, kGemmThreads, (size_t)g.stages * g.stage_bytes + rest, (unsigned)ctas, st, g);
    return check_launch("tc_gemm_kernel");
}

template <typename T, int MODE, bool FP8, int N>
int launch_ctas(GemmArgs<N>& g, int ctas, cudaStream_t st) {
    return ctas == 2 ? launch_gemm<tc_gemm_kernel<T, MODE, FP8, 2, N>, FP8>(g, 2, st)
                     : launch_gemm<tc_gemm_kernel<T, MODE, FP8, 1, N>, FP8>(g, 1, st);
}

int too_large(const char* what) {
    set_error("%s: more than 2^31 tiles or rows", what);
    return LF_ERR_UNSUPPORTED;
}

int join_splits(const JoinJobs& jobs, int count, int dtype, cudaStream_t st) {
    int64_t most = 1;
    for (int i = 0; i < count; ++i) most = std::max(most, (jobs.job[i].rows * (jobs.job[i].ldp / 4) * jobs.job[i].walkers + 255) / 256);
    const dim3 grid((unsigned)std::min<int64_t>(most, (int64_t)num_sms() * 16), (unsigned)count);
    launch_early(dtype == LF_F16 ? split_join_kernel<__half> : split_join_kernel<__nv_bfloat16>, grid, 256, 0, 1, st, jobs);
    return check_launch("split_join_kernel");
}
JoinJob join_of(const Product& q, const float* part, int splits) {
    return {part, q.m * q.msegs, up(q.n, 4), splits, (int)q.n, splits >= 32 ? 8 : splits >= 8 ? 4 : 1, q.e};
}

int fill_problem(Problem& g, const Product& q, const Shape& s, float* part) {
    const int bk = q.op_dtype == LF_F8E4M3 ? 128 : 64;
    g.m = (int)q.m, g.n = (int)q.n;
    g.msegs = q.msegs;
    g.tiles_m = (int)((q.m + kBM * s.ctas - 1) / (kBM * s.ctas));
    g.tiles_n = (int)((q.n + s.bn - 1) / s.bn);
    g.seg_iters = (int)((q.k + bk - 1) / bk);
    g.iters = g.seg_iters * q.ksegs;
    g.split_iters = (g.iters + s.splits - 1) / s.splits;
    g.splits = (g.iters + g.split_iters - 1) / g.split_iters;
    if (q.m > INT32_MAX - 256 || q.n > INT32_MAX - 256 || units_of(g) > INT32_MAX / 4) return too_large("matrix product");
    g.bn = s.bn;
    g.a_mn = q.a_mn, g.b_mn = q.b_mn;
    g.idesc = idesc_of(q.op_dtype, q.a_mn, q.b_mn, s.ctas, s.bn);
    g.e = q.e;
    g.e.tma = !part && tma_ok(q.e.out, q.e.ldo, 2);
    g.e.pairs = q.n % 2 == 0 && q.e.ldo % 2 == 0 && aligned(q.e.out, 4);
    g.e.vec_res = q.n % 8 == 0 && tma_ok(q.e.res, q.e.ldr, 2);  // here: whole 16-byte chunks
    if (g.e.tma && !encode_out(&g.out, {q.e.out, q.n, q.m, q.e.ldo, q.msegs, q.m * q.e.ldo}, q.dtype)) return LF_ERR_CUDA;
    g.part = part;
    g.ldp = up(q.n, 4);
    if (!encode(&g.a, q.a, q.op_dtype, q.a_mn ? 64 : bk, q.a_mn ? bk : kBM)) return LF_ERR_CUDA;
    if (!encode(&g.b, q.b, q.op_dtype, q.b_mn ? 64 : bk, q.b_mn ? bk : s.bn / s.ctas)) return LF_ERR_CUDA;
    set_divisors(g, s.ctas);
    return LF_OK;
}

int stage_bytes_of(const Shape& s) { return (kBM + s.bn / s.ctas) * kRowBytes; }

int run_product(const Product& q, Arena& ws, cudaStream_t st) {
    if (q.m == 0 || q.n == 0) return LF_OK;
    JoinJobs join{};
    if (q.k == 0) {  // an empty sum: the epilogue of zero
        join.job[0] = join_of(q, nullptr, 0);
        return ws.base ? join_splits(join, 1, q.dtype, st) : LF_OK;
    }
    const Shape s = choose(q);
    float* part = s.splits > 1 ? (float*)ws.take(part_bytes(q, s)) : nullptr;
    if (!ws.base) return LF_OK;
    GemmArgs<1> g{};
    if (int rc = fill_problem(g.p[0], q, s, part)) return rc;
    g.first[1] = (int)units_of(g.p[0]);
    g.stage_bytes = stage_bytes_of(s);
    const bool half = q.dtype == LF_F16;
    int rc;
    if (q.op_dtype == LF_F8E4M3)
        rc = half ? launch_ctas<__half, kLinear, true>(g, s.ctas, st) : launch_ctas<__nv_bfloat16, kLinear, true>(g, s.ctas, st);
    else
        rc = half ? launch_ctas<__half, kLinear, false>(g, s.ctas, st) : launch_ctas<__nv_bfloat16, kLinear, false>(g, s.ctas, st);
    if (rc || !part) return rc;
    join.job[0] = join_of(q, part, g.p[0].splits);
    return join_splits(join, 1, q.dtype, st);
}

// Up to three products of 16-bit operands that do not depend on one another,
// in one launch: a gradient's products are often too small to fill the SMs
// one by one, and large ones fill each other's last wave.  Where the estimates
// say so they run apart: over 44 drawn backward passes (16 to 40000 rows) the
// rule measured 1.002 times the better way's time, 1.10 at worst (always shared
// 1.008, always apart 1.15).
int run_products(const Product* in, int given, Arena& ws, cudaStream_t st) {
    Product q[3];
    int count = 0;
    for (int i = 0; i < given; ++i) {
        if (in[i].m == 0 || in[i].n == 0 || in[i].k == 0) {
            if (int rc = run_product(in[i], ws, st)) return rc;
        } else q[count++] = in[i];
    }
    if (count == 0) return LF_OK;
    if (count == 1) return run_product(q[0], ws, st);
    Shape one[3], two[3];
    const double pairs = choose_together(q, count, 2, two), singles = choose_together(q, count, 1, one);
    const Shape* s = pairs <= singles ? two : one;
    double apart = 0;
    for (int i = 0; i < count; ++i) {
        double t;
        choose(q[i], &t);
        apart += t + 2500;  // a launch after the first
    }
    if (apart - 2500 < std::min(pairs, singles)) {
        for (int i = 0; i < count; ++i)
            if (int rc = run_product(q[i], ws, st)) return rc;
        return LF_OK;
    }
    float* part[3] = {};
    for (int i = 0; i < count; ++i)
        if (s[i].splits > 1) part[i] = (float*)ws.take(part_bytes(q[i], s[i]));
    if (!ws.base) return LF_OK;
    // Long units first.
    int order[3] = {0, 1, 2};
    double unit[3];
    for (int i = 0; i < count; ++i) {
        const int64_t iters = (q[i].k + 63) / 64 * q[i].ksegs;
        unit[i] = std::max((double)((iters + s[i].splits - 1) / s[i].splits) * step_cycles(s[i].ctas, s[i].bn, s[i].bn), 500 + s[i].bn * 10.0);
    }
    std::sort(order, order + count, [&](int a, int b) { return unit[a] > unit[b]; });
    GemmArgs<3> g{};
    JoinJobs join{};
    int joins = 0;
    int64_t at = 0;
    for (int i = 0; i < 3; ++i) {
        g.first[i] = (int)at;
        if (i >= count) continue;
        const int k = order[i];
        if (int rc = fill_problem(g.p[i], q[k], s[k], part[k])) return rc;
        if (i == count - 1) g.longer = (int)at;
        at += units_of(g.p[i]);
        if (at > INT32_MAX / 2) return too_large("matrix products");
        g.stage_bytes = std::max(g.stage_bytes, stage_bytes_of(s[k]));
        if (part[k]) join.job[joins++] = join_of(q[k], part[k], g.p[i].splits);
    }
    g.first[3] = (int)at;
    // The long units' last turn is the problem's before the last.
    g.extra = extra_units(g.longer, (int)at - g.longer, std::min((int)at, num_sms() / s[0].ctas),
                          unit[order[count - 2]] / unit[order[count - 1]]);
    const int rc = q[0].dtype == LF_F16 ? launch_ctas<__half, kLinear, false>(g, s[0].ctas, st)
                                        : launch_ctas<__nv_bfloat16, kLinear, false>(g, s[0].ctas, st);
    return rc || !joins ? rc : join_splits(join, joins, q[0].dtype, st);
}

// A dense operand as TMA can read it: itself, or a copy with padded rows.
Mat operand(const void* p, int64_t rows, int64_t cols, int64_t ld, int es, Arena& ws, cudaStream_t st) {
    if (rows == 0 || cols == 0 || tma_ok(p, ld, es)) return {p, cols, rows, ld, 1, 0};
    const int64_t ldo = up(cols, 16 / es);
    void* out = ws.take((size_t)rows * ldo * es);
    if (out) {
        const unsigned grid = (unsigned)std::min<int64_t>((rows * ((ldo * es + 511) / 512) + 7) / 8, (int64_t)num_sms() * 8);
        if (es == 1) launch_early(pack_rows_kernel<uint8_t>, grid, 256, 0, 1, st, (const uint8_t*)p, ld, (uint8_t*)out, ldo, rows, cols);
        else launch_early(pack_rows_kernel<uint16_t>, grid, 256, 0, 1, st, (const uint16_t*)p, ld, (uint16_t*)out, ldo, rows, cols);
    }
    return {out, cols, rows, ldo, 1, 0};
}

void set_out(Epilogue& e, void* out, int64_t ldo) {
    e.out = out;
    e.ldo = ldo;
    e.vec_out = aligned(out, 8) && ldo % 4 == 0;
}
void set_res(Epilogue& e, const void* res, int64_t ldr) {
    e.res = res;
    e.ldr = ldr;
    e.vec_res = aligned(res, 8) && ldr % 4 == 0;
}

int zero(void* p, int64_t rows, int64_t row_bytes, cudaStream_t st) {
    if (p && rows * row_bytes && cudaMemsetAsync(p, 0, (size_t)(rows * row_bytes), st) != cudaSuccess) return check_launch("zero fill");
    return LF_OK;
}

// out[c] = sum of column c of in [rows, cols] (16-bit), for `count` matrices of
// as many rows.  `padded`: whole vectors may be read past cols (our own buffers).
struct Columns {
    const void* in;
    int64_t ld, cols;
    void* out;
    bool padded;
};
int run_colsum(const Columns* c, int count, int64_t rows, int dtype, Arena& ws, cudaStream_t st) {
    ColsumJobs p{};
    int64_t widest = 0;
    bool vec = true;
    int jobs = 0;
    for (int i = 0; i < count; ++i) {
        if (c[i].cols == 0 || !c[i].out) continue;
        if (rows == 0) {
            if (ws.base)
                if (int rc = zero(c[i].out, 1, c[i].cols * 2, st)) return rc;
            continue;
        }
        vec = vec && aligned(c[i].in, 16) && c[i].ld % 8 == 0 && (c[i].padded || c[i].cols % 8 == 0);
        p.job[jobs++] = {c[i].in, c[i].out, nullptr, c[i].ld, c[i].cols};
        widest = std::max(widest, c[i].cols);
    }
    if (!jobs) return LF_OK;
    const int v = vec ? 8 : 1;
    p.tx = 1;
    while (p.tx < 32 && p.tx * v < widest) p.tx *= 2;
    const int64_t wide = (widest + p.tx * v - 1) / (p.tx * v);
    // About four blocks per SM, each at least eight rows per row walker.
    const int64_t most = std::max<int64_t>(1, 4 * num_sms() / (wide * jobs)), least = 8 * 256 / p.tx;
    p.rows = rows;
    p.slice = std::max(least, (rows + most - 1) / most);
    p.slices = (int)((rows + p.slice - 1) / p.slice);
    for (int i = 0; i < jobs; ++i) p.job[i].part = (float*)ws.take((size_t)p.slices * p.job[i].cols * 4);
    if (!ws.base) return LF_OK;
    const dim3 grid((unsigned)wide, (unsigned)p.slices, (unsigned)jobs), join((unsigned)((widest + 31) / 32), 1, (unsigned)jobs);
    if (dtype == LF_F16) {
        launch_early(vec ? colsum_kernel<__half, 8> : colsum_kernel<__half, 1>, grid, 256, 0, 1, st, p);
        launch_early(colsum_join_kernel<__half>, join, 1024, 0, 1, st, p);
    } else {
        launch_early(vec ? colsum_kernel<__nv_bfloat16, 8> : colsum_kernel<__nv_bfloat16, 1>, grid, 256, 0, 1, st, p);
        launch_early(colsum_join_kernel<__nv_bfloat16>, join, 1024, 0, 1, st, p);
    }
    return check_launch("colsum_kernel");
}

// Rows that few_rows_kernel takes: its time grows with them (4096 x 1024 bf16
// weights: 4.1 us for one, 6.8 for four, 10.5 for eight; 512 x 512: 2.1, 2.8
// and 3.9), the tensor cores' does not (8.0 and 4.8 us).
bool few_rows(int64_t m, int64_t n, int64_t k) { return k > 0 && (m <= 4 || (m <= 8 && n * k <= (1 << 19))); }

template <typename T, bool GATED>
void launch_few(const void* x, int64_t ldx, const void* w, int64_t ldw, int m, int n, int k, const Epilogue& e, cudaStream_t st) {
    const bool vec = k % 8 == 0 && ldx % 8 == 0 && ldw % 8 == 0 && aligned(x, 16) && aligned(w, 16);
    int wpr = 1;  // warps per weight row: more where there are too few rows to fill the SMs
    while (wpr < 8 && (int64_t)n * wpr < 32 * (int64_t)num_sms() && k / (256 * wpr) > 1) wpr *= 2;
    const unsigned grid = (unsigned)((n + 8 / wpr - 1) / (8 / wpr));
    const T *xp = (const T*)x, *wp = (const T*)w;
#define LFB_FEW(MT)                                                                                          \
    launch_early(vec ? few_rows_kernel<T, GATED, MT, true> : few_rows_kernel<T, GATED, MT, false>, grid, 256, 0, 1, st, xp, ldx, \
                 wp, ldw, m, n, k, wpr, e)
    if (m == 1) { LFB_FEW(1); }
    else if (m == 2) { LFB_FEW(2); }
    else if (m <= 4) { LFB_FEW(4); }
    else { LFB_FEW(8); }
#undef LFB_FEW
}
template <bool GATED>
int run_few(const void* x, int64_t ldx, const void* w, int64_t ldw, int64_t m, int64_t n, int64_t k, const Epilogue& e,
            int dtype, cudaStream_t st) {
    if (dtype == LF_F16) launch_few<__half, GATED>(x, ldx, w, ldw, (int)m, (int)n, (int)k, e, st);
    else launch_few<__nv_bfloat16, GATED>(x, ldx, w, ldw, (int)m, (int)n, (int)k, e, st);
    return check_launch("few_rows_kernel");
}

int check_common(const char* what, int act, int dtype, std::initializer_list<int64_t> sizes) {
    if (dtype != LF_F16 && dtype != LF_BF16) {
        set_error("%s: unsupported dtype code %d (fp16 and bf16)", what, dtype);
        return LF_ERR_DTYPE;
    }
    if (act < LF_ACT_NONE || act > LF_ACT_SILU) {
        set_error("%s: unknown activation %d", what, act);
        return LF_ERR_INVALID;
    }
    for (int64_t v : sizes)
        if (v < 0) {
            set_error("%s: negative size", what);
            return LF_ERR_INVALID;
        }
    for (int64_t v : sizes)
        if (v > INT32_MAX - 256) {
            set_error("%s: a size passes 2^31", what);
            return LF_ERR_UNSUPPORTED;
        }
    return LF_OK;
}

// Every pointer on its element's boundary (a misaligned access would fault).
int check_aligned(const char* what, std::initializer_list<const void*> ptrs, size_t bytes) {
    for (const void* p : ptrs)
        if (!aligned(p, bytes)) {
            set_error("%s: a pointer is not aligned to its %zu-byte elements", what, bytes);
            return LF_ERR_INVALID;
        }
    return LF_OK;
}

int missing(const char* what, const char* names) {
    set_error("%s: %s required", what, names);
    return LF_ERR_INVALID;
}

Product weight_product(const Mat& x, const Mat& w, int64_t m, int64_t n, int64_t k, int dtype, int op_dtype) {
    Product q;
    q.a = x, q.b = w;
    q.m = m, q.n = n, q.k = k;
    q.dtype = dtype, q.op_dtype = op_dtype;
    return q;
}

// ---- linear ----------------------------------------------------------------
int check_linear(const char* what, const lf_linear_t* a, bool quant) {
    if (!a) return missing(what, "arguments are");
    if (int rc = check_common(what, a->activation, a->dtype, {a->m, a->n, a->k})) return rc;
    if (int rc = check_aligned(what, {a->bias, a->residual, a->y, a->dy, a->dx, a->dw, a->db, quant ? nullptr : a->x, quant ? nullptr : a->w}, 2))
        return rc;
    if (quant)
        if (int rc = check_aligned(what, {a->x_scale, a->w_scale}, 4)) return rc;
    if (a->m == 0 || a->n == 0) return LF_OK;
    if (a->k > 0 && (!a->w || !a->x)) return missing(what, "x and w are");
    if (a->ldx < a->k || a->ldw < a->k || (a->residual && a->ldr < a->n)) {
        set_error("%s: a row stride is shorter than its row", what);
        return LF_ERR_INVALID;
    }
    if (quant && (!a->x_scale || !a->w_scale)) return missing(what, "x_scale and w_scale are");
    return LF_OK;
}

int linear_fwd(const lf_linear_t* a, bool quant, Arena& ws, cudaStream_t st) {
    if (a->m == 0 || a->n == 0) return LF_OK;
    Epilogue e{};
    set_out(e, a->y, a->n);
    e.bias = a->bias;
    if (a->residual) set_res(e, a->residual, a->ldr);
    e.act = a->activation;
    if (quant) e.sa = (const float*)a->x_scale, e.sb = (const float*)a->w_scale;
    if (!quant && few_rows(a->m, a->n, a->k)) return ws.base ? run_few<false>(a->x, a->ldx, a->w, a->ldw, a->m, a->n, a->k, e, a->dtype, st) : LF_OK;
    const int es = quant ? 1 : 2;
    Mat x = operand(a->x, a->m, a->k, a->ldx, es, ws, st), w = operand(a->w, a->n, a->k, a->ldw, es, ws, st);
    Product q = weight_product(x, w, a->m, a->n, a->k, a->dtype, quant ? LF_F8E4M3 : a->dtype);
    q.e = e;
    return run_product(q, ws, st);
}

int linear_bwd(const lf_linear_t* a, Arena& ws, cudaStream_t st) {
    const int64_t m = a->m, n = a->n, k = a->k;
    const bool need_z = a->activation != LF_ACT_NONE;
    Mat x, w, dz;
    if (need_z || a->dw) x = operand(a->x, m, k, a->ldx, 2, ws, st);
    if (need_z || a->dx) w = operand(a->w, n, k, a->ldw, 2, ws, st);
    if (need_z) {
        const int64_t ld = up(n, 8);
        dz = {ws.take((size_t)m * ld * 2), n, m, ld, 1, 0};
        Product q = weight_product(x, w, m, n, k, a->dtype, a->dtype);
        set_out(q.e, const_cast<void*>(dz.p), ld);
        set_res(q.e, a->dy, a->lddy);
        q.e.bias = a->bias;
        q.e.act = a->activation;
        q.e.act_bwd = true;
        if (int rc = run_product(q, ws, st)) return rc;
    } else {
        dz = operand(a->dy, m, n, a->lddy, 2, ws, st);
    }
    Product q[2];
    int count = 0;
    if (a->dx) {  // dx = dz W: W is read with its k contiguous
        Product& p = q[count++] = weight_product(dz, w, m, k, n, a->dtype, a->dtype);
        p.b_mn = true;
        set_out(p.e, a->dx, k);
    }
    if (a->dw) {  // dW = dz^T x: both operands transposed
        Product& p = q[count++] = weight_product(dz, x, n, k, m, a->dtype, a->dtype);
        p.a_mn = p.b_mn = true;
        set_out(p.e, a->dw, k);
    }
    if (int rc = run_products(q, count, ws, st)) return rc;
    const Columns c{dz.p, dz.ld, n, a->db, need_z};
    return run_colsum(&c, 1, m, a->dtype, ws, st);
}

// ---- gated feed-forward block ----------------------------------------------
int check_ffn(const char* what, const lf_gated_ffn_t* a) {
    if (!a) return missing(what, "arguments are");
    if (int rc = check_common(what, a->activation, a->dtype, {a->m, a->c, a->f})) return rc;
    if (2 * a->f > INT32_MAX - 256) return too_large(what);
    if (int rc = check_aligned(what, {a->x, a->w_in, a->b_in, a->w_out, a->b_out, a->residual, a->y, a->dy, a->dx, a->dw_in, a->db_in,
                                      a->dw_out, a->db_out}, 2))
        return rc;
    if (a->m == 0 || a->c == 0) return LF_OK;
    if (!a->x || (a->f > 0 && (!a->w_in || !a->w_out))) return missing(what, "x, w_in and w_out are");
    if (a->ldx < a->c || (a->residual && a->ldr < a->c)) {
        set_error("%s: a row stride is shorter than its row", what);
        return LF_ERR_INVALID;
    }
    return LF_OK;
}

// Win [2F, C] as two planes of F rows, so that a tile that passes F reads zeros.
Mat gate_up(Mat w, int64_t f) { return {w.p, w.inner, f, w.ld, 2, f * w.ld}; }

// Tile of the gated kernels by the same estimate as choose(); bn counts gate
// and up columns.  A tile of the backward has two halves of bn/2 hidden
// columns and a third product that is as wide as bn; about 700 cycles of each
// half's epilogue are not covered by products.
Shape choose_gated(int64_t m, int64_t f, int64_t c, bool bwd) {
    const int64_t iters = (c + 63) / 64, sms = num_sms();
    Shape best{1, 128, 1};
    double least = 1e30;
    for (int ctas : {2, 1})
        for (int bh : {128, 64, 32}) {
            if (bh < (ctas == 2 && !bwd ? 128 : bwd ? 64 : 32)) continue;
            const int64_t width = bwd ? 2 * bh : bh;
            const int64_t tiles = (m + kBM * ctas - 1) / (kBM * ctas) * ((f + width - 1) / width), waves = (tiles * ctas + sms - 1) / sms;
            const double main = iters * step_cycles(ctas, 2 * bh, 2 * bh), epi = 500 + bh * (bwd ? 25.0 : 15.0);
            double t = bwd ? waves * std::max(3 * main + 1400, 2 * epi) + epi : waves * std::max(main, epi) + std::min(main, epi);
            if (t < least) least = t, best = {ctas, 2 * bh, 1};
        }
    return best;
}

int run_gated(const lf_gated_ffn_t* a, const Mat& x, const Mat& win, const Mat* dy, const Mat* wout, void* out, int64_t ldo,
              int64_t plane, cudaStream_t st) {
    const bool bwd = dy != nullptr;
    const Shape s = choose_gated(a->m, a->f, a->c, bwd);
    const int bh = s.bn / 2;
    GemmArgs<1> args{};
    Problem& g = args.p[0];
    g.m = (int)a->m, g.n = (int)a->f;
    g.msegs = g.splits = 1;
    g.tiles_m = (int)((a->m + kBM * s.ctas - 1) / (kBM * s.ctas));
    const int width = bwd ? 2 * bh : bh;  // hidden columns of a tile
    g.tiles_n = (int)((a->f + width - 1) / width);
    if ((int64_t)g.tiles_m * g.tiles_n > INT32_MAX / 2) return too_large("gated feed-forward block");
    g.iters = g.split_iters = g.seg_iters = (int)((a->c + 63) / 64);
    g.bn = s.bn;
    args.stage_bytes = stage_bytes_of(s);
    g.idesc = idesc_of(a->dtype, false, false, s.ctas, s.bn);
    g.idesc2 = idesc_of(a->dtype, false, true, s.ctas, s.bn);
    g.e.out = out, g.e.ldo = ldo, g.e.bias = a->b_in, g.e.act = a->activation;
    if (!encode_out(&g.out, {out, a->f, a->m, ldo, bwd ? 3 : 1, plane}, a->dtype)) return LF_ERR_CUDA;
    if (!encode(&g.a, x, a->dtype, 64, kBM) || !encode(&g.b, gate_up(win, a->f), a->dtype, 64, bh)) return LF_ERR_CUDA;
    if (bwd && (!encode(&g.a2, *dy, a->dtype, 64, kBM) || !encode(&g.b2, *wout, a->dtype, 64, 64))) return LF_ERR_CUDA;
    set_divisors(g, s.ctas);
    args.first[1] = (int)units_of(g);
    if (bwd)
        return a->dtype == LF_F16 ? launch_ctas<__half, kGatedBwd, false>(args, s.ctas, st)
                                  : launch_ctas<__nv_bfloat16, kGatedBwd, false>(args, s.ctas, st);
    return a->dtype == LF_F16 ? launch_ctas<__half, kGated, false>(args, s.ctas, st)
                              : launch_ctas<__nv_bfloat16, kGated, false>(args, s.ctas, st);
}

template <typename T>
int launch_narrow(NarrowArgs& g, cudaStream_t st) {
    constexpr int w_bytes = 3 * kHB * kRowBytes, rest = 4 * kBM * kRowBytes + kEpiWarps * (kStageOut + column_bytes<false>()) + kBarrierBytes;
    g.stages = std::min(6, (kSmemLimit - rest) / w_bytes);
    static std::once_flag once[64];
    int dev = 0;
    cudaGetDevice(&dev);
    std::call_once(once[dev & 63], [] { cudaFuncSetAttribute(narrow_ffn_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemLimit); });
    launch_early(narrow_ffn_kernel<T>, (unsigned)std::min(g.tiles, num_sms()), kGemmThreads, (size_t)g.stages * w_bytes + rest, 1, st, g);
    return check_launch("narrow_ffn_kernel");
}

// Whether the forward runs as one kernel: few channels, and either few hidden
// columns or enough tiles of 128 tokens, since a CTA takes a tile's hidden
// columns one after another (64 channels, bf16, us, one kernel and two:
// 100352 tokens, 256 hidden 31 and 41; 500 tokens 8.0 and 9.3; 100352 tokens,
// 1024 hidden 85 and 126; 9472 tokens 18 and 19; 2000 tokens 18 and 13).  From
// 65 to 128 channels one kernel, with its weights through a ring, was slower than
// two (100352 tokens: 96 channels, 384 hidden 71 and 62; 128, 512 90 and 80; at
// most 4 % faster, 72, 256: 56 and 57).
bool narrow(const lf_gated_ffn_t* a) {
    return a->f > 0 && a->c <= kNarrow && !few_rows(a->m, 3 * a->f, a->c) &&
           (a->f <= 5 * kHB || 2 * ((a->m + kBM - 1) / kBM) >= num_sms());
}

int run_narrow(const lf_gated_ffn_t* a, const Mat& x, const Mat& win, const Mat& wout, const Epilogue& e, cudaStream_t st) {
    NarrowArgs g{};
    g.e = e;
    g.e.act = a->activation;
    g.e.tma = tma_ok(e.out, e.ldo, 2);
    g.e.pairs = a->c % 2 == 0 && e.ldo % 2 == 0 && aligned(e.out, 4);
    g.e.vec_res = a->c % 8 == 0 && tma_ok(e.res, e.ldr, 2);
    g.b_in = a->b_in;
    g.m = (int)a->m, g.c = (int)a->c, g.f = (int)a->f;
    g.tiles = (int)((a->m + kBM - 1) / kBM);
    g.blocks = (int)((a->f + kHB - 1) / kHB);
    if ((int64_t)g.tiles * g.blocks > INT32_MAX / 2) return too_large("gated feed-forward block");
    g.idesc1 = idesc_of(a->dtype, false, false, 1, 2 * kHB);
    g.idesc2 = idesc_of(a->dtype, false, false, 1, kNarrow);
    if (!encode(&g.x, x, a->dtype, 64, kBM) || !encode(&g.win, gate_up(win, a->f), a->dtype, 64, kHB, CU_TENSOR_MAP_SWIZZLE_128B, 2) ||
        !encode(&g.wout, wout, a->dtype, 64, kNarrow))
        return LF_ERR_CUDA;
    if (g.e.tma && !encode_out(&g.out, {e.out, a->c, a->m, e.ldo, 1, 0}, a->dtype)) return LF_ERR_CUDA;
    return a->dtype == LF_F16 ? launch_narrow<__half>(g, st) : launch_narrow<__nv_bfloat16>(g, st);
}

template <typename T, int CTAS>
int launch_narrow_bwd(const NarrowBwdArgs& g, int slots, cudaStream_t st) {
    constexpr int bytes = 10 * kBM * kRowBytes + 6 * kHB * kRowBytes + 16384 + 2048 + 2 * kBwdHidden * (int)sizeof(T) + kBarrierBytes;
    static_assert(bytes <= kSmemLimit, "shared memory");
    static std::once_flag once[64];
    int dev = 0;
    cudaGetDevice(&dev);
    const auto kernel = narrow_ffn_bwd_kernel<T, CTAS>;
    std::call_once(once[dev & 63], [&] { cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemLimit); });
    launch_early(kernel, (unsigned)(slots * CTAS), kBwdThreads, (size_t)bytes, CTAS, st, g);
    return check_launch("narrow_ffn_bwd_kernel");
}

// Whether the backward runs as one kernel and a join: wherever the weights and
// the sums of their gradients fit two SMs, since then it is as fast at the
// smallest sizes and faster above (GPU time in us with bf16, 64 channels,
// against the gated backward, three products and a join: 128 tokens, 64 hidden
// 14.5 and 14.5; 500, 256: 25 and 29; 9472, 256: 22 and 31; 100352, 64: 33 and
// 63; 100352, 256: 64 and 126; 401408, 176: 201 and 377).
bool narrow_bwd(const lf_gated_ffn_t* a) { return a->f > 0 && a->c <= kNarrow && a->f <= 2 * kBwdHidden; }

int run_narrow_bwd(const lf_gated_ffn_t* a, const Mat& x, const Mat& win, const Mat& wout, const Mat& dy, Arena& ws, cudaStream_t st) {
    const int64_t m = a->m, c = a->c, f = a->f;
    if (m > INT32_MAX - 256) return too_large("gated feed-forward block");
    NarrowBwdArgs g{};
    const int ctas = f > kBwdHidden ? 2 : 1;
    g.tiles = (int)((m + kBM - 1) / kBM);
    const int slots = std::min(g.tiles, num_sms() / ctas);
    g.ld_in = (int)up(c, 4), g.ld_out = (int)up(f, 4), g.ld_bi = (int)up(2 * f, 4), g.ld_bo = (int)up(c, 4);
    if (a->dw_in) g.part_in = (float*)ws.take((size_t)slots * 2 * f * g.ld_in * 4);
    if (a->dw_out) g.part_out = (float*)ws.take((size_t)slots * c * g.ld_out * 4);
    if (a->db_in) g.part_bi = (float*)ws.take((size_t)slots * g.ld_bi * 4);
    if (a->db_out) g.part_bo = (float*)ws.take((size_t)slots * g.ld_bo * 4);
    if (!ws.base) return LF_OK;
    g.b_in = a->b_in, g.dx = a->dx, g.act = a->activation;
    g.m = (int)m, g.c = (int)c, g.f = (int)f;
    g.blocks = f > kHB ? 2 : 1;
    g.vec_dx = c % 8 == 0 && aligned(a->dx, 16);
    g.id_gu = idesc_of(a->dtype, false, false, 1, 2 * kHB);
    g.id_n = idesc_of(a->dtype, false, true, 1, 64);
    g.id_w = idesc_of(a->dtype, true, true, 1, 64);
    g.id_b = idesc_of(a->dtype, true, false, 1, 16);
    if (!encode(&g.x, x, a->dtype, 64, kBM) || !encode(&g.dy, dy, a->dtype, 64, kBM) ||
        !encode(&g.win, gate_up(win, f), a->dtype, 64, kHB, CU_TENSOR_MAP_SWIZZLE_128B, 2) || !encode(&g.wout, wout, a->dtype, 64, kNarrow))
        return LF_ERR_CUDA;
    const bool half = a->dtype == LF_F16;
    int rc;
    if (ctas == 2) rc = half ? launch_narrow_bwd<__half, 2>(g, slots, st) : launch_narrow_bwd<__nv_bfloat16, 2>(g, slots, st);
    else rc = half ? launch_narrow_bwd<__half, 1>(g, slots, st) : launch_narrow_bwd<__nv_bfloat16, 1>(g, slots, st);
    if (rc) return rc;
    JoinJobs jobs{};
    int count = 0;
    auto join = [&](const float* part, int64_t rows, int64_t ld, int64_t cols, void* out) {
        if (!part) return;
        JoinJob& j = jobs.job[count++] = {part, rows, ld, slots, (int)cols, slots >= 32 ? 8 : slots >= 8 ? 4 : 1, {}};
        set_out(j.e, out, cols);
    };
    join(g.part_in, 2 * f, g.ld_in, c, a->dw_in);
    join(g.part_out, c, g.ld_out, f, a->dw_out);
    join(g.part_bi, 1, g.ld_bi, 2 * f, a->db_in);
    join(g.part_bo, 1, g.ld_bo, c, a->db_out);
    return count ? join_splits(jobs, count, a->dtype, st) : LF_OK;
}

int ffn_fwd(const lf_gated_ffn_t* a, Arena& ws, cudaStream_t st) {
    const int64_t m = a->m, c = a->c, f = a->f;
    if (m == 0 || c == 0) return LF_OK;
    const int64_t ldh = up(f, 8);
    Mat h{narrow(a) ? nullptr : ws.take((size_t)m * ldh * 2), f, m, ldh, 1, 0};
    Epilogue e{};
    set_out(e, a->y, c);
    e.bias = a->b_out;
    if (a->residual) set_res(e, a->residual, a->ldr);
    if (f > 0 && few_rows(m, 3 * f, c)) {
        if (!ws.base) return LF_OK;
        Epilogue eh{};
        set_out(eh, const_cast<void*>(h.p), ldh);
        eh.bias = a->b_in, eh.act = a->activation;
        if (int rc = run_few<true>(a->x, a->ldx, a->w_in, c, m, f, c, eh, a->dtype, st)) return rc;
        return run_few<false>(h.p, ldh, a->w_out, f, m, c, f, e, a->dtype, st);
    }
    Mat x = operand(a->x, m, c, a->ldx, 2, ws, st), win = operand(a->w_in, 2 * f, c, c, 2, ws, st);
    Mat wout = operand(a->w_out, c, f, f, 2, ws, st);
    if (narrow(a)) return ws.base ? run_narrow(a, x, win, wout, e, st) : LF_OK;
    if (ws.base && f > 0)
        if (int rc = run_gated(a, x, win, nullptr, nullptr, const_cast<void*>(h.p), ldh, 0, st)) return rc;
    Product q = weight_product(h, wout, m, c, f, a->dtype, a->dtype);
    q.e = e;
    return run_product(q, ws, st);
}

int ffn_bwd(const lf_gated_ffn_t* a, Arena& ws, cudaStream_t st) {
    const int64_t m = a->m, c = a->c, f = a->f;
    if (m == 0 || c == 0) return LF_OK;
    const int64_t ld = up(f, 8), plane = m * ld;
    Mat x = operand(a->x, m, c, a->ldx, 2, ws, st), win = operand(a->w_in, 2 * f, c, c, 2, ws, st);
    Mat wout = operand(a->w_out, c, f, f, 2, ws, st), dy = operand(a->dy, m, c, a->lddy, 2, ws, st);
    if (narrow_bwd(a)) return run_narrow_bwd(a, x, win, wout, dy, ws, st);
    uint16_t* dz = (uint16_t*)ws.take((size_t)3 * plane * 2);  // dg, du, h
    if (ws.base && f > 0)
        if (int rc = run_gated(a, x, win, &dy, &wout, dz, ld, plane, st)) return rc;
    const Mat both{dz, f, m, ld, 2, plane}, h{dz + 2 * plane, f, m, ld, 1, 0};
    Product q[3];
    int count = 0;
    if (a->dx) {  // dx = [dg|du] Win: two K segments of F
        Product& p = q[count++] = weight_product(both, gate_up(win, f), m, c, f, a->dtype, a->dtype);
        p.b_mn = true;
        p.ksegs = 2;
        set_out(p.e, a->dx, c);
    }
    if (a->dw_in) {  // two row segments of F
        Product& p = q[count++] = weight_product(both, x, f, c, m, a->dtype, a->dtype);
        p.a_mn = p.b_mn = true;
        p.msegs = 2;
        set_out(p.e, a->dw_in, c);
    }
    if (a->dw_out) {
        Product& p = q[count++] = weight_product(dy, h, c, f, m, a->dtype, a->dtype);
        p.a_mn = p.b_mn = true;
        set_out(p.e, a->dw_out, f);
    }
    if (int rc = run_products(q, count, ws, st)) return rc;
    uint16_t* db_in = (uint16_t*)a->db_in;
    const Columns cols[3] = {{dz, ld, f, db_in, true}, {dz + plane, ld, f, db_in ? db_in + f : nullptr, true}, {a->dy, a->lddy, c, a->db_out, false}};
    return run_colsum(cols, 3, m, a->dtype, ws, st);
}

int check_ws(const char* what, const void* ws, size_t have, size_t need) {
    if (need && (!ws || !aligned(ws, 256) || have < need)) {
        set_error("%s: needs %zu bytes of 256-byte aligned workspace, got %zu", what, need, ws ? have : (size_t)0);
        return LF_ERR_INVALID;
    }
    return LF_OK;
}

// With a counting arena the operators only add up what they would take.
template <class F>
size_t count_of(F&& f) {
    Arena ws{0};
    return f(ws) == LF_OK ? ws.used : 0;
}
constexpr uintptr_t kNoWorkspace = 256;  // stands for a workspace of no bytes

template <class F>
int run_with(const char* what, void* ws, size_t bytes, size_t need, F&& f) {
    if (int rc = check_ws(what, ws, bytes, need)) return rc;
    Arena arena{need ? reinterpret_cast<uintptr_t>(ws) : kNoWorkspace};
    return f(arena);
}

}  // namespace
}  // namespace lfb

using namespace lfb;

extern "C" size_t lf_linear_fwd_workspace_size(const lf_linear_t* a) {
    if (check_linear("lf_linear_fwd", a, false)) return 0;
    return count_of([&](Arena& w) { return linear_fwd(a, false, w, nullptr); });
}

extern "C" int lf_linear_fwd(const lf_linear_t* a, void* workspace, size_t workspace_bytes, lf_stream_t stream) {
    clear_error();
    if (int rc = check_linear("lf_linear_fwd", a, false)) return rc;
    if (a->m && a->n && !a->y) return missing("lf_linear_fwd", "y is");
    return run_with("lf_linear_fwd", workspace, workspace_bytes, lf_linear_fwd_workspace_size(a),
                    [&](Arena& w) { return linear_fwd(a, false, w, (cudaStream_t)stream); });
}

extern "C" size_t lf_linear_quant_fwd_workspace_size(const lf_linear_t* a) {
    if (check_linear("lf_linear_quant_fwd", a, true)) return 0;
    return count_of([&](Arena& w) { return linear_fwd(a, true, w, nullptr); });
}

extern "C" int lf_linear_quant_fwd(const lf_linear_t* a, void* workspace, size_t workspace_bytes, lf_stream_t stream) {
    clear_error();
    if (int rc = check_linear("lf_linear_quant_fwd", a, true)) return rc;
    if (a->m && a->n && !a->y) return missing("lf_linear_quant_fwd", "y is");
    return run_with("lf_linear_quant_fwd", workspace, workspace_bytes, lf_linear_quant_fwd_workspace_size(a),
                    [&](Arena& w) { return linear_fwd(a, true, w, (cudaStream_t)stream); });
}

extern "C" size_t lf_linear_bwd_workspace_size(const lf_linear_t* a) {
    if (check_linear("lf_linear_bwd", a, false)) return 0;
    return count_of([&](Arena& w) { return linear_bwd(a, w, nullptr); });
}

extern "C" int lf_linear_bwd(const lf_linear_t* a, void* workspace, size_t workspace_bytes, lf_stream_t stream) {
    clear_error();
    if (int rc = check_linear("lf_linear_bwd", a, false)) return rc;
    cudaStream_t st = (cudaStream_t)stream;
    if (a->m && a->n && !a->dy) return missing("lf_linear_bwd", "dy is");
    if (a->lddy < a->n) {
        set_error("lf_linear_bwd: lddy is shorter than a row");
        return LF_ERR_INVALID;
    }
    return run_with("lf_linear_bwd", workspace, workspace_bytes, lf_linear_bwd_workspace_size(a),
                    [&](Arena& w) { return linear_bwd(a, w, st); });
}

extern "C" size_t lf_gated_ffn_fwd_workspace_size(const lf_gated_ffn_t* a) {
    if (check_ffn("lf_gated_ffn_fwd", a)) return 0;
    return count_of([&](Arena& w) { return ffn_fwd(a, w, nullptr); });
}

extern "C" int lf_gated_ffn_fwd(const lf_gated_ffn_t* a, void* workspace, size_t workspace_bytes, lf_stream_t stream) {
    clear_error();
    if (int rc = check_ffn("lf_gated_ffn_fwd", a)) return rc;
    if (a->m && a->c && !a->y) return missing("lf_gated_ffn_fwd", "y is");
    return run_with("lf_gated_ffn_fwd", workspace, workspace_bytes, lf_gated_ffn_fwd_workspace_size(a),
                    [&](Arena& w) { return ffn_fwd(a, w, (cudaStream_t)stream); });
}

extern "C" size_t lf_gated_ffn_bwd_workspace_size(const lf_gated_ffn_t* a) {
    if (check_ffn("lf_gated_ffn_bwd", a)) return 0;
    return count_of([&](Arena& w) { return ffn_bwd(a, w, nullptr); });
}

extern "C" int lf_gated_ffn_bwd(const lf_gated_ffn_t* a, void* workspace, size_t workspace_bytes, lf_stream_t stream) {
    clear_error();
    if (int rc = check_ffn("lf_gated_ffn_bwd", a)) return rc;
    cudaStream_t st = (cudaStream_t)stream;
    if (a->m == 0 || a->c == 0) {  // no token or no channel: every gradient is empty or zero
        if (int rc = zero(a->dw_in, 2 * a->f, a->c * 2, st)) return rc;
        if (int rc = zero(a->dw_out, a->c, a->f * 2, st)) return rc;
        if (int rc = zero(a->db_in, 2 * a->f, 2, st)) return rc;
        return zero(a->db_out, 1, a->c * 2, st);
    }
    if (!a->dy) return missing("lf_gated_ffn_bwd", "dy is");
    if (a->lddy < a->c) {
        set_error("lf_gated_ffn_bwd: lddy is shorter than a row");
        return LF_ERR_INVALID;
    }
    return run_with("lf_gated_ffn_bwd", workspace, workspace_bytes, lf_gated_ffn_bwd_workspace_size(a),
                    [&](Arena& w) { return ffn_bwd(a, w, st); });
}
