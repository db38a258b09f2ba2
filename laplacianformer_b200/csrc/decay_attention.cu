// Causal linear attention with a decay per head, its backward pass, and its
// form for single tokens.
//
//   S_t = l S_(t-1) + k_t v_t^T,   o_t = sigma q_t S_t,   l = exp(log_decay[h])
//
// Prompts and training go by chunks of 128 tokens.  Within a chunk, with G the
// state decayed to the chunk's first token (l S before it):
//   o_i = sigma [ sum_(j<=i) l^(i-j) (q_i . k_j) v_j + l^i q_i G ]
//   G'  = l^n G + sum_j l^(n-j) k_j v_j^T            (n tokens, j from 0)
// The gradients are the same recurrence with other operands, so one kernel
// makes all four (out = mix(a, b, c)):
//   o  = mix(q, k, v)    dq = mix(do, v, k)          forwards in time
//   dk = mix(v, do, q)   dv = mix(k, q, do)          backwards
// and the gradient of the first state is the last dv state.
//
// Every power of l is taken of a difference of positions and is at most 1 for
// a decay: nothing is divided by a small power.  Sums and states are fp32.
// Rounded to 16 bits as operands of products, besides the inputs: the weighted
// scores (once), the state that q meets (once), and l^(n-j) b_j, which goes in as
// two 16-bit parts so that the state keeps about 17 bits (bf16) or 22 (fp16) of
// each term.  In fp16, whose range is narrow (gradients of 1e-6 would be
// subnormal, products of large ones infinite), powers of two bring these operands
// into it and are taken out of the sums: one per row of scores, by its largest
// weighted score; one per chunk of b, by its largest weighted row, at most 2^14 (of
// a term 2^-30 of the largest is lost, or 2^-39); one per state.  What it takes to
// find them: 32x2x3136x32 training 170 -> 201 us, 8x16x16384x64 training 1.39 ->
// 1.56 ms, 8 heads of 65536 tokens, size 128, 231 -> 268 us.  (Bounds by the sizes
// of a's rows and b, looked up by the copying warp: 196 us, 1.71 ms, 402 us; by a
// launch of their own: 215 us, 1.93 ms, 335 us.)
//
// What bounds it.  Sequences are cut into segments until every block slot has
// one (two slots per SM for heads up to 64); the state before a segment comes
// from a launch that reads b and c of the segments before.  Where heads fill the
// slots without cuts the main launch is memory bound: 296 heads of 7168 tokens,
// bf16, size 64: 208 us, 5.2 TB/s.  8x16x16384x64: 240 us and 45 us for the
// sums, since 256 segments leave 40 slots empty.  A training step is four mixes
// and two sums (dq takes the forward's, dv those of dk, transposed): 1.21 ms; with
// four sums 1.36.  Few chunks per slot (32x2x3136x32 fp16 201 us, 128x8x196x64 bf16
// 150 us a training step) are bound by a chunk's chain: products, weights, products,
// output, about 5200 cycles for a pair of blocks.
// Between 64 and 128 one block fits an SM and waits on that chain alone: 8 heads
// of 65536 tokens, size 128: 216 us, 2.5 TB/s.
// A token at a time only the state matters: 192x16 heads of 64: 15 us, 6.7 TB/s.
#include <algorithm>
#include <type_traits>
#include <utility>

#include "tc_ptx.cuh"
#include "tma_map.h"

namespace lfb {

// Set by a kernel whose bounded wait expired (merged into lf_device_status).
__device__ int g_decay_status = 0;

int decay_status(bool clear) {
    int v = 0;
    if (cudaMemcpyFromSymbol(&v, g_decay_status, sizeof(int)) != cudaSuccess) return LF_ERR_CUDA;
    if (clear) {
        int z = 0;
        if (cudaMemcpyToSymbol(g_decay_status, &z, sizeof(int)) != cudaSuccess) return LF_ERR_CUDA;
    }
    return v;
}

namespace {

constexpr int kChunk = 128;           // tokens per chunk: rows of a product's tile
constexpr int kRing = 5;              // operand tiles in flight: the chunk's three and the next one's first two
constexpr int kEpi = 256;             // threads that turn accumulators into operands and outputs
constexpr int kThreads = kEpi + 64;   // and a warp for copies, a warp for products
constexpr int kBlock = kChunk * 128;  // bytes of 128 rows of 64 columns
constexpr int kCutChunks = 64;        // chunks whose products may follow one another on a state: with 16 cuts of 2^-23 at most, 2^-13
constexpr uint32_t kNegateA = 1u << 13;  // of an instruction descriptor: the product with -A

struct alignas(64) MixArgs {
    CUtensorMap a, b, c, out;
    const float* log_decay;
    const float* g0;         // state before the first token (to be decayed by l), or with `rev` the gradient of the last state
    float* gout;             // state after the last token, or with `rev` the gradient of the first state
    float* ends;             // [bh][nseg][units][64W][64W]: what each unit of a segment adds to the state
    const int64_t* lengths;  // tokens per sequence, or null
    void* o;                 // rows of dc elements, where TMA cannot write them
    int64_t o_sb, o_sh, o_st;
    int heads, t, da, dc, chunks, nseg, per_seg, items;
    int unit, units;         // chunks per unit, units per segment
    int joined;              // a segment finds the state before it in the slot of its unit that is first in time
    int turned;              // the sums are there already, transposed (of b and c the other way round)
    int g0_row, g0_col;      // strides within a state matrix (transposed for dq and dk)
    float scale, g0_scale, gout_scale;
    int ksteps, nb;          // 16-column steps of da; dc rounded up to 16
    uint32_t id_qk, id_qg, id_pv, id_kv;
    int tma_out;
};

template <int W>
constexpr int mix_smem() {
    // ring, low parts (then the output's staging), state operand, tables and barriers
    return 1024 + (kRing + 1) * W * kBlock + 64 * W * 128 * W + 2048;
}

template <int W>
constexpr int kEndsRing = 4;  // tiles in flight of the sums before a segment
template <int W>
constexpr int ends_smem() {
    return 1024 + (kEndsRing<W> + 2) * W * kBlock + 256;
}

__device__ __forceinline__ void load4d(void* dst, const CUtensorMap* map, uint64_t* bar, int x, int h, int t, int b) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(
                     smem_u32(dst)),
                 "l"(map), "r"(smem_u32(bar)), "r"(x), "r"(h), "r"(t), "r"(b)
                 : "memory");
}
__device__ __forceinline__ void store4d(const CUtensorMap* map, const void* src, int x, int h, int t, int b) {
    asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.tile.bulk_group [%0, {%2, %3, %4, %5}], [%1];" ::"l"(map),
                 "r"(smem_u32(src)), "r"(x), "r"(h), "r"(t), "r"(b)
                 : "memory");
}
__device__ __forceinline__ void expect(uint64_t* bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
// mbar_wait() for waits that are mostly short: the clock is read only after a run of tries, so that waiting warps take few
// issue slots from the working ones (with mbar_wait they took more than half of them).
__device__ __forceinline__ bool wait_for(uint64_t* bar, uint32_t parity) {
    const uint32_t addr = smem_u32(bar);
    uint64_t t0 = 0;
    for (uint32_t spin = 0;; ++spin) {
        uint32_t done;
        asm volatile(
            "{\n\t.reg .pred p, q;\n\t.reg .b32 n;\n\t"
            "mov.b32 n, 0;\n"
            "TRY%=:\n\t"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
            "@p bra DONE%=;\n\t"
            "add.u32 n, n, 1;\n\t"
            "setp.lt.u32 q, n, 64;\n\t"
            "@q bra TRY%=;\n"
            "DONE%=:\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}\n"
            : "=r"(done)
            : "r"(addr), "r"(parity), "r"(20000u)
            : "memory");
        if (done) return true;
        if (spin == 0) t0 = global_ns();
        else if (global_ns() - t0 > 2000000000ull) return false;
    }
}
__device__ __forceinline__ void arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// Barrier of the epilogue's threads; whether `ok` holds for all of them, so that they leave together.
__device__ __forceinline__ bool epi_sync(bool ok) {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %1, 0;\n\t"
        "barrier.cta.red.and.pred q, 1, %2, p;\n\tselp.u32 %0, 1, 0, q;\n\t}\n"
        : "=r"(r)
        : "r"((uint32_t)ok), "n"(kEpi)
        : "memory");
    return r != 0;
}
// Pairs of 16-bit values, each product and sum rounded once.
template <typename T> __device__ __forceinline__ uint32_t mul16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    if constexpr (std::is_same<T, __half>::value) asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    else asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
template <typename T> __device__ __forceinline__ uint32_t fma16x2(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t r;
    if constexpr (std::is_same<T, __half>::value) asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
    else asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
    return r;
}
// (The hardware's power of two, about 2 units in the last place, for factors that meet a 16-bit rounding.)
__device__ __forceinline__ float exp2_of(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// The lowest n bits (none below 0, all from 32 on).
__device__ __forceinline__ uint32_t keep_low(int n) {
    uint32_t r;
    asm("shl.b32 %0, %1, %2;" : "=r"(r) : "r"(0xffffffffu), "r"(max(n, 0)));  // (shifts past the width give 0)
    return ~r;
}
__device__ __forceinline__ void sts16(uint8_t* p, uint4 v) { *reinterpret_cast<uint4*>(p) = v; }

// l^n; 1 for n = 0 whatever l is.
__device__ __forceinline__ float power(float g, int64_t n) { return n == 0 ? 1.f : expf((float)n * g); }

struct Item {
    int bh, b, h, seg, first, n, active;
    int64_t len;
};
__device__ __forceinline__ int64_t tokens_in(const MixArgs& p, int b) {
    if (!p.lengths) return p.t;
    const int64_t n = p.lengths[b];
    return n < 0 ? 0 : n < p.t ? n : p.t;
}
__device__ __forceinline__ Item item_of(const MixArgs& p, int i) {
    Item t;
    t.bh = i / p.nseg;
    t.seg = i - t.bh * p.nseg;
    t.b = t.bh / p.heads;
    t.h = t.bh - t.b * p.heads;
    t.len = tokens_in(p, t.b);
    t.active = (int)((t.len + kChunk - 1) / kChunk);
    t.first = t.seg * p.per_seg;
    const int last = min(min(t.first + p.per_seg, p.chunks), t.active);
    t.n = max(0, last - t.first);
    return t;
}

// Power of two that takes mx into [2^14, 2^15); 1 for 0 and for what is not finite.
__device__ __forceinline__ float range_scale(uint32_t bits) {
    const int e = (int)(bits >> 23);
    if (bits == 0 || e == 0xff) return 1.f;
    return __uint_as_float((uint32_t)max(1, min(127 + 141 - e, 254)) << 23);
}

// fp16 operands of products are brought into fp16's range by powers of two, which the products' sums are freed of again.
// The largest size among fp16 pairs (NaN only where all are).
template <int N>
__device__ __forceinline__ float largest16(const uint4 (&x)[N]) {
    __half2 m = __half2half2(__ushort_as_half(0));
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const uint32_t v[4] = {x[j].x, x[j].y, x[j].z, x[j].w};
#pragma unroll
        for (int q = 0; q < 4; ++q) m = __hmax2(m, __habs2(*reinterpret_cast<const __half2*>(&v[q])));
    }
    return fmaxf(__low2float(m), __high2float(m));
}
// 1 / s of a power of two between 2^-126 and 2^126.
__device__ __forceinline__ float inverse2(float s) { return __uint_as_float(0x7f000000u - __float_as_uint(s)); }
__device__ __forceinline__ float largest8(const float* p) {
    const float4 x = reinterpret_cast<const float4*>(p)[0], y = reinterpret_cast<const float4*>(p)[1];
    return fmaxf(fmaxf(fmaxf(x.x, x.y), fmaxf(x.z, x.w)), fmaxf(fmaxf(y.x, y.y), fmaxf(y.z, y.w)));
}
// For weighted b of sizes up to `top` whose weights are up to `grow`: the weights times it, and b times them, stay below 2^15.
__device__ __forceinline__ float weight_scale(float top, float grow) { return range_scale(__float_as_uint(fmaxf(top, 1.f) * fmaxf(grow, 1.f))); }

// Scales rows of a tile of b, 8 at a time (eight lanes to a row, so that no bank is met twice): b w in two parts, the
// first in place, the second negated in `low`; w0 and w1 are a row's weight in two parts, for the rows 4 apart.
//   high = b w0 rounded;  b w0 - high is exact (it has no more bits than b), and b w1 joins it with one rounding
__device__ __forceinline__ int row_pack(int w, int r, int ch) { return w * kBlock + r * 128 + ((ch ^ (r & 7)) << 4); }
template <int W>
__device__ __forceinline__ void fetch_rows(const uint8_t* tile, int row0, int lane, uint4 (&x)[2][W]) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int w = 0; w < W; ++w) x[i][w] = *reinterpret_cast<const uint4*>(tile + row_pack(w, row0 + (lane >> 3) + 4 * i, lane & 7));
}
template <typename T, int W>
__device__ __forceinline__ void scale_rows(uint8_t* tile, uint8_t* low, int row0, int lane, const uint4 (&x)[2][W], const uint32_t (&wh)[2], const uint32_t (&wl)[2]) {
#pragma unroll
    for (int w = 0; w < W; ++w) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t v[4] = {x[i][w].x, x[i][w].y, x[i][w].z, x[i][w].w};
            uint32_t h[4], l[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                h[q] = mul16x2<T>(v[q], wh[i]);
                l[q] = fma16x2<T>(v[q], wl[i] ^ 0x80008000u, fma16x2<T>(v[q], wh[i] ^ 0x80008000u, h[q]));
            }
            const int at = row_pack(w, row0 + (lane >> 3) + 4 * i, lane & 7);
            sts16(tile + at, make_uint4(h[0], h[1], h[2], h[3]));
            sts16(low + at, make_uint4(l[0], l[1], l[2], l[3]));
        }
    }
}
// A weight in two 16-bit parts, side by side; and each twice for packed arithmetic.
template <typename T>
__device__ __forceinline__ uint32_t split_weight(float w) {
    const T hi = Elem<T>::store(w);
    return pack2<T>(w, w - Elem<T>::load(hi));
}
__device__ __forceinline__ void spread(uint32_t w, uint32_t& wh, uint32_t& wl) {
    wh = __byte_perm(w, w, 0x1010);
    wl = __byte_perm(w, w, 0x3232);
}
// Rows past the sequence's end: zeros, whatever they hold.
template <int W>
__device__ __forceinline__ void clear_rows(uint8_t* tile, int from, int thread, int threads) {
    for (int j = thread; j < (kChunk - from) * 8 * W; j += threads) {
        const int r = from + j / (8 * W), u = j % (8 * W);
        sts16(tile + (u >> 3) * kBlock + r * 128 + ((u & 7) << 4), make_uint4(0u, 0u, 0u, 0u));
    }
}

// Whether nothing is left of unit u of a segment where the next segment (in time) begins: such units are neither summed nor read.
__device__ __forceinline__ bool forgotten(const MixArgs& p, float g, int u, bool rev) {
    return power(g, (int64_t)(rev ? u * p.unit : max(0, p.per_seg - (u + 1) * p.unit)) * kChunk) == 0.f;
}

// What units of chunks add to the state, for the segments that go on after them: sum_j l^(n-j) b_j c_j^T.  A chunk's products
// start from 0, with weights to the chunk's end, and are added to the unit's sum in registers while the next chunk's run: a
// product cuts its sum off at the accumulator's last bit, so that sums of many chunks on one accumulator would lose more the
// longer a unit is (units of 111 chunks: 7e-5 of the state, 6e-7 so).  Two warps copy and multiply, eight scale b and add up.
// Blocks for heads above 64 take at most 144 registers a thread (as 448 threads would), so that the join's blocks are placed
// beside them (8 heads of 65536 tokens, size 128: 216 us, 225 without).
template <typename T, int W, bool REV>
__global__ void __launch_bounds__(W == 1 ? kThreads : 448, W == 1 ? 2 : 1) decay_ends_kernel(const __grid_constant__ MixArgs p) {
    constexpr int kTile = W * kBlock, kState = 64 * W, kTiles = kEndsRing<W>;
    constexpr bool F16 = std::is_same<T, __half>::value;
    extern __shared__ uint8_t raw[];
    uint8_t* const ring = raw + (-smem_u32(raw) & 1023u);  // (keeps the pointer one to shared memory)
    uint8_t* const lows = ring + kTiles * kTile;
    uint64_t* const bars = reinterpret_cast<uint64_t*>(lows + 2 * kTile);
    uint64_t *full = bars, *empty = bars + kTiles, *ready = empty + kTiles, *used = ready + 2, *read = used + 2, *drain = read + 2;
    uint32_t* const tmem_ptr = reinterpret_cast<uint32_t*>(drain + 1);
    float* const tops = reinterpret_cast<float*>(drain + 2);  // [2][8], largest weighted b that a warp has seen
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    grid_release();
    if (tid == 0) {
        for (int i = 0; i < kTiles; ++i) mbar_init(&full[i], 1), mbar_init(&empty[i], 1);
        for (int i = 0; i < 2; ++i) mbar_init(&ready[i], kEpi), mbar_init(&used[i], 1), mbar_init(&read[i], kEpi);
        mbar_init(drain, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 9) tmem_alloc(tmem_ptr, 2 * kState);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    grid_wait();
    const uint32_t tmem = *tmem_ptr;
    bool ok = true;
    // Unit i of the segments that others follow.
    struct Unit {
        int b, h, first, n;  // chunks
        int64_t len, slot;
    };
    auto unit_of = [&](int i) {
        const int per = (p.nseg - 1) * p.units, bh = i / per, r = i - bh * per, seg = r / p.units + (REV ? 1 : 0), u = r % p.units;
        Unit x;
        x.b = bh / p.heads, x.h = bh - x.b * p.heads;
        x.len = tokens_in(p, x.b);
        x.slot = ((int64_t)bh * p.nseg + seg) * p.units + u;
        x.first = seg * p.per_seg + u * p.unit;
        const int end = min(min(x.first + p.unit, (seg + 1) * p.per_seg), p.chunks), active = (int)((x.len + kChunk - 1) / kChunk);
        // Forwards only whole units are asked for.
        x.n = REV ? max(0, min(end, active) - x.first) : end > x.first && (int64_t)end * kChunk <= x.len ? end - x.first : 0;
        if (forgotten(p, p.log_decay[x.h], u, REV)) x.n = 0;
        return x;
    };
    const int count = p.items;
    if (warp == 8) {
        if (elect_one()) {
            int n = 0;
            for (int i = blockIdx.x; ok && i < count; i += gridDim.x) {
                const Unit x = unit_of(i);
                for (int k = 0; ok && k < x.n; ++k)
                    for (int j = 0; j < 2; ++j, ++n) {
                        const int s = n % kTiles;
                        if (!(ok = wait_for(&empty[s], (n / kTiles & 1) ^ 1))) break;
                        expect(&full[s], kTile);
                        for (int w = 0; w < W; ++w)
                            load4d(ring + s * kTile + w * kBlock, j ? &p.c : &p.b, &full[s], w * 64, x.h, (x.first + k) * kChunk, x.b);
                    }
            }
            if (!ok)
                for (int k = max(0, n - kTiles); k < n; ++k) mbar_wait(&full[k % kTiles], k / kTiles & 1, 100000000ull);
        }
        __syncwarp();
    } else if (warp == 9) {
        const uint32_t go = elect_one() ? 1u : 0u;
        int m = 0;
        for (int i = blockIdx.x; ok && i < count; i += gridDim.x) {
            const Unit x = unit_of(i);
            for (int k = 0; k < x.n; ++k, ++m) {
                const int nb = 2 * m % kTiles, nc = (2 * m + 1) % kTiles;
                if (!(ok = wait_for(&full[nc], (2 * m + 1) / kTiles & 1) && wait_for(&ready[m & 1], m >> 1 & 1))) break;
                if (m > 1 && !(ok = wait_for(&read[m & 1], (m >> 1 & 1) ^ 1))) break;  // the sum before the last has been read
                tc_fence_after();
                const uint64_t dh = make_desc(smem_u32(ring + nb * kTile), kBlock, 1024), dl = make_desc(smem_u32(lows + (m & 1) * kTile), kBlock, 1024);
                const uint64_t dv = make_desc(smem_u32(ring + nc * kTile), kBlock, 1024);
                const uint32_t sum = tmem + (m & 1) * kState;
#pragma unroll
                for (int s = 0; s < 8; ++s) mma_f16(sum, dl + (uint64_t)(s * 128), dv + (uint64_t)(s * 128), p.id_kv | kNegateA, s > 0 ? 1u : 0u, go);
#pragma unroll
                for (int s = 0; s < 8; ++s) mma_f16(sum, dh + (uint64_t)(s * 128), dv + (uint64_t)(s * 128), p.id_kv, 1u, go);
                if (go) mma_commit(&empty[nb]), mma_commit(&empty[nc]), mma_commit(&used[m & 1]);
            }
        }
        if (!ok) {
            if (go) mma_commit(drain);
            mbar_wait(drain, 0, 100000000ull);
        }
        __syncwarp();
    } else {
        const int quad = warp & 3, half = warp >> 2, col0 = half * 32 * W;
        const uint32_t tq = tmem + ((uint32_t)(quad * 32) << 16);
        int m = 0;
        for (int i = blockIdx.x; i < count; i += gridDim.x) {
            const Unit x = unit_of(i);
            if (x.n == 0) continue;
            const float g = p.log_decay[x.h], whole = power(g, kChunk);
            float w[4], scale = 1.f, held = 1.f;  // fp16: the scale of b, and, forwards, of what `acc` holds
            uint32_t wh[2][2], wl[2][2];  // of the 16 rows of this warp
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int r = warp * 16 + (j >> 1) * 8 + (j & 1) * 4 + (lane >> 3);
                w[j] = power(g, REV ? r + 1 : kChunk - r);
                spread(split_weight<T>(w[j]), wh[j >> 1][j & 1], wl[j >> 1][j & 1]);
            }
            float acc[32 * W];
#pragma unroll
            for (int j = 0; j < 32 * W; ++j) acc[j] = 0.f;
            // Chunk k of the unit, the mk-th of this block, whose b was scaled by s.  (A power that overflows meets no 0.)
            auto add = [&](int k, int mk, float s) {
                ok = ok && wait_for(&used[mk & 1], mk >> 1 & 1);
                tc_fence_after();
                float w = REV ? power(g, (int64_t)k * kChunk) : k == 0 ? 0.f : whole;
                if constexpr (F16) w *= REV ? inverse2(s) : s * inverse2(held);
                held = s;
#pragma unroll
                for (int c = 0; c < 32 * W; c += 16)
                    if (col0 + c < p.nb) {
                        float v[16];
                        tmem_ld16(tq + (mk & 1) * kState + col0 + c, v);
                        tmem_wait_ld();
                        reg_fence(v);
#pragma unroll
                        for (int j = 0; j < 16; ++j) acc[c + j] = REV ? __fmaf_rn(w, v[j], acc[c + j]) : __fmaf_rn(w, acc[c + j], v[j]);
                    }
                tc_fence_before();
                arrive(&read[mk & 1]);
            };
            for (int k = 0; k < x.n; ++k, ++m) {
                const int nb = 2 * m % kTiles, nc = (2 * m + 1) % kTiles;
                const int L = (int)min((int64_t)kChunk, x.len - (int64_t)(x.first + k) * kChunk);
                uint8_t* const low = lows + (m & 1) * kTile;  // (its last products' sum has been read)
                const float last = scale;
                ok = ok && wait_for(&full[nb], 2 * m / kTiles & 1);
                uint4 rows[2][2][W];
                if constexpr (F16) {
                    float size = 0.f;
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        fetch_rows<W>(ring + nb * kTile, warp * 16 + u * 8, lane, rows[u]);
#pragma unroll
                        for (int i = 0; i < 2; ++i)
                            if (warp * 16 + u * 8 + (lane >> 3) + 4 * i < L) size = fmaxf(size, largest16(rows[u][i]) * w[2 * u + i]);
                    }
                    const uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(size));
                    if (lane == 0) tops[(m & 1) * 8 + warp] = __uint_as_float(top);
                    epi_sync(true);
                    scale = weight_scale(largest8(tops + (m & 1) * 8), whole);
#pragma unroll
                    for (int j = 0; j < 4; ++j) spread(split_weight<T>(w[j] * scale), wh[j >> 1][j & 1], wl[j >> 1][j & 1]);
                }
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    if constexpr (!F16) fetch_rows<W>(ring + nb * kTile, warp * 16 + u * 8, lane, rows[u]);
                    scale_rows<T, W>(ring + nb * kTile, low, warp * 16 + u * 8, lane, rows[u], wh[u], wl[u]);
                }
                if (L < kChunk) {
                    ok = ok && wait_for(&full[nc], (2 * m + 1) / kTiles & 1);
                    epi_sync(true);  // (the rows that others scaled)
                    clear_rows<W>(ring + nb * kTile, L, tid, kEpi), clear_rows<W>(low, L, tid, kEpi), clear_rows<W>(ring + nc * kTile, L, tid, kEpi);
                }
                fence_async_smem();
                arrive(&ready[m & 1]);
                if (k > 0) add(k - 1, m - 1, last);
            }
            add(x.n - 1, m - 1, scale);
            if constexpr (F16 && !REV)
#pragma unroll
                for (int j = 0; j < 32 * W; ++j) acc[j] *= inverse2(held);
            // The accumulators of 64 rows are 16 in each quarter of the lanes.
            if (W == 2 || lane < 16) {
                float* const dst = p.ends + (x.slot * kState + (W == 1 ? quad * 16 + lane : quad * 32 + lane)) * kState + col0;
#pragma unroll
                for (int j = 0; j < 32 * W; j += 4)
                    *reinterpret_cast<float4*>(dst + j) =
                        col0 + j < p.nb ? make_float4(acc[j], acc[j + 1], acc[j + 2], acc[j + 3]) : make_float4(0.f, 0.f, 0.f, 0.f);
            }
        }
    }
    if (!ok) atomicExch(&g_decay_status, (int)LF_ERR_TIMEOUT);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 9) tmem_dealloc(tmem, 2 * kState);
}

// From the units' sums the state before each segment, in the slot of its unit that is first in time: four elements of a head's
// state per thread, its units read eight at a time and joined in the order of time.  (Segments that summed their
// predecessors' units themselves read up to 34 x 64 KB each before their first chunk.)
template <int W, bool REV>
__global__ void __launch_bounds__(256) decay_join_kernel(const __grid_constant__ MixArgs p) {
    constexpr int kState = 64 * W, kQuads = kState * kState / 4;
    grid_release();
    grid_wait();
    const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int bh = (int)(at / kQuads), b = bh / p.heads;
    const float g = p.log_decay[bh - b * p.heads];
    const int64_t len = tokens_in(p, b);
    const int active = (int)((len + kChunk - 1) / kChunk), total = p.nseg * p.units;
    float4* const slots = reinterpret_cast<float4*>(p.ends) + (int64_t)bh * total * kQuads + at % kQuads;
    // Units are counted in time; the first chunk of one, its chunks (before another), whether its sum was made.
    auto place = [&](int i) { return REV ? total - 1 - i : i; };
    auto first = [&](int u) { return u / p.units * p.per_seg + u % p.units * p.unit; };
    auto length = [&](int u) { return min(p.unit, p.per_seg - u % p.units * p.unit); };
    auto there = [&](int u) {
        const int seg = u / p.units, from = first(u);
        if (forgotten(p, g, u % p.units, REV)) return false;
        return REV ? seg > 0 && from < active : seg < p.nseg - 1 && (int64_t)(from + length(u)) * kChunk <= len;
    };
    const float wu = power(g, (int64_t)p.unit * kChunk), wl = power(g, (int64_t)length(p.units - 1) * kChunk);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    bool any = false;  // (a power that overflows meets no 0)
    for (int i0 = 0; i0 < total; i0 += 8) {
        float4 x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (i0 + j < total && there(place(i0 + j))) x[j] = slots[(int64_t)place(i0 + j) * kQuads];
            else x[j] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int u = place(i0 + j), v = u % p.units;
            if (i0 + j >= total) break;
            if (v == (REV ? p.units - 1 : 0)) slots[(int64_t)u * kQuads] = acc;  // (its own sum is in x)
            if (!there(u)) continue;
            const float w = !any ? 0.f : v == p.units - 1 ? wl : wu;
            acc.x = __fmaf_rn(w, acc.x, x[j].x), acc.y = __fmaf_rn(w, acc.y, x[j].y), acc.z = __fmaf_rn(w, acc.z, x[j].z), acc.w = __fmaf_rn(w, acc.w, x[j].w);
            any = true;
        }
    }
}

// W: 64-column blocks per operand row (head sizes up to 64 W).  REV: backwards
// in time.  EXACT: the state is an output, or a segment is longer than kCutChunks.
// Products that add to a state cut it off at its last bit 16 times a chunk, always
// downwards: 1.2e-5 of a slow head's state, which 16-bit outputs do not see; but
// in a head that forgets nothing the cuts add up (65536 tokens in one segment:
// outputs 4.2e-4 too small, an fp16 rounding).  With EXACT a chunk's products start
// from 0 and are added to the decayed state in registers (8x16x16384x64 takes 8 %
// longer so); it waits in columns of its own, or, since the accumulators of 64
// rows leave lanes 16 to 31 of each quarter free, there.
template <typename T, int W, bool REV, bool EXACT>
__global__ void __launch_bounds__(kThreads, W == 1 ? 2 : 1) decay_mix_kernel(const __grid_constant__ MixArgs p) {
    constexpr int kTile = W * kBlock, kState = 64 * W;                        // state rows
    constexpr int kO = 128, kKv = 128 + 64 * W, kCols = W == 1 ? 256 : 512;   // tensor memory columns; scores from 0 on
    constexpr int kOld = W == 1 || !EXACT ? kKv : kKv + 128;                  // the decayed state
    constexpr bool F16 = std::is_same<T, __half>::value;
    extern __shared__ uint8_t raw[];
    uint8_t* const ring = raw + (-smem_u32(raw) & 1023u);  // (keeps the pointer one to shared memory)
    uint8_t* const low = ring + kRing * kTile;
    uint8_t* const gop = low + kTile;                                         // [state row][dc], 64 columns a block
    float* const pw = reinterpret_cast<float*>(gop + kState * 128 * W);       // l^n, n = 0..128
    uint32_t* const gmax = reinterpret_cast<uint32_t*>(pw + 132);             // largest size in the state; two in turn
    float* const tops = pw + 136;                                             // largest weighted b that a warp has seen
    float* const most = pw + 144;                                             // [2][128], largest score in each half of a row
    uint64_t* const bars = reinterpret_cast<uint64_t*>(pw + 400);
    uint64_t *full = bars, *empty = bars + kRing, *s_full = bars + 2 * kRing, *k_ready = s_full + 1, *p_ready = s_full + 2,
             *kv_full = s_full + 3, *o_full = s_full + 4, *g_ready = s_full + 5, *qg_full = s_full + 6, *drain = s_full + 7;
    uint32_t* const tmem_ptr = reinterpret_cast<uint32_t*>(s_full + 8);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    grid_release();
    if (tid == 0) {
        for (int i = 0; i < kRing; ++i) mbar_init(&full[i], 1), mbar_init(&empty[i], 1);
        mbar_init(s_full, 1), mbar_init(kv_full, 1), mbar_init(o_full, 1), mbar_init(qg_full, 1), mbar_init(drain, 1);
        mbar_init(k_ready, kEpi), mbar_init(p_ready, kEpi), mbar_init(g_ready, kEpi);
        gmax[0] = gmax[1] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 9) tmem_alloc(tmem_ptr, kCols);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    grid_wait();
    const uint32_t tmem = *tmem_ptr;
    bool ok = true;

    if (warp == 8) {  // copies
        if (elect_one()) {
            int n = 0;
            for (int i = blockIdx.x; ok && i < p.items; i += gridDim.x) {
                const Item t = item_of(p, i);
                for (int k = 0; ok && k < t.n; ++k) {
                    const int t0 = (REV ? t.first + t.n - 1 - k : t.first + k) * kChunk;
                    for (int j = 0; j < 3; ++j) {
                        const int s = n % kRing;
                        if (!(ok = wait_for(&empty[s], (n / kRing & 1) ^ 1))) break;
                        expect(&full[s], kTile);
                        const CUtensorMap* m = j == 0 ? &p.a : j == 1 ? &p.b : &p.c;
                        for (int w = 0; w < W; ++w) load4d(ring + s * kTile + w * kBlock, m, &full[s], w * 64, t.h, t0, t.b);
                        ++n;
                    }
                }
            }
            if (!ok)  // a wait ran out: let the copies in flight land
                for (int k = max(0, n - kRing); k < n; ++k) mbar_wait(&full[k % kRing], k / kRing & 1, 100000000ull);
        }
        __syncwarp();
    } else if (warp == 9) {  // products
        const uint32_t go = elect_one() ? 1u : 0u;
        int n = 0, cc = 0;
        for (int i = blockIdx.x; ok && i < p.items; i += gridDim.x) {
            const Item t = item_of(p, i);
            for (int k = 0; k < t.n; ++k, ++cc, n += 3) {
                const int na = n, nk = n + 1, nv = n + 2;
                const uint32_t sk = smem_u32(ring + nk % kRing * kTile), sv = smem_u32(ring + nv % kRing * kTile);
                if (!(ok = wait_for(&full[nk % kRing], nk / kRing & 1))) break;
                const int first = REV ? (t.active - 1) / p.per_seg : 0;  // the segment that the sequence starts with
                const bool has_g = k > 0 || p.g0 || t.seg != first;      // there is a state before this chunk
                const uint32_t sa = smem_u32(ring + na % kRing * kTile);
                if (!(ok = wait_for(&full[na % kRing], na / kRing & 1))) break;
                if (cc > 0 && !(ok = wait_for(o_full, (cc - 1) & 1))) break;  // the scores' columns hold its operand
                tc_fence_after();
                const uint64_t da = make_desc(sa, 16, 1024), db = make_desc(sk, 16, 1024);
#pragma unroll
                for (int s = 0; s < 4 * W; ++s) {  // (unrolled: an address that the loop computes costs more than the product)
                    const uint64_t at = (uint64_t)((s >> 2) * (kBlock >> 4) + (s & 3) * 2);
                    if (s < p.ksteps) mma_f16(tmem, da + at, db + at, p.id_qk, s > 0 ? 1u : 0u, go);
                }
                if (go) mma_commit(s_full);
                if (!(ok = wait_for(g_ready, cc & 1))) break;
                tc_fence_after();
                if (has_g) {
                    const uint64_t dg = make_desc(smem_u32(gop), kState * 128, 1024);
#pragma unroll
                    for (int s = 0; s < 4 * W; ++s) {
                        const uint64_t at = (uint64_t)((s >> 2) * (kBlock >> 4) + (s & 3) * 2);
                        if (s < p.ksteps) mma_f16(tmem + kO, da + at, dg + (uint64_t)(s * 128), p.id_qg, s > 0 ? 1u : 0u, go);
                    }
                    if (go) mma_commit(qg_full);
                }
                if (go) mma_commit(&empty[na % kRing]);
                if (!(ok = wait_for(k_ready, cc & 1) && wait_for(&full[nv % kRing], nv / kRing & 1))) break;
                tc_fence_after();
                const uint64_t dh = make_desc(sk, kBlock, 1024), dl = make_desc(smem_u32(low), kBlock, 1024);
                const uint64_t dv = make_desc(sv, kBlock, 1024);
#pragma unroll
                for (int s = 0; s < 8; ++s) mma_f16(tmem + kKv, dl + (uint64_t)(s * 128), dv + (uint64_t)(s * 128), p.id_kv | kNegateA, (has_g && !EXACT) || s > 0 ? 1u : 0u, go);
#pragma unroll
                for (int s = 0; s < 8; ++s) mma_f16(tmem + kKv, dh + (uint64_t)(s * 128), dv + (uint64_t)(s * 128), p.id_kv, 1u, go);
                if (go) mma_commit(kv_full), mma_commit(&empty[nk % kRing]);
                if (!(ok = wait_for(p_ready, cc & 1))) break;
                tc_fence_after();
#pragma unroll
                for (int s = 0; s < 8; ++s)  // scores of columns 64 on lie 64 columns further
                    mma_f16_ts(tmem + kO, tmem + (s >> 2) * 64 + (s & 3) * 8, dv + (uint64_t)(s * 128), p.id_pv, has_g || s > 0 ? 1u : 0u, go);
                if (go) mma_commit(o_full), mma_commit(&empty[nv % kRing]);
            }
        }
        if (!ok) {  // products in flight end before the tensor memory is freed
            if (go) mma_commit(drain);
            mbar_wait(drain, 0, 100000000ull);
        }
        __syncwarp();
    } else {
        const int quad = warp & 3, half = warp >> 2;
        const uint32_t tq = tmem + ((uint32_t)(quad * 32) << 16);
        const int row = quad * 32 + lane;                         // of a chunk
        // The state: the accumulators of 64 rows are 16 in each quarter of the lanes.
        const int srow = W == 1 ? quad * 16 + lane : row;
        const bool live = W == 2 || lane < 16;
        const int col0 = half * 32 * W;                           // this thread's columns of the state and of the output
        const int kr = tid >> 1, kpart = tid & 1;                 // the row of b, and half of it, that this thread scales
        int n = 0, cc = 0, qg = 0, puts = 0;
        for (int i = blockIdx.x; ok && i < p.items; i += gridDim.x) {
            const Item t = item_of(p, i);
            const float g = p.log_decay[t.h];
            const float g2 = (g < -1e30f ? -1e30f : g) * 1.44269504f, l1 = exp2_of(g2);  // (times 0 steps: 0; NaN stays)
            const int first_seg = REV ? (t.active - 1) / p.per_seg : 0;
            bool has_g = (p.g0 || (t.n > 0 && t.seg != first_seg));
            float G[32 * W], unscale = 1.f;      // fp16: one over the scale of the state's operand,
            float bscale = 1.f;                  // and b's scale, which without EXACT the state has too
            const float grow = F16 ? fmaxf(exp2_of(15.f * g2), 1.f) : 1.f;
            // Chunk k of the item, its tokens, and 1 where the state shall not be decayed past its last token.
            auto chunk_of = [&](int k) { return REV ? t.first + t.n - 1 - k : t.first + k; };
            auto tokens_of = [&](int k) { return (int)min((int64_t)kChunk, t.len - (int64_t)chunk_of(k) * kChunk); };
            auto last_of = [&](int k) { return !REV && p.gout && chunk_of(k) == t.active - 1 ? 1 : 0; };
            // G before chunk k: as an operand (rows of dc columns, in fp16 times a power of two that keeps the largest in
            // range), and decayed over the chunk to where the chunk's products, or their sum, add to it.
            auto put_state = [&](int k) {
                float s = 1.f;
                if constexpr (F16) {
                    float m = 0.f;
#pragma unroll
                    for (int j = 0; j < 32 * W; ++j) m = fmaxf(m, fabsf(G[j]));
                    const uint32_t wm = __reduce_max_sync(0xffffffffu, live ? __float_as_uint(m) : 0u);
                    const int slot = puts++ & 1;
                    if (lane == 0) atomicMax(&gmax[slot], wm);
                    epi_sync(true);
                    s = range_scale(gmax[slot]);
                    if (tid == 0) gmax[slot ^ 1] = 0;
                    unscale = inverse2(s) * (EXACT ? 1.f : inverse2(bscale));
                }
                if (live) {
                    uint8_t* const dst = gop + (W == 2 ? half * kState * 128 : 0) + srow * 128;
#pragma unroll
                    for (int j = 0; j < 4 * W; ++j) {
                        const float* v = &G[8 * j];
                        const int ch = (W == 1 ? half * 4 : 0) + j;
                        const uint4 o = F16 ? make_uint4(pack2<T>(v[0] * s, v[1] * s), pack2<T>(v[2] * s, v[3] * s), pack2<T>(v[4] * s, v[5] * s),
                                                         pack2<T>(v[6] * s, v[7] * s))
                                            : make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
                        sts16(dst + ((ch ^ (srow & 7)) << 4), o);
                    }
                }
                fence_async_smem();
                const float w = pw[tokens_of(k) - last_of(k)];
                const uint64_t w2 = pk2(w, w);
#pragma unroll
                for (int c = 0; c < 2 * W; ++c)
                    if (col0 + 16 * c < p.nb) {
                        float v[16];
#pragma unroll
                        for (int j = 0; j < 16; j += 2) upk2(mul2(pk2(G[16 * c + j], G[16 * c + j + 1]), w2), v[j], v[j + 1]);
                        tmem_st16(tq + kOld + col0 + 16 * c, reinterpret_cast<const uint32_t(&)[16]>(v));
                    }
                tmem_wait_st();
                tc_fence_before();
            };
            epi_sync(true);  // the tables' last readers are done
            if (tid <= kChunk) pw[tid] = power(g, tid);
            // ---- the state before this segment
#pragma unroll
            for (int j = 0; j < 32 * W; ++j) G[j] = 0.f;
            if (has_g && live) {
                if (p.g0 && srow < p.da) {
                    // tokens that come before, and one step more into the chunk's terms
                    const int64_t before = REV ? t.len - min(t.len, (int64_t)(t.first + t.n) * kChunk) : (int64_t)t.first * kChunk;
                    const float w = (t.n > 0 ? power(g, before) * (REV ? 1.f : power(g, 1)) : 1.f) * p.g0_scale;
                    const float* src = p.g0 + (int64_t)t.bh * p.da * p.dc + (int64_t)srow * p.g0_row;
#pragma unroll
                    for (int j = 0; j < 32 * W; ++j)
                        if (col0 + j < p.dc) G[j] = w * src[(int64_t)(col0 + j) * p.g0_col];
                }
                if (t.n > 0 && t.seg != first_seg) {
                    // The sums of the units before this segment (forwards to its start, backwards from the last token), or what
                    // they were joined to.
                    const int here = REV ? t.first + t.n : t.first, mine = REV ? p.units - 1 : 0;
                    const int u0 = p.joined ? t.seg : REV ? t.seg + 1 : 0, u1 = p.joined ? t.seg : REV ? first_seg : t.seg - 1;
                    for (int u = u0; u <= u1; ++u) {
                        const int from = u * p.per_seg, to = min(from + p.per_seg, REV ? t.active : p.chunks);
                        for (int v = p.joined ? mine : 0; p.joined ? v == mine : from + v * p.unit < to; ++v) {
                            const int64_t after = REV ? from + v * p.unit - here : here - min(from + (v + 1) * p.unit, to);
                            const float w = p.joined ? 1.f : power(g, after * kChunk);
                            if (w == 0.f) continue;  // forgotten: not summed either
                            const float* const e = p.ends + (((int64_t)t.bh * p.nseg + u) * p.units + v) * (kState * kState);
                            if (p.turned) {
#pragma unroll
                                for (int j = 0; j < 32 * W; ++j) G[j] = __fmaf_rn(w, e[(col0 + j) * kState + srow], G[j]);
                            } else {
#pragma unroll
                                for (int j = 0; j < 8 * W; ++j) {
                                    const float4 x = reinterpret_cast<const float4*>(e + srow * kState + col0)[j];
                                    G[4 * j] = __fmaf_rn(w, x.x, G[4 * j]), G[4 * j + 1] = __fmaf_rn(w, x.y, G[4 * j + 1]);
                                    G[4 * j + 2] = __fmaf_rn(w, x.z, G[4 * j + 2]), G[4 * j + 3] = __fmaf_rn(w, x.w, G[4 * j + 3]);
                                }
                            }
                        }
                    }
                }
            }
            epi_sync(true);  // the tables are written
            if (t.n > 0) {
                if (has_g) {
                    if (W == 1 && EXACT)  // (the other lanes are 0)
#pragma unroll
                        for (int j = 0; j < 32 * W; ++j) G[j] += __shfl_xor_sync(0xffffffffu, G[j], 16);
                    put_state(0);
                }
                arrive(g_ready);
            }
            // ---- chunks
            for (int k = 0; k < t.n; ++k, ++cc, n += 3) {
                const int chunk = chunk_of(k), L = tokens_of(k), e = last_of(k), nk = n + 1, nv = n + 2;
                // ---- b_j times its power of l, in two parts
                uint8_t *hi = ring + nk % kRing * kTile + kr * 128, *lo = low + kr * 128;
                if (W == 2) hi += kpart * kBlock, lo += kpart * kBlock;
                uint4 x[4];
                int at[4];
                const float wj = kr >= L ? 0.f : REV ? pw[kr + 1] : pw[L - e - kr];
                auto fetch = [&](int j0) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        at[j] = ((W == 1 ? kpart * 4 + j : (j0 + j) ^ (kpart << 2)) ^ (kr & 7)) << 4;
                        x[j] = *reinterpret_cast<const uint4*>(hi + at[j]);
                    }
                };
                ok = wait_for(&full[nk % kRing], nk / kRing & 1) && ok;
                if constexpr (F16) {
                    float m = 0.f;
                    if (W == 2) fetch(4), m = largest16(x);
                    fetch(0), m = fmaxf(m, largest16(x));
                    const uint32_t top = __reduce_max_sync(0xffffffffu, kr < L ? __float_as_uint(m * wj) : 0u);
                    if (lane == 0) tops[warp] = __uint_as_float(top);
                } else {
                    fetch(0);
                }
                ok = wait_for(s_full, cc & 1) && ok;  // the scores are done: b may be overwritten
                if (tid == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                if (!(ok = epi_sync(ok))) break;      // and the last output has left the staging
                tc_fence_after();
                if constexpr (F16) {
                    // b's scale stays while its weighted rows are between 2^5 and 2^15; a state that has it follows a new one.
                    const float top = largest8(tops);
                    if (top > 0.f && !(top * bscale >= 32.f && top * bscale < 32768.f)) {
                        const float s = weight_scale(top, pw[kChunk]);
                        if (!EXACT && has_g && s != bscale) {
                            const float f = s * inverse2(bscale);
                            for (int c = 0; c < 32 * W; c += 16)
                                if (col0 + c < p.nb) {
                                    float v[16];
                                    tmem_ld16(tq + kOld + col0 + c, v);
                                    tmem_wait_ld();
                                    reg_fence(v);
#pragma unroll
                                    for (int j = 0; j < 16; ++j) v[j] *= f;
                                    tmem_st16(tq + kOld + col0 + c, reinterpret_cast<const uint32_t(&)[16]>(v));
                                }
                            tmem_wait_st();
                            tc_fence_before();
                        }
                        bscale = s;
                    }
                }
                const float w = wj * bscale;
                const T w0 = Elem<T>::store(w);
                const uint32_t wh = pack2<T>(w, w), nh = wh ^ 0x80008000u, nl = pack2<T>(Elem<T>::load(w0) - w, Elem<T>::load(w0) - w);
#pragma unroll
                for (int j0 = 0; j0 < 4 * W; j0 += 4) {
                    if (j0 > 0) fetch(j0);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint32_t v[4] = {x[j].x, x[j].y, x[j].z, x[j].w};
                        uint32_t h[4], l[4];
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            // high = b wh rounded; b wh - high is exact (it has no more bits than b); b wl joins with one rounding.
                            // The second part is negated.
                            h[q] = mul16x2<T>(v[q], wh);
                            l[q] = fma16x2<T>(v[q], nl, fma16x2<T>(v[q], nh, h[q]));
                        }
                        sts16(hi + at[j], make_uint4(h[0], h[1], h[2], h[3]));
                        sts16(lo + at[j], make_uint4(l[0], l[1], l[2], l[3]));
                    }
                }
                if (L < kChunk) {  // rows past the sequence: zeros, whatever they hold
                    const uint4 none = make_uint4(0u, 0u, 0u, 0u);
                    if (kr >= L)
                        for (int j = 0; j < 4 * W; ++j) {
                            const int here = ((W == 1 ? kpart * 4 + j : j) ^ (kr & 7)) << 4;  // (what this thread has written)
                            sts16(hi + here, none), sts16(lo + here, none);
                        }
                    ok = wait_for(&full[nv % kRing], nv / kRing & 1) && ok;
                    uint8_t* const tv = ring + nv % kRing * kTile;
                    for (int j = tid; j < (kChunk - L) * 8 * W; j += kEpi) {
                        const int r = L + j / (8 * W), u = j % (8 * W);
                        sts16(tv + (u >> 3) * kBlock + r * 128 + ((u & 7) << 4), none);
                    }
                }
                fence_async_smem();
                arrive(k_ready);
                // ---- weighted scores: row `row`, columns 64 half on, in blocks of 32.  Their factors scale l^(i-j) are made
                // here: loads from a table in shared memory wait for the products' operands, which go first (a block of 32
                // columns took 1100 cycles so, 700 now; 8 heads of 65536 tokens, size 128: 228 -> 217 us; with two blocks
                // per SM, which wait in turn, no difference).
                float unit = p.scale, back = 1.f;
                if constexpr (F16) {
                    // The row's scale: its largest score, each 16 columns weighted as the nearest (for weights above 1: the furthest) of
                    // them, goes to between 2^14 and 2^15; the output's undoes it.  The other half of the row is another warp's.
                    float m = 0.f;
#pragma unroll 1
                    for (int bl = 0; bl < 2; ++bl) {
                        const int blk = half * 2 + bl;
                        if (REV ? blk < quad : blk > quad) continue;
                        float v[32];
                        tmem_ld32(tq + blk * 32, v);
                        tmem_wait_ld();
                        reg_fence(v);
                        if (blk == quad || L < kChunk) {
                            const uint32_t seen = (blk != quad ? 0xffffffffu : REV ? 0xffffffffu << lane : 0xffffffffu >> (31 - lane)) & keep_low(L - blk * 32);
#pragma unroll
                            for (int j = 0; j < 32; ++j)
                                if (!(seen & 1u << j)) v[j] = 0.f;
                        }
                        float near = 0.f, far = 0.f;
#pragma unroll
                        for (int j = 0; j < 16; ++j) near = fmaxf(near, fabsf(v[j])), far = fmaxf(far, fabsf(v[j + 16]));
                        const int d = REV ? blk * 32 - row : row - blk * 32 - 15, d2 = REV ? d + 16 : d - 16;
                        m = fmaxf(m, fmaxf(near * exp2_of((float)max(d, 0) * g2), far * exp2_of((float)max(d2, 0) * g2)));
                    }
                    most[half * kChunk + row] = m * grow;
                    asm volatile("barrier.cta.sync %0, 64;" ::"r"(2 + quad) : "memory");
                    m = fmaxf(most[row], most[kChunk + row]);
                    unit = fminf(range_scale(__float_as_uint(m)), 0x1p40f), back = p.scale * inverse2(unit);
                }
#pragma unroll 1
                for (int bl = 0; bl < 2; ++bl) {
                    const int blk = half * 2 + bl;
                    uint32_t u[16];
                    if (REV ? blk < quad : blk > quad) {
#pragma unroll
                        for (int j = 0; j < 16; ++j) u[j] = 0u;
                    } else {
                        float v[32];
                        tmem_ld32(tq + blk * 32, v);
                        tmem_wait_ld();
                        reg_fence(v);
                        // Two factors at once, of columns 16 apart, from the nearest columns on (so that one which underflows takes
                        // none of a nearer column along): each is l times the last, and `unit` on the diagonal (0 before it).
                        const int d = REV ? blk * 32 - row : row - blk * 32 - 15;  // steps to the first of the two columns
                        const int d2 = REV ? d + 16 : d - 16;
                        const float x0 = exp2_of((float)max(d, 0) * g2) * unit, y0 = exp2_of((float)max(d2, 0) * g2) * unit;
                        uint64_t f = pk2(d >= 0 ? x0 : 0.f, d2 >= 0 ? y0 : 0.f);
                        if (blk == quad) {
#pragma unroll
                            for (int i = 0; i < 16; ++i) {
                                const int j = REV ? i : 15 - i;
                                upk2(mul2(pk2(v[j], v[j + 16]), f), v[j], v[j + 16]);
                                float x, y;
                                upk2(mul2(f, pk2(l1, l1)), x, y);
                                const int next = REV ? j + 1 : j - 1;
                                f = pk2(lane == next ? unit : x, lane == next + 16 ? unit : y);
                            }
                        } else {
#pragma unroll
                            for (int i = 0; i < 16; ++i) {
                                const int j = REV ? i : 15 - i;
                                upk2(mul2(pk2(v[j], v[j + 16]), f), v[j], v[j + 16]);
                                f = mul2(f, pk2(l1, l1));
                            }
                        }
#pragma unroll
                        for (int j = 0; j < 16; ++j) u[j] = pack2<T>(v[2 * j], v[2 * j + 1]);
                        if (L < kChunk) {  // (a product with what lies past the sequence may not be finite)
#pragma unroll
                            for (int j = 0; j < 16; ++j) u[j] &= keep_low(16 * (L - blk * 32) - 32 * j);
                        }
                    }
                    tmem_st16(tq + half * 64 + bl * 16, u);
                }
                if (has_g) {  // what the state gives, times the row's power
                    ok = wait_for(qg_full, qg++ & 1) && ok;
                    tc_fence_after();
                    const int d = REV ? L - 1 - row : row;
                    const float w = (d >= 0 ? pw[d] : 0.f) * unit * unscale;
                    const uint64_t w2 = pk2(w, w);
#pragma unroll
                    for (int c = 0; c < W; ++c) {
                        if (col0 + 32 * c < p.nb) {
                            float v[32];
                            tmem_ld32(tq + kO + col0 + 32 * c, v);
                            tmem_wait_ld();
                            reg_fence(v);
#pragma unroll
                            for (int j = 0; j < 16; ++j) upk2(mul2(pk2(v[2 * j], v[2 * j + 1]), w2), v[2 * j], v[2 * j + 1]);
                            tmem_st32(tq + kO + col0 + 32 * c, v);
                        }
                    }
                }
                tmem_wait_st();
                tc_fence_before();
                arrive(p_ready);
                // ---- the state after this chunk
                ok = wait_for(kv_full, cc & 1) && ok;
                tc_fence_after();
#pragma unroll
                for (int c = 0; c < W; ++c)
                    if (col0 + 32 * c < p.nb) tmem_ld32(tq + kKv + col0 + 32 * c, reinterpret_cast<float(&)[32]>(G[32 * c]));
                tmem_wait_ld();
                reg_fence(G);
                const float un = EXACT ? inverse2(bscale) : 1.f;
                if constexpr (F16 && EXACT && W == 2)
#pragma unroll
                    for (int j = 0; j < 32 * W; ++j) G[j] *= un;
                if constexpr (EXACT) {
                    if constexpr (W == 1) {
#pragma unroll
                        for (int j = 0; j < 32; ++j) {
                            const float x = has_g || lane < 16 ? (F16 && lane < 16 ? G[j] * un : G[j]) : 0.f;
                            G[j] = x + __shfl_xor_sync(0xffffffffu, x, 16);
                        }
                    } else if (has_g) {
#pragma unroll
                        for (int c = 0; c < W; ++c)
                            if (col0 + 32 * c < p.nb) {
                                float v[32];
                                tmem_ld32(tq + kOld + col0 + 32 * c, v);
                                tmem_wait_ld();
                                reg_fence(v);
#pragma unroll
                                for (int j = 0; j < 32; ++j) G[32 * c + j] += v[j];
                            }
                    }
                }
                if (p.nb & 16) {  // the last columns of 32 are nobody's
#pragma unroll
                    for (int j = 16; j < 32 * W; j += 32)
#pragma unroll
                        for (int m = 0; m < 16; ++m)
                            if (col0 + j >= p.nb) G[j + m] = 0.f;
                }
                has_g = true;
                if (k + 1 < t.n) put_state(k + 1);
                // ---- the output
                ok = wait_for(o_full, cc & 1) && ok;
                tc_fence_after();
#pragma unroll
                for (int c = 0; c < W; ++c) {
                    if (col0 + 32 * c < p.nb) {
                        float v[32];
                        tmem_ld32(tq + kO + col0 + 32 * c, v);
                        tmem_wait_ld();
                        reg_fence(v);
                        if constexpr (F16)
#pragma unroll
                            for (int j = 0; j < 32; j += 2) upk2(mul2(pk2(v[j], v[j + 1]), pk2(back, back)), v[j], v[j + 1]);
                        uint8_t* const dst = low + (W == 2 ? half * kBlock : 0) + row * 128;
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const float* x = &v[8 * j];
                            sts16(dst + ((((W == 1 ? half * 4 : 0) + 4 * c + j) ^ (row & 7)) << 4),
                                  make_uint4(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]), pack2<T>(x[4], x[5]), pack2<T>(x[6], x[7])));
                        }
                        if (L < kChunk && row >= L)
#pragma unroll
                            for (int j = 0; j < 4; ++j) sts16(dst + ((((W == 1 ? half * 4 : 0) + 4 * c + j) ^ (row & 7)) << 4), make_uint4(0u, 0u, 0u, 0u));
                    }
                }
                tc_fence_before();
                if (k + 1 < t.n) arrive(g_ready);  // the state operand is written and the output's columns are read
                fence_async_smem();
                if (!(ok = epi_sync(ok))) break;
                if (p.tma_out) {
                    if (tid == 0) {
                        for (int w = 0; w < W; ++w)
                            if (w * 64 < p.dc) store4d(&p.out, low + w * kBlock, w * 64, t.h, chunk * kChunk, t.b);
                        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                    }
                } else {
                    T* const o = (T*)p.o + t.b * p.o_sb + t.h * p.o_sh + (int64_t)chunk * kChunk * p.o_st;
                    const int rows = min(kChunk, p.t - chunk * kChunk);
                    for (int r = warp; r < rows; r += kEpi / 32)
                        for (int c = lane; c < p.dc; c += 32)
                            o[r * p.o_st + c] = *reinterpret_cast<const T*>(low + (c >> 6) * kBlock + r * 128 + ((((c >> 3) & 7) ^ (r & 7)) << 4) + (c & 7) * 2);
                }
            }
            if (!ok) break;
            // ---- rows past the sequence in this segment's whole chunks
            const int end = min(t.first + p.per_seg, p.chunks);
            const int64_t z0 = (int64_t)max(t.first + t.n, t.first) * kChunk, z1 = min((int64_t)end * kChunk, (int64_t)p.t);
            T* const o = (T*)p.o + t.b * p.o_sb + t.h * p.o_sh;
            for (int64_t r = z0 + warp; r < z1; r += kEpi / 32)
                for (int c = lane; c < p.dc; c += 32) o[r * p.o_st + c] = Elem<T>::store(0.f);
            // ---- the state at the end, from the segment that got there (without tokens: as it was)
            const bool mine = t.active == 0 ? t.seg == 0 : REV ? t.seg == 0 : t.n > 0 && t.first + t.n == t.active;
            if (p.gout && mine && live && srow < p.da) {
                float* const dst = p.gout + (int64_t)t.bh * p.da * p.dc + (int64_t)srow * p.dc;
#pragma unroll
                for (int j = 0; j < 32 * W; ++j)
                    if (col0 + j < p.dc) dst[col0 + j] = G[j] * p.gout_scale;
            }
        }
        if (tid == 0 && p.tma_out) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }
    if (!ok) atomicExch(&g_decay_status, (int)LF_ERR_TIMEOUT);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 9) tmem_dealloc(tmem, kCols);
}

// Copies heads that TMA cannot address to [b][t][h][dp], dp a multiple of 8: 16 bytes of output per thread.
struct PackArgs {
    const uint16_t* in;
    uint16_t* out;
    int64_t sb, sh, st, rows;
    int heads, t, d, dp;
};
__global__ void __launch_bounds__(256) pack_heads_kernel(const PackArgs p) {
    grid_release();
    grid_wait();
    const int per = p.dp / 8;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < p.rows * per; i += (int64_t)gridDim.x * 256) {
        const int64_t r = i / per, bt = r / p.heads, b = bt / p.t;
        const int c = (int)(i - r * per) * 8;
        const uint16_t* src = p.in + b * p.sb + (r - bt * p.heads) * p.sh + (bt - b * p.t) * p.st;
        uint16_t v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = c + j < p.d ? src[c + j] : (uint16_t)0;
        *reinterpret_cast<uint4*>(p.out + i * 8) = *reinterpret_cast<const uint4*>(v);
    }
}

// One token: S = l S + k v^T in place, o = sigma q S.  A block per head: the
// threads cover rows of dv columns (VEC each), so the state is read and written
// once, coalesced, and each thread sums q S over the rows it holds; the row
// groups' sums join in order.
struct StepArgs {
    const void *q, *k, *v;
    const float* log_decay;
    float* state;
    void* o;
    int64_t q_sb, q_sh, k_sb, k_sh, v_sb, v_sh;
    int heads, dk, dv, tx;
    float scale;
};
template <typename T, int VEC>
__global__ void __launch_bounds__(256) decay_step_kernel(const StepArgs p) {
    __shared__ float sum[256 * VEC], qk[2][128];
    grid_release();
    grid_wait();
    const int64_t bh = blockIdx.x, b = bh / p.heads, h = bh - b * p.heads;
    const int c = (threadIdx.x % p.tx) * VEC, rg = threadIdx.x / p.tx, groups = 256 / p.tx;
    const T *q = (const T*)p.q + b * p.q_sb + h * p.q_sh, *k = (const T*)p.k + b * p.k_sb + h * p.k_sh;
    const T* v = (const T*)p.v + b * p.v_sb + h * p.v_sh;
    float* S = p.state + bh * p.dk * p.dv + c;
    const bool in = c < p.dv;
    float x[4][VEC], vv[VEC], acc[VEC];
    // The first rows are on their way while the small operands come.
    auto fetch = [&](int r0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = r0 + i * groups;
            if (in && r < p.dk) {
                if constexpr (VEC == 4) *reinterpret_cast<float4*>(x[i]) = *reinterpret_cast<const float4*>(S + r * p.dv);
                else x[i][0] = S[r * p.dv];
            }
        }
    };
    fetch(rg);
    const float l = expf(p.log_decay[h]);
    if (threadIdx.x < p.dk) qk[0][threadIdx.x] = Elem<T>::load(q[threadIdx.x]) * p.scale;
    else if (threadIdx.x >= 128 && threadIdx.x - 128 < p.dk) qk[1][threadIdx.x - 128] = Elem<T>::load(k[threadIdx.x - 128]);
#pragma unroll
    for (int j = 0; j < VEC; ++j) vv[j] = in ? Elem<T>::load(v[c + j]) : 0.f, acc[j] = 0.f;
    __syncthreads();
    for (int r0 = rg; r0 < p.dk; r0 += 4 * groups) {
        if (r0 != rg) fetch(r0);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = r0 + i * groups;
            if (in && r < p.dk) {
                const float kr = qk[1][r], qr = qk[0][r];
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    x[i][j] = __fmaf_rn(x[i][j], l, kr * vv[j]);
                    acc[j] = __fmaf_rn(qr, x[i][j], acc[j]);
                }
                if constexpr (VEC == 4) *reinterpret_cast<float4*>(S + r * p.dv) = *reinterpret_cast<const float4*>(x[i]);
                else S[r * p.dv] = x[i][0];
            }
        }
    }
#pragma unroll
    for (int j = 0; j < VEC; ++j) sum[threadIdx.x * VEC + j] = acc[j];
    __syncthreads();
    if (threadIdx.x < p.dv) {
        float t = 0.f;
        for (int i = 0; i < groups; ++i) t += sum[i * p.tx * VEC + threadIdx.x];
        ((T*)p.o)[bh * p.dv + threadIdx.x] = Elem<T>::store(t);
    }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
// Heads of d elements: strides of sequences, heads and tokens in elements.
struct Heads {
    const void* p;
    int64_t sb, sh, st, d;
};
struct Sizes {
    int64_t b, h, t;
};

bool tma_heads(const Heads& x, const Sizes& z) {
    const int64_t n[3] = {z.b, z.h, z.t}, s[3] = {x.sb, x.sh, x.st};
    if (!aligned(x.p, 16)) return false;
    for (int i = 0; i < 3; ++i)
        if (n[i] > 1 && (s[i] <= 0 || s[i] % 8 != 0 || s[i] >= (int64_t)1 << 38)) return false;
    return true;
}
int64_t padded(int64_t d) { return (d + 7) / 8 * 8; }
size_t packed_bytes(const Heads& x, const Sizes& z) {
    return tma_heads(x, z) ? 0 : (size_t)(z.b * z.h * z.t * padded(x.d) * 2 + 255) / 256 * 256;
}

// x itself, or a copy at `at` (moved on) that TMA can read.
Heads addressable(const Heads& x, const Sizes& z, uint8_t*& at, cudaStream_t st) {
    if (tma_heads(x, z)) return x;
    const int64_t dp = padded(x.d), rows = z.b * z.h * z.t;
    PackArgs a{(const uint16_t*)x.p, (uint16_t*)at, x.sb, x.sh, x.st, rows, (int)z.h, (int)z.t, (int)x.d, (int)dp};
    const int64_t blocks = std::min<int64_t>((rows * (dp / 8) + 255) / 256, (int64_t)num_sms() * 8);
    launch_early(pack_heads_kernel, (unsigned)blocks, 256, 0, 1, st, a);
    Heads y{at, z.t * z.h * dp, dp, z.h * dp, x.d};
    at += packed_bytes(x, z);
    return y;
}

bool encode_heads(CUtensorMap* map, const Heads& x, const Sizes& z, int dtype) {
    const cuuint64_t dims[4] = {(cuuint64_t)x.d, (cuuint64_t)z.h, (cuuint64_t)z.t, (cuuint64_t)z.b};
    const cuuint64_t strides[3] = {(cuuint64_t)(z.h > 1 ? x.sh * 2 : 16), (cuuint64_t)(z.t > 1 ? x.st * 2 : 16),
                                   (cuuint64_t)(z.b > 1 ? x.sb * 2 : 16)};
    const cuuint32_t box[4] = {64, 1, kChunk, 1};
    return encode_tiled(map, dtype == LF_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, x.p, dims,
                        strides, box, CU_TENSOR_MAP_SWIZZLE_128B,
                        x.d > 64 ? CU_TENSOR_MAP_L2_PROMOTION_L2_256B : CU_TENSOR_MAP_L2_PROMOTION_L2_128B);  // (a row, not its neighbours')
}

// Sums before a head's last segment (of 16 KB) from which a launch of their own joins them: at 6 (64 heads of 3136 tokens)
// the three launches of a training step cost more than the segments' own loops, 208 against 200 us; at 136 (8 heads of
// 65536 tokens, size 128) they save, 277 -> 225 us.
constexpr int kJoinFrom = 16;

int blocks_of(int64_t da, int64_t dc) { return da <= 64 && dc <= 64 ? 1 : 2; }

// Segments per sequence, and units of the sums that segments need of those before them.
struct Deal {
    int nseg, per_seg, unit, units;
};
Deal deal(const Sizes& z, int w) {
    const int64_t chunks = (z.t + kChunk - 1) / kChunk, bh = z.b * z.h, slots = (int64_t)num_sms() * (w == 1 ? 2 : 1);
    double least = 1e30;
    int64_t best = 1;
    for (int64_t n = 1; n <= std::min<int64_t>(chunks, 64); ++n) {
        const int64_t per = (chunks + n - 1) / n;
        if ((chunks + per - 1) / per != n) continue;
        // In times of a chunk: rounds of blocks, and a launch that reads b and c of all segments but one.
        const double t = (double)((bh * n + slots - 1) / slots) * (per + 1.0) + (n > 1 ? 0.5 * (double)(bh * (n - 1) * per) / slots + 3.0 : 0.0);
        if (t < least) least = t, best = n;
    }
    Deal d{};
    d.nseg = (int)best, d.per_seg = (int)((chunks + best - 1) / best), d.unit = d.per_seg, d.units = 1;
    if (best > 1) {  // units so short that every slot has work, and not shorter than 4 chunks
        const int64_t want = std::max<int64_t>(1, 2 * slots / (bh * (best - 1)));
        d.unit = (int)std::max<int64_t>(std::min<int64_t>(4, d.per_seg), (d.per_seg + want - 1) / want);
        d.units = (d.per_seg + d.unit - 1) / d.unit;
    }
    return d;
}

size_t ends_bytes(const Sizes& z, int w) {
    const Deal d = deal(z, w);
    return d.nseg > 1 ? (size_t)z.b * z.h * d.nseg * d.units * (64 * w) * (64 * w) * 4 : 0;
}

uint32_t idesc(int dtype, bool a_mn, bool b_mn, int m, int n) {
    const uint32_t f = dtype == LF_BF16 ? 1u : 0u;
    return (1u << 4) | (f << 7) | (f << 10) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) |
           ((uint32_t)(m >> 4) << 24);
}

template <auto Kernel>
void allow_smem(int bytes) {
    static std::once_flag once[64];
    int dev = 0;
    cudaGetDevice(&dev);
    std::call_once(once[dev & 63], [&] { cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes); });
}

template <typename T, int W, bool REV>
void launch_mix(MixArgs a, int64_t bh, cudaStream_t st) {
    const int slots = num_sms() * (W == 1 ? 2 : 1);
    if (a.nseg > 1 && !a.turned) {
        constexpr auto sums = decay_ends_kernel<T, W, REV>;
        allow_smem<sums>(ends_smem<W>());
        a.items = (int)(bh * (a.nseg - 1) * a.units);
        launch_early(sums, (unsigned)std::min(a.items, slots), kThreads, ends_smem<W>(), 1, st, a);
        constexpr auto join = decay_join_kernel<W, REV>;
        if (a.joined) launch_early(join, (unsigned)(bh * (4 * W * W)), 256, 0, 1, st, a);
    }
    a.items = (int)(bh * a.nseg);
    auto mix = [&](auto exact) {
        constexpr auto kernel = decay_mix_kernel<T, W, REV, decltype(exact)::value>;
        allow_smem<kernel>(mix_smem<W>());
        launch_early(kernel, (unsigned)std::min(a.items, slots), kThreads, mix_smem<W>(), 1, st, a);
    };
    a.gout || a.per_seg > kCutChunks ? mix(std::true_type()) : mix(std::false_type());
}

struct Mix {
    Heads a, b, c, out;
    const float *g0 = nullptr;
    float* gout = nullptr;
    bool transposed = false;  // the state matrices are [dc][da]
    bool rev = false;
    bool turned = false;      // a call before has left the sums of c_j b_j^T
};

int run_mix(const Mix& m, const Sizes& z, const float* log_decay, const int64_t* lengths, double scale, int dtype, float* ends,
            cudaStream_t st) {
    const int w = blocks_of(m.a.d, m.c.d);
    MixArgs p{};
    p.log_decay = log_decay, p.lengths = lengths, p.g0 = m.g0, p.gout = m.gout, p.ends = ends;
    p.o = const_cast<void*>(m.out.p), p.o_sb = m.out.sb, p.o_sh = m.out.sh, p.o_st = m.out.st;
    p.heads = (int)z.h, p.t = (int)z.t, p.da = (int)m.a.d, p.dc = (int)m.c.d;
    p.chunks = (int)((z.t + kChunk - 1) / kChunk);
    const Deal d = deal(z, w);
    p.nseg = d.nseg, p.per_seg = d.per_seg, p.unit = d.unit, p.units = d.units;
    p.turned = m.turned;
    p.joined = (d.nseg - 1) * d.units * w * w > kJoinFrom;
    p.g0_row = m.transposed ? 1 : p.dc, p.g0_col = m.transposed ? p.da : 1;
    p.scale = (float)scale, p.g0_scale = m.rev ? (float)(1.0 / scale) : 1.f, p.gout_scale = m.rev ? (float)scale : 1.f;
    p.ksteps = (p.da + 15) / 16, p.nb = (p.dc + 15) / 16 * 16;
    p.id_qk = idesc(dtype, false, false, 128, 128), p.id_qg = idesc(dtype, false, true, 128, p.nb);
    p.id_pv = p.id_qg, p.id_kv = idesc(dtype, true, true, 64 * w, p.nb);
    p.tma_out = tma_heads(m.out, z) ? 1 : 0;
    if (!encode_heads(&p.a, m.a, z, dtype) || !encode_heads(&p.b, m.b, z, dtype) || !encode_heads(&p.c, m.c, z, dtype)) return LF_ERR_CUDA;
    if (p.tma_out && !encode_heads(&p.out, m.out, z, dtype)) return LF_ERR_CUDA;
    const int64_t bh = z.b * z.h;
#define LFB_MIX(T, W) (m.rev ? launch_mix<T, W, true>(p, bh, st) : launch_mix<T, W, false>(p, bh, st))
    if (dtype == LF_F16) {
        if (w == 1) LFB_MIX(__half, 1);
        else LFB_MIX(__half, 2);
    } else {
        if (w == 1) LFB_MIX(__nv_bfloat16, 1);
        else LFB_MIX(__nv_bfloat16, 2);
    }
#undef LFB_MIX
    return check_launch("decay_attention");
}

int refuse(const char* what, const char* why) {
    set_error("%s: %s", what, why);
    return LF_ERR_INVALID;
}

int check_sizes(const char* what, int64_t b, int64_t h, int64_t t, int64_t dk, int64_t dv) {
    if (b < 0 || h < 0 || t < 0 || dk < 1 || dv < 1) return refuse(what, "bad sizes");
    if (dk > 128 || dv > 128) {
        set_error("%s: head sizes up to 128 are supported, got %lld and %lld", what, (long long)dk, (long long)dv);
        return LF_ERR_UNSUPPORTED;
    }
    // Work units and token numbers are 32-bit.
    if (t > INT32_MAX - kChunk || (b > 0 && h > INT32_MAX / 64 / b)) {
        set_error("%s: b*h up to 2^25 and t up to 2^31 - 129 are supported", what);
        return LF_ERR_UNSUPPORTED;
    }
    return LF_OK;
}

int check_attention(const char* what, const lf_decay_attention_t* a, bool bwd) {
    if (!a) return refuse(what, "no arguments");
    if (a->dtype != LF_F16 && a->dtype != LF_BF16) {
        set_error("%s: unsupported dtype code %d (fp16 and bf16)", what, a->dtype);
        return LF_ERR_DTYPE;
    }
    if (int rc = check_sizes(what, a->b, a->h, a->t, a->key_size, a->value_size)) return rc;
    if (!(a->scale > 0) || !(a->scale < 1e30) || a->scale < 1e-30) return refuse(what, "scale must be between 1e-30 and 1e30");
    for (const void* p : {(const void*)a->q, (const void*)a->k, (const void*)a->v, (const void*)a->o, a->d_o, (const void*)a->dq,
                          (const void*)a->dk, (const void*)a->dv})
        if (!aligned(p, 2)) return refuse(what, "a pointer is not aligned to its elements");
    for (const void* p : {(const void*)a->log_decay, (const void*)a->state, (const void*)a->state_out, (const void*)a->d_state_out,
                          (const void*)a->d_state})
        if (!aligned(p, 4)) return refuse(what, "a pointer is not aligned to its elements");
    if (!aligned(a->lengths, 8)) return refuse(what, "a pointer is not aligned to its elements");
    if (!aligned(a->sums, 256)) return refuse(what, "sums must be 256-byte aligned");
    if (a->b == 0 || a->h == 0) return LF_OK;
    const uintptr_t n = (uintptr_t)(a->b * a->h * a->key_size * a->value_size) * 4;
    for (const auto& x : {std::make_pair(a->state, a->state_out), std::make_pair(a->d_state_out, a->d_state)}) {
        const uintptr_t from = (uintptr_t)x.first, to = (uintptr_t)x.second;
        if (from && to && from != to && from < to + n && to < from + n) return refuse(what, "a state and the one that is written overlap without being the same");
    }
    if (!a->log_decay) return refuse(what, "log_decay is required");
    if (a->t > 0 && (!a->q || !a->k || !a->v || (!bwd && !a->o) || (bwd && !a->d_o))) return refuse(what, "q, k, v and the output or its gradient are required");
    if (bwd && a->t > 0 && a->d_state && !a->dv) return refuse(what, "the state's gradient comes with dv");
    return LF_OK;
}

// A state updated in place where a sequence is cut: several blocks read what one of them writes, so they read a copy.
size_t state_bytes(const lf_decay_attention_t* a) { return (size_t)(a->b * a->h * a->key_size * a->value_size) * 4; }
size_t copy_bytes(const lf_decay_attention_t* a, const float* from, const float* to) {
    return from && from == to && deal({a->b, a->h, a->t}, blocks_of(a->key_size, a->value_size)).nseg > 1 ? (state_bytes(a) + 255) / 256 * 256 : 0;
}
// `from`, or its copy at `at` (moved on).
const float* read_apart(const lf_decay_attention_t* a, const float* from, const float* to, uint8_t*& at, cudaStream_t st) {
    const size_t n = copy_bytes(a, from, to);
    if (n == 0) return from;
    cudaMemcpyAsync(at, from, state_bytes(a), cudaMemcpyDeviceToDevice, st);
    const float* const copy = (const float*)at;
    at += n;
    return copy;
}

Heads heads_of(const void* p, const int64_t* s, int64_t d) { return {p, s[0], s[1], s[2], d}; }
Heads dense_heads(void* p, const Sizes& z, int64_t d) { return {p, z.t * z.h * d, d, z.h * d, d}; }

// T = 0: the state passes through.
int pass_state(const char* what, const float* from, float* to, size_t bytes, cudaStream_t st) {
    if (to && to != from && (from ? cudaMemcpyAsync(to, from, bytes, cudaMemcpyDeviceToDevice, st) : cudaMemsetAsync(to, 0, bytes, st)) != cudaSuccess)
        return check_launch(what);
    return LF_OK;
}

}  // namespace
}  // namespace lfb

using namespace lfb;

extern "C" size_t lf_decay_attention_sums_size(const lf_decay_attention_t* a) {
    if (!a || check_sizes("lf_decay_attention_sums_size", a->b, a->h, a->t, a->key_size, a->value_size) || a->b == 0 || a->h == 0 || a->t == 0) return 0;
    return ends_bytes({a->b, a->h, a->t}, blocks_of(a->key_size, a->value_size));
}

extern "C" size_t lf_decay_attention_fwd_workspace_size(const lf_decay_attention_t* a) {
    if (!a || check_attention("lf_decay_attention_fwd", a, false) || a->b == 0 || a->h == 0 || a->t == 0) return 0;
    const Sizes z{a->b, a->h, a->t};
    return packed_bytes(heads_of(a->q, a->q_strides, a->key_size), z) + packed_bytes(heads_of(a->k, a->k_strides, a->key_size), z) +
           packed_bytes(heads_of(a->v, a->v_strides, a->value_size), z) + copy_bytes(a, a->state, a->state_out) +
           (a->sums ? 0 : ends_bytes(z, blocks_of(a->key_size, a->value_size)));
}

extern "C" int lf_decay_attention_fwd(const lf_decay_attention_t* a, void* workspace, size_t workspace_bytes, lf_stream_t stream) {
    clear_error();
    const char* what = "lf_decay_attention_fwd";
    if (int rc = check_attention(what, a, false)) return rc;
    cudaStream_t st = (cudaStream_t)stream;
    if (a->b == 0 || a->h == 0) return LF_OK;
    if (a->t == 0) return pass_state(what, a->state, a->state_out, state_bytes(a), st);
    const size_t need = lf_decay_attention_fwd_workspace_size(a);
    if (need && (!workspace || !aligned(workspace, 256) || workspace_bytes < need)) {
        set_error("%s: needs %zu bytes of 256-byte aligned workspace, got %zu", what, need, workspace ? workspace_bytes : (size_t)0);
        return LF_ERR_INVALID;
    }
    const Sizes z{a->b, a->h, a->t};
    uint8_t* at = (uint8_t*)workspace;
    Mix m;
    m.a = addressable(heads_of(a->q, a->q_strides, a->key_size), z, at, st);
    m.b = addressable(heads_of(a->k, a->k_strides, a->key_size), z, at, st);
    m.c = addressable(heads_of(a->v, a->v_strides, a->value_size), z, at, st);
    m.out = dense_heads(a->o, z, a->value_size);
    m.g0 = read_apart(a, a->state, a->state_out, at, st), m.gout = a->state_out;
    return run_mix(m, z, a->log_decay, a->lengths, a->scale, a->dtype, a->sums ? a->sums : (float*)at, st);
}

extern "C" size_t lf_decay_attention_bwd_workspace_size(const lf_decay_attention_t* a) {
    if (!a || check_attention("lf_decay_attention_bwd", a, true) || a->b == 0 || a->h == 0 || a->t == 0) return 0;
    const Sizes z{a->b, a->h, a->t};
    return packed_bytes(heads_of(a->q, a->q_strides, a->key_size), z) + packed_bytes(heads_of(a->k, a->k_strides, a->key_size), z) +
           packed_bytes(heads_of(a->v, a->v_strides, a->value_size), z) + packed_bytes(heads_of(a->d_o, a->do_strides, a->value_size), z) +
           copy_bytes(a, a->d_state_out, a->d_state) + ends_bytes(z, blocks_of(a->key_size, a->value_size));
}

extern "C" int lf_decay_attention_bwd(const lf_decay_attention_t* a, void* workspace, size_t workspace_bytes, lf_stream_t stream) {
    clear_error();
    const char* what = "lf_decay_attention_bwd";
    if (int rc = check_attention(what, a, true)) return rc;
    cudaStream_t st = (cudaStream_t)stream;
    if (a->b == 0 || a->h == 0) return LF_OK;
    if (a->t == 0) return pass_state(what, a->d_state_out, a->d_state, state_bytes(a), st);
    const size_t need = lf_decay_attention_bwd_workspace_size(a);
    if (need && (!workspace || !aligned(workspace, 256) || workspace_bytes < need)) {
        set_error("%s: needs %zu bytes of 256-byte aligned workspace, got %zu", what, need, workspace ? workspace_bytes : (size_t)0);
        return LF_ERR_INVALID;
    }
    const Sizes z{a->b, a->h, a->t};
    uint8_t* at = (uint8_t*)workspace;
    const Heads q = addressable(heads_of(a->q, a->q_strides, a->key_size), z, at, st);
    const Heads k = addressable(heads_of(a->k, a->k_strides, a->key_size), z, at, st);
    const Heads v = addressable(heads_of(a->v, a->v_strides, a->value_size), z, at, st);
    const Heads g = addressable(heads_of(a->d_o, a->do_strides, a->value_size), z, at, st);
    const float* const d_state_out = read_apart(a, a->d_state_out, a->d_state, at, st);
    auto mix = [&](const Heads& x, const Heads& y, const Heads& w, void* out, const float* g0, float* gout, bool transposed, bool rev,
                   bool turned) {
        Mix m;
        m.a = x, m.b = y, m.c = w, m.out = dense_heads(out, z, w.d), m.g0 = g0, m.gout = gout, m.transposed = transposed, m.rev = rev, m.turned = turned;
        return run_mix(m, z, a->log_decay, a->lengths, a->scale, a->dtype, turned && !rev ? a->sums : (float*)at, st);
    };
    // The segments' sums for dq are the forward's, those for dv are dk's, transposed.
    if (a->dq)
        if (int rc = mix(g, v, k, a->dq, a->state, nullptr, true, false, a->sums != nullptr)) return rc;
    if (a->dk)
        if (int rc = mix(v, g, q, a->dk, d_state_out, nullptr, true, true, false)) return rc;
    if (a->dv)
        if (int rc = mix(k, q, g, a->dv, d_state_out, a->d_state, false, true, a->dk != nullptr)) return rc;
    return LF_OK;
}

extern "C" int lf_decay_attention_step(const lf_decay_step_t* a, lf_stream_t stream) {
    clear_error();
    const char* what = "lf_decay_attention_step";
    if (!a) return refuse(what, "no arguments");
    if (a->dtype != LF_F32 && a->dtype != LF_F16 && a->dtype != LF_BF16) {
        set_error("%s: unsupported dtype code %d (fp32, fp16 and bf16)", what, a->dtype);
        return LF_ERR_DTYPE;
    }
    if (int rc = check_sizes(what, a->b, a->h, 1, a->key_size, a->value_size)) return rc;
    if (!(a->scale > 0) || !(a->scale < 1e30) || a->scale < 1e-30) return refuse(what, "scale must be between 1e-30 and 1e30");
    if (a->b == 0 || a->h == 0) return LF_OK;
    if (!a->q || !a->k || !a->v || !a->o || !a->state || !a->log_decay) return refuse(what, "every operand is required");
    for (const void* p : {a->q, a->k, a->v, (const void*)a->o})
        if (!aligned(p, dtype_size(a->dtype))) return refuse(what, "a pointer is not aligned to its elements");
    for (const void* p : {(const void*)a->state, (const void*)a->log_decay})
        if (!aligned(p, 4)) return refuse(what, "a pointer is not aligned to its elements");
    const bool vec = a->value_size % 4 == 0 && aligned(a->state, 16);
    StepArgs p{a->q, a->k, a->v, a->log_decay, a->state, a->o, a->q_strides[0], a->q_strides[1], a->k_strides[0], a->k_strides[1],
               a->v_strides[0], a->v_strides[1], (int)a->h, (int)a->key_size, (int)a->value_size, 1, (float)a->scale};
    while (p.tx * (vec ? 4 : 1) < p.dv) p.tx *= 2;
    const unsigned grid = (unsigned)(a->b * a->h);
    cudaStream_t st = (cudaStream_t)stream;
#define LFB_STEP(T) (vec ? launch_early(decay_step_kernel<T, 4>, grid, 256, 0, 1, st, p) : launch_early(decay_step_kernel<T, 1>, grid, 256, 0, 1, st, p))
    if (a->dtype == LF_F32) LFB_STEP(float);
    else if (a->dtype == LF_F16) LFB_STEP(__half);
    else LFB_STEP(__nv_bfloat16);
#undef LFB_STEP
    return check_launch(what);
}
