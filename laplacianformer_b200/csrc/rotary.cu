// Rotary positions: each pair (x, y) of a head turns by angle = position * frequency,
//   x' = m (x cos - y sin),   y' = m (x sin + y cos),
// pairs being the two halves of the first 2 P channels or neighbours; the rest
// of the head is copied.  The backward turns by the opposite angle.
//
// Memory bound: queries and keys are read and written once, in one launch.  A
// block takes a few tokens with all their heads, so that an angle is computed
// once for all of them: in turns, position * (frequency / 2 pi).  The factor is
// held in two parts and a far product's rounding error is added to its
// fraction, so that the fraction is exact to fp32 at any position that 53 bits
// hold (a 64-bit product alone is 2^-52 of the angle off: 5e-6 radians at 2^35,
// where all digits are gone at 2^53); then the sine and cosine of the fraction
// in 32 bits.
//
// Measured, bf16, queries and keys of 8x16x16384x64: 215 us a pass, 5.0 TB/s
// (the copies of the next two tiles are in flight while one is turned; with
// loads when a tile's turn came 330 us).
#include <math.h>

#include <algorithm>
#include <mutex>

#include "lf_common.cuh"

namespace lfb {
namespace {

constexpr int kPairs = 128;      // pairs that a head may have
constexpr int kAngles = 512;     // sines and cosines of a tile
constexpr int kUnits = 4;        // units of a thread in a tile

struct RotaryArgs {
    const void* x[2];
    void* y[2];
    int64_t sb[2], sh[2], st[2];
    const int64_t* positions;
    int64_t position_stride, offset, tokens;   // tokens of all sequences
    double turns[kPairs], rest[kPairs];        // frequency / 2 pi in two parts
    Divisor per_token, per_head, per_pair, per_t;  // units of a token, of a head; pairs; tokens of a sequence
    int heads[2], t, size, pairs, rotated, per_block;
    float magnitude, sign;
};

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Vec {
    T v[VEC];
};
template <typename T, int VEC>
constexpr int rotary_stages() {
    return sizeof(T) * VEC == 16 ? 3 : 0;
}
__device__ __forceinline__ void copy16(void* dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(dst))), "l"(src) : "memory");
}

// A unit is VEC pairs (HALVES), VEC/2 pairs (neighbours; one pair when VEC is 1), or VEC copied elements.  A block walks
// over tiles of `per_block` tokens, up to kUnits units to a thread.  With vectors of 16 bytes the units of the next tiles
// are on their way to places of each thread's own in shared memory while one is turned.
template <typename T, int VEC, bool HALVES>
__global__ void __launch_bounds__(256) rotary_kernel(const __grid_constant__ RotaryArgs p) {
    constexpr int PAIRS = HALVES ? VEC : VEC == 1 ? 1 : VEC / 2;   // of a unit
    constexpr bool TWO = HALVES || VEC == 1;                       // a unit's pairs lie in two places
    constexpr int S = rotary_stages<T, VEC>();
    using V = Vec<T, VEC>;
    extern __shared__ __align__(16) uint8_t staged[];              // [stage][unit][place][thread]
    __shared__ __align__(16) float2 table[2][kAngles];             // cosine and sine of a tile's tokens, by turns
    grid_release();
    grid_wait();
    const int tiles = (int)((p.tokens + p.per_block - 1) / p.per_block);
    // Unit u of the tile that starts at token tok0: its elements, how much further the second place is (0: none), its
    // first angle (-1: copied).
    struct Unit {
        const T* src;
        T* dst;
        int off, pair;
    };
    auto unit_of = [&](int tok0, int u) {
        Unit x;
        const int tok = p.per_token.of(u), r = u - tok * (int)p.per_token.d;
        int h = p.per_head.of(r);
        const int e = r - h * (int)p.per_head.d;
        const int which = h >= p.heads[0] ? 1 : 0;
        if (which) h -= p.heads[0];
        const int n = tok0 + tok, s = p.per_t.of(n), t = n - s * p.t;
        int c;
        if (e < p.rotated) {
            x.pair = tok * p.pairs + e * PAIRS;
            c = HALVES ? e * VEC : e * PAIRS * 2;
            x.off = HALVES ? p.pairs : VEC == 1 ? 1 : 0;
        } else {
            x.pair = -1;
            c = 2 * p.pairs + (e - p.rotated) * VEC;
            x.off = 0;
        }
        x.src = (const T*)p.x[which] + s * p.sb[which] + h * p.sh[which] + t * p.st[which] + c;
        x.dst = (T*)p.y[which] + ((int64_t)n * p.heads[which] + h) * p.size + c;
        return x;
    };
    auto units_in = [&](int tok0) { return min(p.per_block, (int)(p.tokens - tok0)) * (int)p.per_token.d; };
    auto place = [&](int stage, int i, int j) { return staged + (((stage * kUnits + i) * 2 + j) * 256 + threadIdx.x) * 16; };
    auto fetch = [&](int64_t tile, int stage) {
        if (tile < tiles) {
            const int tok0 = (int)tile * p.per_block, units = units_in(tok0);
#pragma unroll
            for (int i = 0; i < kUnits; ++i) {
                const int u = threadIdx.x + i * 256;
                if (u >= units) break;
                const Unit x = unit_of(tok0, u);
                copy16(place(stage, i, 0), x.src);
                if (TWO && x.off) copy16(place(stage, i, 1), x.src + x.off);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    if constexpr (S > 0) {
#pragma unroll
        for (int k = 0; k + 1 < S; ++k) fetch((int64_t)blockIdx.x + (int64_t)k * gridDim.x, k);
    }
    int stage = 0, turn = 0;
    for (int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x, turn ^= 1) {
        const int tok0 = (int)tile * p.per_block, units = units_in(tok0), toks = min(p.per_block, (int)(p.tokens - tok0));
        float2* const cs = table[turn];
        for (int i = threadIdx.x; i < toks * p.pairs; i += 256) {
            const int tok = p.per_pair.of(i), k = i - tok * p.pairs;
            const int n = tok0 + tok, s = p.per_t.of(n), t = n - s * p.t;
            const int64_t pos = p.positions ? p.positions[(int64_t)s * p.position_stride + t] : p.offset + t;
            const double at = (double)pos, whole = at * p.turns[k];
            double turns = whole - rint(whole);
            if (fabs(whole) > 0x1p24) {  // (nearer the product's error is below 2^-29 of a turn)
                turns += fma(at, p.rest[k], fma(at, p.turns[k], -whole));  // far out up to half a turn
                turns -= rint(turns);
            }
            float sn, c;
            sincospif(2.f * (float)turns, &sn, &c);
            cs[i] = make_float2(c * p.magnitude, sn * p.magnitude * p.sign);
        }
        if constexpr (S > 0) {
            fetch(tile + (int64_t)(S - 1) * gridDim.x, stage == 0 ? S - 1 : stage - 1);
            asm volatile("cp.async.wait_group %0;" ::"n"(S > 0 ? S - 1 : 0) : "memory");
        }
        __syncthreads();  // the angles are there; whoever still reads the last tile's has the other table
        for (int i0 = 0; i0 * 256 < units; i0 += kUnits) {
#pragma unroll
            for (int i = 0; i < kUnits; ++i) {
                const int u = threadIdx.x + (i0 + i) * 256;
                if (u >= units) break;
                const Unit x = unit_of(tok0, u);
                V a, b;
                if constexpr (S > 0) {
                    a = *reinterpret_cast<const V*>(place(stage, i, 0));
                    if (TWO && x.off) b = *reinterpret_cast<const V*>(place(stage, i, 1));
                } else {
                    a = *reinterpret_cast<const V*>(x.src);
                    if (TWO && x.off) b = *reinterpret_cast<const V*>(x.src + x.off);
                }
                if (x.pair >= 0) {
                    const float2* f = cs + x.pair;
                    if constexpr (TWO) {
#pragma unroll
                        for (int j = 0; j < VEC; ++j) {
                            const float p0 = Elem<T>::load(a.v[j]), p1 = Elem<T>::load(b.v[j]);
                            a.v[j] = Elem<T>::store(p0 * f[j].x - p1 * f[j].y);
                            b.v[j] = Elem<T>::store(p0 * f[j].y + p1 * f[j].x);
                        }
                    } else {
#pragma unroll
                        for (int j = 0; j < VEC / 2; ++j) {
                            const float p0 = Elem<T>::load(a.v[2 * j]), p1 = Elem<T>::load(a.v[2 * j + 1]);
                            a.v[2 * j] = Elem<T>::store(p0 * f[j].x - p1 * f[j].y);
                            a.v[2 * j + 1] = Elem<T>::store(p0 * f[j].y + p1 * f[j].x);
                        }
                    }
                }
                *reinterpret_cast<V*>(x.dst) = a;
                if (TWO && x.off) *reinterpret_cast<V*>(x.dst + x.off) = b;
            }
        }
        if constexpr (S > 0) stage = stage + 1 == S ? 0 : stage + 1;
    }
}

template <typename T, int VEC, bool HALVES>
void launch_tiles(const RotaryArgs& p, int64_t tiles, cudaStream_t st) {
    constexpr auto kernel = rotary_kernel<T, VEC, HALVES>;
    constexpr int smem = rotary_stages<T, VEC>() * kUnits * 2 * 256 * 16;
    static std::once_flag once[64];
    static int per_sm[64];
    int dev = 0;
    cudaGetDevice(&dev);
    dev &= 63;
    std::call_once(once[dev], [&] {
        int v = 0;
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&v, kernel, 256, smem) != cudaSuccess || v < 1) v = 1;
        per_sm[dev] = v;
    });
    launch_early(kernel, (unsigned)std::min<int64_t>(tiles, (int64_t)per_sm[dev] * num_sms()), 256, smem, 1, st, p);
}

template <typename T, bool HALVES>
void launch_rotary(RotaryArgs& p, bool vec, cudaStream_t st) {
    constexpr int V = 16 / sizeof(T);
    const int v = vec ? V : 1, pairs = HALVES ? v : vec ? v / 2 : 1;
    p.rotated = p.pairs / pairs;
    const int per_head = p.rotated + (p.size - 2 * p.pairs) / v;
    p.per_head = Divisor(per_head), p.per_token = Divisor(per_head * (p.heads[0] + p.heads[1])), p.per_pair = Divisor(std::max(1, p.pairs)), p.per_t = Divisor(p.t);
    // With vectors a tile is what the stages hold; otherwise as many tokens as there is room for angles of, up to 16 units a thread.
    const int most = (vec ? 1 : 4) * kUnits * 256;
    p.per_block = std::max(1, std::min(kAngles / std::max(1, p.pairs), most / (int)p.per_token.d));
    const int64_t tiles = (p.tokens + p.per_block - 1) / p.per_block;
    if (vec && (int)p.per_token.d <= kUnits * 256) launch_tiles<T, V, HALVES>(p, tiles, st);
    else if (vec) {  // a token of more units than a tile has places for: by single elements
        launch_rotary<T, HALVES>(p, false, st);
    } else launch_tiles<T, 1, HALVES>(p, tiles, st);
}

}  // namespace
}  // namespace lfb

using namespace lfb;

extern "C" int lf_rotary(const lf_rotary_t* a, lf_stream_t stream) {
    clear_error();
    auto refuse = [](const char* why) {
        set_error("lf_rotary: %s", why);
        return LF_ERR_INVALID;
    };
    if (!a) return refuse("no arguments");
    if (a->dtype != LF_F32 && a->dtype != LF_F16 && a->dtype != LF_BF16) {
        set_error("lf_rotary: unsupported dtype code %d (fp32, fp16 and bf16)", a->dtype);
        return LF_ERR_DTYPE;
    }
    const int64_t heads = a->heads[0] + a->heads[1];
    if (a->b < 0 || a->t < 0 || a->heads[0] < 0 || a->heads[1] < 0 || a->size < 0 || a->pairs < 0 || 2 * a->pairs > a->size) return refuse("bad sizes");
    if (a->b == 0 || a->t == 0 || heads == 0 || a->size == 0) return LF_OK;
    // A token's units are counted in 22 bits, blocks in 31.
    if (a->pairs > kPairs || a->size > 65536 || heads > 65536 || heads * a->size > 1 << 22 || a->t > INT32_MAX || a->b > INT32_MAX / a->t) {
        set_error("lf_rotary: up to %d pairs, 2^22 elements of a token and 2^31 - 1 tokens are supported", kPairs);
        return LF_ERR_UNSUPPORTED;
    }
    if (a->pairs > 0 && !a->frequencies) return refuse("frequencies are required");
    const int es = (int)dtype_size(a->dtype), v = 16 / es;
    bool vec = a->size % v == 0 && (2 * a->pairs) % v == 0 && (a->interleaved || a->pairs % v == 0);
    RotaryArgs p{};
    for (int i = 0; i < 2; ++i) {
        if (a->heads[i] == 0) continue;
        if (!a->x[i] || !a->y[i]) return refuse("an operand or its output is missing");
        if (!aligned(a->x[i], es) || !aligned(a->y[i], es)) return refuse("a pointer is not aligned to its elements");
        p.x[i] = a->x[i], p.y[i] = a->y[i], p.heads[i] = (int)a->heads[i];
        p.sb[i] = a->strides[i][0], p.sh[i] = a->strides[i][1], p.st[i] = a->strides[i][2];
        vec = vec && aligned(a->x[i], 16) && aligned(a->y[i], 16) && (a->b == 1 || p.sb[i] % v == 0) && (a->heads[i] == 1 || p.sh[i] % v == 0) &&
              (a->t == 1 || p.st[i] % v == 0);
    }
    if (!aligned(a->positions, 8)) return refuse("a pointer is not aligned to its elements");
    p.positions = a->positions, p.position_stride = a->position_stride, p.offset = a->offset, p.tokens = a->b * a->t;
    for (int64_t k = 0; k < a->pairs; ++k) {
        const double f = a->frequencies[k], head = 0.15915494309189535, tail = -9.839338337591243e-18;  // 1 / 2 pi
        p.turns[k] = f * head;
        p.rest[k] = fma(f, tail, fma(f, head, -p.turns[k]));
    }
    p.t = (int)a->t, p.size = (int)a->size, p.pairs = (int)a->pairs;
    p.magnitude = (float)a->magnitude, p.sign = a->inverse ? -1.f : 1.f;
    cudaStream_t st = (cudaStream_t)stream;
#define LFB_ROTARY(T) (a->interleaved ? launch_rotary<T, false>(p, vec, st) : launch_rotary<T, true>(p, vec, st))
    if (a->dtype == LF_F32) LFB_ROTARY(float);
    else if (a->dtype == LF_F16) LFB_ROTARY(__half);
    else LFB_ROTARY(__nv_bfloat16);
#undef LFB_ROTARY
    return check_launch("lf_rotary");
}
