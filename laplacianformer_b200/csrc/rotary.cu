// Rotary positions: each pair (x, y) of a head turns by angle = position * frequency,
//   x' = m (x cos - y sin),   y' = m (x sin + y cos),
// pairs being the two halves of the first 2 P channels or neighbours; the rest
// of the head is copied.  The backward turns by the opposite angle.
//
// Memory bound: queries and keys are read and written once, in one launch.  A
// block takes a few tokens with all their heads, so that an angle is computed
// once for all of them: in turns, position * (frequency / 2 pi) in 64 bits,
// whose fraction is exact enough at any position that fits 2^53 (a 32-bit
// product at position 10^6 is off by up to 0.06 radians), then the sine and
// cosine of the fraction in 32 bits.
#include <algorithm>

#include "lf_common.cuh"

namespace lfb {
namespace {

constexpr int kPairs = 128;      // pairs that a head may have
constexpr int kAngles = 2048;    // sines and cosines that a block holds
constexpr int kUnits = 4;        // units of a thread in flight

struct RotaryArgs {
    const void* x[2];
    void* y[2];
    int64_t sb[2], sh[2], st[2];
    const int64_t* positions;
    int64_t position_stride, offset, tokens;   // tokens of all sequences
    double turns[kPairs];                      // frequency / 2 pi
    Divisor per_token, per_head, per_pair;     // units of a token, of a head; pairs
    int heads[2], t, size, pairs, rotated, per_block;
    float magnitude, sign;
};

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Vec {
    T v[VEC];
};

// A unit is VEC pairs (HALVES), VEC/2 pairs (neighbours; one pair when VEC is 1), or VEC copied elements.
template <typename T, int VEC, bool HALVES>
__global__ void __launch_bounds__(256) rotary_kernel(const __grid_constant__ RotaryArgs p) {
    constexpr int PAIRS = HALVES ? VEC : VEC == 1 ? 1 : VEC / 2;   // of a unit
    constexpr bool TWO = HALVES || VEC == 1;                       // a unit's pairs lie in two places
    __shared__ float2 cs[kAngles];
    grid_release();
    grid_wait();
    const int64_t tok0 = (int64_t)blockIdx.x * p.per_block;
    const int toks = (int)min((int64_t)p.per_block, p.tokens - tok0), units = toks * (int)p.per_token.d;
    const int turning = p.rotated;                                 // units of a head that turn; the others are copied
    Vec<T, VEC> a[kUnits], b[kUnits];
    int off[kUnits], pair[kUnits];
    T* dst[kUnits];
    // Where the unit's elements are: its (first) place, how much further the second is (0: none), and its first angle (-1: copied).
    auto fetch = [&](int i0) {
#pragma unroll
        for (int i = 0; i < kUnits; ++i) {
            const int u = i0 + i * 256;
            off[i] = -1;
            if (u >= units) continue;
            const int tok = p.per_token.of(u), r = u - tok * (int)p.per_token.d;
            int h = p.per_head.of(r);
            const int e = r - h * (int)p.per_head.d;
            const int which = h >= p.heads[0] ? 1 : 0;
            if (which) h -= p.heads[0];
            const int64_t n = tok0 + tok, s = n / p.t, t = n - s * p.t;
            int c;
            if (e < turning) {
                pair[i] = tok * p.pairs + e * PAIRS;
                c = HALVES ? e * VEC : e * PAIRS * 2;
                off[i] = HALVES ? p.pairs : VEC == 1 ? 1 : 0;
            } else {
                pair[i] = -1;
                c = 2 * p.pairs + (e - turning) * VEC;
                off[i] = 0;
            }
            const T* src = (const T*)p.x[which] + s * p.sb[which] + h * p.sh[which] + t * p.st[which] + c;
            dst[i] = (T*)p.y[which] + (n * p.heads[which] + h) * p.size + c;
            a[i] = *reinterpret_cast<const Vec<T, VEC>*>(src);
            if (TWO && off[i]) b[i] = *reinterpret_cast<const Vec<T, VEC>*>(src + off[i]);
        }
    };
    fetch(threadIdx.x);  // on their way while the angles are computed
    for (int i = threadIdx.x; i < toks * p.pairs; i += 256) {
        const int tok = p.per_pair.of(i), k = i - tok * p.pairs;
        const int64_t n = tok0 + tok, s = n / p.t, t = n - s * p.t;
        const int64_t pos = p.positions ? p.positions[s * p.position_stride + t] : p.offset + t;
        double turn = (double)pos * p.turns[k];
        turn -= rint(turn);
        float sn, c;
        sincospif(2.f * (float)turn, &sn, &c);
        cs[i] = make_float2(c * p.magnitude, sn * p.magnitude * p.sign);
    }
    __syncthreads();
    for (int i0 = threadIdx.x; i0 < units; i0 += kUnits * 256) {
        if (i0 != threadIdx.x) fetch(i0);
#pragma unroll
        for (int i = 0; i < kUnits; ++i) {
            if (off[i] < 0) continue;
            if (pair[i] >= 0) {
                const float2* f = cs + pair[i];
                if constexpr (TWO) {
#pragma unroll
                    for (int j = 0; j < VEC; ++j) {
                        const float x = Elem<T>::load(a[i].v[j]), y = Elem<T>::load(b[i].v[j]);
                        a[i].v[j] = Elem<T>::store(x * f[j].x - y * f[j].y);
                        b[i].v[j] = Elem<T>::store(x * f[j].y + y * f[j].x);
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < VEC / 2; ++j) {
                        const float x = Elem<T>::load(a[i].v[2 * j]), y = Elem<T>::load(a[i].v[2 * j + 1]);
                        a[i].v[2 * j] = Elem<T>::store(x * f[j].x - y * f[j].y);
                        a[i].v[2 * j + 1] = Elem<T>::store(x * f[j].y + y * f[j].x);
                    }
                }
            }
            *reinterpret_cast<Vec<T, VEC>*>(dst[i]) = a[i];
            if (TWO && off[i]) *reinterpret_cast<Vec<T, VEC>*>(dst[i] + off[i]) = b[i];
        }
    }
}

template <typename T, bool HALVES>
void launch_rotary(RotaryArgs& p, bool vec, cudaStream_t st) {
    constexpr int V = 16 / sizeof(T);
    const int v = vec ? V : 1, pairs = HALVES ? v : vec ? v / 2 : 1;
    p.rotated = p.pairs / pairs;
    const int per_head = p.rotated + (p.size - 2 * p.pairs) / v;
    p.per_head = Divisor(per_head), p.per_token = Divisor(per_head * (p.heads[0] + p.heads[1])), p.per_pair = Divisor(std::max(1, p.pairs));
    // A block's threads get kUnits units each where the angles allow it.
    p.per_block = std::max(1, std::min(kAngles / std::max(1, p.pairs), 256 * kUnits / (int)p.per_token.d));
    const unsigned grid = (unsigned)((p.tokens + p.per_block - 1) / p.per_block);
    if (vec) launch_early(rotary_kernel<T, V, HALVES>, grid, 256, 0, 1, st, p);
    else launch_early(rotary_kernel<T, 1, HALVES>, grid, 256, 0, 1, st, p);
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
    for (int64_t k = 0; k < a->pairs; ++k) p.turns[k] = a->frequencies[k] / 6.283185307179586476925286766559;
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
