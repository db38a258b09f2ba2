// Division of row numbers by a constant.  Plain C++ too, so that the host can
// replay it.
#pragma once
#include <stdint.h>

#ifdef __CUDACC__
#define LFB_DIVISOR_CALL __host__ __device__ __forceinline__
#else
#define LFB_DIVISOR_CALL inline
#endif

namespace lfb {

// n / d for 0 <= n < 2^31 and 0 < d < 2^31 by a multiplication (Granlund and Montgomery 1994).
struct Divisor {
    uint32_t d, mul, shift;
    Divisor() = default;
    explicit Divisor(uint32_t v) : d(v), shift(0) {
        while ((1u << shift) < d) ++shift;
        mul = (uint32_t)((((uint64_t)1 << 32) * (((uint64_t)1 << shift) - d)) / d + 1);
    }
    LFB_DIVISOR_CALL int of(int n) const {
#ifdef __CUDA_ARCH__
        const uint32_t high = __umulhi((uint32_t)n, mul);
#else
        const uint32_t high = (uint32_t)(((uint64_t)(uint32_t)n * mul) >> 32);
#endif
        return (int)((high + (uint32_t)n) >> shift);
    }
};

// r / d for 0 <= r < 2^40 and 0 < d < 2^40: with 2^s >= d > 2^(s-1) and m = floor(2^(40+s) / d) + 1, m d exceeds 2^(40+s) by
// at most 2^s, so r m / 2^(40+s) has r / d for its floor (the same paper).  r 2^23 and m fit 64 bits.
struct LongDivisor {
    uint64_t mul;
    uint32_t shift;  // s - 1
    LongDivisor() = default;
    explicit LongDivisor(int64_t d) {
        uint32_t s = 1;
        while (((int64_t)1 << s) < d) ++s;
        uint64_t q = 0, rest = 1;  // 2^(40+s) / d bit by bit: the dividend may not fit 64 bits
        for (uint32_t i = 0; i < 40 + s; ++i) {
            rest *= 2, q *= 2;
            if (rest >= (uint64_t)d) rest -= (uint64_t)d, ++q;
        }
        mul = q + 1, shift = s - 1;
    }
    LFB_DIVISOR_CALL int64_t of(int64_t r) const {
#ifdef __CUDA_ARCH__
        const uint64_t high = __umul64hi((uint64_t)r << 23, mul);
#else
        const uint64_t high = (uint64_t)(((unsigned __int128)((uint64_t)r << 23) * mul) >> 64);
#endif
        return (int64_t)(high >> shift);
    }
};

}  // namespace lfb
