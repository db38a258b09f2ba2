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

// The group of row r where each takes `each` of `rows` rows in turn: by the multiplication while rows are counted in 31 bits
// (its d is 0 otherwise), else by a 64-bit division.
struct RowGroups {
    Divisor by;
    int64_t each;
    RowGroups() = default;
    RowGroups(int64_t rows, int64_t each_) : by{}, each(each_) {
        if (rows <= INT32_MAX && each <= rows && each > 0) by = Divisor((uint32_t)each);
    }
    LFB_DIVISOR_CALL int64_t of(int64_t r) const { return by.d ? (int64_t)by.of((int)r) : r / each; }
};

}  // namespace lfb
