// Rows of a norm in the registers of thread groups: packs of elements, group
// reductions, the tables of group sizes, and the checks of their operands.
#pragma once

#include <initializer_list>
#include <mutex>

#include "lf_common.cuh"

namespace lfb {
namespace {

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

template <int G>
constexpr int block_of() {
    return G <= 32 ? 256 : G;
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

}  // namespace
}  // namespace lfb
