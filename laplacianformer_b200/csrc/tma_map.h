// Tensor maps for TMA copies (host side).
#pragma once

#include <cuda.h>

#include <mutex>

#include "lf_common.cuh"

namespace lfb {

typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                             const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                             CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeFn encode_fn() {
    static std::once_flag once;
    static EncodeFn fn = nullptr;
    std::call_once(once, [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = (EncodeFn)p;
    });
    return fn;
}

// Whether the map of `rank` dimensions (innermost first, strides in bytes from the second on) could be made.
inline bool encode_tiled(CUtensorMap* map, CUtensorMapDataType type, int rank, const void* p, const cuuint64_t* dims,
                         const cuuint64_t* strides, const cuuint32_t* box, CUtensorMapSwizzle swizzle,
                         CUtensorMapL2promotion promotion = CU_TENSOR_MAP_L2_PROMOTION_L2_256B) {
    const cuuint32_t step[5] = {1, 1, 1, 1, 1};
    EncodeFn fn = encode_fn();
    if (!fn) {
        set_error("cuTensorMapEncodeTiled is not available");
        return false;
    }
    auto call = [&] {
        return fn(map, type, (cuuint32_t)rank, const_cast<void*>(p), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  swizzle, promotion, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    };
    CUresult r = call();
    if (r == CUDA_ERROR_INVALID_CONTEXT) {  // the first call of a host thread (an autograd worker): bind the device's context
        int dev = 0;
        if (cudaGetDevice(&dev) == cudaSuccess && cudaSetDevice(dev) == cudaSuccess) r = call();
    }
    if (r != CUDA_SUCCESS) set_error("cuTensorMapEncodeTiled failed (%d)", (int)r);
    return r == CUDA_SUCCESS;
}

}  // namespace lfb
