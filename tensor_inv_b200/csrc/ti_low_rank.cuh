// ti_low_rank.cuh -- what the kernels of the low-rank products share.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "ti_philox.cuh"

namespace ti {

// A matrix of 16-bit elements: element (i, j) at p[i*s0 + j*s1].
struct Matrix16 {
    const void *p;
    int64_t s0, s1;
};

// The adapters' factor that meets a dimension of the shared matrix: element (c, j) of adapter s
// (c along that dimension, j < r) at p[s*ss + c*sc + j*sr].
struct Factor16 {
    const void *p;
    int64_t ss, sc, sr;
};

// Which adapter a row takes.
struct RowIndex {
    const void *p;  // null: adapter 0 for every row
    int is64;
    int64_t s;      // number of adapters
    // adapter of row t, or -1
    __device__ __forceinline__ int at(int64_t t) const {
        if (!p) return 0;
        const int64_t i = is64 ? static_cast<const int64_t *>(p)[t]
                               : static_cast<int64_t>(static_cast<const int32_t *>(p)[t]);
        return i >= 0 && i < s ? static_cast<int>(i) : -1;
    }
};

template <typename T>
__device__ __forceinline__ float to_float(T v);
template <>
__device__ __forceinline__ float to_float<__half>(__half v) {
    return __half2float(v);
}
template <>
__device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) {
    return __bfloat162float(v);
}

template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ __half from_float<__half>(float v) {
    return __float2half_rn(v);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) {
    return __float2bfloat16_rn(v);
}

}  // namespace ti
