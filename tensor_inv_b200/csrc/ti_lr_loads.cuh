// ti_lr_loads.cuh -- loads and small pieces shared by the kernels of the low-rank products.
#pragma once

#include <type_traits>

#include "ti_common.cuh"
#include "ti_low_rank.cuh"

namespace ti {

// 8 consecutive elements at `p`, of which the first n exist (n <= 0: none)
__device__ __forceinline__ uint4 load8(const uint16_t *p, int64_t n) {
    if (n >= 8) return __ldg(reinterpret_cast<const uint4 *>(p));
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (e < n) w[e >> 1] |= static_cast<uint32_t>(p[e]) << (16 * (e & 1));
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// 8 elements of a row with the dropout mask applied.
__device__ __forceinline__ uint4 masked(uint4 v, const Dropout &d, const DropoutKeys &keys,
                                        uint32_t row, uint32_t block) {
    if (d.cut > 65535u) return make_uint4(0, 0, 0, 0);  // everything is dropped
    const uint4 b = dropout_bits(d, keys, row, block);
    const uint32_t cut16 = d.cut << 16;
    return make_uint4(keep_pair(v.x, b.x, cut16), keep_pair(v.y, b.y, cut16),
                      keep_pair(v.z, b.z, cut16), keep_pair(v.w, b.w, cut16));
}

template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
    if constexpr (std::is_same<T, __nv_bfloat16>::value)
        return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
    else
        return __half22float2(*reinterpret_cast<const __half2 *>(&w));
}

template <typename T>
__device__ __forceinline__ void unpack8(uint4 v, float (&f)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float2 h = unpack2<T>(w[e]);
        f[2 * e] = h.x;
        f[2 * e + 1] = h.y;
    }
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    return v;
}

// Writes a float into the shared memory of CTA `rank`, at this CTA's address `p`.
__device__ __forceinline__ void store_remote(float *p, uint32_t rank, float v) {
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(map_to_rank(smem_u32(p), rank)), "f"(v));
}

__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t n;
    asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(n));
    return n;
}

}  // namespace ti
