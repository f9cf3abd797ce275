// ti_lr_dot.cuh -- one row times its adapter's factor over a slice of the inner dimension, by
// a group of warps; 16-bit loads shared by the kernels of the low-rank products.
#pragma once

#include <type_traits>

#include "ti_common.cuh"
#include "ti_low_rank.cuh"

namespace ti {

// How a factor is read: element by element, in 16-byte vectors along c, or along the rank.
enum { kFScalar = 0, kFC = 1, kFR = 2 };

__host__ inline int factor_mode(const Factor16 &F) {
    const bool base = (reinterpret_cast<uintptr_t>(F.p) & 15) == 0 && F.ss % 8 == 0;
    if (base && F.sc == 1 && F.sr % 8 == 0) return kFC;
    if (base && F.sr == 1 && F.sc % 8 == 0) return kFR;
    return kFScalar;
}

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
__device__ __forceinline__ uint4 masked(uint4 v, const Dropout &d, uint64_t key, uint32_t row,
                                        uint32_t block) {
    if (d.cut > 65535u) return make_uint4(0, 0, 0, 0);  // everything is dropped
    const uint4 b = dropout_bits(d, key, row, block);
    const uint32_t cut2 = d.cut * 0x10001u;
    return make_uint4(v.x & __vcmpgeu2(b.x, cut2), v.y & __vcmpgeu2(b.y, cut2),
                      v.z & __vcmpgeu2(b.z, cut2), v.w & __vcmpgeu2(b.w, cut2));
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

// A float in the shared memory of CTA `rank` of the cluster, at this CTA's address `p`.
__device__ __forceinline__ float load_remote(const float *p, uint32_t rank) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];"
                 : "=f"(v)
                 : "r"(map_to_rank(smem_u32(p), rank))
                 : "memory");
    return v;
}

__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t n;
    asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(n));
    return n;
}

// part[w][j] (w < kWarps) such that its sum over w is sum_{c in [begin, end)} m(t, c) x[c] F[c][j].
// Called by kWarps whole warps; begin is a multiple of 8.  The caller synchronises afterwards.
//   vectors along c:    a warp takes a rank at a time, its lanes 8 elements of c each
//   vectors along rank: a warp takes a part of the slice, its lanes one element of c each
template <typename T, bool kDrop, int kWarps>
__device__ __forceinline__ void dot_slice(const uint16_t *x, const uint16_t *F, int64_t sc,
                                          int64_t sr, int mode, int r, int64_t begin, int64_t end,
                                          const Dropout &drop, uint64_t key, uint32_t row,
                                          int warp, int lane, float *part, int part_stride) {
    if (mode == kFR) {
        const int64_t share = ((end - begin + kWarps - 1) / kWarps + 7) / 8 * 8;
        const int64_t lo = begin + warp * share, hi = min(end, lo + share);
        for (int jb = 0; jb < r; jb += 8) {
            float acc[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) acc[j] = 0.0f;
#pragma unroll 8
            for (int64_t c = lo + lane; c < hi; c += 32) {
                float f[8];
                unpack8<T>(load8(F + c * sc + jb, r - jb), f);
                float v = to_float(*reinterpret_cast<const T *>(x + c));
                if (kDrop)
                    if (!dropout_kept(dropout_bits(drop, key, row, static_cast<uint32_t>(c >> 3)),
                                      static_cast<int>(c & 7), drop.cut))
                        v = 0.0f;
#pragma unroll
                for (int j = 0; j < 8; ++j) acc[j] += v * f[j];
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float v = warp_sum(acc[j]);
                if (lane == 0 && jb + j < r) part[warp * part_stride + jb + j] = v;
            }
        }
        return;
    }
    for (int j = warp; j < r; j += kWarps) {
        float acc = 0.0f;
#pragma unroll 4
        for (int64_t c = begin + 8 * lane; c < end; c += 256) {
            uint4 xv = load8(x + c, end - c);
            if (kDrop) xv = masked(xv, drop, key, row, static_cast<uint32_t>(c >> 3));
            float v[8], f[8];
            unpack8<T>(xv, v);
            if (mode == kFC) {
                unpack8<T>(load8(F + j * sr + c, end - c), f);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    f[e] = c + e < end
                               ? to_float(*reinterpret_cast<const T *>(F + (c + e) * sc + j * sr))
                               : 0.0f;
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) acc += v[e] * f[e];
        }
        acc = warp_sum(acc);
        if (lane < kWarps) part[lane * part_stride + j] = lane == 0 ? acc : 0.0f;
    }
}

}  // namespace ti
