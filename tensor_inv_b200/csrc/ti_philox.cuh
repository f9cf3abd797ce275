// ti_philox.cuh -- the counter-based generator of dropout.
//
// Philox4x32-10 (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as 1, 2, 3",
// 2011): ten rounds of two 32 x 32 -> 64-bit products, key bumped by the Weyl constants.  One
// block of 128 bits serves the 8 consecutive columns of one 16-byte vector of 16-bit elements,
// 16 bits each: half the integer work of 32 bits per element, for a drop probability in steps
// of 2^-16 (the scale of the kept elements uses the probability so rounded, so the mean is kept).
#pragma once

#include <stdint.h>

namespace ti {

struct Dropout {
    uint32_t cut;  // 0..65536: an element is kept when its 16 bits are >= cut
    uint64_t seed;
    const uint64_t *seed_ptr;
    uint64_t offset;
};

__device__ __forceinline__ uint64_t dropout_key(const Dropout &d) {
    return d.seed_ptr ? *d.seed_ptr : d.seed;
}

// The key of every round.  Kept in registers by kernels that make many blocks: it saves a third
// of a block's integer work.
struct DropoutKeys {
    uint32_t k0[10], k1[10];
    __device__ __forceinline__ explicit DropoutKeys(uint64_t key) {
#pragma unroll
        for (int i = 0; i < 10; ++i) {
            k0[i] = static_cast<uint32_t>(key) + i * 0x9E3779B9u;
            k1[i] = static_cast<uint32_t>(key >> 32) + i * 0xBB67AE85u;
        }
    }
};

__device__ __forceinline__ uint4 philox(uint4 c, const DropoutKeys &k) {
#pragma unroll
    for (int i = 0; i < 10; ++i) {
        const uint64_t a = static_cast<uint64_t>(c.x) * 0xD2511F53u;
        const uint64_t b = static_cast<uint64_t>(c.z) * 0xCD9E8D57u;
        c = make_uint4(static_cast<uint32_t>(b >> 32) ^ c.y ^ k.k0[i], static_cast<uint32_t>(b),
                       static_cast<uint32_t>(a >> 32) ^ c.w ^ k.k1[i], static_cast<uint32_t>(a));
    }
    return c;
}

// The 128 bits of columns [8*block, 8*block + 8) of a row.
__device__ __forceinline__ uint4 dropout_bits(const Dropout &d, const DropoutKeys &keys,
                                              uint32_t row, uint32_t block) {
    return philox(make_uint4(block, row, static_cast<uint32_t>(d.offset),
                             static_cast<uint32_t>(d.offset >> 32)),
                  keys);
}

// Whether column j (0..7) of the block is kept.
__device__ __forceinline__ bool dropout_kept(const uint4 &bits, int j, uint32_t cut) {
    const uint32_t w = j < 2 ? bits.x : j < 4 ? bits.y : j < 6 ? bits.z : bits.w;
    return ((j & 1) ? w >> 16 : w & 0xFFFFu) >= cut;
}

// Two packed 16-bit elements with the dropped ones cleared: `bits` holds their numbers, `cut16` is
// the cut in the upper half (cut < 65536).
__device__ __forceinline__ uint32_t keep_pair(uint32_t x, uint32_t bits, uint32_t cut16) {
    if (bits < cut16) x &= 0x0000FFFFu;
    if ((bits << 16) < cut16) x &= 0xFFFF0000u;
    return x;
}

__host__ __device__ __forceinline__ float dropout_scale(uint32_t cut) {
    return cut >= 65536u ? 0.0f : 65536.0f / (65536.0f - static_cast<float>(cut));
}

}  // namespace ti
