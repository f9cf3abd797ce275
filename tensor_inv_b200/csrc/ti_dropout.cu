// ti_dropout.cu -- Y = dropout(X) with a mask made from a counter-based generator.
//
// Each element is read once and written once, the mask exists in registers only.  A generator
// block costs 20 wide multiplications and 20 three-input xors for 8 elements, so the integer pipes
// are nearly as busy as the memory; everything around the rounds is kept short.  A warp takes 32 or
// 128 consecutive blocks of a row, one or four per lane, in 16-byte copies where both matrices allow
// them; the four blocks' copies and rounds overlap.  Measured on a B200: 16384 x 8192 bf16 96 us
// (5.6 TB/s of 6.5 measured); 143 us with two blocks in flight and the keys made in each round.
#include "tensor_inv_crt.h"
#include "ti_common.cuh"
#include "ti_lr_launch.cuh"

namespace ti {

namespace {

constexpr int kThreads = 256;

// Elements of one generator block (8 columns) of type T.
template <typename T>
struct alignas(16) Block {
    T v[8];
};

template <typename T, bool kVec>
__device__ __forceinline__ void load(Block<T> &x, const T *p, int64_t s1, int64_t n) {
    if (kVec && n >= 8) {
        constexpr int kWords = sizeof(x) / 16;
#pragma unroll
        for (int w = 0; w < kWords; ++w)
            reinterpret_cast<uint4 *>(&x)[w] = __ldcs(reinterpret_cast<const uint4 *>(p) + w);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < n) x.v[j] = p[j * s1];
    }
}

template <typename T, bool kVec>
__device__ __forceinline__ void store(const Block<T> &x, T *p, int64_t n) {
    if (kVec && n >= 8) {
        constexpr int kWords = sizeof(x) / 16;
#pragma unroll
        for (int w = 0; w < kWords; ++w)
            reinterpret_cast<uint4 *>(p)[w] = reinterpret_cast<const uint4 *>(&x)[w];
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < n) p[j] = x.v[j];
    }
}

template <typename T>
__device__ __forceinline__ uint32_t scale_pair(uint32_t w, float scale);
template <>
__device__ __forceinline__ uint32_t scale_pair<__nv_bfloat16>(uint32_t w, float scale) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(__uint_as_float(w << 16) * scale,
                                                   __uint_as_float(w & 0xFFFF0000u) * scale);
    return *reinterpret_cast<const uint32_t *>(&v);
}
template <>
__device__ __forceinline__ uint32_t scale_pair<__half>(uint32_t w, float scale) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w));
    const __half2 v = __floats2half2_rn(f.x * scale, f.y * scale);
    return *reinterpret_cast<const uint32_t *>(&v);
}

// Masks and scales a block (0 < cut < 65536).
template <typename T>
__device__ __forceinline__ void apply(Block<T> &x, const uint4 &bits, uint32_t cut, float scale32,
                                      double scale64) {
    const uint32_t w[4] = {bits.x, bits.y, bits.z, bits.w};
    const uint32_t cut16 = cut << 16;
    if constexpr (sizeof(T) == 2) {
        uint32_t *p = reinterpret_cast<uint32_t *>(&x);
#pragma unroll
        for (int k = 0; k < 4; ++k) p[k] = scale_pair<T>(keep_pair(p[k], w[k], cut16), scale32);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const bool kept = ((j & 1) ? w[j >> 1] : w[j >> 1] << 16) >= cut16;
            const T y = sizeof(T) == 8 ? static_cast<T>(x.v[j] * scale64)
                                       : static_cast<T>(x.v[j] * scale32);
            x.v[j] = kept ? y : T(0);
        }
    }
}

template <typename T, bool kVec, int kUnroll>
__global__ void __launch_bounds__(kThreads)
    dropout_kernel(const T *X, int64_t sx0, int64_t sx1, T *Y, int64_t ldy, int64_t rows,
                   int64_t cols, Dropout drop) {
    const DropoutKeys keys(dropout_key(drop));
    const double scale64 = drop.cut > 65535u ? 0.0 : 65536.0 / (65536.0 - drop.cut);
    const float scale32 = dropout_scale(drop.cut);
    const int lane = threadIdx.x & 31;
    // a warp's tile: row i, blocks [32 * kUnroll * b, ...); all warps' step is (step_i, step_b)
    const int64_t tiles = (cols + 256 * kUnroll - 1) / (256 * kUnroll);
    const int64_t step = int64_t(gridDim.x) * (kThreads / 32);
    const int64_t step_i = step / tiles, step_b = step % tiles;
    const int64_t first = blockIdx.x * int64_t(kThreads / 32) + (threadIdx.x >> 5);
    int64_t i = first / tiles, b = first % tiles;
    while (i < rows) {
        const int64_t c0 = 256 * kUnroll * b + 8 * lane;
        const T *src = X + i * sx0 + c0 * sx1;
        T *dst = Y + i * ldy + c0;
        Block<T> x[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
            load<T, kVec>(x[u], src + 256 * u * sx1, sx1, cols - c0 - 256 * u);
        // cut = 0 copies the bits (a product with 1 would change a NaN's), 65536 drops everything
        if (drop.cut > 65535u) {
#pragma unroll
            for (int u = 0; u < kUnroll; ++u)
#pragma unroll
                for (int j = 0; j < 8; ++j) x[u].v[j] = T(0.0f);
        } else if (drop.cut) {
#pragma unroll
            for (int u = 0; u < kUnroll; ++u)
                apply<T>(x[u],
                         dropout_bits(drop, keys, static_cast<uint32_t>(i),
                                      static_cast<uint32_t>((c0 >> 3) + 32 * u)),
                         drop.cut, scale32, scale64);
        }
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
            store<T, kVec>(x[u], dst + 256 * u, cols - c0 - 256 * u);
        i += step_i;
        b += step_b;
        if (b >= tiles) {
            b -= tiles;
            ++i;
        }
    }
}

template <typename T, bool kVec>
void run(const T *X, int64_t sx0, int64_t sx1, T *Y, int64_t ldy, int64_t rows, int64_t cols,
         const Dropout &drop, int sms, cudaStream_t st) {
    // four blocks per lane where that leaves every SM work and few idle lanes; else one
    constexpr int kMany = sizeof(T) == 2 ? 4 : sizeof(T) == 4 ? 2 : 1;
    const int64_t wide = (cols + 256 * kMany - 1) / (256 * kMany), narrow = (cols + 255) / 256;
    const bool many = rows * wide >= int64_t(sms) * 16 && wide * kMany <= narrow + narrow / 4;
    const int64_t want = (rows * (many ? wide : narrow) + kThreads / 32 - 1) / (kThreads / 32);
    const int64_t most = int64_t(sms) * 8;
    const unsigned grid = static_cast<unsigned>(want < most ? want : most);
    if (many)
        dropout_kernel<T, kVec, kMany><<<grid, kThreads, 0, st>>>(X, sx0, sx1, Y, ldy, rows, cols, drop);
    else
        dropout_kernel<T, kVec, 1><<<grid, kThreads, 0, st>>>(X, sx0, sx1, Y, ldy, rows, cols, drop);
}

template <typename T>
cudaError_t launch(const void *X, int64_t sx0, int64_t sx1, void *Y, int64_t ldy, int64_t rows,
                   int64_t cols, const Dropout &drop, int sms, cudaStream_t st) {
    constexpr int64_t kPer16 = 16 / sizeof(T);
    const bool vec =
        sx1 == 1 && ((reinterpret_cast<uintptr_t>(X) | reinterpret_cast<uintptr_t>(Y)) & 15) == 0 &&
        (rows == 1 || (sx0 % kPer16 == 0 && ldy % kPer16 == 0));
    const T *x = static_cast<const T *>(X);
    T *y = static_cast<T *>(Y);
    if (vec)
        run<T, true>(x, sx0, sx1, y, ldy, rows, cols, drop, sms, st);
    else
        run<T, false>(x, sx0, sx1, y, ldy, rows, cols, drop, sms, st);
    return cudaGetLastError();
}

}  // namespace
}  // namespace ti

using namespace ti;

extern "C" int ti_dropout(int dtype, const void *X, int64_t sx0, int64_t sx1, void *Y, int64_t ldy,
                          int64_t rows, int64_t cols, const ti_dropout_spec_t *drop,
                          void *stream) {
    if (dtype < TI_TYPE_F16 || dtype > TI_TYPE_F64 || rows < 0 || cols < 0 || !drop)
        return TI_ERR_INVALID_ARGUMENT;
    if (drop->cut < 0 || drop->cut > 65536 || ldy < cols) return TI_ERR_INVALID_ARGUMENT;
    if (rows >= int64_t(1) << 32 || cols >= int64_t(1) << 34) return TI_ERR_UNSUPPORTED;
    int sms = 0, *err = nullptr;
    const int rc = low_rank_context(&sms, &err);
    if (rc != TI_OK) return rc;
    if (rows == 0 || cols == 0) return TI_OK;
    if (!X || !Y) return TI_ERR_INVALID_ARGUMENT;
    const Dropout d{static_cast<uint32_t>(drop->cut), drop->seed, drop->seed_ptr, drop->offset};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    cudaError_t e;
    switch (dtype) {
        case TI_TYPE_F16: e = launch<__half>(X, sx0, sx1, Y, ldy, rows, cols, d, sms, st); break;
        case TI_TYPE_BF16:
            e = launch<__nv_bfloat16>(X, sx0, sx1, Y, ldy, rows, cols, d, sms, st);
            break;
        case TI_TYPE_F32: e = launch<float>(X, sx0, sx1, Y, ldy, rows, cols, d, sms, st); break;
        default: e = launch<double>(X, sx0, sx1, Y, ldy, rows, cols, d, sms, st); break;
    }
    return e == cudaSuccess ? TI_OK : TI_ERR_CUDA;
}
