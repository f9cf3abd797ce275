// ti_dropout.cu -- Y = dropout(X) with a mask made from a counter-based generator.
//
// Memory bound: each element is read once and written once, the mask exists in registers only.
// One thread takes the 8 columns of one generator block at a time -- 16, 32 or 64 bytes of a row,
// in 16-byte copies where both matrices allow them -- and two blocks are in flight per thread, so
// that the loads of one hide behind the ten rounds of the other.
#include "tensor_inv_crt.h"
#include "ti_common.cuh"
#include "ti_low_rank.cuh"

namespace ti {

int device_context(int *num_sms, int **err);

namespace {

constexpr int kThreads = 256, kUnroll = 2;

template <typename T>
__device__ __forceinline__ T scaled(T v, double, float scale) {
    return from_float<T>(to_float(v) * scale);
}
template <>
__device__ __forceinline__ double scaled<double>(double v, double scale, float) {
    return v * scale;
}

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

template <typename T, bool kVec>
__global__ void __launch_bounds__(kThreads)
    dropout_kernel(const T *X, int64_t sx0, int64_t sx1, T *Y, int64_t ldy, int64_t rows,
                   int64_t cols, Dropout drop) {
    const int64_t blocks = (cols + 7) >> 3;
    const uint64_t key = dropout_key(drop);
    const double scale64 = drop.cut > 65535u ? 0.0 : 65536.0 / (65536.0 - drop.cut);
    const float scale32 = dropout_scale(drop.cut);
    // unit (i, b): row i, columns 8b ..; a step of the whole grid is (step_i, step_b)
    const int64_t step = int64_t(gridDim.x) * kThreads;
    const int64_t step_i = step / blocks, step_b = step % blocks;
    const int64_t first = blockIdx.x * int64_t(kThreads) + threadIdx.x;
    int64_t i = first / blocks, b = first % blocks;
    while (i < rows) {
        Block<T> x[kUnroll];
        int64_t ui[kUnroll], ub[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            ui[u] = i;
            ub[u] = b;
            if (i < rows) load<T, kVec>(x[u], X + i * sx0 + 8 * b * sx1, sx1, cols - 8 * b);
            i += step_i;
            b += step_b;
            if (b >= blocks) {
                b -= blocks;
                ++i;
            }
        }
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            if (ui[u] >= rows) break;
            if (drop.cut) {  // cut = 0 copies the bits: a product with 1 would change a NaN's
                const uint4 bits = dropout_bits(drop, key, static_cast<uint32_t>(ui[u]),
                                                static_cast<uint32_t>(ub[u]));
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    x[u].v[j] = dropout_kept(bits, j, drop.cut)
                                    ? scaled<T>(x[u].v[j], scale64, scale32)
                                    : T(0.0f);
            }
            store<T, kVec>(x[u], Y + ui[u] * ldy + 8 * ub[u], cols - 8 * ub[u]);
        }
    }
}

template <typename T>
cudaError_t launch(const void *X, int64_t sx0, int64_t sx1, void *Y, int64_t ldy, int64_t rows,
                   int64_t cols, const Dropout &drop, int sms, cudaStream_t st) {
    constexpr int64_t kPer16 = 16 / sizeof(T);
    const bool vec = sx1 == 1 && ((reinterpret_cast<uintptr_t>(X) | reinterpret_cast<uintptr_t>(Y)) & 15) == 0 &&
                     (rows == 1 || (sx0 % kPer16 == 0 && ldy % kPer16 == 0));
    const int64_t units = rows * ((cols + 7) / 8);
    const int64_t want = (units + kThreads - 1) / kThreads, most = int64_t(sms) * 8;
    const unsigned grid = static_cast<unsigned>(want < most ? want : most);
    const T *x = static_cast<const T *>(X);
    T *y = static_cast<T *>(Y);
    if (vec)
        dropout_kernel<T, true><<<grid, kThreads, 0, st>>>(x, sx0, sx1, y, ldy, rows, cols, drop);
    else
        dropout_kernel<T, false><<<grid, kThreads, 0, st>>>(x, sx0, sx1, y, ldy, rows, cols, drop);
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
    const int rc = device_context(&sms, &err);
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
