// ti_dropout.cu -- Y = dropout(X) with a mask made from a counter-based generator.
//
// Memory bound: each element is read once and written once, the mask exists in registers only.
#include "tensor_inv_crt.h"
#include "ti_common.cuh"
#include "ti_low_rank.cuh"

namespace ti {

int device_context(int *num_sms, int **err);

namespace {

template <typename T>
__device__ __forceinline__ T scaled(T v, uint32_t cut) {
    return from_float<T>(to_float(v) * dropout_scale(cut));
}
template <>
__device__ __forceinline__ double scaled<double>(double v, uint32_t cut) {
    return v * (65536.0 / (65536.0 - cut));
}

// One thread per block of 8 columns.
template <typename T>
__global__ void dropout_kernel(const T *X, int64_t sx0, int64_t sx1, T *Y, int64_t ldy,
                               int64_t rows, int64_t cols, Dropout drop) {
    const int64_t blocks = (cols + 7) >> 3;
    const uint64_t key = dropout_key(drop);
    for (int64_t u = blockIdx.x * int64_t(blockDim.x) + threadIdx.x; u < rows * blocks;
         u += int64_t(gridDim.x) * blockDim.x) {
        const int64_t i = u / blocks, b = u % blocks;
        const uint4 bits =
            dropout_bits(drop, key, static_cast<uint32_t>(i), static_cast<uint32_t>(b));
        for (int j = 0; j < 8; ++j) {
            const int64_t c = 8 * b + j;
            if (c >= cols) break;
            T y = T(0.0f);
            // cut = 0 copies the bits: a product with 1 would make a NaN canonical
            if (dropout_kept(bits, j, drop.cut))
                y = drop.cut ? scaled(X[i * sx0 + c * sx1], drop.cut) : X[i * sx0 + c * sx1];
            Y[i * ldy + c] = y;
        }
    }
}

template <typename T>
cudaError_t launch(const void *X, int64_t sx0, int64_t sx1, void *Y, int64_t ldy, int64_t rows,
                   int64_t cols, const Dropout &drop, int sms, cudaStream_t st) {
    const int64_t units = rows * ((cols + 7) / 8);
    const int64_t want = (units + 255) / 256, most = int64_t(sms) * 8;
    dropout_kernel<T><<<static_cast<unsigned>(want < most ? want : most), 256, 0, st>>>(
        static_cast<const T *>(X), sx0, sx1, static_cast<T *>(Y), ldy, rows, cols, drop);
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
