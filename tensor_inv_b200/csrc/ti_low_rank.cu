// ti_low_rank.cu -- low-rank products beside a shared one: the C entry points and the kernels.
//
//   forward   P[t] = f (M X)[t] A[i]     Y[t] = X[t] W + P[t] B[i]          i = index[t]
//   backward  dP[t] = f dY[t] B[i]^T     dX[t] = dY[t] W^T + M (dP[t] A[i]^T)
//             dA[i] = sum_t (M X)[t]^T dP[t]        dB[i] = sum_t P[t]^T dY[t]
// with f = alpha * scale[i] * 65536 / (65536 - cut) and M the dropout mask (ti_philox.cuh).
// Three forms serve both directions: project (a row times its adapter's factor), expand (the
// shared product plus a row of P times a factor) and wgrad (sums over an adapter's rows).
#include "tensor_inv_crt.h"
#include "ti_common.cuh"
#include "ti_low_rank.cuh"

namespace ti {

int device_context(int *num_sms, int **err);

namespace {

// P[t][j] = f * sum_c m(t, c) M[t][c] F[i][c][j], one warp per (t, j).
template <typename T>
__global__ void project_kernel(Matrix16 M, int64_t rows, int64_t cols, Factor16 F, int64_t r,
                               RowIndex index, const float *scale, float alpha, Dropout drop,
                               float *P) {
    const int64_t w = (blockIdx.x * int64_t(blockDim.x) + threadIdx.x) >> 5;
    const int lane = threadIdx.x & 31;
    if (w >= rows * r) return;
    const int64_t t = w / r, j = w % r;
    const int i = index.at(t);
    float acc = 0.0f;
    if (i >= 0) {
        const T *x = static_cast<const T *>(M.p) + t * M.s0;
        const T *f = static_cast<const T *>(F.p) + i * F.ss + j * F.sr;
        const uint64_t key = drop.cut ? dropout_key(drop) : 0;
        for (int64_t c = lane; c < cols; c += 32) {
            if (drop.cut) {
                const uint4 bits = dropout_bits(drop, key, static_cast<uint32_t>(t),
                                                static_cast<uint32_t>(c >> 3));
                if (!dropout_kept(bits, static_cast<int>(c & 7), drop.cut)) continue;
            }
            acc += to_float(x[c * M.s1]) * to_float(f[c * F.sc]);
        }
        for (int o = 16; o; o >>= 1) acc += __shfl_xor_sync(0xFFFFFFFFu, acc, o);
        acc *= alpha * (scale ? scale[i] : 1.0f);
    }
    if (lane == 0) P[w] = acc;
}

// out[t][c] = sum_k M[t][k] W[k][c] + m(t, c) sum_j P[t][j] F[i][c][j], one thread per (t, c).
template <typename T>
__global__ void expand_kernel(Matrix16 M, int64_t rows, int64_t inner, Matrix16 W, int64_t cols,
                              const float *P, Factor16 F, int64_t r, RowIndex index,
                              Dropout drop, T *out, int64_t ldo) {
    const int64_t e = blockIdx.x * int64_t(blockDim.x) + threadIdx.x;
    if (e >= rows * cols) return;
    const int64_t t = e / cols, c = e % cols;
    const T *x = static_cast<const T *>(M.p) + t * M.s0;
    const T *w = static_cast<const T *>(W.p) + c * W.s1;
    float acc = 0.0f;
    for (int64_t k = 0; k < inner; ++k) acc += to_float(x[k * M.s1]) * to_float(w[k * W.s0]);
    const int i = index.at(t);
    bool kept = i >= 0;
    if (kept && drop.cut)
        kept = dropout_kept(dropout_bits(drop, dropout_key(drop), static_cast<uint32_t>(t),
                                         static_cast<uint32_t>(c >> 3)),
                            static_cast<int>(c & 7), drop.cut);
    if (kept) {
        const T *f = static_cast<const T *>(F.p) + i * F.ss + c * F.sc;
        float low = 0.0f;
        for (int64_t j = 0; j < r; ++j) low += P[t * r + j] * to_float(f[j * F.sr]);
        acc += low;
    }
    out[t * ldo + c] = from_float<T>(acc);
}

// out[s][c][j] = sum over the rows t of adapter s of m(t, c) M[t][c] V[t][j].
template <typename T>
__global__ void wgrad_kernel(Matrix16 M, int64_t rows, int64_t cols, const float *V, int64_t r,
                             RowIndex index, Dropout drop, T *out, int64_t ss, int64_t sc,
                             int64_t sr) {
    const int64_t e = blockIdx.x * int64_t(blockDim.x) + threadIdx.x;
    if (e >= index.s * cols * r) return;
    const int64_t j = e % r, c = e / r % cols, s = e / (r * cols);
    const uint64_t key = drop.cut ? dropout_key(drop) : 0;
    float acc = 0.0f;
    for (int64_t t = 0; t < rows; ++t) {
        if (index.at(t) != s) continue;
        if (drop.cut && !dropout_kept(dropout_bits(drop, key, static_cast<uint32_t>(t),
                                                   static_cast<uint32_t>(c >> 3)),
                                      static_cast<int>(c & 7), drop.cut))
            continue;
        acc += to_float(static_cast<const T *>(M.p)[t * M.s0 + c * M.s1]) * V[t * r + j];
    }
    out[s * ss + c * sc + j * sr] = from_float<T>(acc);
}

constexpr int64_t kMaxRank = 256;

size_t align256(size_t x) { return (x + 255) & ~size_t(255); }

int check_op(const ti_low_rank_t *op) {
    if (!op || (op->dtype != TI_TYPE_F16 && op->dtype != TI_TYPE_BF16)) return TI_ERR_INVALID_ARGUMENT;
    if (op->t < 0 || op->k < 0 || op->n < 0 || op->s < 1 || op->r < 1) return TI_ERR_INVALID_ARGUMENT;
    if (op->r > kMaxRank || op->t >= int64_t(1) << 31 || op->k >= int64_t(1) << 31 ||
        op->n >= int64_t(1) << 31 || op->s >= int64_t(1) << 31)
        return TI_ERR_UNSUPPORTED;
    if (op->index && op->index_bytes != 4 && op->index_bytes != 8) return TI_ERR_INVALID_ARGUMENT;
    if (op->drop.cut < 0 || op->drop.cut > 65536) return TI_ERR_INVALID_ARGUMENT;
    return TI_OK;
}

Dropout device_spec(const ti_dropout_spec_t &d) {
    return Dropout{static_cast<uint32_t>(d.cut), d.seed, d.seed_ptr, d.offset};
}

unsigned blocks_for(int64_t n, int per) { return static_cast<unsigned>((n + per - 1) / per); }

int status(cudaError_t e) { return e == cudaSuccess ? TI_OK : TI_ERR_CUDA; }

template <typename T>
int forward(const ti_low_rank_t &op, void *Y, int64_t ldy, float *P, cudaStream_t st) {
    const Matrix16 X{op.x, op.sx0, op.sx1}, W{op.w, op.sw0, op.sw1};
    const RowIndex index{op.index, op.index_bytes == 8, op.s};
    const Dropout drop = device_spec(op.drop);
    project_kernel<T><<<blocks_for(op.t * op.r, 4), 128, 0, st>>>(
        X, op.t, op.k, Factor16{op.a, op.sa0, op.sa1, op.sa2}, op.r, index, op.scale,
        op.alpha * dropout_scale(drop.cut), drop, P);
    if (op.n)
        expand_kernel<T><<<blocks_for(op.t * op.n, 256), 256, 0, st>>>(
            X, op.t, op.k, W, op.n, P, Factor16{op.b, op.sb0, op.sb2, op.sb1}, op.r, index,
            Dropout{}, static_cast<T *>(Y), ldy);
    return status(cudaGetLastError());
}

template <typename T>
int backward(const ti_low_rank_t &op, const Matrix16 &dY, const float *P, void *dX, int64_t lddx,
             void *dA, const int64_t (&sda)[3], void *dB, const int64_t (&sdb)[3], float *dP,
             cudaStream_t st) {
    const Matrix16 X{op.x, op.sx0, op.sx1};
    const RowIndex index{op.index, op.index_bytes == 8, op.s};
    const Dropout drop = device_spec(op.drop);
    if ((dX || dA) && op.t)
        project_kernel<T><<<blocks_for(op.t * op.r, 4), 128, 0, st>>>(
            dY, op.t, op.n, Factor16{op.b, op.sb0, op.sb2, op.sb1}, op.r, index, op.scale,
            op.alpha * dropout_scale(drop.cut), Dropout{}, dP);
    if (dX && op.t && op.k)
        expand_kernel<T><<<blocks_for(op.t * op.k, 256), 256, 0, st>>>(
            dY, op.t, op.n, Matrix16{op.w, op.sw1, op.sw0}, op.k, dP,
            Factor16{op.a, op.sa0, op.sa1, op.sa2}, op.r, index, drop, static_cast<T *>(dX), lddx);
    if (dA && op.k)
        wgrad_kernel<T><<<blocks_for(op.s * op.k * op.r, 256), 256, 0, st>>>(
            X, op.t, op.k, dP, op.r, index, drop, static_cast<T *>(dA), sda[0], sda[1], sda[2]);
    if (dB && op.n)
        wgrad_kernel<T><<<blocks_for(op.s * op.n * op.r, 256), 256, 0, st>>>(
            dY, op.t, op.n, P, op.r, index, Dropout{}, static_cast<T *>(dB), sdb[0], sdb[2],
            sdb[1]);
    return status(cudaGetLastError());
}

}  // namespace
}  // namespace ti

using namespace ti;

extern "C" {

int ti_low_rank_workspace_size(const ti_low_rank_t *op, int backward, size_t *bytes) {
    const int rc = check_op(op);
    if (rc != TI_OK || !bytes) return rc != TI_OK ? rc : TI_ERR_INVALID_ARGUMENT;
    (void)backward;
    *bytes = align256(sizeof(float) * static_cast<size_t>(op->t * op->r));
    return TI_OK;
}

int ti_low_rank_matmul(const ti_low_rank_t *op, void *Y, int64_t ldy, float *P, void *workspace,
                       size_t workspace_bytes, void *stream) {
    size_t need = 0;
    int rc = ti_low_rank_workspace_size(op, 0, &need);
    if (rc != TI_OK) return rc;
    int sms = 0, *err = nullptr;
    if ((rc = device_context(&sms, &err)) != TI_OK) return rc;
    if (op->t == 0) return TI_OK;
    if ((op->k && (!op->x || !op->a || (op->n && !op->w))) || (op->n && (!op->b || !Y)) ||
        ldy < op->n)
        return TI_ERR_INVALID_ARGUMENT;
    if (need && (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 255)))
        return TI_ERR_WORKSPACE;
    float *proj = P ? P : static_cast<float *>(workspace);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return op->dtype == TI_TYPE_F16 ? forward<__half>(*op, Y, ldy, proj, st)
                                    : forward<__nv_bfloat16>(*op, Y, ldy, proj, st);
}

int ti_low_rank_backward(const ti_low_rank_t *op, const void *dY, int64_t sdy0, int64_t sdy1,
                         const float *P, void *dX, int64_t lddx, void *dA, int64_t sda0,
                         int64_t sda1, int64_t sda2, void *dB, int64_t sdb0, int64_t sdb1,
                         int64_t sdb2, void *workspace, size_t workspace_bytes, void *stream) {
    size_t need = 0;
    int rc = ti_low_rank_workspace_size(op, 1, &need);
    if (rc != TI_OK) return rc;
    int sms = 0, *err = nullptr;
    if ((rc = device_context(&sms, &err)) != TI_OK) return rc;
    if ((op->k && !op->a) || (op->n && !op->b) ||
        (op->t && ((op->k && !op->x) || (op->n && !dY) || (op->k && op->n && dX && !op->w) ||
                   (dB && !P))))
        return TI_ERR_INVALID_ARGUMENT;
    if (dX && lddx < op->k) return TI_ERR_INVALID_ARGUMENT;
    if (need && (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 255)))
        return TI_ERR_WORKSPACE;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const Matrix16 G{dY, sdy0, sdy1};
    const int64_t sda[3] = {sda0, sda1, sda2}, sdb[3] = {sdb0, sdb1, sdb2};
    float *dP = static_cast<float *>(workspace);
    return op->dtype == TI_TYPE_F16
               ? backward<__half>(*op, G, P, dX, lddx, dA, sda, dB, sdb, dP, st)
               : backward<__nv_bfloat16>(*op, G, P, dX, lddx, dA, sda, dB, sdb, dP, st);
}

}  // extern "C"
