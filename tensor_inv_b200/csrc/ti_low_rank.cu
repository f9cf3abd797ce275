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
#include "ti_lr_launch.cuh"

namespace ti {

int device_context(int *num_sms, int **err);

namespace {

// dst[z][i][j] = src[z][i][j], rows of `ld` elements: operands that a copy engine cannot read (odd
// strides or addresses) are copied once, all of a call's in one launch.  32 x 64 tiles through
// shared memory, so that both sides are coalesced whichever stride of src is 1.
struct PackJob {
    Matrix16 src;
    int64_t batch, s_batch, rows, cols;
    uint16_t *dst;
    int64_t ld, first;  // the job's first tile
};
constexpr int kMaxJobs = 4;
struct PackJobs {
    PackJob job[kMaxJobs];
    int n;
    int64_t tiles;
};

__global__ void __launch_bounds__(256) pack_kernel(const __grid_constant__ PackJobs jobs) {
    __shared__ uint16_t tile[32][66];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int64_t u = blockIdx.x; u < jobs.tiles; u += gridDim.x) {
        int k = 0;
        while (k + 1 < jobs.n && u >= jobs.job[k + 1].first) ++k;
        const PackJob &J = jobs.job[k];
        const int64_t tiles_c = (J.cols + 63) / 64, tiles = (J.rows + 31) / 32 * tiles_c;
        const int64_t v = u - J.first, z = v / tiles;
        const int64_t r0 = v % tiles / tiles_c * 32, c0 = v % tiles_c * 64;
        const uint16_t *s = static_cast<const uint16_t *>(J.src.p) + z * J.s_batch;
        const int nr = static_cast<int>(min(int64_t(32), J.rows - r0));
        const int nc = static_cast<int>(min(int64_t(64), J.cols - c0));
        if (J.src.s0 == 1 && J.src.s1 != 1) {  // a warp reads columns
            const uint16_t *p = s + r0 + lane + (c0 + warp) * J.src.s1;
#pragma unroll
            for (int c = 0; c < 8; ++c)
                if (lane < nr && warp + 8 * c < nc) tile[lane][warp + 8 * c] = p[8 * c * J.src.s1];
        } else {
            const uint16_t *p = s + (r0 + warp) * J.src.s0 + (c0 + lane) * J.src.s1;
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    if (warp + 8 * r < nr && lane + 32 * h < nc)
                        tile[warp + 8 * r][lane + 32 * h] = p[8 * r * J.src.s0 + 32 * h * J.src.s1];
        }
        __syncthreads();
        // two columns per lane; the padding behind the last column belongs to the copy
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (warp + 8 * r < nr && 2 * lane < nc)
                *reinterpret_cast<uint32_t *>(J.dst + (z * J.rows + r0 + warp + 8 * r) * J.ld + c0 +
                                              2 * lane) =
                    *reinterpret_cast<const uint32_t *>(&tile[warp + 8 * r][2 * lane]);
        __syncthreads();
    }
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

int status(cudaError_t e) { return e == cudaSuccess ? TI_OK : TI_ERR_CUDA; }

int64_t round8(int64_t x) { return (x + 7) / 8 * 8; }

// Hands out parts of the workspace; with no base it only counts bytes.  Operands that the copy
// engine cannot read are noted and packed together by pack().
struct Arena {
    uint8_t *base;
    size_t used;
    PackJobs jobs;
    void *take(size_t bytes) {
        void *p = base ? base + used : nullptr;
        used += align256(bytes);
        return p;
    }
    void *packed(const Matrix16 &M, int64_t batch, int64_t s_batch, int64_t rows, int64_t cols,
                 int64_t ld) {
        void *dst = take(sizeof(uint16_t) * static_cast<size_t>(batch * rows * ld));
        if (batch && rows && cols) {
            jobs.job[jobs.n++] = PackJob{M,  batch, s_batch, rows, cols, static_cast<uint16_t *>(dst),
                                         ld, jobs.tiles};
            jobs.tiles += batch * ((rows + 31) / 32) * ((cols + 63) / 64);
        }
        return dst;
    }
    cudaError_t pack(int sms, cudaStream_t st) const {
        if (!jobs.n) return cudaSuccess;
        const int64_t most = int64_t(sms) * 8;
        pack_kernel<<<static_cast<unsigned>(jobs.tiles < most ? jobs.tiles : most), 256, 0, st>>>(jobs);
        return cudaGetLastError();
    }
};

// The matrix as `rows` rows of contiguous elements that a copy engine can read: itself, or a
// packed copy in the workspace.
Matrix16 readable(const Matrix16 &M, int64_t rows, int64_t cols, Arena &arena) {
    const int64_t ld = round8(cols);
    if (copyable(M.p, rows, M.s0, M.s1, cols)) return Matrix16{M.p, rows <= 1 ? ld : M.s0, 1};
    return Matrix16{arena.packed(M, 1, 0, rows, cols, ld), ld, 1};
}

// A projecting factor (s adapters, cols x r) as it is, or, where the copy engine has to read it and
// cannot, packed in rows of one rank.
Factor16 readable_factor(const Factor16 &F, int64_t s, int64_t cols, int64_t r, int64_t rows,
                         Arena &arena) {
    if (rows <= project_rows_limit(s) || factor_mode(F) != kFScalar) return F;
    const int64_t ld = round8(cols), batch = F.ss == 0 ? 1 : s;
    return Factor16{arena.packed(Matrix16{F.p, F.sr, F.sc}, batch, F.ss, r, cols, ld),
                    F.ss == 0 ? 0 : r * ld, 1, ld};
}

// W (inner x cols) with one unit stride, readable in that orientation.
Matrix16 readable_w(const Matrix16 &W, int64_t inner, int64_t cols, Arena &arena) {
    if (copyable(W.p, cols, W.s1, W.s0, inner))
        return Matrix16{W.p, 1, cols <= 1 ? round8(inner) : W.s1};
    if (W.s0 == 1 && W.s1 != 1) {
        const Matrix16 t = readable(Matrix16{W.p, W.s1, W.s0}, cols, inner, arena);
        return Matrix16{t.p, 1, t.s0};
    }
    return readable(W, inner, cols, arena);
}

struct Gradient {
    const void *dY;
    int64_t sdy0, sdy1;
    const float *P;
    void *dX;
    int64_t lddx;
    void *dA;
    int64_t sda[3];
    void *dB;
    int64_t sdb[3];
};

// out = 0 where the inner dimension is empty (the low-rank term is then zero too)
cudaError_t clear(void *out, int64_t ldo, int64_t rows, int64_t cols, cudaStream_t st) {
    return cudaMemset2DAsync(out, 2 * ldo, 0, 2 * cols, rows, st);
}

// The projection, then the expansion that reads it.
cudaError_t project_expand(bool half, const ProjectOperands &p, const ExpandOperands *x, int sms,
                           int *err, cudaStream_t st) {
    const cudaError_t e = lr_project(half, p, sms, err, st);
    if (e != cudaSuccess || !x) return e;
    if (!x->inner) return clear(x->out, x->ldo, x->rows, x->cols, st);
    return x->rows <= expand_rows_limit(x->index.s) ? lr_expand_rows(half, *x, sms, err, st)
                                       : lr_expand_pairs(half, *x, err, st);
}

int forward(const ti_low_rank_t &op, void *Y, int64_t ldy, float *P, Arena &arena, int sms,
            int *err, cudaStream_t st) {
    const RowIndex index{op.index, op.index_bytes == 8, op.s};
    const Dropout drop = device_spec(op.drop);
    float *own = static_cast<float *>(arena.take(sizeof(float) * op.t * op.r));
    if (!P) P = own;
    const Matrix16 X = readable(Matrix16{op.x, op.sx0, op.sx1}, op.t, op.k, arena);
    const Matrix16 W = readable_w(Matrix16{op.w, op.sw0, op.sw1}, op.k, op.n, arena);
    const Factor16 A = readable_factor(Factor16{op.a, op.sa0, op.sa1, op.sa2}, op.s, op.k, op.r,
                                       op.t, arena);
    if (!arena.base) return TI_OK;
    const cudaError_t packed = arena.pack(sms, st);
    if (packed != cudaSuccess) return status(packed);
    const ProjectOperands p{X,     op.t,     op.k,
                            A,
                            op.r,  index,    op.scale,
                            op.alpha * dropout_scale(drop.cut),
                            drop,  P};
    const ExpandOperands x{X,    op.t,  op.k,      W,  op.n, P, Factor16{op.b, op.sb0, op.sb2, op.sb1},
                           op.r, index, Dropout{}, Y,  ldy};
    return status(project_expand(op.dtype == TI_TYPE_F16, p, op.n ? &x : nullptr, sms, err, st));
}

int backward(const ti_low_rank_t &op, const Gradient &g, Arena &arena, int sms, int *err,
             cudaStream_t st) {
    const RowIndex index{op.index, op.index_bytes == 8, op.s};
    const Dropout drop = device_spec(op.drop);
    float *dP = static_cast<float *>(arena.take(sizeof(float) * op.t * op.r));
    const Matrix16 dY = readable(Matrix16{g.dY, g.sdy0, g.sdy1}, op.t, op.n, arena);
    // what a missing gradient alone would read is left alone; the size counts everything
    Matrix16 X{}, Wt{};
    if (!arena.base || g.dA) X = readable(Matrix16{op.x, op.sx0, op.sx1}, op.t, op.k, arena);
    if (!arena.base || g.dX) Wt = readable_w(Matrix16{op.w, op.sw1, op.sw0}, op.n, op.k, arena);
    const WgradPlan plan = lr_wgrad_plan(op.t, op.r, op.s, op.k, op.n,
                                         index.p != nullptr && op.s > 1, drop.cut != 0);
    void *lists = arena.take(plan.list_bytes);
    float *part_a = plan.part[0] ? static_cast<float *>(arena.take(plan.part[0])) : nullptr;
    float *part_b = plan.part[1] ? static_cast<float *>(arena.take(plan.part[1])) : nullptr;
    const Factor16 Bt = readable_factor(Factor16{op.b, op.sb0, op.sb2, op.sb1}, op.s, op.n, op.r,
                                        op.t, arena);
    if (!arena.base) return TI_OK;
    const cudaError_t packed = arena.pack(sms, st);
    if (packed != cudaSuccess) return status(packed);
    const bool half = op.dtype == TI_TYPE_F16;
    if ((g.dX || g.dA) && op.t) {
        const ProjectOperands p{dY,    op.t,     op.n,
                                Bt,
                                op.r,  index,    op.scale,
                                op.alpha * dropout_scale(drop.cut),
                                Dropout{}, dP};
        const ExpandOperands x{dY,   op.t,  op.n, Wt,   op.k, dP, Factor16{op.a, op.sa0, op.sa1, op.sa2},
                               op.r, index, drop, g.dX, g.lddx};
        const cudaError_t e =
            project_expand(half, p, g.dX && op.k ? &x : nullptr, sms, err, st);
        if (e != cudaSuccess) return status(e);
    }
    return status(lr_wgrad(
        half,
        WgradOperand{X, op.k, dP, drop, part_a, g.dA, g.sda[0], g.sda[1], g.sda[2]},
        WgradOperand{dY, op.n, g.P, Dropout{}, part_b, g.dB, g.sdb[0], g.sdb[2], g.sdb[1]}, op.t,
        op.r, index, plan, lists, sms, err, st));
}

bool bad_workspace(const void *ws, size_t have, size_t need) {
    return need && (!ws || have < need || (reinterpret_cast<uintptr_t>(ws) & 255));
}

}  // namespace

int low_rank_context(int *num_sms, int **err) {
    static PerDevice<int> sms;
    static PerDevice<int *> words;
    std::atomic<int> *n = sms.here();
    std::atomic<int *> *w = words.here();
    if (!n || !w) return TI_ERR_NO_DEVICE;
    *err = w->load(std::memory_order_acquire);
    *num_sms = n->load(std::memory_order_acquire);
    if (*err && *num_sms) return TI_OK;
    const int rc = device_context(num_sms, err);
    if (rc != TI_OK) return rc;
    n->store(*num_sms, std::memory_order_release);
    w->store(*err, std::memory_order_release);
    return TI_OK;
}

}  // namespace ti

using namespace ti;

extern "C" {

int ti_low_rank_workspace_size(const ti_low_rank_t *op, size_t *bytes) {
    const int rc = check_op(op);
    if (rc != TI_OK || !bytes) return rc != TI_OK ? rc : TI_ERR_INVALID_ARGUMENT;
    Arena count{};
    forward(*op, nullptr, 0, nullptr, count, 0, nullptr, nullptr);
    *bytes = count.used;
    return TI_OK;
}

int ti_low_rank_backward_workspace_size(const ti_low_rank_t *op, const void *dY, int64_t sdy0,
                                        int64_t sdy1, size_t *bytes) {
    const int rc = check_op(op);
    if (rc != TI_OK || !bytes) return rc != TI_OK ? rc : TI_ERR_INVALID_ARGUMENT;
    Arena count{};
    Gradient g{};
    g.dY = dY;
    g.sdy0 = sdy0;
    g.sdy1 = sdy1;
    backward(*op, g, count, 0, nullptr, nullptr);
    *bytes = count.used;
    return TI_OK;
}

int ti_low_rank_matmul(const ti_low_rank_t *op, void *Y, int64_t ldy, float *P, void *workspace,
                       size_t workspace_bytes, void *stream) {
    size_t need = 0;
    int rc = ti_low_rank_workspace_size(op, &need);
    if (rc != TI_OK) return rc;
    int sms = 0, *err = nullptr;
    if ((rc = low_rank_context(&sms, &err)) != TI_OK) return rc;
    if (op->t == 0) return TI_OK;
    if ((op->k && (!op->x || !op->a || (op->n && !op->w))) || (op->n && (!op->b || !Y)) ||
        ldy < op->n)
        return TI_ERR_INVALID_ARGUMENT;
    if (bad_workspace(workspace, workspace_bytes, need)) return TI_ERR_WORKSPACE;
    Arena arena{static_cast<uint8_t *>(workspace), 0, {}};
    return forward(*op, Y, ldy, P, arena, sms, err, static_cast<cudaStream_t>(stream));
}

int ti_low_rank_backward(const ti_low_rank_t *op, const void *dY, int64_t sdy0, int64_t sdy1,
                         const float *P, void *dX, int64_t lddx, void *dA, int64_t sda0,
                         int64_t sda1, int64_t sda2, void *dB, int64_t sdb0, int64_t sdb1,
                         int64_t sdb2, void *workspace, size_t workspace_bytes, void *stream) {
    size_t need = 0;
    int rc = ti_low_rank_backward_workspace_size(op, dY, sdy0, sdy1, &need);
    if (rc != TI_OK) return rc;
    int sms = 0, *err = nullptr;
    if ((rc = low_rank_context(&sms, &err)) != TI_OK) return rc;
    if ((op->k && !op->a) || (op->n && !op->b) ||
        (op->t && ((op->k && !op->x) || (op->n && !dY) || (op->k && op->n && dX && !op->w) ||
                   (dB && !P))))
        return TI_ERR_INVALID_ARGUMENT;
    if (dX && lddx < op->k) return TI_ERR_INVALID_ARGUMENT;
    if (bad_workspace(workspace, workspace_bytes, need)) return TI_ERR_WORKSPACE;
    const Gradient g{dY, sdy0, sdy1, P, dX, lddx, dA, {sda0, sda1, sda2}, dB, {sdb0, sdb1, sdb2}};
    // a call without rows may come without a workspace: there is nothing to pack then
    alignas(256) static uint8_t none[256];
    Arena arena{workspace ? static_cast<uint8_t *>(workspace) : none, 0, {}};
    return backward(*op, g, arena, sms, err, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
