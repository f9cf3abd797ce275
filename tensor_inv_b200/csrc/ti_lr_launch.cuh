// ti_lr_launch.cuh -- the launchers of the low-rank products' kernels.
#pragma once

#include <cuda.h>

#include <atomic>

#include "ti_low_rank.cuh"

namespace ti {

// One word per device, zero at first: what a launcher has set up or found out there.  Threads that
// race on the first call of a device do the same work twice, which is harmless.
template <typename T>
struct PerDevice {
    static constexpr int kMaxDev = 64;
    std::atomic<T> word[kMaxDev] = {};
    // the current device's word, or null
    std::atomic<T> *here() {
        int dev = 0;
        if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDev) return nullptr;
        return &word[dev];
    }
};

// SM count and error word of the current device (asked for once per device); a TI_* status.
int low_rank_context(int *num_sms, int **err);

// Tensor map of a matrix of 16-bit elements, `outer` rows of `inner` contiguous ones `ld` apart,
// 128-byte swizzle; base and rows 16-byte aligned.
bool make_map16(CUtensorMap *map, const void *base, int64_t inner, int64_t outer, int64_t ld,
                int box_inner, int box_outer);

// Whether a copy engine can read the matrix as `rows` rows of contiguous elements.
inline bool copyable(const void *p, int64_t rows, int64_t ld, int64_t s_inner, int64_t inner) {
    return (inner <= 1 || s_inner == 1) && (reinterpret_cast<uintptr_t>(p) & 15) == 0 &&
           (rows <= 1 || (ld % 8 == 0 && ld >= inner));
}

// Up to these many rows, project runs a cluster per row and expand streams W past the rows; above
// them, project takes tiles of 128 rows and expand tiles of 256 on CTA pairs.
// One adapter: 4096 x 4096, r = 16, expand on pairs against rows: 128 rows 32 against 21 us, 256 rows
// 34 against 33 us.
// Several: a tile multiplies with every adapter that any of its rows takes, which in a batch of short
// requests is all of them, while the rows' cost does not depend on it.  Both kernels together, tiles
// against rows, r = 16: 512 rows of 64 adapters in any order 205 against 78 us, in order (8 rows each)
// 108 against 78 us; of 16 adapters 89 against 77 us and 55 against 76 us; r = 64, 64 adapters: 462
// against 298 us and 231 against 254 us.  1024 rows of 64 adapters in order: 80 against 147 us.
// The index is on the device, so the rule goes by the adapters passed, not by those that rows take,
// and leaves the rank out: 512 rows that all take one of 64 adapters lose by it, 70 us against the 34 us
// of tiles at r = 16, 230 against 41 us at r = 64, 787 against 55 us at r = 256 (passing that adapter
// alone gives the tiles).
inline int64_t many_adapter_rows(int64_t adapters) {
    return adapters < 32 ? 256 : adapters < 64 ? 8 * adapters : 512;
}
inline int64_t project_rows_limit(int64_t adapters) { return many_adapter_rows(adapters); }
inline int64_t expand_rows_limit(int64_t adapters) {
    return adapters > 1 ? many_adapter_rows(adapters) : 128;
}

// How a factor is read: element by element, in 16-byte vectors along c, or along the rank.
enum { kFScalar = 0, kFC = 1, kFR = 2 };

inline int factor_mode(const Factor16 &F) {
    // (a copy engine's strides are not negative)
    const bool base = (reinterpret_cast<uintptr_t>(F.p) & 15) == 0 && F.ss % 8 == 0 && F.ss >= 0;
    if (base && F.sc == 1 && F.sr % 8 == 0 && F.sr > 0) return kFC;
    if (base && F.sr == 1 && F.sc % 8 == 0 && F.sc > 0) return kFR;
    return kFScalar;
}

// P = f (m M) F: the rows' projections, F a factor along M's inner dimension.
struct ProjectOperands {
    Matrix16 M;  // unit s1, copyable
    int64_t rows, cols;
    Factor16 F;
    int64_t r;
    RowIndex index;
    const float *scale;
    float alpha;
    Dropout drop;
    float *P;
};
// With more than project_rows_limit rows the copy engine reads F: factor_mode(F) != kFScalar.
cudaError_t lr_project(bool half, const ProjectOperands &o, int num_sms, int *err,
                       cudaStream_t stream);

// out = M W + m (P F), F a factor along out's columns.
struct ExpandOperands {
    Matrix16 M;  // unit s1, copyable
    int64_t rows, inner;
    Matrix16 W;  // one unit stride, copyable
    int64_t cols;
    float *P;
    Factor16 F;
    int64_t r;
    RowIndex index;
    Dropout drop;
    void *out;
    int64_t ldo;
};
// 256-row tiles on CTA pairs (ti_lr_gemm.cu)
cudaError_t lr_expand_pairs(bool half, const ExpandOperands &o, int *err, cudaStream_t stream);
// W streamed past a few rows (ti_lr_rows.cu); launched directly behind the projection that makes
// o.P, whose other operands it reads before that has finished.
cudaError_t lr_expand_rows(bool half, const ExpandOperands &o, int num_sms, int *err,
                           cudaStream_t stream);

// The gradients of the adapters (ti_lr_wgrad.cu).
struct WgradPlan {
    int64_t chunk[2], chunks[2];      // rows per chunk and their number, for dA and dB
    size_t list_bytes, part[2];       // workspace
};
WgradPlan lr_wgrad_plan(int64_t rows, int64_t r, int64_t s, int64_t cols_a, int64_t cols_b,
                        bool listed, bool dropped);

// out[s][c][j] = sum over adapter s's rows of m(t, c) M[t][c] V[t][j]; out null: not computed
struct WgradOperand {
    Matrix16 M;  // unit s1, copyable
    int64_t cols;
    const float *V;
    Dropout drop;
    float *part;
    void *out;
    int64_t ss, sc, sr;
};
cudaError_t lr_wgrad(bool half, const WgradOperand &a, const WgradOperand &b, int64_t rows,
                     int64_t r, const RowIndex &index, const WgradPlan &plan, void *lists,
                     int num_sms, int *err, cudaStream_t stream);

}  // namespace ti
