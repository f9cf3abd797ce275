// ti_lr_rows.cu -- the expand form for few rows: out = M W + P F with W's bytes as the bound.
//
// With few rows every element of W is read once and meets a handful of rows, so the kernel is a
// stream of W: its columns stand on the 128-row side of the MMA (D[c][t] = sum_k W[k][c] M[t][k]),
// the rows fill the narrow side (16 to 128 of them), and the inner dimension is split over a
// cluster so that about every SM streams a share.  The partial tiles meet in distributed shared
// memory: each CTA adds the cluster's parts of some rows, in rank order, and stores them.
//
// The low-rank term is a few multiply-adds per output and runs on the plain cores while the copies
// of W are in flight: each CTA of the cluster takes every C-th row, thread c holds column c, and
// the row's P meets its adapter's F in float32.  It reads only the adapters that rows ask for, each
// once per row, and nothing of one row's adapter can reach another row.
//
// The kernel may start before the projection has finished (programmatic launch): copies of M and W,
// which the projection only reads, begin at once, and P is waited for where it is needed.
//
// Roles: warp 0 copies, warp 1 TMEM and MMA issue, warps 2..5 low-rank term and epilogue.
#include <atomic>
#include <cstring>
#include <type_traits>

#include "ti_common.cuh"
#include "ti_lr_launch.cuh"

namespace ti {
namespace {

constexpr int kCols = 128, kBK = 64;
constexpr int kThreads = 192;
constexpr int kWBytes = kCols * kBK * 2;  // 16 KB

template <int kNT>
struct Shape {
    static constexpr int kMBytes = kNT * kBK * 2;
    static constexpr int kStageBytes = kWBytes + kMBytes;
    static constexpr int kPartBytes = kNT * kCols * 4;
    static constexpr int kStages = kNT <= 32 ? 9 : kNT == 64 ? 7 : 4;
    static constexpr size_t kSmem = size_t(kStages) * kStageBytes + kPartBytes + 1024 + 256;
    static constexpr uint32_t kTmemCols = kNT < 32 ? 32 : kNT;
};

struct Params {
    int64_t rows, cols;
    int num_kb, per_rank;  // steps of the inner dimension, and how many each rank takes
    int row_tiles;
    int w_nmajor;
    uint32_t idesc;
    const float *P;
    int64_t r;
    Factor16 F;
    int fmode;             // 2: vectors of 8 along the rank, 0: element by element
    RowIndex index;
    Dropout drop;
    void *out;
    int64_t ldo;
    int *err;
};

__device__ __forceinline__ void umma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                         uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}

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

__device__ __forceinline__ void raise(const Params &P, volatile int *abort, int code) {
    *abort = 1;
    atomicCAS(P.err, 0, code);
}

__device__ __forceinline__ void drain_wait(const Params &P, uint64_t *bar, uint32_t parity) {
    const uint32_t a = smem_u32(bar);
    const unsigned long long t0 = globaltimer_ns();
    while (!mbar_try_wait(a, parity)) {
        if (globaltimer_ns() - t0 > kWaitTimeoutNs) {
            atomicCAS(P.err, 0, kErrTimeoutDrain);
            return;
        }
    }
}

template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
    if constexpr (std::is_same<T, __nv_bfloat16>::value)
        return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
    else
        return __half22float2(*reinterpret_cast<const __half2 *>(&w));
}

// sum_j P[t][j] F[i][c][j] for up to four rows at once (their loads overlap); rows without an
// adapter, or a column past the end, give 0.
template <typename T>
__device__ __forceinline__ void low_rank(const Params &P, const int64_t (&t)[4], const int (&i)[4],
                                         int64_t c, float (&acc)[4]) {
    const T *f[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        acc[u] = 0.0f;
        f[u] = static_cast<const T *>(P.F.p) + max(i[u], 0) * P.F.ss + c * P.F.sc;
    }
    if (c >= P.cols) return;
    for (int64_t j0 = 0; j0 < P.r; j0 += 8) {
        float v[4][8];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            if (P.fmode == 2 && j0 + 8 <= P.r) {
                uint4 x = make_uint4(0, 0, 0, 0);
                if (i[u] >= 0) x = __ldg(reinterpret_cast<const uint4 *>(f[u] + j0));
                const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float2 h = unpack2<T>(w[e]);
                    v[u][2 * e] = h.x;
                    v[u][2 * e + 1] = h.y;
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    v[u][e] = i[u] >= 0 && j0 + e < P.r ? to_float(f[u][(j0 + e) * P.F.sr]) : 0.0f;
            }
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (i[u] >= 0) {
                const float *p = P.P + t[u] * P.r + j0;
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (j0 + e < P.r) acc[u] += p[e] * v[u][e];
            }
    }
}

template <typename T, int kNT, bool kDrop>
__global__ void __launch_bounds__(kThreads, 1)
    lr_rows_kernel(const __grid_constant__ CUtensorMap tmM, const __grid_constant__ CUtensorMap tmW,
                   const __grid_constant__ Params P) {
    using S = Shape<kNT>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>(
        (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *sW = smem;
    uint8_t *sM = sW + S::kStages * kWBytes;
    float *part = reinterpret_cast<float *>(sM + S::kStages * S::kMBytes);  // [kNT][128]
    uint64_t *full = reinterpret_cast<uint64_t *>(part + kNT * kCols);
    uint64_t *empty = full + S::kStages;
    uint64_t *tfull = empty + S::kStages;
    uint64_t *drain = tfull + 1;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(drain + 1);
    volatile int *abort = reinterpret_cast<volatile int *>(tmem_slot + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank(), csize = cluster_size();
    const int64_t tile = blockIdx.x / csize;
    // neighbouring clusters share W's columns, so a second row tile finds them in L2
    const int64_t row0 = tile % P.row_tiles * kNT, col0 = tile / P.row_tiles * kCols;
    const int kb0 = static_cast<int>(rank) * P.per_rank;
    const int steps = max(0, min(P.num_kb, kb0 + P.per_rank) - kb0);

    if (threadIdx.x == 0) {
        for (int s = 0; s < S::kStages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        mbar_init(tfull, 1);
        mbar_init(drain, 1);
        *abort = 0;
        fence_barrier_init();
        prefetch_tensormap(&tmM);
        prefetch_tensormap(&tmW);
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, S::kTmemCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;

    if (warp == 0) {
        if (lane == 0) {
            // ---------------- copies ----------------
            int stage = 0;
            uint32_t phase = 0, issued_mask = 0, issued_phase = 0;
            bool ok = true;
            for (int k = 0; k < steps; ++k) {
                if (!mbar_wait(&empty[stage], phase ^ 1, abort)) {
                    raise(P, abort, kErrTimeoutProducer);
                    ok = false;
                    break;
                }
                mbar_arrive_expect_tx(&full[stage], S::kStageBytes);
                const int k0 = (kb0 + k) * kBK;
                uint8_t *w = sW + stage * kWBytes;
                if (P.w_nmajor) {
                    tma_load_2d(w, &tmW, &full[stage], static_cast<int>(col0), k0);
                    tma_load_2d(w + 8192, &tmW, &full[stage], static_cast<int>(col0) + 64, k0);
                } else {
                    tma_load_2d(w, &tmW, &full[stage], k0, static_cast<int>(col0));
                }
                tma_load_2d(sM + stage * S::kMBytes, &tmM, &full[stage], k0, static_cast<int>(row0));
                issued_mask |= 1u << stage;
                issued_phase = (issued_phase & ~(1u << stage)) | (phase << stage);
                if (++stage == S::kStages) {
                    stage = 0;
                    phase ^= 1;
                }
            }
            if (!ok)
                for (int s = 0; s < S::kStages; ++s)
                    if ((issued_mask >> s) & 1) drain_wait(P, &full[s], (issued_phase >> s) & 1);
        }
    } else if (warp == 1) {
        if (lane == 0) {
            // ---------------- MMA issuer ----------------
            int stage = 0;
            uint32_t phase = 0;
            bool ok = true;
            int k = 0;
            for (; k < steps; ++k) {
                if (!mbar_wait(&full[stage], phase, abort)) {
                    raise(P, abort, kErrTimeoutMma);
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint32_t sw = smem_u32(sW + stage * kWBytes);
                const uint64_t wdesc = P.w_nmajor ? make_sw128_mnmajor_desc(sw, 8192)
                                                  : make_sw128_kmajor_desc(sw);
                const uint32_t wstep = P.w_nmajor ? 128 : 2;
                const uint64_t mdesc = make_sw128_kmajor_desc(smem_u32(sM + stage * S::kMBytes));
#pragma unroll
                for (int kk = 0; kk < kBK / 16; ++kk)
                    umma_f16(tmem_base, wdesc + wstep * kk, mdesc + 2 * kk, P.idesc,
                             (k | kk) != 0 ? 1u : 0u);
                umma_commit(&empty[stage]);
                if (++stage == S::kStages) {
                    stage = 0;
                    phase ^= 1;
                }
            }
            if (ok) {
                umma_commit(tfull);
            } else if (k > 0) {
                umma_commit(drain);
                drain_wait(P, drain, 0);
            }
        }
    } else {
        // ---------------- low-rank term, then this CTA's part of the tile ----------------
        const int q = warp & 3, lc = q * 32 + lane;  // TMEM lane = column of the tile
        const int64_t col = col0 + lc;
        asm volatile("griddepcontrol.wait;" ::: "memory");  // the projection is complete
        const uint64_t key = kDrop ? dropout_key(P.drop) : 0;
        const int here = static_cast<int>(min(int64_t(kNT), P.rows - row0));
        for (int t = 0; t < here; ++t)
            if (t % csize != rank) part[t * kCols + lc] = 0.0f;
        for (int t0 = static_cast<int>(rank); t0 < here; t0 += 4 * csize) {
            int64_t t[4];
            int i[4];
            float acc[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int lt = t0 + u * static_cast<int>(csize);
                t[u] = row0 + lt;
                i[u] = lt < here ? P.index.at(t[u]) : -1;
            }
            low_rank<T>(P, t, i, col, acc);
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int lt = t0 + u * static_cast<int>(csize);
                if (lt >= here) break;
                if (kDrop && i[u] >= 0) {
                    const uint4 bits = dropout_bits(P.drop, key, static_cast<uint32_t>(t[u]),
                                                    static_cast<uint32_t>(col >> 3));
                    if (!dropout_kept(bits, static_cast<int>(col & 7), P.drop.cut)) acc[u] = 0.0f;
                }
                part[lt * kCols + lc] = acc[u];
            }
        }
        bool ok = true;
        if (!mbar_wait(tfull, 0, abort)) {
            raise(P, abort, kErrTimeoutEpilogue);
            ok = false;
        }
        __syncwarp();
        tc_fence_after();
        if (__all_sync(0xFFFFFFFFu, ok) && steps > 0) {
            const uint32_t tbase = tmem_base + (static_cast<uint32_t>(q * 32) << 16);
            constexpr int kLoad = kNT < 32 ? kNT : 32;
            for (int c = 0; c < here; c += kLoad) {
                uint32_t v[32];
                tmem_ld_32x32b_x32(tbase + c, v);
                tmem_wait_ld();
#pragma unroll
                for (int e = 0; e < kLoad; ++e)
                    if (c + e < here) part[(c + e) * kCols + lc] += __uint_as_float(v[e]);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem_base, S::kTmemCols);
    }
    cluster_sync_all();  // every CTA's part is written
    if (warp >= 2) {
        const int lc = threadIdx.x - 64;
        const int64_t col = col0 + lc;
        const int here = static_cast<int>(min(int64_t(kNT), P.rows - row0));
        T *out = static_cast<T *>(P.out);
        if (col < P.cols)
            for (int t = static_cast<int>(rank); t < here; t += csize) {
                float v = 0.0f;
                for (uint32_t k = 0; k < csize; ++k) v += load_remote(part + t * kCols + lc, k);
                out[(row0 + t) * P.ldo + col] = from_float<T>(v);
            }
    }
    cluster_sync_all();  // nobody leaves while its part is being read
}

template <typename T, int kNT, bool kDrop>
cudaError_t launch(const CUtensorMap &tmM, const CUtensorMap &tmW, const Params &P, int64_t tiles,
                   int ranks, cudaStream_t stream) {
    using S = Shape<kNT>;
    auto kernel = lr_rows_kernel<T, kNT, kDrop>;
    constexpr int kMaxDev = 64;
    static std::atomic<int> configured[kMaxDev];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= kMaxDev) return cudaErrorInvalidDevice;
    if (!configured[dev].load(std::memory_order_acquire)) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 static_cast<int>(S::kSmem));
        if (e != cudaSuccess) return e;
        configured[dev].store(1, std::memory_order_release);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(tiles * ranks));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = S::kSmem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ranks;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kernel, tmM, tmW, P);
}

template <typename T, int kNT>
cudaError_t expand(const Matrix16 &M, int64_t rows, int64_t inner, const Matrix16 &W, int64_t cols,
                   const float *Pj, const Factor16 &F, int64_t r, const RowIndex &index,
                   const Dropout &drop, void *out, int64_t ldo, int num_sms, int *err,
                   cudaStream_t stream) {
    Params P;
    std::memset(&P, 0, sizeof(P));
    P.rows = rows;
    P.cols = cols;
    P.num_kb = static_cast<int>((inner + kBK - 1) / kBK);
    P.row_tiles = static_cast<int>((rows + kNT - 1) / kNT);
    const int64_t tiles = (cols + kCols - 1) / kCols * P.row_tiles;
    // as many CTAs per tile as fit in one wave of one CTA per SM, each with some steps to take
    int ranks = 1;
    while (ranks < 8 && tiles * (ranks + 1) <= num_sms && P.num_kb >= 2 * (ranks + 1)) ++ranks;
    P.per_rank = (P.num_kb + ranks - 1) / ranks;
    P.w_nmajor = W.s0 != 1;
    const int type = std::is_same<T, __half>::value ? 0 : 1;
    P.idesc = (1u << 4) | (static_cast<uint32_t>(type) << 7) | (static_cast<uint32_t>(type) << 10) |
              (P.w_nmajor ? 1u << 15 : 0u) | (static_cast<uint32_t>(kNT >> 3) << 17) |
              (static_cast<uint32_t>(kCols >> 4) << 24);
    P.P = Pj;
    P.r = r;
    P.F = F;
    P.fmode = F.sr == 1 && F.sc % 8 == 0 && F.ss % 8 == 0 &&
                      (reinterpret_cast<uintptr_t>(F.p) & 15) == 0
                  ? 2
                  : 0;
    P.index = index;
    P.drop = drop;
    P.out = out;
    P.ldo = ldo;
    P.err = err;
    CUtensorMap tmM, tmW;
    if (!make_map16(&tmM, M.p, inner, rows, M.s0, kBK, kNT)) return cudaErrorInvalidValue;
    if (P.w_nmajor ? !make_map16(&tmW, W.p, cols, inner, W.s0, 64, kBK)
                   : !make_map16(&tmW, W.p, inner, cols, W.s1, kBK, kCols))
        return cudaErrorInvalidValue;
    return drop.cut ? launch<T, kNT, true>(tmM, tmW, P, tiles, ranks, stream)
                    : launch<T, kNT, false>(tmM, tmW, P, tiles, ranks, stream);
}

template <typename T, typename... Args>
cudaError_t by_rows(int64_t rows, Args &&...args) {
    return rows <= 16   ? expand<T, 16>(args...)
           : rows <= 32 ? expand<T, 32>(args...)
           : rows <= 64 ? expand<T, 64>(args...)
                        : expand<T, 128>(args...);
}

}  // namespace

cudaError_t lr_expand_rows(bool half, const Matrix16 &M, int64_t rows, int64_t inner,
                           const Matrix16 &W, int64_t cols, const float *P, const Factor16 &F,
                           int64_t r, const RowIndex &index, const Dropout &drop, void *out,
                           int64_t ldo, int num_sms, int *err, cudaStream_t stream) {
    return half ? by_rows<__half>(rows, M, rows, inner, W, cols, P, F, r, index, drop, out, ldo,
                                  num_sms, err, stream)
                : by_rows<__nv_bfloat16>(rows, M, rows, inner, W, cols, P, F, r, index, drop, out,
                                         ldo, num_sms, err, stream);
}

}  // namespace ti
