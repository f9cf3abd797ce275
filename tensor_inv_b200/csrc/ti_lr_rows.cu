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
// For up to kFuseRows rows the projection is made here as well: each CTA of a cluster takes its
// share of the inner dimension, and the one that serves a row adds the shares.  Every column tile
// repeats that work, but for so few rows it is small against W and hides behind its copies, and
// one launch is left of two.  Otherwise the projection runs before, and this kernel may start
// before it has finished (programmatic launch): copies of M and W, which the projection only
// reads, begin at once, and P is waited for where it is needed.
//
// Roles: warp 0 copies, warp 1 TMEM and MMA issue, warps 2..9 low-rank term and epilogue (two
// groups of 128 threads, one thread per column, that share the rows).
#include <atomic>
#include <cstring>
#include <type_traits>

#include "ti_lr_dot.cuh"
#include "ti_lr_launch.cuh"

namespace ti {
namespace {

constexpr int kCols = 128, kBK = 64;
constexpr int kLowWarps = 8, kLowThreads = 32 * kLowWarps;
constexpr int kThreads = 64 + kLowThreads;
constexpr int kMaxRank = 256;
constexpr int kWBytes = kCols * kBK * 2;  // 16 KB

template <int kNT, bool kFused>
struct Shape {
    static constexpr int kMBytes = kNT * kBK * 2;
    static constexpr int kStageBytes = kWBytes + kMBytes;
    static constexpr int kPartBytes = kNT * kCols * 4;
    // the projection's sums by warp and in all, for the rows of the fused form
    static constexpr int kFuseBytes = kFused ? kFuseRows * kMaxRank * 4 * (kLowWarps + 2) : 0;
    static constexpr int kStages = kFused ? 8 : kNT <= 32 ? 9 : kNT == 64 ? 7 : 4;
    static constexpr size_t kSmem = size_t(kStages) * kStageBytes + kPartBytes + kFuseBytes + 1024 +
                                    512 + sizeof(int) * kNT;
    static constexpr uint32_t kTmemCols = kNT < 32 ? 32 : kNT;
};

struct Params {
    int64_t rows, cols;
    int num_kb, per_rank;  // steps of the inner dimension, and how many each rank takes
    int row_tiles;
    int w_nmajor;
    uint32_t idesc;
    float *P;              // the projection; fused: written if not null
    int64_t r;
    Factor16 F;
    int fmode, pvec;       // F in vectors along the rank (kFR); P's rows in vectors of 4
    // fused form: the projection's own operands
    const void *M;
    int64_t ldm, inner;
    Factor16 G;
    int gmode;
    const float *scale;
    float alpha;
    Dropout gdrop;
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

__device__ __forceinline__ void low_sync() {
    asm volatile("bar.sync 1, %0;" ::"n"(kLowThreads) : "memory");
}

// sum_j p[u][j] F[i[u]][c][j] for up to four rows at once (their loads overlap); rows without an
// adapter, or a column past the end, give 0.
template <typename T>
__device__ __forceinline__ void low_rank(const Params &P, const float *const (&p)[4],
                                         const int (&i)[4], int64_t c, float (&acc)[4]) {
    const T *f[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        acc[u] = 0.0f;
        f[u] = static_cast<const T *>(P.F.p) + max(i[u], 0) * P.F.ss + c * P.F.sc;
    }
    if (c >= P.cols) return;
    const int r = static_cast<int>(P.r);
#pragma unroll 2
    for (int j0 = 0; j0 < r; j0 += 8) {
        const bool whole = j0 + 8 <= r;
        uint4 x[4];
        float v[4][8], w[4][8];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            if (P.fmode == kFR) {
                x[u] = make_uint4(0, 0, 0, 0);
                if (i[u] >= 0)
                    x[u] = load8(reinterpret_cast<const uint16_t *>(f[u] + j0), r - j0);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    v[u][e] = i[u] >= 0 && j0 + e < r ? to_float(f[u][(j0 + e) * P.F.sr]) : 0.0f;
            }
            if (P.pvec && whole) {
                const float4 a = *reinterpret_cast<const float4 *>(p[u] + j0);
                const float4 b = *reinterpret_cast<const float4 *>(p[u] + j0 + 4);
                w[u][0] = a.x, w[u][1] = a.y, w[u][2] = a.z, w[u][3] = a.w;
                w[u][4] = b.x, w[u][5] = b.y, w[u][6] = b.z, w[u][7] = b.w;
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) w[u][e] = j0 + e < r ? p[u][j0 + e] : 0.0f;
            }
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            if (i[u] < 0) continue;
            if (P.fmode == kFR) unpack8<T>(x[u], v[u]);
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[u] += w[u][e] * v[u][e];
        }
    }
}

template <typename T, int kNT, bool kDrop, bool kFused>
__global__ void __launch_bounds__(kThreads, 1)
    lr_rows_kernel(const __grid_constant__ CUtensorMap tmM, const __grid_constant__ CUtensorMap tmW,
                   const __grid_constant__ Params P) {
    using S = Shape<kNT, kFused>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>(
        (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *sW = smem;
    uint8_t *sM = sW + S::kStages * kWBytes;
    float *part = reinterpret_cast<float *>(sM + S::kStages * S::kMBytes);  // [kNT][128]
    float *fuse = part + kNT * kCols;                // [kLowWarps][kFuseRows][kMaxRank]
    float *slice_sum = fuse + kLowWarps * kFuseRows * kMaxRank;  // [kFuseRows][kMaxRank]
    float *projection = slice_sum + kFuseRows * kMaxRank;        // [kFuseRows][kMaxRank]
    uint64_t *full = reinterpret_cast<uint64_t *>(fuse + S::kFuseBytes / 4);
    uint64_t *empty = full + S::kStages;
    uint64_t *tfull = empty + S::kStages;
    uint64_t *drain = tfull + 1;
    uint64_t *sums = drain + 1;  // fused: every CTA's slice of the projection is in place
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(sums + 1);
    volatile int *abort = reinterpret_cast<volatile int *>(tmem_slot + 1);
    int *sidx = const_cast<int *>(abort) + 1;  // [kNT] adapters of the tile's rows

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
        mbar_init(sums, csize);
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
    if (kFused) cluster_sync_all();  // every `sums` is ready for the other CTAs' arrivals
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
        const int group = (warp - 2) >> 2, lt = threadIdx.x - 64;
        const int64_t col = col0 + lc;
        const int here = static_cast<int>(min(int64_t(kNT), P.rows - row0));
        const int c4 = static_cast<int>(csize);
        for (int t = lt; t < here; t += kLowThreads) sidx[t] = P.index.at(row0 + t);
        for (int t = group; t < here; t += 2)
            if (t % c4 != static_cast<int>(rank)) part[t * kCols + lc] = 0.0f;
        low_sync();
        // this group's rows: rank + c4 * (group + 2 * n); their adapters' factors come into L2
        const int first = static_cast<int>(rank) + c4 * group;
        if (P.fmode == kFR && col < P.cols)
            for (int t = first; t < here; t += 2 * c4) {
                const int i = sidx[t];
                if (i < 0) continue;
                const T *f = static_cast<const T *>(P.F.p) + i * P.F.ss + col * P.F.sc;
                for (int j = 0; j < P.r; j += 16)
                    asm volatile("prefetch.global.L2 [%0];" ::"l"(f + j));
            }
        if constexpr (kFused) {
            const int64_t begin = int64_t(kb0) * kBK;
            const int64_t end = min(P.inner, begin + int64_t(steps) * kBK);
            const uint64_t gkey = P.gdrop.cut ? dropout_key(P.gdrop) : 0;
            const int r = static_cast<int>(P.r);
            for (int t = 0; t < here; ++t) {
                const int i = sidx[t];
                if (i < 0) continue;
                const uint16_t *x = static_cast<const uint16_t *>(P.M) + (row0 + t) * P.ldm;
                const uint16_t *g = static_cast<const uint16_t *>(P.G.p) + i * P.G.ss;
                float *dst = fuse + t * kMaxRank;
                if (P.gdrop.cut)
                    dot_slice<T, true, kLowWarps>(x, g, P.G.sc, P.G.sr, P.gmode, r, begin, end,
                                                  P.gdrop, gkey, static_cast<uint32_t>(row0 + t),
                                                  warp - 2, lane, dst, kFuseRows * kMaxRank);
                else
                    dot_slice<T, false, kLowWarps>(x, g, P.G.sc, P.G.sr, P.gmode, r, begin, end,
                                                   P.gdrop, 0, 0, warp - 2, lane, dst,
                                                   kFuseRows * kMaxRank);
            }
            low_sync();
            for (int e = lt; e < here * r; e += kLowThreads) {
                const int t = e / r, j = e % r;
                float v = 0.0f;
                if (sidx[t] >= 0)
                    for (int w = 0; w < kLowWarps; ++w)
                        v += fuse[(w * kFuseRows + t) * kMaxRank + j];
                slice_sum[t * kMaxRank + j] = v;
            }
            low_sync();
            // tell every CTA of the cluster, then add the slices of the rows served here
            if (lt < c4) mbar_arrive_remote(map_to_rank(smem_u32(sums), lt));
            bool ok = mbar_wait_cluster(sums, 0, abort);
            if (!ok) raise(P, abort, kErrTimeoutEpilogue);
            for (int e = lt; ok && e < here * r; e += kLowThreads) {
                const int t = e / r, j = e % r;
                if (t % c4 != static_cast<int>(rank)) continue;
                const int i = sidx[t];
                float v = 0.0f;
                if (i >= 0) {
                    for (int k = 0; k < c4; ++k) v += load_remote(slice_sum + t * kMaxRank + j, k);
                    v *= P.alpha * (P.scale ? P.scale[i] : 1.0f);
                }
                projection[t * kMaxRank + j] = v;
                if (P.P && col0 == 0) P.P[(row0 + t) * P.r + j] = v;
            }
            low_sync();
        } else {
            asm volatile("griddepcontrol.wait;" ::: "memory");  // the projection is complete
        }
        const uint64_t key = kDrop ? dropout_key(P.drop) : 0;
        for (int t0 = first; t0 < here; t0 += 8 * c4) {
            const float *p[4];
            int i[4];
            float acc[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int t = t0 + 2 * c4 * u;
                i[u] = t < here ? sidx[t] : -1;
                const int tc = t < here ? t : t0;
                p[u] = kFused ? projection + tc * kMaxRank : P.P + (row0 + tc) * P.r;
            }
            low_rank<T>(P, p, i, col, acc);
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int t = t0 + 2 * c4 * u;
                if (t >= here) break;
                if (kDrop && i[u] >= 0) {
                    const uint4 bits = dropout_bits(P.drop, key, static_cast<uint32_t>(row0 + t),
                                                    static_cast<uint32_t>(col >> 3));
                    if (!dropout_kept(bits, static_cast<int>(col & 7), P.drop.cut)) acc[u] = 0.0f;
                }
                part[t * kCols + lc] = acc[u];
            }
        }
        low_sync();  // the low-rank parts of both groups are in place
        bool ok = true;
        if (!mbar_wait(tfull, 0, abort)) {
            raise(P, abort, kErrTimeoutEpilogue);
            ok = false;
        }
        __syncwarp();
        tc_fence_after();
        if (__all_sync(0xFFFFFFFFu, ok) && steps > 0) {
            const uint32_t tbase = tmem_base + (static_cast<uint32_t>(q * 32) << 16);
            for (int c = 32 * group; c < here; c += 64) {  // the groups take 32 rows in turn
                uint32_t v[32];
                tmem_ld_32x32b_x32(tbase + c, v);
                tmem_wait_ld();
#pragma unroll
                for (int e = 0; e < 32; ++e)
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
        const int lc = (threadIdx.x - 64) % kCols, group = (threadIdx.x - 64) / kCols;
        const int64_t col = col0 + lc;
        const int here = static_cast<int>(min(int64_t(kNT), P.rows - row0));
        T *out = static_cast<T *>(P.out);
        if (col < P.cols)
            for (int t = static_cast<int>(rank + csize * group); t < here; t += 2 * csize) {
                float v = 0.0f;
                for (uint32_t k = 0; k < csize; ++k) v += load_remote(part + t * kCols + lc, k);
                out[(row0 + t) * P.ldo + col] = from_float<T>(v);
            }
    }
    cluster_sync_all();  // nobody leaves while its part is being read
}

template <typename T, int kNT, bool kDrop, bool kFused>
cudaError_t launch(const CUtensorMap &tmM, const CUtensorMap &tmW, const Params &P, int64_t tiles,
                   int ranks, cudaStream_t stream) {
    using S = Shape<kNT, kFused>;
    auto kernel = lr_rows_kernel<T, kNT, kDrop, kFused>;
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
    cfg.numAttrs = kFused ? 1 : 2;  // the fused form reads what earlier work wrote at once
    return cudaLaunchKernelEx(&cfg, kernel, tmM, tmW, P);
}

template <typename T, int kNT>
cudaError_t expand(const ExpandOperands &o, const ProjectOperands *fuse, int num_sms, int *err,
                   cudaStream_t stream) {
    Params P;
    std::memset(&P, 0, sizeof(P));
    P.rows = o.rows;
    P.cols = o.cols;
    P.num_kb = static_cast<int>((o.inner + kBK - 1) / kBK);
    P.row_tiles = static_cast<int>((o.rows + kNT - 1) / kNT);
    const int64_t tiles = (o.cols + kCols - 1) / kCols * P.row_tiles;
    // as many CTAs per tile as fit in one wave of one CTA per SM, each with some steps to take
    int ranks = 1;
    while (ranks < 8 && tiles * (ranks + 1) <= num_sms && P.num_kb >= 2 * (ranks + 1)) ++ranks;
    P.per_rank = (P.num_kb + ranks - 1) / ranks;
    P.w_nmajor = o.W.s0 != 1;
    const int type = std::is_same<T, __half>::value ? 0 : 1;
    P.idesc = (1u << 4) | (static_cast<uint32_t>(type) << 7) | (static_cast<uint32_t>(type) << 10) |
              (P.w_nmajor ? 1u << 15 : 0u) | (static_cast<uint32_t>(kNT >> 3) << 17) |
              (static_cast<uint32_t>(kCols >> 4) << 24);
    P.P = o.P;
    P.r = o.r;
    P.F = o.F;
    P.fmode = factor_mode(o.F) == kFR ? kFR : kFScalar;
    P.pvec = o.r % 4 == 0 && (reinterpret_cast<uintptr_t>(o.P) & 15) == 0;
    P.index = o.index;
    P.drop = o.drop;
    P.out = o.out;
    P.ldo = o.ldo;
    P.err = err;
    CUtensorMap tmM, tmW;
    if (!make_map16(&tmM, o.M.p, o.inner, o.rows, o.M.s0, kBK, kNT)) return cudaErrorInvalidValue;
    if (P.w_nmajor ? !make_map16(&tmW, o.W.p, o.cols, o.inner, o.W.s0, 64, kBK)
                   : !make_map16(&tmW, o.W.p, o.inner, o.cols, o.W.s1, kBK, kCols))
        return cudaErrorInvalidValue;
    if constexpr (kNT == 16)
        if (fuse) {
            P.M = o.M.p;
            P.ldm = o.M.s0;
            P.inner = o.inner;
            P.G = fuse->F;
            P.gmode = factor_mode(fuse->F);
            P.scale = fuse->scale;
            P.alpha = fuse->alpha;
            P.gdrop = fuse->drop;
            return o.drop.cut ? launch<T, kNT, true, true>(tmM, tmW, P, tiles, ranks, stream)
                              : launch<T, kNT, false, true>(tmM, tmW, P, tiles, ranks, stream);
        }
    return o.drop.cut ? launch<T, kNT, true, false>(tmM, tmW, P, tiles, ranks, stream)
                      : launch<T, kNT, false, false>(tmM, tmW, P, tiles, ranks, stream);
}

template <typename T>
cudaError_t by_rows(const ExpandOperands &o, const ProjectOperands *fuse, int num_sms, int *err,
                    cudaStream_t stream) {
    return o.rows <= 16   ? expand<T, 16>(o, fuse, num_sms, err, stream)
           : o.rows <= 32 ? expand<T, 32>(o, fuse, num_sms, err, stream)
           : o.rows <= 64 ? expand<T, 64>(o, fuse, num_sms, err, stream)
                          : expand<T, 128>(o, fuse, num_sms, err, stream);
}

}  // namespace

cudaError_t lr_expand_rows(bool half, const ExpandOperands &o, const ProjectOperands *fuse,
                           int num_sms, int *err, cudaStream_t stream) {
    return half ? by_rows<__half>(o, fuse, num_sms, err, stream)
                : by_rows<__nv_bfloat16>(o, fuse, num_sms, err, stream);
}

}  // namespace ti
