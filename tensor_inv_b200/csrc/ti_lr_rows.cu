// ti_lr_rows.cu -- the expand form for few rows: out = M W + P F with W's bytes as the bound.
//
// With few rows every element of W is read once and meets a handful of rows, so the kernel is a
// stream of W: its columns stand on the 128-row side of the MMA (D[c][t] = sum_k W[k][c] M[t][k]),
// the rows fill the narrow side (16 to 128 of them), and the inner dimension is split over a
// cluster so that about every SM streams a share.  Rows are served by the cluster's CTAs in turn: a
// CTA sends its part of a row into the serving CTA's shared memory, which adds the parts in rank
// order and stores the row.
//
// The low-rank term is a few multiply-adds per output and runs on the plain cores while the copies
// of W are in flight: thread c of the serving CTA holds column c, and the row's P meets its
// adapter's F in float32.  (Where F's vectors run along the columns, a lane reads four columns of a
// quarter of the ranks: 48 x 4096 x 8192, r = 16, 29 us where 16-bit reads took 49 us, projection not
// counted.)  It reads only the adapters that rows ask for, each once per row, and
// nothing of one row's adapter can reach another row.
//
// The kernel starts while the projection still runs (programmatic launch): W, M, the indices and F,
// which the projection only reads or does not touch, are asked for at once, and P is waited for
// where it is needed.  A stream of W fills the memory system's queues, and a read behind them
// takes several microseconds; so all but the first copies wait until the first rows of F, the one
// dependent chain of reads here, have been asked for.
//
// Measured on a B200, projection and launches included, replayed from a graph over weights larger
// than L2: 4096 x 4096, r = 16: 1 row 13.4 us, 8 rows of 8 adapters 13.6 us, 24 rows 14.6 us;
// 8192 x 8192, 8 rows: 32.5 us (4.1 TB/s of W); 4096 x 8192, 48 rows of 64 adapters: 25 us.
//
// Roles: warp 0 copies, warp 1 TMEM and MMA issue, warps 2..9 low-rank term and epilogue (two
// groups of 128 threads, one thread per column, that share the rows).
#include <atomic>
#include <cstring>
#include <type_traits>

#include "ti_lr_loads.cuh"
#include "ti_lr_launch.cuh"

namespace ti {
namespace {

constexpr int kCols = 128, kBK = 64;
constexpr int kLowWarps = 8, kLowThreads = 32 * kLowWarps;
constexpr int kThreads = 64 + kLowThreads;
constexpr int kWBytes = kCols * kBK * 2;  // 16 KB
constexpr int kEarly = 2;                 // copies that do not wait for the reads of F
constexpr int kBatch = 4;                 // rows of a group whose reads of F overlap
constexpr int kProjBytes = 24 * 1024;     // the served rows' projections, as far as they fit

template <int kNT>
struct Shape {
    static constexpr int kMBytes = kNT * kBK * 2;
    static constexpr int kStageBytes = kWBytes + kMBytes;
    // Parts: [sending CTA][rows served][128], for up to 8 CTAs.  The low-rank term is one more
    // sender, so that nothing is read back to be added to; at 128 rows there is no room for that,
    // and the serving CTA adds its own part to it.
    static constexpr bool kLowApart = kNT < 128;
    static constexpr int kPartBytes = (kLowApart ? 2 * kNT : kNT + 8) * kCols * 4;
    // four stages stream W as fast as nine do
    static constexpr int kStages = 4;
    static constexpr size_t kSmem = size_t(kStages) * kStageBytes + kPartBytes + kProjBytes + 1024 +
                                    256 + sizeof(int) * kNT;
    static constexpr uint32_t kTmemCols = kNT < 32 ? 32 : kNT;
};

struct Params {
    int64_t rows, cols;
    int num_kb, per_rank;  // steps of the inner dimension, and how many each rank takes
    int row_tiles;
    int w_nmajor;
    uint32_t idesc;
    const float *P;
    int r;
    Factor16 F;
    int fvec, pvec;        // F in vectors of 8 along the rank; P's rows in vectors of 4
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

// 16 bytes, in program order with the barriers around it.
__device__ __forceinline__ uint4 load_ordered(const void *p) {
    uint4 v;
    asm volatile("ld.global.nc.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(p)
                 : "memory");
    return v;
}

// F[i][c][j0 .. j0+16) of kBatch rows' adapters, as 16-bit values; zeros where there are none.
template <typename T>
__device__ __forceinline__ void load_factors(const Params &P, const int (&i)[kBatch], int64_t c,
                                             int j0, uint4 (&f)[kBatch][2]) {
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
        const uint16_t *src = static_cast<const uint16_t *>(P.F.p) + max(i[u], 0) * P.F.ss +
                              c * P.F.sc + j0 * P.F.sr;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int n = i[u] >= 0 && c < P.cols ? P.r - j0 - 8 * h : 0;
            f[u][h] = make_uint4(0, 0, 0, 0);
            if (P.fvec && n >= 8) {
                f[u][h] = load_ordered(src + 8 * h);
            } else if (n > 0) {
                uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (e < n)
                        w[e >> 1] |= static_cast<uint32_t>(__ldg(src + (8 * h + e) * P.F.sr))
                                     << (16 * (e & 1));
                f[u][h] = make_uint4(w[0], w[1], w[2], w[3]);
            }
        }
    }
}

// F[i][c .. c+4)[j .. j+4) of kBatch rows' adapters (F's vectors run along the columns).
__device__ __forceinline__ void load_columns(const Params &P, const int (&i)[kBatch], int64_t c,
                                             int j, uint2 (&f)[kBatch][4]) {
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
        const uint16_t *src = static_cast<const uint16_t *>(P.F.p) + max(i[u], 0) * P.F.ss + c;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            f[u][e] = make_uint2(0, 0);
            if (i[u] < 0 || j + e >= P.r) continue;
            const uint16_t *q = src + (j + e) * P.F.sr;
            if (c + 4 <= P.cols) {
                asm volatile("ld.global.nc.v2.u32 {%0, %1}, [%2];"
                             : "=r"(f[u][e].x), "=r"(f[u][e].y)
                             : "l"(q)
                             : "memory");
            } else {
#pragma unroll
                for (int d = 0; d < 3; ++d)
                    if (c + d < P.cols)
                        (d < 2 ? f[u][e].x : f[u][e].y) |= static_cast<uint32_t>(__ldg(q + d))
                                                           << (16 * (d & 1));
            }
        }
    }
}

// (Registers are held to what lets a CTA start beside two CTAs of the projection.)
template <typename T, int kNT, bool kDrop, bool kCol>
__global__ void __launch_bounds__(kThreads, 2)
    lr_rows_kernel(const __grid_constant__ CUtensorMap tmM, const __grid_constant__ CUtensorMap tmW,
                   const __grid_constant__ Params P) {
    using S = Shape<kNT>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>(
        (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *sW = smem;
    uint8_t *sM = sW + S::kStages * kWBytes;
    float *part = reinterpret_cast<float *>(sM + S::kStages * S::kMBytes);
    float *proj = part + S::kPartBytes / 4;
    uint64_t *full = reinterpret_cast<uint64_t *>(proj + kProjBytes / 4);
    uint64_t *empty = full + S::kStages;
    uint64_t *tfull = empty + S::kStages;
    uint64_t *drain = tfull + 1;
    uint64_t *asked = drain + 1;  // the first reads of F are on their way
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(asked + 1);
    volatile int *abort = reinterpret_cast<volatile int *>(tmem_slot + 1);
    int *sidx = const_cast<int *>(abort) + 1;  // [kNT] adapters of the tile's rows

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = static_cast<int>(cluster_rank()), csize = static_cast<int>(cluster_size());
    const int64_t tile = blockIdx.x / csize;
    // neighbouring clusters share W's columns, so a second row tile finds them in L2
    const int64_t row0 = tile % P.row_tiles * kNT, col0 = tile / P.row_tiles * kCols;
    const int kb0 = rank * P.per_rank;
    const int steps = max(0, min(P.num_kb, kb0 + P.per_rank) - kb0);
    const int here = static_cast<int>(min(int64_t(kNT), P.rows - row0));
    // row t of the tile is the k-th that CTA t % csize serves, k = t / csize; there the parts lie
    // [sending CTA][k][column]
    const int part_rows = (kNT + csize - 1) / csize;

    if (threadIdx.x == 0) {
        prefetch_tensormap(&tmW);
        prefetch_tensormap(&tmM);
        for (int s = 0; s < S::kStages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        mbar_init(tfull, 1);
        mbar_init(drain, 1);
        mbar_init(asked, kLowWarps);
        *abort = 0;
        fence_barrier_init();
    }
    // a row's adapter is asked for now and awaited behind the barrier
    int adapter = -1;
    if (warp >= 2 && static_cast<int>(threadIdx.x) - 64 < here)
        adapter = P.index.at(row0 + threadIdx.x - 64);
    if (warp == 1) {
        tmem_alloc(tmem_slot, S::kTmemCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    cluster_arrive();  // awaited before anything is written to another CTA: it must have started

    if (warp == 0) {
        if (lane == 0) {
            // ---------------- copies ----------------
            int stage = 0, issued = 0;
            uint32_t phase = 0;
            for (; issued < steps; ++issued) {
                if ((issued == kEarly && !mbar_wait(asked, 0, abort)) ||
                    !mbar_wait(&empty[stage], phase ^ 1, abort)) {
                    raise(P, abort, kErrTimeoutProducer);
                    break;
                }
                mbar_arrive_expect_tx(&full[stage], S::kStageBytes);
                const int k0 = (kb0 + issued) * kBK;
                uint8_t *w = sW + stage * kWBytes;
                if (P.w_nmajor) {
                    tma_load_2d(w, &tmW, &full[stage], static_cast<int>(col0), k0);
                    tma_load_2d(w + 8192, &tmW, &full[stage], static_cast<int>(col0) + 64, k0);
                } else {
                    tma_load_2d(w, &tmW, &full[stage], k0, static_cast<int>(col0));
                }
                tma_load_2d(sM + stage * S::kMBytes, &tmM, &full[stage], k0, static_cast<int>(row0));
                if (++stage == S::kStages) {
                    stage = 0;
                    phase ^= 1;
                }
            }
            if (issued < steps)  // gave up: every copy lands before the CTA may exit
                for (int k = max(0, issued - S::kStages); k < issued; ++k)
                    drain_wait(P, &full[k % S::kStages], static_cast<uint32_t>(k / S::kStages) & 1);
        }
        __syncwarp();
        cluster_wait();
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
        __syncwarp();
        cluster_wait();
    } else {
        // ---------------- low-rank term, then this CTA's part of the tile ----------------
        const int q = warp & 3, lc = q * 32 + lane;  // TMEM lane = column of the tile
        const int group = (warp - 2) >> 2, lt = threadIdx.x - 64;
        const int64_t col = col0 + lc;
        float *send = part + rank * part_rows * kCols + lc;
        float *low = S::kLowApart ? part + csize * part_rows * kCols + lc : send;
        const DropoutKeys key(kDrop ? dropout_key(P.drop) : 0);
        if (lt < kNT) sidx[lt] = adapter;
        low_sync();
        // Served row k's projection lies at proj[k * r]; where they do not all fit they are read from
        // memory each time (and every read of a step is waited for).
        const int served = (here - rank + csize - 1) / csize;
        const bool staged = served * P.r * 4 <= kProjBytes;
        // the served rows k = group, group + 2, ..., kBatch of them at a time
        bool waited = false;
        for (int k0 = group; rank + csize * k0 < here || !waited; k0 += 2 * kBatch) {
            int i[kBatch];
            // kCol: a lane takes four columns and a quarter of the ranks
            float acc[kBatch][kCol ? 4 : 1] = {};
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
                const int t = rank + csize * (k0 + 2 * u);
                i[u] = t < here ? sidx[t] : -1;
            }
#pragma unroll 1
            for (int j0 = 0; j0 < P.r; j0 += 16) {
                uint4 f[kBatch][2];
                uint2 fc[kBatch][4];
                const int jc = j0 + 4 * (lane >> 3);  // kCol: the lane's ranks
                if constexpr (kCol)
                    load_columns(P, i, col0 + q * 32 + 4 * (lane & 7), jc, fc);
                else
                    load_factors<T>(P, i, col, j0, f);
                if (!waited) {
                    waited = true;
                    __syncwarp();
                    if (lane == 0) mbar_arrive(asked);
                    // the factors of later rows come as far as L2
                    if (P.fvec && col < P.cols)
                        for (int k = k0 + 2 * kBatch; rank + csize * k < here; k += 2) {
                            const int later = sidx[rank + csize * k];
                            if (later >= 0)
                                asm volatile("prefetch.global.L2 [%0];" ::"l"(
                                    static_cast<const uint16_t *>(P.F.p) + later * P.F.ss +
                                    col * P.F.sc));
                        }
                    asm volatile("griddepcontrol.wait;" ::: "memory");  // the projection is complete
                    if (staged) {
                        for (int e = lt; e < served * P.r; e += kLowThreads)
                            proj[e] = P.P[(row0 + rank + csize * (e / P.r)) * P.r + e % P.r];
                        low_sync();
                    }
                }
#pragma unroll
                for (int u = 0; u < kBatch; ++u) {
                    if (i[u] < 0) continue;
                    const float *p =
                        staged ? proj + (k0 + 2 * u) * P.r + j0
                               : P.P + (row0 + rank + csize * (k0 + 2 * u)) * P.r + j0;
                    if constexpr (kCol) {
                        float w[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            w[e] = jc + e < P.r ? p[4 * (lane >> 3) + e] : 0.0f;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float2 lo = unpack2<T>(fc[u][e].x), hi = unpack2<T>(fc[u][e].y);
                            if (jc + e < P.r) {
                                acc[u][0] += w[e] * lo.x;
                                acc[u][1] += w[e] * lo.y;
                                acc[u][2] += w[e] * hi.x;
                                acc[u][3] += w[e] * hi.y;
                            }
                        }
                        continue;
                    }
                    float v[16];
                    unpack8<T>(f[u][0], *reinterpret_cast<float(*)[8]>(&v[0]));
                    unpack8<T>(f[u][1], *reinterpret_cast<float(*)[8]>(&v[8]));
#pragma unroll
                    for (int e = 0; e < 16; e += 4) {
                        if (P.pvec) {  // r is a multiple of 4
                            if (j0 + e < P.r) {
                                const float4 w = *reinterpret_cast<const float4 *>(p + e);
                                acc[u][0] += w.x * v[e];
                                acc[u][0] += w.y * v[e + 1];
                                acc[u][0] += w.z * v[e + 2];
                                acc[u][0] += w.w * v[e + 3];
                            }
                        } else {
#pragma unroll
                            for (int d = 0; d < 4; ++d)
                                if (j0 + e + d < P.r) acc[u][0] += p[e + d] * v[e + d];
                        }
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
                const int t = rank + csize * (k0 + 2 * u);
                if (t >= here) break;
                float sum = acc[u][0];
                if constexpr (kCol) {
                    // the ranks' quarters added, then each lane its own column
#pragma unroll
                    for (int d = 0; d < 4; ++d) {
                        float x = acc[u][d];
                        x += __shfl_xor_sync(0xFFFFFFFFu, x, 8);
                        x += __shfl_xor_sync(0xFFFFFFFFu, x, 16);
                        x = __shfl_sync(0xFFFFFFFFu, x, lane >> 2);
                        if ((lane & 3) == d) sum = x;
                    }
                }
                if (kDrop && i[u] >= 0) {
                    const uint4 bits = dropout_bits(P.drop, key, static_cast<uint32_t>(row0 + t),
                                                    static_cast<uint32_t>(col >> 3));
                    if (!dropout_kept(bits, static_cast<int>(col & 7), P.drop.cut)) sum = 0.0f;
                }
                low[(k0 + 2 * u) * kCols] = sum;
            }
        }
        cluster_wait();
        if (!S::kLowApart) low_sync();  // both groups' low-rank terms are in place
        bool ok = true;
        if (!mbar_wait(tfull, 0, abort)) {
            raise(P, abort, kErrTimeoutEpilogue);
            ok = false;
        }
        __syncwarp();
        tc_fence_after();
        if (__all_sync(0xFFFFFFFFu, ok)) {
            const uint32_t tbase = tmem_base + (static_cast<uint32_t>(q * 32) << 16);
            for (int c = 32 * group; c < here; c += 64) {  // the groups take 32 rows in turn
                uint32_t v[32];
                tmem_ld_32x32b_x32(tbase + c, v);
                tmem_wait_ld();
                int to = c % csize, k = c / csize;  // row c + e: served by CTA `to`, its k-th
#pragma unroll
                for (int e = 0; e < 32; ++e) {
                    // a CTA without steps has nothing in TMEM
                    const float x = steps > 0 ? __uint_as_float(v[e]) : 0.0f;
                    if (c + e < here) {
                        if (to == rank)
                            send[k * kCols] = S::kLowApart ? x : send[k * kCols] + x;
                        else
                            store_remote(send + k * kCols, to, x);
                    }
                    if (++to == csize) {
                        to = 0;
                        ++k;
                    }
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem_base, S::kTmemCols);
    }
    cluster_sync_all();  // every part has arrived; no remote access follows
    if (warp >= 2) {
        const int lc = (threadIdx.x - 64) % kCols, group = (threadIdx.x - 64) / kCols;
        const int64_t col = col0 + lc;
        T *out = static_cast<T *>(P.out);
        if (col < P.cols)
#pragma unroll 4
            for (int k = group; rank + csize * k < here; k += 2) {
                const float *src = part + k * kCols + lc;
                float v = 0.0f;
#pragma unroll
                for (int c = 0; c < 9; ++c)
                    if (c < csize + S::kLowApart) v += src[c * part_rows * kCols];
                out[(row0 + rank + csize * k) * P.ldo + col] = from_float<T>(v);
            }
    }
}

template <typename T, int kNT, bool kDrop, bool kCol>
cudaError_t launch(const CUtensorMap &tmM, const CUtensorMap &tmW, const Params &P, int64_t tiles,
                   int ranks, cudaStream_t stream) {
    using S = Shape<kNT>;
    auto kernel = lr_rows_kernel<T, kNT, kDrop, kCol>;
    static PerDevice<int> ready;
    std::atomic<int> *set = ready.here();
    if (!set) return cudaErrorInvalidDevice;
    if (!set->load(std::memory_order_acquire)) {
        const cudaError_t e = cudaFuncSetAttribute(
            kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(S::kSmem));
        if (e != cudaSuccess) return e;
        set->store(1, std::memory_order_release);
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
cudaError_t expand(const ExpandOperands &o, int num_sms, int *err, cudaStream_t stream) {
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
    P.r = static_cast<int>(o.r);
    P.F = o.F;
    P.fvec = factor_mode(o.F) == kFR;
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
    if (factor_mode(o.F) == kFC)
        return o.drop.cut ? launch<T, kNT, true, true>(tmM, tmW, P, tiles, ranks, stream)
                          : launch<T, kNT, false, true>(tmM, tmW, P, tiles, ranks, stream);
    return o.drop.cut ? launch<T, kNT, true, false>(tmM, tmW, P, tiles, ranks, stream)
                      : launch<T, kNT, false, false>(tmM, tmW, P, tiles, ranks, stream);
}

template <typename T>
cudaError_t by_rows(const ExpandOperands &o, int num_sms, int *err, cudaStream_t stream) {
    return o.rows <= 16   ? expand<T, 16>(o, num_sms, err, stream)
           : o.rows <= 32 ? expand<T, 32>(o, num_sms, err, stream)
           : o.rows <= 64 ? expand<T, 64>(o, num_sms, err, stream)
                          : expand<T, 128>(o, num_sms, err, stream);
}

}  // namespace

cudaError_t lr_expand_rows(bool half, const ExpandOperands &o, int num_sms, int *err,
                           cudaStream_t stream) {
    return half ? by_rows<__half>(o, num_sms, err, stream)
                : by_rows<__nv_bfloat16>(o, num_sms, err, stream);
}

}  // namespace ti
