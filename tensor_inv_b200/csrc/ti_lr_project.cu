// ti_lr_project.cu -- the project form: P[t] = f * (m M)[t] F[i], i = index[t].
//
//   P[t][j] = alpha * scale[i] * sum_c m(t, c) M[t][c] F[i][c][j]        (float32, t x r)
//
// One pass over M, 2 r operations per element against 2 bytes: M's bytes bound it.
//   tiles: 128 rows x a slice of the inner dimension per CTA, M and F staged by the copy engine, the
//          products on tcgen05 with up to 64 ranks per MMA.  Each distinct adapter among the rows
//          has its own accumulator columns, so M is read once for all of them (those that fit a
//          stage: four at 64 ranks, more at fewer; the rest take further passes, from L2); a row
//          keeps the columns of its own adapter, and nothing
//          of another reaches it.  With dropout, the mask is applied to the staged tile between
//          the copy and the MMA.  A cluster of up to 8 CTAs shares the rows; each sends its sums
//          to the CTA that finishes the row, which adds them in rank order.
//   rows:  one row per cluster, plain multiply-adds: for few rows each with an adapter of its own
//          F's bytes bound it, and no product is shared between rows.
//
// Measured on a B200, launch included: 4096 x 4096, r = 16: 14.4 us (2.3 TB/s of M), with dropout
// 20.6 us (the mask's integer work); 16384 x 4096, r = 16: 35 us (3.8 TB/s); 8192 x 8192, r = 32: 36 us.
// What holds the shorter ones back is the few stages that each CTA runs through, not the memory.  Rows
// of 16 adapters in random order (4096 x 4096, r = 16) take 51 us: every tile meets every adapter.
#include <atomic>
#include <cstring>

#include "ti_lr_loads.cuh"
#include "ti_lr_launch.cuh"

namespace ti {
namespace {

struct ProjectParams {
    const void *M;
    int64_t ld, rows, cols;
    Factor16 F;
    int64_t r;
    RowIndex index;
    const float *scale;
    float alpha;
    Dropout drop;
    float *P;
    int64_t slice;  // inner elements per CTA, a multiple of 256
    int mode;       // how F is read: kFC vectors along c, kFR vectors along j, kFScalar
};

constexpr int kTileRows = 128, kBK = 64;
constexpr int kWorkers = 256, kTileThreads = 64 + kWorkers;  // copies, MMA issue, 8 workers
constexpr int kMBytes = kTileRows * kBK * 2, kFBytes = 32768;  // per stage
constexpr int kStageBytes = kMBytes + kFBytes, kStages = 4;
constexpr int kBlockRanks = 64;  // ranks of one CTA
constexpr uint32_t kTmemCols = 256;  // kFBytes / 128 ranks
constexpr size_t kTileSmem = size_t(kStages) * kStageBytes + sizeof(float) * kTileRows * kBlockRanks +
                             1024 + 1024 + 512;

struct TileParams {
    int64_t rows, r;
    RowIndex index;
    const float *scale;
    float alpha;
    Dropout drop;
    float *P;
    int num_kb, per_rank;   // steps of the inner dimension, and how many each rank takes
    int rp;                 // ranks per adapter in TMEM: r, or the block's part, rounded up to 16
    int slots, slot_bytes;  // adapters per pass, and their bytes in a stage
    int along_rank;         // F's vectors run along the rank (N-major operand)
    int one_adapter;        // all adapters are the same memory
    uint32_t idesc;
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

__device__ __forceinline__ void store_cluster4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c,
                                               uint32_t d) {
    asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b),
                 "r"(c), "r"(d));
}

__device__ __forceinline__ void raise(const TileParams &P, volatile int *abort, int code) {
    *abort = 1;
    atomicCAS(P.err, 0, code);
}

__device__ __forceinline__ void drain_wait(const TileParams &P, uint64_t *bar, uint32_t parity) {
    const uint32_t a = smem_u32(bar);
    const unsigned long long t0 = globaltimer_ns();
    while (!mbar_try_wait(a, parity)) {
        if (globaltimer_ns() - t0 > kWaitTimeoutNs) {
            atomicCAS(P.err, 0, kErrTimeoutDrain);
            return;
        }
    }
}

// Roles: warp 0 copies, warp 1 TMEM and MMA issue, warps 2..9 the mask and the epilogue.
template <typename T, bool kDrop>
__global__ void __launch_bounds__(kTileThreads, 1)
    project_tiles_kernel(const __grid_constant__ CUtensorMap tmM,
                         const __grid_constant__ CUtensorMap tmF,
                         const __grid_constant__ TileParams P) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t *ring = reinterpret_cast<uint8_t *>(
        (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    // what this CTA finishes: [sending CTA][row of its share][rp]
    float *sum = reinterpret_cast<float *>(ring + kStages * kStageBytes);
    int *sidx = reinterpret_cast<int *>(sum + kTileRows * kBlockRanks);  // [128] rows' adapters
    int *list = sidx + kTileRows;                                        // [128] distinct ones
    uint64_t *full = reinterpret_cast<uint64_t *>(list + kTileRows);
    uint64_t *ready = full + kStages;   // with dropout: the tile is masked
    uint64_t *empty = ready + kStages;
    uint64_t *tfull = empty + kStages;
    uint64_t *tempty = tfull + 1;
    uint64_t *drain = tempty + 1;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(drain + 1);
    volatile int *abort = reinterpret_cast<volatile int *>(tmem_slot + 1);
    int *distinct = const_cast<int *>(abort) + 1;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = static_cast<int>(cluster_rank()), csize = static_cast<int>(cluster_size());
    const int share = kTileRows / csize;  // rows that each CTA finishes
    const int64_t row0 = int64_t(blockIdx.x / csize) * kTileRows;
    const int j0 = static_cast<int>(blockIdx.y) * kBlockRanks;
    const int kb0 = rank * P.per_rank;
    const int steps = max(0, min(P.num_kb, kb0 + P.per_rank) - kb0);

    if (threadIdx.x == 0) {
        prefetch_tensormap(&tmM);
        prefetch_tensormap(&tmF);
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&ready[s], kWorkers / 32);
            mbar_init(&empty[s], 1);
        }
        mbar_init(tfull, 1);
        mbar_init(tempty, 4);
        mbar_init(drain, 1);
        *abort = 0;
        fence_barrier_init();
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, kTmemCols);
        tmem_relinquish();
    }
    if (warp == 2) {
        // the rows' adapters, and the distinct ones in increasing order
        int idx[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int64_t t = row0 + 32 * q + lane;
            idx[q] = t < P.rows ? P.index.at(t) : -1;
            sidx[32 * q + lane] = idx[q];
        }
        int cur = -1, n = 0;
        while (true) {
            unsigned least = 0x7FFFFFFFu;
#pragma unroll
            for (int q = 0; q < 4; ++q)
                if (idx[q] > cur) least = min(least, static_cast<unsigned>(idx[q]));
            least = __reduce_min_sync(0xFFFFFFFFu, least);
            if (least == 0x7FFFFFFFu) break;
            cur = static_cast<int>(least);
            if (lane == 0) list[n] = cur;
            ++n;
        }
        if (lane == 0) *distinct = n;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    const int nd = *distinct;
    cluster_arrive();  // awaited before anything is written to another CTA: it must have started

    if (warp == 0) {
        if (lane == 0) {
            // ---------------- copies ----------------
            int stage = 0;
            uint32_t phase = 0, issued_mask = 0, issued_phase = 0;
            bool ok = true;
            for (int a0 = 0; ok && a0 < nd; a0 += P.slots) {
                const int n = min(P.slots, nd - a0);
                for (int k = 0; k < steps; ++k) {
                    if (!mbar_wait(&empty[stage], phase ^ 1, abort)) {
                        raise(P, abort, kErrTimeoutProducer);
                        ok = false;
                        break;
                    }
                    mbar_arrive_expect_tx(&full[stage], kMBytes + n * P.slot_bytes);
                    const int k0 = (kb0 + k) * kBK;
                    uint8_t *m = ring + stage * kStageBytes;
                    tma_load_2d(m, &tmM, &full[stage], k0, static_cast<int>(row0));
                    for (int a = 0; a < n; ++a) {
                        const int s = P.one_adapter ? 0 : list[a0 + a];
                        uint8_t *f = m + kMBytes + a * P.slot_bytes;
                        if (P.along_rank)
                            tma_load_3d(f, &tmF, &full[stage], j0, k0, s);
                        else
                            tma_load_3d(f, &tmF, &full[stage], k0, j0, s);
                    }
                    issued_mask |= 1u << stage;
                    issued_phase = (issued_phase & ~(1u << stage)) | (phase << stage);
                    if (++stage == kStages) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
            }
            if (!ok)  // every copy lands before the CTA may exit
                for (int s = 0; s < kStages; ++s)
                    if ((issued_mask >> s) & 1) drain_wait(P, &full[s], (issued_phase >> s) & 1);
        }
        __syncwarp();
        cluster_wait();
    } else if (warp == 1) {
        if (lane == 0) {
            // ---------------- MMA issuer ----------------
            int stage = 0;
            uint32_t phase = 0, pass = 0;
            bool ok = true, any_issued = false;
            for (int a0 = 0; ok && a0 < nd; a0 += P.slots, ++pass) {
                const int n = min(P.slots, nd - a0);
                if (!mbar_wait(tempty, (pass & 1) ^ 1, abort)) {
                    raise(P, abort, kErrTimeoutMma);
                    ok = false;
                    break;
                }
                tc_fence_after();
                for (int k = 0; k < steps; ++k) {
                    if (!mbar_wait(kDrop ? &ready[stage] : &full[stage], phase, abort)) {
                        raise(P, abort, kErrTimeoutMma);
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t sm = smem_u32(ring + stage * kStageBytes);
                    const uint64_t mdesc = make_sw128_kmajor_desc(sm);
                    for (int a = 0; a < n; ++a) {
                        const uint32_t sf = sm + kMBytes + a * P.slot_bytes;
                        const uint64_t fdesc = P.along_rank ? make_sw128_mnmajor_desc(sf, 8192)
                                                            : make_sw128_kmajor_desc(sf);
                        const uint32_t fstep = P.along_rank ? 128 : 2;
#pragma unroll
                        for (int kk = 0; kk < kBK / 16; ++kk)
                            umma_f16(tmem_base + a * P.rp, mdesc + 2 * kk, fdesc + fstep * kk,
                                     P.idesc, (k | kk) != 0 ? 1u : 0u);
                    }
                    any_issued = true;
                    umma_commit(&empty[stage]);
                    if (++stage == kStages) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
                if (ok) umma_commit(tfull);
            }
            if (!ok && any_issued) {
                umma_commit(drain);
                drain_wait(P, drain, 0);
            }
        }
        __syncwarp();
        cluster_wait();
    } else {
        // ---------------- the mask, then the epilogue ----------------
        const int wt = threadIdx.x - 64;
        const int q = warp & 3, lr = q * 32 + lane;  // TMEM lane = row of the tile
        const DropoutKeys key(kDrop ? dropout_key(P.drop) : 0);
        const int own = sidx[lr];
        float *dst = sum + (rank * share + lr % share) * P.rp;
        bool started = false;
        int stage = 0;
        uint32_t phase = 0, pass = 0;
        bool ok = true;
        for (int a0 = 0; ok && a0 < nd; a0 += P.slots, ++pass) {
            const int n = min(P.slots, nd - a0);
            if (kDrop) {
                for (int k = 0; k < steps; ++k) {
                    ok = mbar_wait(&full[stage], phase, abort);
                    if (!ok) {
                        raise(P, abort, kErrTimeoutEpilogue);
                        break;
                    }
                    uint8_t *m = ring + stage * kStageBytes;
                    // a thread takes chunk wt % 8 of rows wt / 8, wt / 8 + 32, ...
                    const int chunk = wt & 7;
#pragma unroll
                    for (int h = 0; h < kTileRows / 32; ++h) {
                        const int mr = (wt >> 3) + 32 * h;
                        uint4 *p = reinterpret_cast<uint4 *>(m + mr * 128 + ((chunk ^ (mr & 7)) << 4));
                        *p = masked(*p, P.drop, key, static_cast<uint32_t>(row0 + mr),
                                    static_cast<uint32_t>((kb0 + k) * (kBK / 8) + chunk));
                    }
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&ready[stage]);
                    if (++stage == kStages) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
            }
            // Only the warps that arrive on tempty may wait here: nothing would hold the next pass
            // back for another, and a phase that it missed would leave it two passes behind.
            ok = ok && (warp >= 6 || mbar_wait(tfull, pass & 1, abort));
            if (!ok) raise(P, abort, kErrTimeoutEpilogue);
            ok = __all_sync(0xFFFFFFFFu, ok);
            if (!started) {
                started = true;
                cluster_wait();
            }
            if (ok && warp < 6) {
                tc_fence_after();
                const uint32_t tbase = tmem_base + (static_cast<uint32_t>(q * 32) << 16);
                const uint32_t to = map_to_rank(smem_u32(dst), lr / share);
                for (int a = 0; a < n; ++a) {
                    const bool mine = own == list[a0 + a];
                    if (!__any_sync(0xFFFFFFFFu, mine)) continue;
                    for (int j = 0; j < P.rp; j += 16) {
                        uint32_t v[16];
                        tmem_ld_32x32b_x16(tbase + a * P.rp + j, v);
                        tmem_wait_ld();
                        if (mine) {
                            const uint32_t zero = steps > 0 ? 0xFFFFFFFFu : 0u;  // nothing in TMEM
#pragma unroll
                            for (int e = 0; e < 16; e += 4)
                                store_cluster4(to + 4 * (j + e), v[e] & zero, v[e + 1] & zero,
                                               v[e + 2] & zero, v[e + 3] & zero);
                        }
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(tempty);
            }
        }
        if (!started) cluster_wait();
    }
    // the kernel that reads P may prepare itself now; it waits for this grid before P
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem_base, kTmemCols);
    }
    cluster_sync_all();  // every sum has arrived; no remote access follows
    // the cluster's slices, added in order
    for (int e = threadIdx.x; e < share * P.rp; e += kTileThreads) {
        const int lr = rank * share + e / P.rp, j = j0 + e % P.rp;
        const int64_t t = row0 + lr;
        if (t >= P.rows || j >= P.r) continue;
        const int i = sidx[lr];
        float v = 0.0f;
        if (i >= 0) {
            for (int c = 0; c < csize; ++c) v += sum[c * share * P.rp + e];
            v *= P.alpha * (P.scale ? P.scale[i] : 1.0f);
        }
        P.P[t * P.r + j] = v;
    }
}

// ---------------------------------------------------------------------------------------
// few rows: a cluster per row
// ---------------------------------------------------------------------------------------
constexpr int kRowThreads = 256, kRowWarps = kRowThreads / 32;
constexpr int kMaxRankRows = 256;

// part[w][j] such that its sum over the warps w is sum_{c in [begin, end)} m(t, c) x[c] F[c][j].
// begin is a multiple of 8; the caller synchronises afterwards.  All reads of a step are issued
// before the first is used: a step covers 1024 elements and 16 ranks, the whole of a usual slice.
//   vectors along c, or element by element: a warp takes two ranks, its lanes 8 elements each
//   vectors along the rank: a warp takes an eighth of the slice, its lanes one element each
template <typename T, bool kDrop>
__device__ __forceinline__ void dot_slice(const ProjectParams &P, const uint16_t *x,
                                          const uint16_t *F, int64_t begin, int64_t end,
                                          const DropoutKeys &key, uint32_t row, int warp, int lane,
                                          float (*part)[kMaxRankRows]) {
    const int r = static_cast<int>(P.r);
    if (P.mode == kFR) {
        const int64_t share = (end - begin + 8 * kRowWarps - 1) / (8 * kRowWarps) * 8;
        const int64_t lo = begin + warp * share, hi = min(end, lo + share);
        for (int jb = 0; jb < r; jb += 16) {
            float acc[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) acc[j] = 0.0f;
            for (int64_t c0 = lo + lane; c0 - lane < hi; c0 += 128) {
                uint4 f[4][2];
                float v[4];
#pragma unroll
                for (int s = 0; s < 4; ++s) {
                    const int64_t c = c0 + 32 * s;
                    const bool in = c < hi;
                    v[s] = in ? to_float(*reinterpret_cast<const T *>(x + c)) : 0.0f;
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        f[s][h] = load8(F + (in ? c : lo) * P.F.sc + jb + 8 * h,
                                        in ? r - jb - 8 * h : 0);
                }
#pragma unroll
                for (int s = 0; s < 4; ++s) {
                    const int64_t c = c0 + 32 * s;
                    if (kDrop && c < hi)
                        if (!dropout_kept(dropout_bits(P.drop, key, row, static_cast<uint32_t>(c >> 3)),
                                          static_cast<int>(c & 7), P.drop.cut))
                            v[s] = 0.0f;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float w[8];
                        unpack8<T>(f[s][h], w);
                        // an element past the end is skipped, not multiplied by zero
                        if (c < hi)
#pragma unroll
                            for (int j = 0; j < 8; ++j) acc[8 * h + j] += v[s] * w[j];
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const float v = warp_sum(acc[j]);
                if (lane == 0 && jb + j < r) part[warp][jb + j] = v;
            }
        }
        return;
    }
    for (int jb = 0; jb < r; jb += 2 * kRowWarps) {
        const int j[2] = {jb + warp, jb + warp + kRowWarps};
        float acc[2] = {0.0f, 0.0f};
        for (int64_t c0 = begin + 8 * lane; c0 - 8 * lane < end; c0 += 1024) {
            uint4 xv[4], f[2][4];
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const int64_t c = c0 + 256 * s, n = end - c;
                xv[s] = load8(x + c, n);
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    if (P.mode == kFC) {
                        f[k][s] = load8(F + j[k] * P.F.sr + c, j[k] < r ? n : 0);
                    } else {
                        uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            if (j[k] < r && e < n)
                                w[e >> 1] |= static_cast<uint32_t>(
                                                 __ldg(F + (c + e) * P.F.sc + j[k] * P.F.sr))
                                             << (16 * (e & 1));
                        f[k][s] = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                }
            }
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const int64_t c = c0 + 256 * s;
                if (kDrop) xv[s] = masked(xv[s], P.drop, key, row, static_cast<uint32_t>(c >> 3));
                float v[8], w[8];
                unpack8<T>(xv[s], v);
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    unpack8<T>(f[k][s], w);
#pragma unroll
                    for (int e = 0; e < 8; ++e) acc[k] += v[e] * w[e];
                }
            }
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const float v = warp_sum(acc[k]);
            if (j[k] < r && lane < kRowWarps) part[lane][j[k]] = lane == 0 ? v : 0.0f;
        }
    }
}

template <typename T, bool kDrop>
__global__ void __launch_bounds__(kRowThreads, 3)
    project_rows_kernel(const __grid_constant__ ProjectParams P) {
    __shared__ float part[kRowWarps][kMaxRankRows];
    __shared__ float sum[8][kMaxRankRows];  // in CTA 0: every CTA's slice
    cluster_arrive();  // awaited before anything is written to another CTA: it must have started
    // the kernel that reads P may start its own reads now; it waits for this grid before P
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t crank = cluster_rank(), csize = cluster_size();
    const int64_t t = blockIdx.x / csize;
    const int i = P.index.at(t);
    const int64_t begin = int64_t(crank) * P.slice, end = min(P.cols, begin + P.slice);
    const int r = static_cast<int>(P.r);
    if (i >= 0)
        dot_slice<T, kDrop>(P, static_cast<const uint16_t *>(P.M) + t * P.ld,
                            static_cast<const uint16_t *>(P.F.p) + i * P.F.ss, begin, end,
                            DropoutKeys(kDrop ? dropout_key(P.drop) : 0),
                            static_cast<uint32_t>(t), warp, lane,
                            part);
    cluster_wait();
    __syncthreads();
    for (int j = threadIdx.x; j < r; j += kRowThreads) {
        float v = 0.0f;
        if (i >= 0)
            for (int w = 0; w < kRowWarps; ++w) v += part[w][j];
        store_remote(&sum[crank][j], 0, v);
    }
    cluster_sync_all();
    if (crank == 0)
        for (int j = threadIdx.x; j < r; j += kRowThreads) {
            float v = 0.0f;
            for (uint32_t q = 0; q < csize; ++q) v += sum[q][j];
            P.P[t * P.r + j] = i < 0 ? 0.0f : v * (P.alpha * (P.scale ? P.scale[i] : 1.0f));
        }
}

// Launches a kernel in clusters of `parts`; `ready` is the kernel's own.
template <typename K, typename... Args>
cudaError_t launch_cluster(K kernel, PerDevice<int> &ready, int parts, dim3 grid, int threads,
                           size_t smem, cudaStream_t stream, const Args &...args) {
    std::atomic<int> *set = ready.here();
    if (!set) return cudaErrorInvalidDevice;
    if (!set->load(std::memory_order_acquire)) {
        // An SM whose shared memory is carved out small would have to drain before the
        // expanding kernel's CTAs fit beside this one.
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout,
                                             cudaSharedmemCarveoutMaxShared);
        if (e == cudaSuccess && smem > 48 * 1024)
            e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     static_cast<int>(smem));
        if (e != cudaSuccess) return e;
        set->store(1, std::memory_order_release);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = parts;
    attr.val.clusterDim.y = 1;
    attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

bool make_factor_map(CUtensorMap *map, const Factor16 &F, int mode, int64_t cols, int64_t r,
                     int64_t adapters, int rp) {
    EncodeTiledFn enc = get_encode_fn();
    if (!enc) return false;
    const bool along = mode == kFR;
    const int64_t n_in = along ? r : cols, n_mid = along ? cols : r;
    // (a dimension of one element has no stride of its own)
    const int64_t s_mid = n_mid > 1 ? (along ? F.sc : F.sr) : (n_in + 7) / 8 * 8;
    cuuint64_t dims[3] = {static_cast<cuuint64_t>(n_in), static_cast<cuuint64_t>(n_mid),
                          static_cast<cuuint64_t>(adapters)};
    cuuint64_t strides[2] = {static_cast<cuuint64_t>(2 * s_mid),
                             static_cast<cuuint64_t>(2 * (adapters > 1 ? F.ss : s_mid * n_mid))};
    cuuint32_t box[3] = {64, static_cast<cuuint32_t>(along ? kBK : rp), 1};
    cuuint32_t estr[3] = {1, 1, 1};
    return enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 3, const_cast<void *>(F.p), dims, strides, box,
               estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T>
cudaError_t project_tiles(const ProjectOperands &o, int num_sms, int *err, cudaStream_t stream) {
    const int mode = factor_mode(o.F);
    if (mode == kFScalar) return cudaErrorInvalidValue;  // the caller packs such a factor
    TileParams P;
    std::memset(&P, 0, sizeof(P));
    P.rows = o.rows;
    P.r = o.r;
    P.index = o.index;
    P.scale = o.scale;
    P.alpha = o.alpha;
    P.drop = o.drop;
    P.P = o.P;
    P.err = err;
    P.num_kb = static_cast<int>((o.cols + kBK - 1) / kBK);
    const int64_t blocks = (o.r + kBlockRanks - 1) / kBlockRanks;
    P.rp = o.r >= kBlockRanks ? kBlockRanks : static_cast<int>((o.r + 15) / 16 * 16);
    P.along_rank = mode == kFR;
    P.one_adapter = o.F.ss == 0 || o.index.s == 1;
    P.slot_bytes = P.along_rank ? 128 * kBK : 128 * P.rp;
    P.slots = kFBytes / P.slot_bytes;
    const int type = std::is_same<T, __half>::value ? 0 : 1;
    P.idesc = (1u << 4) | (static_cast<uint32_t>(type) << 7) | (static_cast<uint32_t>(type) << 10) |
              (P.along_rank ? 1u << 16 : 0u) | (static_cast<uint32_t>(P.rp >> 3) << 17) |
              (static_cast<uint32_t>(kTileRows >> 4) << 24);
    // 1, 2, 4 or 8 CTAs share a tile's inner dimension, as long as all fit one per SM.  (Clusters
    // of 8 find room in fewer places: 16 of them do not fit at once, and 2048 x 4096 took 17.6 us
    // with 16 clusters of 8, 4096 x 4096 14.5 us with 32 of 4.)
    const int64_t tile_count = (o.rows + kTileRows - 1) / kTileRows;
    int parts = 1;
    while (parts < 8 && tile_count * blocks * 2 * parts <= (parts == 4 ? num_sms / 2 : num_sms) &&
           P.num_kb >= 4 * parts)
        parts *= 2;
    P.per_rank = (P.num_kb + parts - 1) / parts;
    CUtensorMap tmM, tmF;
    if (!make_map16(&tmM, o.M.p, o.cols, o.rows, o.M.s0, kBK, kTileRows) ||
        !make_factor_map(&tmF, o.F, mode, o.cols, o.r, P.one_adapter ? 1 : o.index.s, P.rp))
        return cudaErrorInvalidValue;
    const dim3 grid(static_cast<unsigned>(parts * tile_count), static_cast<unsigned>(blocks));
    static PerDevice<int> ready[2];
    return o.drop.cut ? launch_cluster(project_tiles_kernel<T, true>, ready[1], parts, grid,
                                       kTileThreads, kTileSmem, stream, tmM, tmF, P)
                      : launch_cluster(project_tiles_kernel<T, false>, ready[0], parts, grid,
                                       kTileThreads, kTileSmem, stream, tmM, tmF, P);
}

template <typename T>
cudaError_t project(const ProjectOperands &o, int num_sms, int *err, cudaStream_t stream) {
    if (o.rows > project_rows_limit(o.index.s) && o.cols > 0)
        return project_tiles<T>(o, num_sms, err, stream);
    ProjectParams P{o.M.p,   o.M.s0,  o.rows,  o.cols, o.F, o.r,
                    o.index, o.scale, o.alpha, o.drop, o.P, 0, factor_mode(o.F)};
    // slices of 1024 (8 elements for each of 128 lanes) until 8 CTAs share a row
    int parts = 1;
    while (parts < 8 && P.cols > 1024 * parts) ++parts;
    P.slice = ((P.cols + parts - 1) / parts + 255) / 256 * 256;
    const dim3 grid(static_cast<unsigned>(parts * P.rows));
    static PerDevice<int> ready[2];
    return P.drop.cut ? launch_cluster(project_rows_kernel<T, true>, ready[1], parts, grid,
                                       kRowThreads, 0, stream, P)
                      : launch_cluster(project_rows_kernel<T, false>, ready[0], parts, grid,
                                       kRowThreads, 0, stream, P);
}

}  // namespace

cudaError_t lr_project(bool half, const ProjectOperands &o, int num_sms, int *err,
                       cudaStream_t stream) {
    return half ? project<__half>(o, num_sms, err, stream)
                : project<__nv_bfloat16>(o, num_sms, err, stream);
}

}  // namespace ti
