// ti_lr_wgrad.cu -- the gradients of the adapters: sums over each adapter's rows.
//
//   dA[s][c][j] = sum_{t: index[t] = s} m(t, c) X[t][c] dP[t][j]
//   dB[s][j][c] = sum_{t: index[t] = s} dY[t][c] P[t][j]
//
// Both are out[s] = M^T V with a wide 16-bit M (rows x cols) and a thin float32 V (rows x r); both
// run in one launch.  M's bytes bound them: each element is read once and meets r values of V.
//
//   lists  one CTA per adapter writes the positions of its rows, in order, so that an adapter's rows
//          are consecutive; no atomics, so the sums have one order.  A single adapter needs none.
//   wgrad  a CTA takes a chunk of that order and 256 columns, in stages of 64 rows.  The copy engine
//          gathers the rows (four row numbers per copy; places without a row get one past the end,
//          which reads as zeros, so that no row of another adapter enters).  M stays as it lies in
//          memory: its columns are the 128-row side of the MMA, read in the orientation whose
//          consecutive elements run along the columns.  Eight warps turn V into the other operand:
//          16-bit values in parts, the rounded value and what is left of it.  Three parts of bf16 hold
//          all 24 bits of V, two of fp16 hold 22 (a sum whose terms cancel keeps what float32 values
//          give it).  For fp16, whose exponents V may leave, each rank's column is first scaled by a
//          power of two that brings its largest value of the CTA's rows to 2^14; the sums are scaled
//          back.  With dropout the same warps mask the staged tile.  Where a chunk crosses from one adapter to
//          the next the sums go to another slot: chunk + adapter numbers the (chunk, adapter) pairs
//          that occur without gaps in either direction.
//   join   adds an adapter's slots in order and rounds once.  One chunk needs no join.
//
// Measured on a B200, the wgrad kernel alone behind the dX pass: 4096 rows, 4096 + 4096 columns, r = 16:
// 27 us (2.5 TB/s of M), 39 us with dropout, 40 us for fp16 (its scales take a pass over V); 8192 rows,
// r = 64: 71 us (25, 38 and 58 us with two parts of bf16).  Copies of four rows at a time cost more than boxes, so 64
// consecutive rows go as one box: the first case's shape with rows of 16 adapters in random order,
// which cannot, takes 57 us.
//
// Infinities and NaN: an infinity in M meets every part of V, and infinity * 0 or infinity - infinity
// is NaN where the formula has an infinity (and a V near float32's end rounds to one).  So a CTA that
// meets a sum that is not finite forms those sums again at its end, by multiply-adds of M and V as
// they are.  A sum that is finite met no infinity in any part.  (8192 rows, 8192 + 8192 columns,
// r = 64, bf16: 218 us; 554 us where all of M is NaN; up to some ms with infinities.)
#include <cstring>

#include "ti_lr_loads.cuh"
#include "ti_lr_launch.cuh"

namespace ti {
namespace {

constexpr int kCtaCols = 256, kRows = 64;     // columns of a CTA, rows of a stage
constexpr int kAtomBytes = kRows * 128;       // 64 columns of a stage
constexpr int kMBytes = 4 * kAtomBytes;
constexpr int kBlockRanks = 64;               // ranks of a CTA
constexpr int kPartBytes = kBlockRanks * 128; // one part of V's stage
constexpr int kStages = 4;
constexpr int kWorkers = 256, kThreads = 64 + kWorkers;
constexpr uint32_t kTmemCols = 128;           // two halves of the columns, 64 ranks each

template <typename T>
struct Stage {
    static constexpr int kParts = std::is_same<T, __half>::value ? 2 : 3;  // of V
    static constexpr int kBytes = kMBytes + kParts * kPartBytes;
    static constexpr size_t kSmem = size_t(kStages) * kBytes + 1024 + 1024;
};

struct Side {
    const void *M;
    int64_t ld, cols;
    const float *V;
    Dropout drop;
    float *part;      // [slot][r][round8(cols)], or null: one chunk, straight to out
    void *out;
    int64_t ss, sc, sr;
    int64_t blocks;   // column blocks of this side; 0: not computed
    int64_t chunk, chunks;  // rows per chunk, and how many
};

struct WgradParams {
    Side side[2];
    int rp;                 // ranks per CTA in TMEM: r, or the block's part, rounded up to 16
    uint32_t idesc;
    int *err;
    int64_t rows, r, s;
    RowIndex index;         // of a single adapter: rows of others are left out
    const int32_t *order;   // row numbers grouped by adapter, or null: all rows, adapter 0
    const int32_t *start;   // [s + 1] first position of each adapter, or null
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

// Four rows of a matrix whose map's box is one row high, 64 columns from c0, one below the other.
__device__ __forceinline__ void tma_gather4(void *dst, const CUtensorMap *map, uint64_t *bar, int c0,
                                            const int (&row)[4]) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %5, %6, %7}], [%2];" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(row[0]), "r"(row[1]),
        "r"(row[2]), "r"(row[3])
        : "memory");
}

__device__ __forceinline__ void raise(const WgradParams &P, volatile int *abort, int code) {
    *abort = 1;
    atomicCAS(P.err, 0, code);
}

__device__ __forceinline__ void drain_wait(const WgradParams &P, uint64_t *bar, uint32_t parity) {
    const uint32_t a = smem_u32(bar);
    const unsigned long long t0 = globaltimer_ns();
    while (!mbar_try_wait(a, parity)) {
        if (globaltimer_ns() - t0 > kWaitTimeoutNs) {
            atomicCAS(P.err, 0, kErrTimeoutDrain);
            return;
        }
    }
}

__device__ __forceinline__ void worker_sync() {
    asm volatile("bar.sync 1, %0;" ::"n"(kWorkers) : "memory");
}

// worker_sync that also tells every worker whether any of them saw `flag`.
__device__ __forceinline__ bool worker_sync_or(bool flag) {
    uint32_t any;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.u32 p, %1, 0;\n\t"
        "bar.red.or.pred q, 1, %2, p;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(any)
        : "r"(static_cast<uint32_t>(flag)), "n"(kWorkers)
        : "memory");
    return any != 0;
}

// The row at position p of the order, or `rows` (one past the end) where there is none.
__device__ __forceinline__ int row_at(const WgradParams &P, int64_t p, int64_t stop) {
    if (p >= stop) return static_cast<int>(P.rows);
    if (P.order) return P.order[p];
    return P.index.at(p) == 0 ? static_cast<int>(p) : static_cast<int>(P.rows);
}

// The first adapter whose rows reach past pos (P.s: none), found by a whole warp, 32 at a time.
__device__ __forceinline__ int64_t first_adapter(const WgradParams &P, int64_t pos, int lane) {
    int64_t lo = 0, n = P.s;
    while (n > 0) {
        const int64_t step = (n + 31) / 32;
        const int64_t last = lo + min((lane + 1) * step, n) - 1;  // of this lane's share
        const unsigned past = __ballot_sync(0xFFFFFFFFu, P.start[last + 1] > pos);
        if (!past) return P.s;
        const int64_t skip = (__ffs(past) - 1) * step;
        lo += skip;
        if (step == 1) return lo;
        n = min(step, n - skip);
    }
    return P.s;
}

// The segments of a chunk, adapter by adapter from `s` on: f(s, from, to) for positions [from, to);
// returns false to stop.  With `every`, adapters without rows too.
template <class Fn>
__device__ __forceinline__ void segments(const WgradParams &P, int64_t s, int64_t pos, int64_t stop,
                                         bool every, Fn &&f) {
    for (; s < P.s && (every || pos < stop); ++s) {
        const int64_t end = P.start ? min(stop, int64_t(P.start[s + 1])) : stop;
        if ((end > pos || every) && !f(s, pos, max(pos, end))) return;
        pos = max(pos, end);
    }
}

template <typename T>
__device__ __forceinline__ uint16_t bits16(float v) {
    const T h = from_float<T>(v);
    return *reinterpret_cast<const uint16_t *>(&h);
}

// Forms the sums of the CTA's segments that are not finite again, as sums of M's and V's own products
// in the order of the rows.  For results that hold infinities or NaN only: each thread takes a column
// and 16 ranks at a time, and reads M once for them.
template <typename T>
__device__ __noinline__ void add_nonfinite(const WgradParams &P, const Side &S, int64_t chunk,
                                           int64_t s0, int64_t first, int64_t stop, int64_t c0,
                                           int j0) {
    const int64_t ldc = (S.cols + 7) / 8 * 8;
    const bool direct = S.part == nullptr;
    const int ranks = static_cast<int>(min(int64_t(kBlockRanks), P.r - j0));
    const DropoutKeys key(S.drop.cut ? dropout_key(S.drop) : 0);
    auto finite = [](float x) { return fabsf(x) < __int_as_float(0x7F800000); };
    segments(P, s0, first, stop, direct, [&](int64_t s, int64_t from, int64_t to) {
        for (int64_t c = c0 + threadIdx.x; c < min(c0 + kCtaCols, S.cols); c += kThreads) {
            T *out = static_cast<T *>(S.out) + s * S.ss + c * S.sc + j0 * S.sr;
            float *part = S.part + ((chunk + s) * P.r + j0) * ldc + c;
            for (int jb = 0; jb < ranks; jb += 16) {
                const int n = min(16, ranks - jb);
                uint32_t wrong = 0;
                for (int e = 0; e < n; ++e)
                    if (!finite(direct ? to_float(out[(jb + e) * S.sr]) : part[(jb + e) * ldc]))
                        wrong |= 1u << e;
                if (!wrong) continue;
                float sum[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) sum[e] = 0.0f;
                uint32_t open = wrong;  // a sum that is NaN stays so
                for (int64_t b = from; b < to && open; b += 32) {
                    const int64_t end = min(to, b + 32);
#pragma unroll 4
                    for (int64_t p = b; p < end; ++p) {
                        const int64_t row = row_at(P, p, to);
                        if (row >= P.rows) continue;
                        float m = to_float(static_cast<const T *>(S.M)[row * S.ld + c]);
                        if (S.drop.cut &&
                            !dropout_kept(dropout_bits(S.drop, key, static_cast<uint32_t>(row),
                                                       static_cast<uint32_t>(c >> 3)),
                                          static_cast<int>(c & 7), S.drop.cut))
                            m = 0.0f;
                        const float *v = S.V + row * P.r + j0 + jb;
#pragma unroll
                        for (int e = 0; e < 16; ++e)
                            if (e < n) sum[e] += m * v[e];
                    }
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        if (sum[e] != sum[e]) open &= ~(1u << e);
                }
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    if (!((wrong >> e) & 1)) continue;
                    if (direct)
                        out[(jb + e) * S.sr] = from_float<T>(sum[e]);
                    else
                        part[(jb + e) * ldc] = sum[e];
                }
            }
        }
        return true;
    });
}

// order[] and start[]: rows grouped by adapter, ascending within one.  CTA s compacts the rows of
// adapter s behind those of smaller adapters, which it counts first; up to 8192 indices stay in
// registers between the two passes.
__global__ void __launch_bounds__(1024) lists_kernel(RowIndex index, int64_t rows, int32_t *order,
                                                     int32_t *start) {
    constexpr int kHeld = 8;
    __shared__ int warp_sum[32];
    const int s = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int held[kHeld];
    int below = 0;
#pragma unroll
    for (int h = 0; h < kHeld; ++h) {
        const int64_t t = int64_t(h) * 1024 + threadIdx.x;
        held[h] = t < rows ? index.at(t) : -1;
    }
#pragma unroll
    for (int h = 0; h < kHeld; ++h) below += held[h] >= 0 && held[h] < s;
    for (int64_t t = int64_t(kHeld) * 1024 + threadIdx.x; t < rows; t += 1024) {
        const int i = index.at(t);
        below += i >= 0 && i < s;
    }
    below = __reduce_add_sync(0xFFFFFFFFu, below);
    if (lane == 0) warp_sum[warp] = below;
    __syncthreads();
    int at = __reduce_add_sync(0xFFFFFFFFu, warp_sum[lane]);
    if (threadIdx.x == 0) start[s] = at;
    __syncthreads();
    // its own rows, 1024 at a time
    auto place = [&](int64_t t, bool own) {
        const unsigned ballot = __ballot_sync(0xFFFFFFFFu, own);
        if (lane == 0) warp_sum[warp] = __popc(ballot);
        __syncthreads();
        const int n = warp_sum[lane];
        const int before = __reduce_add_sync(0xFFFFFFFFu, lane < warp ? n : 0);
        const int all = __reduce_add_sync(0xFFFFFFFFu, n);
        if (own) order[at + before + __popc(ballot & ((1u << lane) - 1))] = static_cast<int32_t>(t);
        at += all;
        __syncthreads();
    };
#pragma unroll
    for (int h = 0; h < kHeld; ++h)
        if (int64_t(h) * 1024 < rows) place(int64_t(h) * 1024 + threadIdx.x, held[h] == s);
    for (int64_t t0 = int64_t(kHeld) * 1024; t0 < rows; t0 += 1024) {
        const int64_t t = t0 + threadIdx.x;
        place(t, t < rows && index.at(t) == s);
    }
    if (s == gridDim.x - 1 && threadIdx.x == 0) start[s + 1] = at;
}

// Maps of dA's and dB's matrices: boxes of 64 rows, and of one row for gathering.
struct Maps {
    CUtensorMap tile[2], row[2];
};

// Roles: warp 0 copies (16 lanes, four rows each), warp 1 TMEM and MMA issue, warps 2..9 V, the
// mask and the epilogue.
template <typename T>
__global__ void __launch_bounds__(kThreads, 1)
    wgrad_kernel(const __grid_constant__ Maps maps, const __grid_constant__ WgradParams P) {
    constexpr bool kScaled = std::is_same<T, __half>::value;
    constexpr int kParts = Stage<T>::kParts, kStageBytes = Stage<T>::kBytes;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *ring = reinterpret_cast<uint8_t *>(
        (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    float *scale = reinterpret_cast<float *>(ring + kStages * kStageBytes);  // [64] 2^-e by rank
    uint64_t *full = reinterpret_cast<uint64_t *>(scale + kBlockRanks);
    uint64_t *ready = full + kStages;   // V is in place, and M masked
    uint64_t *empty = ready + kStages;
    uint64_t *tfull = empty + kStages;
    uint64_t *tempty = tfull + 1;
    uint64_t *drain = tempty + 1;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(drain + 1);
    volatile int *abort = reinterpret_cast<volatile int *>(tmem_slot + 1);
    int *start_at = const_cast<int *>(abort) + 1;
    volatile int *fix = start_at + 1;  // some sum is not finite

    const int64_t units_a = P.side[0].blocks * P.side[0].chunks;
    const int which = blockIdx.x < units_a ? 0 : 1;
    const Side &S = P.side[which];
    const CUtensorMap *tile_map = &maps.tile[which], *row_map = &maps.row[which];
    const int64_t unit = blockIdx.x - (which ? units_a : 0), chunk = unit / S.blocks;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t c0 = unit % S.blocks * kCtaCols;
    const int j0 = static_cast<int>(blockIdx.y) * kBlockRanks;
    const int64_t total = P.start ? P.start[P.s] : P.rows;
    const bool direct = S.part == nullptr;
    const int64_t first = chunk * S.chunk, stop = min(total, first + S.chunk);

    if (threadIdx.x == 0) {
        if (P.rows) prefetch_tensormap(tile_map);
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&ready[s], kWorkers / 32);
            mbar_init(&empty[s], 1);
        }
        mbar_init(tfull, 1);
        mbar_init(tempty, kWorkers / 32);
        mbar_init(drain, 1);
        *abort = 0;
        *fix = 0;
        fence_barrier_init();
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, kTmemCols);
        tmem_relinquish();
    }
    if (warp == 2) {
        const int64_t s = P.start && !direct ? first_adapter(P, first, lane) : 0;
        if (lane == 0) *start_at = static_cast<int>(s);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    const int64_t s0 = *start_at;

    if (warp == 0) {
        // ---------------- copies ----------------
        int stage = 0;
        uint32_t phase = 0, issued_mask = 0, issued_phase = 0;
        bool ok = true;
        segments(P, s0, first, stop, direct, [&](int64_t, int64_t from, int64_t to) {
            int row[4];
            auto ask = [&](int64_t b) {
#pragma unroll
                for (int e = 0; e < 4; ++e) row[e] = row_at(P, b + 4 * (lane & 15) + e, to);
            };
            ask(from);
            for (int64_t b = from; b < to; b += kRows) {
                if (!mbar_wait(&empty[stage], phase ^ 1, abort)) {
                    raise(P, abort, kErrTimeoutProducer);
                    ok = false;
                }
                ok = __all_sync(0xFFFFFFFFu, ok);
                if (!ok) return false;
                if (lane == 0) mbar_arrive_expect_tx(&full[stage], kMBytes);
                __syncwarp();
                // 64 consecutive rows are one box; a copy of four rows at a time is much slower
                const int row0 = __shfl_sync(0xFFFFFFFFu, row[0], 0);
                bool run = true;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    run = run && row[e] == row0 + 4 * (lane & 15) + e && row[e] < P.rows;
                run = __all_sync(0xFFFFFFFFu, run);
                uint8_t *dst = ring + stage * kStageBytes;
                if (run) {
                    if (lane < 4)
                        tma_load_2d(dst + lane * kAtomBytes, tile_map, &full[stage],
                                    static_cast<int>(c0) + 64 * lane, row0);
                } else if (lane < 16) {
#pragma unroll
                    for (int a = 0; a < 4; ++a)
                        tma_gather4(dst + 512 * lane + a * kAtomBytes, row_map, &full[stage],
                                    static_cast<int>(c0) + 64 * a, row);
                }
                ask(b + kRows);  // the next stage's rows are on their way
                issued_mask |= 1u << stage;
                issued_phase = (issued_phase & ~(1u << stage)) | (phase << stage);
                if (++stage == kStages) {
                    stage = 0;
                    phase ^= 1;
                }
            }
            return true;
        });
        if (!ok && lane == 0)  // every copy lands before the CTA may exit
            for (int s = 0; s < kStages; ++s)
                if ((issued_mask >> s) & 1) drain_wait(P, &full[s], (issued_phase >> s) & 1);
    } else if (warp == 1) {
        if (lane == 0) {
            // ---------------- MMA issuer ----------------
            int stage = 0;
            uint32_t phase = 0, seg = 0;
            bool ok = true, any_issued = false;
            segments(P, s0, first, stop, direct, [&](int64_t, int64_t from, int64_t to) {
                if (from == to) return true;
                if (!mbar_wait(tempty, (seg & 1) ^ 1, abort)) {
                    raise(P, abort, kErrTimeoutMma);
                    ok = false;
                    return false;
                }
                ++seg;
                tc_fence_after();
                for (int64_t b = from; b < to; b += kRows) {
                    if (!mbar_wait(&full[stage], phase, abort) ||
                        !mbar_wait(&ready[stage], phase, abort)) {
                        raise(P, abort, kErrTimeoutMma);
                        ok = false;
                        return false;
                    }
                    tc_fence_after();
                    const uint32_t sm = smem_u32(ring + stage * kStageBytes);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint64_t mdesc =
                            make_sw128_mnmajor_desc(sm + 2 * h * kAtomBytes, kAtomBytes);
#pragma unroll
                        for (int part = 0; part < kParts; ++part) {
                            const uint64_t vdesc =
                                make_sw128_kmajor_desc(sm + kMBytes + part * kPartBytes);
#pragma unroll
                            for (int kk = 0; kk < kRows / 16; ++kk)
                                umma_f16(tmem_base + h * kBlockRanks, mdesc + 128 * kk,
                                         vdesc + 2 * kk, P.idesc,
                                         b > from || part > 0 || kk > 0 ? 1u : 0u);
                        }
                    }
                    any_issued = true;
                    umma_commit(&empty[stage]);
                    if (++stage == kStages) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
                umma_commit(tfull);
                return true;
            });
            if (!ok && any_issued) {
                umma_commit(drain);
                drain_wait(P, drain, 0);
            }
        }
    } else {
        // ---------------- V, the mask, the epilogue ----------------
        const int wt = threadIdx.x - 64, w = warp - 2;
        const int half = w & 1;                  // this warp's 32 rows of a stage
        const int quads = P.rp / 4;              // and every fourth quad of ranks from w / 2
        const DropoutKeys key(S.drop.cut ? dropout_key(S.drop) : 0);
        const bool vec = P.r % 4 == 0 && (reinterpret_cast<uintptr_t>(S.V) & 15) == 0;
        auto load_v = [&](int row, int quad) {
            float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            const int64_t j = j0 + 4 * quad;
            if (row >= P.rows || j >= P.r) return v;
            const float *p = S.V + row * P.r + j;
            if (vec) return *reinterpret_cast<const float4 *>(p);
            v.x = p[0];
            if (j + 1 < P.r) v.y = p[1];
            if (j + 2 < P.r) v.z = p[2];
            if (j + 3 < P.r) v.w = p[3];
            return v;
        };
        int stage = 0;
        uint32_t phase = 0, seg = 0;
        bool ok = true;  // a wait that gave up ends all workers at their next barrier
        segments(P, s0, first, stop, direct, [&](int64_t s, int64_t from, int64_t to) {
            if (kScaled) {
                // 2^-e with the largest finite value of the segment's column near 2^14
                if (worker_sync_or(!ok)) return false;  // the previous scales have been read
                for (int q = w; q < quads; q += kWorkers / 32) {
                    float m[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                    for (int64_t b = from + lane; b - lane < to; b += 32 * 8) {
                        int row[8];
                        float4 v[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) row[i] = row_at(P, b + 32 * i, to);
#pragma unroll
                        for (int i = 0; i < 8; ++i) v[i] = load_v(row[i], q);
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const float x[4] = {fabsf(v[i].x), fabsf(v[i].y), fabsf(v[i].z),
                                                fabsf(v[i].w)};
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                if (x[e] < __int_as_float(0x7F800000)) m[e] = fmaxf(m[e], x[e]);
                        }
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t top = __reduce_max_sync(0xFFFFFFFFu, __float_as_uint(m[e]));
                        // exponent of the largest value; the power stays a normal number
                        const int x = static_cast<int>(top >> 23);  // biased
                        const int y = top ? min(max(127 + 14 + 127 - x, 1), 253) : 127;
                        if (lane == 0) scale[4 * q + e] = __int_as_float(y << 23);
                    }
                }
                worker_sync();
            }
            // row numbers are read two stages ahead and values one, so that neither is waited for
            const int t = 32 * half + lane;
            float4 v[4], ahead[4];
            auto fetch = [&](int r, float4(&x)[4]) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if ((w >> 1) + 4 * i < quads) x[i] = load_v(r, (w >> 1) + 4 * i);
            };
            fetch(row_at(P, from + t, to), v);
            int row = row_at(P, from + kRows + t, to);
            int mask_next = S.drop.cut ? row_at(P, from + (wt >> 2), to) : 0;
            for (int64_t b = from; b < to; b += kRows) {
                const int mask_row = mask_next;
                fetch(row, ahead);
                row = row_at(P, b + 2 * kRows + t, to);
                if (S.drop.cut) mask_next = row_at(P, b + kRows + (wt >> 2), to);
                if (!mbar_wait(&empty[stage], phase ^ 1, abort)) {
                    raise(P, abort, kErrTimeoutProducer);
                    ok = false;
                    break;
                }
                uint8_t *m = ring + stage * kStageBytes;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int quad = (w >> 1) + 4 * i;
                    if (quad >= quads) break;
                    const float x[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int j = 4 * quad + e;
                        float y = kScaled ? x[e] * scale[j] : x[e];
                        const uint32_t at = j * 128 + ((((t >> 3) ^ (j & 7)) << 4) | ((t & 7) << 1));
#pragma unroll
                        for (int part = 0; part < kParts; ++part) {
                            const uint16_t h = bits16<T>(y);
                            const float up = to_float(*reinterpret_cast<const T *>(&h));
                            // infinities and NaN stay whole in the first part
                            y = fabsf(up) < __int_as_float(0x7F800000) ? y - up : 0.0f;
                            *reinterpret_cast<uint16_t *>(m + kMBytes + part * kPartBytes + at) = h;
                        }
                    }
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = ahead[i];
                if (S.drop.cut) {
                    if (!mbar_wait(&full[stage], phase, abort)) {
                        raise(P, abort, kErrTimeoutEpilogue);
                        ok = false;
                        break;
                    }
                    // a thread takes 64 columns of one row
                    const int mr = wt >> 2, a = wt & 3;
                    uint8_t *p = m + a * kAtomBytes + mr * 128;
#pragma unroll
                    for (int c = 0; c < 8; ++c) {
                        uint4 *x = reinterpret_cast<uint4 *>(p + ((c ^ (mr & 7)) << 4));
                        *x = masked(*x, S.drop, key, static_cast<uint32_t>(mask_row),
                                    static_cast<uint32_t>(c0 >> 3) + 8 * a + c);
                    }
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&ready[stage]);
                if (++stage == kStages) {
                    stage = 0;
                    phase ^= 1;
                }
            }
            // ---------------- the segment's sums ----------------
            const int q = warp & 3, h = w >> 2;  // TMEM lane quadrant, half of the columns
            const int64_t c = c0 + 128 * h + 32 * q + lane;
            const bool some = from < to;
            if (ok && some && !mbar_wait(tfull, seg & 1, abort)) {
                raise(P, abort, kErrTimeoutEpilogue);
                ok = false;
            }
            ok = __all_sync(0xFFFFFFFFu, ok);
            if (!ok) return kScaled;  // on to the barrier, where there is one
            tc_fence_after();
            const int64_t ldc = (S.cols + 7) / 8 * 8;
            for (int jb = 0; jb < P.rp; jb += 16) {
                uint32_t x[16];
                if (some) {
                    tmem_ld_32x32b_x16(tmem_base + (static_cast<uint32_t>(q * 32) << 16) +
                                           h * kBlockRanks + jb,
                                       x);
                    tmem_wait_ld();
                }
                if (c < S.cols)
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const int64_t j = j0 + jb + e;
                        if (j >= P.r) continue;
                        float y = some ? __uint_as_float(x[e]) : 0.0f;
                        if (!(fabsf(y) < __int_as_float(0x7F800000))) *fix = 1;
                        // (a power of two, and its inverse by exponent arithmetic)
                        if (kScaled && some)
                            y *= __int_as_float((254 << 23) - __float_as_int(scale[jb + e]));
                        if (direct)
                            static_cast<T *>(S.out)[s * S.ss + c * S.sc + j * S.sr] = from_float<T>(y);
                        else
                            S.part[((chunk + s) * P.r + j) * ldc + c] = y;
                    }
            }
            if (some) {
                ++seg;
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(tempty);
            }
            return true;
        });
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem_base, kTmemCols);
    }
    if (*fix && !*abort) add_nonfinite<T>(P, S, chunk, s0, first, stop, c0, j0);
}

// out[s][c][j] = the sum of adapter s's slots, in order.  A block takes 32 ranks x 32 columns, reads
// them along the columns and writes them along whichever of the two is consecutive in out.
template <typename T>
__global__ void __launch_bounds__(256) join_kernel(const __grid_constant__ WgradParams P) {
    const Side &S = P.side[blockIdx.y];
    if (!S.part) return;
    __shared__ float tile[32][33];
    const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
    const int64_t ldc = (S.cols + 7) / 8 * 8;
    const int64_t total = P.start ? P.start[P.s] : P.rows;
    const int64_t blocks_c = (S.cols + 31) / 32, blocks_j = (P.r + 31) / 32;
    for (int64_t u = blockIdx.x; u < P.s * blocks_j * blocks_c; u += gridDim.x) {
        const int64_t c0 = u % blocks_c * 32, j0 = u / blocks_c % blocks_j * 32;
        const int64_t s = u / (blocks_c * blocks_j);
        const int64_t first = P.start ? P.start[s] : 0;
        const int64_t end = P.start ? P.start[s + 1] : s == 0 ? total : 0;
        const int64_t k0 = first / S.chunk, k1 = end > first ? (end - 1) / S.chunk : k0 - 1;
        T *out = static_cast<T *>(S.out) + s * S.ss;
        const int64_t c = c0 + x;
        float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int64_t k = k0; k <= k1; ++k)
#pragma unroll
            for (int h = 0; h < 4; ++h) {
                const int64_t j = j0 + y + 8 * h;
                if (c < S.cols && j < P.r) v[h] += S.part[((k + s) * P.r + j) * ldc + c];
            }
        if (S.sr == 1 && S.sc != 1) {
#pragma unroll
            for (int h = 0; h < 4; ++h) tile[y + 8 * h][x] = v[h];
            __syncthreads();
#pragma unroll
            for (int h = 0; h < 4; ++h)
                if (c0 + y + 8 * h < S.cols && j0 + x < P.r)
                    out[(c0 + y + 8 * h) * S.sc + j0 + x] = from_float<T>(tile[x][y + 8 * h]);
            __syncthreads();
        } else {
#pragma unroll
            for (int h = 0; h < 4; ++h) {
                const int64_t j = j0 + y + 8 * h;
                if (c < S.cols && j < P.r) out[c * S.sc + j * S.sr] = from_float<T>(v[h]);
            }
        }
    }
}

}  // namespace

// Chunks of rows: one wave of CTAs, one per SM, so that the partial sums, which are written and
// read once for each chunk, stay few.
WgradPlan lr_wgrad_plan(int64_t rows, int64_t r, int64_t s, int64_t cols_a, int64_t cols_b,
                        bool listed, bool dropped) {
    constexpr int64_t kCtas = 148;  // fixed: the workspace is sized without a device
    WgradPlan p{};
    // with a mask a row of dA costs more than a row of dB
    const int64_t cols[2] = {cols_a, cols_b}, weight[2] = {dropped ? 3 : 2, 2};
    int64_t cost = 0;
    for (int w = 0; w < 2; ++w)
        cost += weight[w] * ((cols[w] + kCtaCols - 1) / kCtaCols) * ((r + kBlockRanks - 1) / kBlockRanks);
    for (int w = 0; w < 2; ++w) {
        int64_t chunks = cost ? weight[w] * kCtas / cost : 1;
        const int64_t most = (rows + 127) / 128;  // 128 rows are worth a chunk
        if (chunks > most) chunks = most;
        if (chunks < 1) chunks = 1;
        p.chunk[w] = ((rows + chunks - 1) / chunks + kRows - 1) / kRows * kRows;
        if (p.chunk[w] == 0) p.chunk[w] = kRows;
        p.chunks[w] = rows ? (rows + p.chunk[w] - 1) / p.chunk[w] : 1;
        if (p.chunks[w] > 1)
            p.part[w] = sizeof(float) * static_cast<size_t>((p.chunks[w] + s - 1) * r *
                                                            ((cols[w] + 7) / 8 * 8));
    }
    p.list_bytes = listed ? sizeof(int32_t) * static_cast<size_t>(rows + s + 1) : 0;
    return p;
}

template <typename T>
static cudaError_t wgrad(WgradParams &P, int num_sms, cudaStream_t stream) {
    P.rp = P.r >= kBlockRanks ? kBlockRanks : static_cast<int>((P.r + 15) / 16 * 16);
    const int type = std::is_same<T, __half>::value ? 0 : 1;
    P.idesc = (1u << 4) | (static_cast<uint32_t>(type) << 7) | (static_cast<uint32_t>(type) << 10) |
              (1u << 15) | (static_cast<uint32_t>(P.rp >> 3) << 17) | ((128u >> 4) << 24);
    Maps maps;
    std::memset(&maps, 0, sizeof(maps));
    int64_t units = 0;
    for (int w = 0; w < 2; ++w) {
        const Side &S = P.side[w];
        units += S.blocks * S.chunks;
        // (without rows the sums are zeros and nothing is copied)
        if (S.blocks && P.rows &&
            (!make_map16(&maps.tile[w], S.M, S.cols, P.rows, S.ld, 64, kRows) ||
             !make_map16(&maps.row[w], S.M, S.cols, P.rows, S.ld, 64, 1)))
            return cudaErrorInvalidValue;
    }
    static PerDevice<int> ready;
    std::atomic<int> *set = ready.here();
    if (!set) return cudaErrorInvalidDevice;
    if (!set->load(std::memory_order_acquire)) {
        const cudaError_t e = cudaFuncSetAttribute(
            wgrad_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
            static_cast<int>(Stage<T>::kSmem));
        if (e != cudaSuccess) return e;
        set->store(1, std::memory_order_release);
    }
    const dim3 grid(static_cast<unsigned>(units),
                    static_cast<unsigned>((P.r + kBlockRanks - 1) / kBlockRanks));
    wgrad_kernel<T><<<grid, kThreads, Stage<T>::kSmem, stream>>>(maps, P);
    if (P.side[0].part || P.side[1].part) {
        const int64_t cols = P.side[0].cols > P.side[1].cols ? P.side[0].cols : P.side[1].cols;
        const int64_t want = P.s * ((P.r + 31) / 32) * ((cols + 31) / 32), most = int64_t(num_sms) * 8;
        join_kernel<T><<<dim3(static_cast<unsigned>(want < most ? want : most), 2), 256, 0, stream>>>(P);
    }
    return cudaGetLastError();
}

cudaError_t lr_wgrad(bool half, const WgradOperand &a, const WgradOperand &b, int64_t rows,
                     int64_t r, const RowIndex &index, const WgradPlan &plan, void *lists,
                     int num_sms, int *err, cudaStream_t stream) {
    WgradParams P{};
    P.err = err;
    P.rows = rows;
    P.r = r;
    P.s = index.s;
    const WgradOperand *ops[2] = {&a, &b};
    for (int w = 0; w < 2; ++w) {
        const WgradOperand &o = *ops[w];
        const int64_t blocks = o.out ? (o.cols + kCtaCols - 1) / kCtaCols : 0;
        P.side[w] = Side{o.M.p, o.M.s0, o.cols, o.V, o.drop, blocks ? o.part : nullptr, o.out,
                         o.ss,  o.sc,   o.sr,   blocks, plan.chunk[w], plan.chunks[w]};
    }
    if (P.side[0].blocks + P.side[1].blocks == 0) return cudaSuccess;
    P.index = index;
    if (index.p && index.s > 1) {
        int32_t *start = static_cast<int32_t *>(lists);
        int32_t *order = start + index.s + 1;
        lists_kernel<<<static_cast<unsigned>(index.s), 1024, 0, stream>>>(index, rows, order, start);
        P.order = order;
        P.start = start;
    }
    return half ? wgrad<__half>(P, num_sms, stream) : wgrad<__nv_bfloat16>(P, num_sms, stream);
}

}  // namespace ti
