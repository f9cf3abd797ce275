// ti_lr_gemm.cu -- the expand form on CTA pairs: out = M W + P F, one persistent kernel.
//
//   out[t][c] = sum_k M[t][k] W[k][c] + m(t, c) sum_j P[t][j] F[i][c][j],   i = index[t]
//
// The shared product is a 16-bit GEMM on tcgen05 (kind::f16, float32 accumulators in TMEM) with
// the shape of ti_gemm2.cu: a cluster of two CTAs owns a 256 x 256 output tile, CTA r loads rows
// [128r, 128r+128) of M's tile and columns [128r, 128r+128) of W's per 64-deep stage, and CTA 0
// issues M = 256, N = 256 MMAs for both.  W is read in either orientation (K-major or N-major
// descriptors), so a transposed view costs nothing.
//
// The low-rank term joins the same accumulator as extra steps of the inner dimension: for every
// distinct adapter among the tile's 256 rows and every 16 of its ranks, one step multiplies the
// rows' P (zero for the rows of other adapters) by the adapter's F.  A step costs as much as one
// 64-deep step of the product, so r = 16 adds 1/64 at k = 4096.  P is float32: it enters as
// kind::tf32 in two parts (its upper 11 bits and the rest; 2^-21 relative error) against F, whose
// 16-bit values are exact in tf32.  That keeps fp16's range out of the projection, and the exact
// zeros of foreign rows keep adapters apart -- except for 0 * inf: entries of P or F that are not
// finite enter the MMA as zero and raise a flag, and the epilogue of such a tile adds their
// products itself.
//
// With dropout (dX) the mask applies to the low-rank term alone, so that term has its own 256
// accumulator columns and the epilogue joins the two.  The 512 TMEM columns then hold one tile
// instead of two, and the next tile's MMAs wait for the epilogue; so it prepares its mask bits
// while the MMAs run, holds its results in registers, and gives TMEM back before it stores.
// (128-column tiles would keep both accumulators double buffered, but need half as much again of
// L2 reads per product: 171 us against 109 us without dropout at 4096^3.)
//
// Roles (both CTAs): warp 0 TMA producer; warp 1 TMEM allocation and, in CTA 0, the MMA issuer;
// warps 2..9 epilogue, two per TMEM lane quadrant with 128 columns each; warps 10..13 loaders of the
// low-rank steps, which have two stages of their own and fill them while the product's steps run.  A
// low-rank step is taken after every `every` steps of the product while any are left: a fixed
// order, so results repeat bit for bit, and far enough apart that the loaders are ready (8192^3,
// r = 32, whole call: 990 us with 4, 935 us with 16).  The kernel may start before the projection has finished
// (programmatic launch); the loaders wait for it.
// Measured on a B200 (bf16, this kernel alone): 8192^3 787 to 800 us without adapters (1398 TFLOP/s;
// cuBLAS on the plain product 680 us), 802 to 840 us with rank 32, fp16 880 us (the power cap; a whole
// call in a long run takes 887 to 1058 us); 4096^3 110 us (cuBLAS 92 us), 114 to 117 us with rank 16,
// 126 us with rank 64, 135 us with rank 16 and dropout; 4096 x 4096 x 4097 122 us.  4096^3 is 256 tiles on 74 pairs: the fourth wave is half
// empty.
// All waits are bounded; on timeout the error word is raised and the CTA leaves its loops.
#include <atomic>
#include <cstring>
#include <type_traits>

#include "ti_lr_loads.cuh"
#include "ti_lr_launch.cuh"

namespace ti {
namespace {

constexpr int kBM = 256, kBN = 256, kBK = 64;
constexpr int kHalf = 128;                       // rows of M and columns of W per CTA
constexpr int kABytes = kHalf * kBK * 2, kBBytes = kHalf * kBK * 2;
constexpr int kStageBytes = kABytes + kBBytes, kStages = 5;
constexpr int kLowBytes = 2 * kHalf * 128;       // one low-rank step per CTA: rows of P, rows of F
constexpr int kEpiWarps = 8, kLoaders = 128;
constexpr int kThreads = 64 + 32 * kEpiWarps + kLoaders;
constexpr uint32_t kTmemCols = 512;
constexpr int kGroupM = 8;                       // raster: 8 row tiles (2048 rows) at a time
constexpr int kRankStep = 16;
constexpr int kFixSlots = 16;
constexpr size_t kSmem = size_t(kStages) * kStageBytes + 2 * kLowBytes + 1024 + 512;
// Rows that leave through shared memory: a warp's 32 rows of 16 words, in the last stage of sA; such
// calls use a ring of kStages - 1 stages.
constexpr int kTurnWords = 32 * 16;
static_assert(kEpiWarps * kTurnWords * 4 <= kABytes,
              "the warps' rows do not fit the stage that is left to them");

struct Params {
    int64_t rows, cols;
    int num_kb, tiles_m, tiles_n;
    int every;      // product steps between two low-rank steps
    int64_t total;
    int w_nmajor;
    uint32_t idesc16, idesc32;
    const float *P;
    int64_t r;
    Factor16 F;
    RowIndex index;
    Dropout drop;
    void *out;
    int64_t ldo;
    int align;      // bytes to which the rows of out are aligned: 16, 8, 4 or 2
    int stages;     // of the ring: kStages, or one less where the epilogue takes its space
    int pvec, fvec; // P's rows in vectors of 4, F's in vectors of 8 along the rank
    int *err;
};

__device__ __forceinline__ void tma_load_2d_pair(void *dst, const CUtensorMap *map, uint32_t bar,
                                                 int c0, int c1) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4}], [%2];" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1)
        : "memory");
}

__device__ __forceinline__ void umma_f16_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                              uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}

__device__ __forceinline__ void umma_tf32_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                               uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::tf32 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}

__device__ __forceinline__ void loader_sync() {
    asm volatile("bar.sync 1, %0;" ::"n"(kLoaders) : "memory");
}

// loader_sync that also tells every loader whether any of them saw `flag`.
__device__ __forceinline__ bool loader_sync_or(bool flag) {
    uint32_t any;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.u32 p, %1, 0;\n\t"
        "bar.red.or.pred q, 1, %2, p;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(any)
        : "r"(static_cast<uint32_t>(flag)), "n"(kLoaders)
        : "memory");
    return any != 0;
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

// Tiles of the pair (both CTAs walk the same sequence); f(tm, tn) returns false to stop.
template <class Fn>
__device__ __forceinline__ void tiles(const Params &P, Fn &&f) {
    const int64_t per_group = int64_t(kGroupM) * P.tiles_n;
    for (int64_t u = blockIdx.x >> 1; u < P.total; u += gridDim.x >> 1) {
        const int g = static_cast<int>(u / per_group);
        const int first = g * kGroupM, size = min(kGroupM, P.tiles_m - first);
        const int64_t in = u - g * per_group;
        if (!f(first + static_cast<int>(in % size), static_cast<int>(in / size))) return;
    }
}

__device__ __forceinline__ bool finite(float x) {
    return (__float_as_uint(x) & 0x7F800000u) != 0x7F800000u;
}

// 16-byte chunk `c` (0..7) of 128-byte row `row` in a 128-byte-swizzled tile.
__device__ __forceinline__ float4 *swizzled(uint8_t *tile, int row, int c) {
    return reinterpret_cast<float4 *>(tile + row * 128 + ((c ^ (row & 7)) << 4));
}

// Columns [c0, c0 + 16) of one row of a tile whose P or F holds entries that are not finite:
// adds the products that the MMA left out.
template <typename T>
__device__ __noinline__ void add_nonfinite(const Params &P, int64_t row, int64_t c0, float *acc) {
    const int i = P.index.at(row);
    if (i < 0) return;
    const T *f = static_cast<const T *>(P.F.p) + i * P.F.ss;
    for (int c = 0; c < 16 && c0 + c < P.cols; ++c)
        for (int64_t j = 0; j < P.r; ++j) {
            const float p = P.P[row * P.r + j];
            const float b = to_float(f[(c0 + c) * P.F.sc + j * P.F.sr]);
            if (!finite(p) || !finite(b)) acc[c] += p * b;
        }
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
    __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t *>(&v);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
    __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t *>(&v);
}

__device__ __forceinline__ void store_flag(uint32_t addr) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(1) : "memory");
}

// Stores a warp's 32 rows x 32 packed columns (lane = row), as far as they exist.  Rows that are
// not 16-byte aligned would leave in pieces of 8, 4 or 2 bytes, 32 rows at a time; they go through
// `turn` (32 rows of 16 words, this warp's own) instead, so that a store covers consecutive bytes.
// Word j of row r lies at j ^ (r / 2), which keeps both directions free of bank conflicts.
template <typename T>
__device__ __forceinline__ void store_block(const Params &P, T *out, uint32_t *turn, int64_t row0,
                                            int64_t col0, int lane, const uint32_t (&pk)[16]) {
    if (col0 >= P.cols) return;  // the same for the whole warp
    if (P.align == 16) {
        const int64_t row = row0 + lane;
        if (row >= P.rows) return;
        T *dst = out + row * P.ldo + col0;
        if (col0 + 32 <= P.cols) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                reinterpret_cast<uint4 *>(dst)[j] =
                    make_uint4(pk[4 * j], pk[4 * j + 1], pk[4 * j + 2], pk[4 * j + 3]);
        } else {
            uint16_t *d = reinterpret_cast<uint16_t *>(dst);
#pragma unroll
            for (int j = 0; j < 32; ++j)
                if (col0 + j < P.cols) d[j] = static_cast<uint16_t>(pk[j >> 1] >> (16 * (j & 1)));
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < 16; ++j) turn[lane * 16 + (j ^ (lane >> 1))] = pk[j];
    __syncwarp();
    const int rows = static_cast<int>(min(int64_t(32), P.rows - row0));
    if (P.align >= 4 && col0 + 32 <= P.cols) {  // words: two rows at a time
        uint32_t *dst = reinterpret_cast<uint32_t *>(out + row0 * P.ldo + col0) + (lane & 15);
#pragma unroll 4
        for (int r = lane >> 4; r < rows; r += 2)
            dst[r * (P.ldo >> 1)] = turn[r * 16 + ((lane ^ (r >> 1)) & 15)];
    } else {
        uint16_t *dst = reinterpret_cast<uint16_t *>(out + row0 * P.ldo + col0) + lane;
        const uint16_t *src = reinterpret_cast<const uint16_t *>(turn);
        if (col0 + lane < P.cols)
#pragma unroll 4
            for (int r = 0; r < rows; ++r) dst[r * P.ldo] = src[r * 32 + (lane ^ (r & ~1))];
    }
    __syncwarp();
}

template <typename T, bool kDrop>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    lr_gemm_kernel(const __grid_constant__ CUtensorMap tmM, const __grid_constant__ CUtensorMap tmW,
                   const __grid_constant__ Params P) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>(
        (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *sA = smem;
    uint8_t *sB = sA + kStages * kABytes;
    uint8_t *sLow = sB + kStages * kBBytes;  // two low-rank steps: 128 rows of P, hi | lo, then
                                             // 128 rows of F
    uint64_t *full = reinterpret_cast<uint64_t *>(sLow + 2 * kLowBytes);  // CTA 0
    uint64_t *empty = full + kStages;
    uint64_t *tfull = empty + kStages;   // [2] both CTAs: accumulator ready
    uint64_t *tempty = tfull + 2;           // [2] CTA 0: drained by both epilogues
    uint64_t *lfull = tempty + 2;           // [2] CTA 0: low-rank step written in both CTAs
    uint64_t *lempty = lfull + 2;           // [2] both CTAs: low-rank step taken
    uint64_t *drain = lempty + 2;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(drain + 1);
    volatile int *abort = reinterpret_cast<volatile int *>(tmem_slot + 1);
    volatile int *message = abort + 1;      // [2] CTA 0: 8-wide steps in a low-rank step, 0: no more
    volatile int *fix = message + 2;        // [kFixSlots] by tile: entries that are not finite
    int *least = const_cast<int *>(fix) + kFixSlots;  // [2][4] loaders' smallest adapter, by warp

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();
    constexpr int kBuffers = kDrop ? 1 : 2;  // tiles in TMEM

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(&tfull[a], 1);
            mbar_init(&tempty[a], 2 * kEpiWarps);
            mbar_init(&lfull[a], 2);
            mbar_init(&lempty[a], 1);
        }
        mbar_init(drain, 1);
        *abort = 0;
        for (int f = 0; f < kFixSlots; ++f) fix[f] = 0;
        fence_barrier_init();
        prefetch_tensormap(&tmM);
        prefetch_tensormap(&tmW);
    }
    if (warp == 1) {
        tmem_alloc_pair(tmem_slot, kTmemCols);
        tmem_relinquish_pair();
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;

    if (warp == 0) {
        if (lane == 0) {
            // ---------------- TMA producer (both CTAs) ----------------
            int stage = 0;
            uint32_t phase = 0, issued_mask = 0, issued_phase = 0;
            bool ok = true;
            tiles(P, [&](int tm, int tn) {
                const int row0 = tm * kBM + static_cast<int>(rank) * kHalf;
                const int col0 = tn * kBN + static_cast<int>(rank) * kHalf;
                for (int kb = 0; kb < P.num_kb; ++kb) {
                    if (!mbar_wait(&empty[stage], phase ^ 1, abort)) {
                        raise(P, abort, kErrTimeoutProducer);
                        ok = false;
                        return false;
                    }
                    if (rank == 0) mbar_arrive_expect_tx(&full[stage], 2 * kStageBytes);
                    const uint32_t fb = map_to_rank(smem_u32(&full[stage]), 0);
                    tma_load_2d_pair(sA + stage * kABytes, &tmM, fb, kb * kBK, row0);
                    uint8_t *b = sB + stage * kBBytes;
                    if (P.w_nmajor) {
#pragma unroll
                        for (int h = 0; h < kHalf / 64; ++h)
                            tma_load_2d_pair(b + h * 8192, &tmW, fb, col0 + 64 * h, kb * kBK);
                    } else {
                        tma_load_2d_pair(b, &tmW, fb, kb * kBK, col0);
                    }
                    issued_mask |= 1u << stage;
                    issued_phase = (issued_phase & ~(1u << stage)) | (phase << stage);
                    if (++stage == P.stages) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
                return true;
            });
            if (!ok) {
                // every issued copy lands before the pair may exit; CTA 0 sees both CTAs' bytes
                if (rank == 0) {
                    for (int s = 0; s < kStages; ++s)
                        if ((issued_mask >> s) & 1) drain_wait(P, &full[s], (issued_phase >> s) & 1);
                } else {
                    const unsigned long long t0 = globaltimer_ns();
                    while (globaltimer_ns() - t0 < 1000000ull) {
                    }
                }
            }
        }
    } else if (warp == 1) {
        if (lane == 0 && rank == 0) {
            // ---------------- MMA issuer (CTA 0) ----------------
            int stage = 0;
            uint32_t phase = 0, taken = 0;  // low-rank steps taken: stage taken % 2
            bool ok = true, any_issued = false;
            int64_t unit = 0;
            tiles(P, [&](int, int) {
                const int acc = static_cast<int>(unit % kBuffers);
                const uint32_t acc_phase = static_cast<uint32_t>((unit / kBuffers) & 1);
                ++unit;
                if (!mbar_wait(&tempty[acc], acc_phase ^ 1, abort)) {
                    raise(P, abort, kErrTimeoutMma);
                    ok = false;
                    return false;
                }
                tc_fence_after();
                const uint32_t d = tmem_base + static_cast<uint32_t>(acc * kBN);
                const uint32_t dlow = kDrop ? d + kBN : d;
                bool more = true;         // low-rank steps may follow
                int until = P.every;
                uint32_t have_low = kDrop ? 0u : 1u;  // the low-rank accumulator holds something
                // takes one low-rank step, or the loaders' word that there are no more
                auto low_step = [&]() {
                    const uint32_t at = taken & 1;
                    if (!mbar_wait_cluster(&lfull[at], (taken >> 1) & 1, abort)) {
                        raise(P, abort, kErrTimeoutMma);
                        ok = false;
                        return false;
                    }
                    ++taken;
                    tc_fence_after();
                    const int n8 = message[at];
                    const uint32_t low = smem_u32(sLow + at * kLowBytes);
                    const uint64_t pdesc = make_sw128_kmajor_desc(low);
                    const uint64_t fdesc = make_sw128_kmajor_desc(low + kHalf * 128);
                    for (int part = 0; part < 2; ++part)  // upper bits, then the rest
                        for (int h = 0; h < n8; ++h) {
                            umma_tf32_pair(dlow, pdesc + 4 * part + 2 * h, fdesc + 2 * h,
                                           P.idesc32, have_low);
                            have_low = 1;
                        }
                    umma_commit_pair(&lempty[at]);
                    more = n8 != 0;
                    return true;
                };
                for (int kb = 0; kb < P.num_kb; ++kb) {
                    if (!mbar_wait(&full[stage], phase, abort)) {
                        raise(P, abort, kErrTimeoutMma);
                        ok = false;
                        return false;
                    }
                    tc_fence_after();
                    const uint64_t adesc = make_sw128_kmajor_desc(smem_u32(sA + stage * kABytes));
                    const uint32_t sb = smem_u32(sB + stage * kBBytes);
                    const uint64_t bdesc = P.w_nmajor ? make_sw128_mnmajor_desc(sb, 8192)
                                                      : make_sw128_kmajor_desc(sb);
                    const uint32_t bstep = P.w_nmajor ? 128 : 2;  // 16 inner elements further
#pragma unroll
                    for (int kk = 0; kk < kBK / 16; ++kk)
                        umma_f16_pair(d, adesc + 2 * kk, bdesc + bstep * kk, P.idesc16,
                                      (kb | kk) != 0 ? 1u : 0u);
                    any_issued = true;
                    umma_commit_pair(&empty[stage]);
                    if (++stage == P.stages) {
                        stage = 0;
                        phase ^= 1;
                    }
                    if (more && --until == 0) {
                        until = P.every;
                        if (!low_step()) return false;
                    }
                }
                while (more)
                    if (!low_step()) return false;
                umma_commit_pair(&tfull[acc]);
                return true;
            });
            if (!ok && any_issued) {
                umma_commit_pair(drain);
                drain_wait(P, drain, 0);
            }
        }
    } else if (warp < 2 + kEpiWarps) {
        // ---------------- epilogue (warps 2..9, both CTAs) ----------------
        const int q = warp & 3;              // TMEM lane quadrant this warp may access
        const int part = (warp - 2) >> 2;    // its 128 columns of the tile
        int64_t unit = 0;
        const DropoutKeys key(kDrop ? dropout_key(P.drop) : 0);
        T *out = static_cast<T *>(P.out);
        uint32_t *turn = reinterpret_cast<uint32_t *>(sA + (kStages - 1) * kABytes) +
                         (warp - 2) * kTurnWords;
        // the whole warp has read its accumulator rows: one arrive per warp on CTA 0
        auto release = [&](int acc) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_remote(map_to_rank(smem_u32(&tempty[acc]), 0));
        };
        tiles(P, [&](int tm, int tn) {
            const int acc = static_cast<int>(unit % kBuffers);
            const uint32_t acc_phase = static_cast<uint32_t>((unit / kBuffers) & 1);
            const int slot = static_cast<int>(unit % kFixSlots);
            ++unit;
            const int64_t row = int64_t(tm) * kBM + int64_t(rank) * kHalf + q * 32 + lane;
            const int64_t first = int64_t(tn) * kBN + part * kHalf;
            uint32_t keep[kHalf / 32];  // with dropout: which columns take the low-rank term
            if constexpr (kDrop) {
                const bool has_low = row < P.rows && P.index.at(row) >= 0;
#pragma unroll
                for (int c = 0; c < kHalf / 32; ++c) {
                    uint32_t w = 0;
                    if (has_low) {
#pragma unroll
                        for (int b = 0; b < 4; ++b) {
                            const uint4 bits =
                                dropout_bits(P.drop, key, static_cast<uint32_t>(row),
                                             static_cast<uint32_t>(first >> 3) + 4 * c + b);
#pragma unroll
                            for (int j = 0; j < 8; ++j)
                                w |= static_cast<uint32_t>(dropout_kept(bits, j, P.drop.cut))
                                     << (8 * b + j);
                        }
                    }
                    keep[c] = w;
                }
            }
            if (!mbar_wait(&tfull[acc], acc_phase, abort)) {
                raise(P, abort, kErrTimeoutEpilogue);
                return false;
            }
            __syncwarp();
            tc_fence_after();
            const bool fixup = fix[slot] != 0;
            const uint32_t tbase = tmem_base + (static_cast<uint32_t>(q * 32) << 16) +
                                   static_cast<uint32_t>(acc * kBN + part * kHalf);
            if constexpr (kDrop) {
                uint32_t pk[kHalf / 32][16];
#pragma unroll
                for (int c = 0; c < kHalf / 16; ++c) {
                    uint32_t v[16], low[16];
                    tmem_ld_32x32b_x16(tbase + c * 16, v);
                    tmem_ld_32x32b_x16(tbase + kBN + c * 16, low);
                    tmem_wait_ld();
                    float *y = reinterpret_cast<float *>(v), *l = reinterpret_cast<float *>(low);
                    if (fixup && row < P.rows) add_nonfinite<T>(P, row, first + c * 16, l);
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        if ((keep[c >> 1] >> (16 * (c & 1) + j)) & 1) y[j] += l[j];
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        pk[c >> 1][8 * (c & 1) + j] = pack2<T>(y[2 * j], y[2 * j + 1]);
                }
                release(acc);
#pragma unroll
                for (int c = 0; c < kHalf / 32; ++c)
                    store_block<T>(P, out, turn, row - lane, first + c * 32, lane, pk[c]);
            } else {
#pragma unroll 1
                for (int c = 0; c < kHalf / 32; ++c) {
                    uint32_t v[32], pk[16];
                    float *y = reinterpret_cast<float *>(v);
                    tmem_ld_32x32b_x32(tbase + c * 32, v);
                    tmem_wait_ld();
                    if (fixup && row < P.rows) {
                        add_nonfinite<T>(P, row, first + c * 32, y);
                        add_nonfinite<T>(P, row, first + c * 32 + 16, y + 16);
                    }
#pragma unroll
                    for (int j = 0; j < 16; ++j) pk[j] = pack2<T>(y[2 * j], y[2 * j + 1]);
                    store_block<T>(P, out, turn, row - lane, first + c * 32, lane, pk);
                }
                release(acc);
            }
            return true;
        });
    } else {
        // ---------------- loaders of the low-rank steps (warps 10..13, both CTAs) ----------------
        const int lt = threadIdx.x - 32 * (2 + kEpiWarps);
        int64_t unit = 0;
        uint32_t sent = 0;  // low-rank steps and closing words sent: stage sent % 2
        int turn = 0;
        const uint16_t *F = static_cast<const uint16_t *>(P.F.p);
        const int r = static_cast<int>(P.r);
        asm volatile("griddepcontrol.wait;" ::: "memory");  // the projection is complete
        tiles(P, [&](int tm, int tn) {
            const int slot = static_cast<int>(unit % kFixSlots);
            // Cleared half a round ahead: the other CTA's loaders may be two tiles ahead and raise
            // their flag already, and the epilogue is past the tile that used this slot before.
            if (lt == 0) fix[(unit + kFixSlots / 2) % kFixSlots] = 0;
            ++unit;
            const int64_t row0 = int64_t(tm) * kBM + lt;  // this thread's rows of the pair's tile
            const int i0 = row0 < P.rows ? P.index.at(row0) : -1;
            const int i1 = row0 + kHalf < P.rows ? P.index.at(row0 + kHalf) : -1;
            const int mine = rank ? i1 : i0;
            const int64_t row = row0 + int64_t(rank) * kHalf;
            const int64_t col = int64_t(tn) * kBN + int64_t(rank) * kHalf + lt;
            // a step's reads: 16 ranks of the thread's row and column, as they lie in memory
            struct Reads {
                float4 p[4];
                uint32_t f[kRankStep];  // 8 packed words, or 16 elements
                int nj;
            };
            int cur = -1, j0 = r;
            // The next step: 16 ranks further, or the next adapter in increasing order (the smallest
            // index above `cur` among the pair's rows).
            auto advance = [&]() {
                j0 += kRankStep;
                if (j0 < r) return true;
                j0 = 0;
                const unsigned none = 0x7FFFFFFFu;
                const unsigned c0 = i0 > cur ? static_cast<unsigned>(i0) : none;
                const unsigned c1 = i1 > cur ? static_cast<unsigned>(i1) : none;
                const unsigned m = __reduce_min_sync(0xFFFFFFFFu, min(c0, c1));
                if (lane == 0) least[4 * turn + (lt >> 5)] = static_cast<int>(m);
                loader_sync();
                const int *l = least + 4 * turn;
                turn ^= 1;
                cur = min(min(l[0], l[1]), min(l[2], l[3]));
                return cur != static_cast<int>(none);
            };
            auto fetch = [&](Reads &x) {
                x.nj = min(kRankStep, r - j0);
                const float *prow = P.P + row * P.r + j0;
                const bool take = mine == cur;
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int j = 4 * q;
                    x.p[q] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    if (P.pvec) {  // r is a multiple of 4
                        if (take && j < x.nj) x.p[q] = *reinterpret_cast<const float4 *>(prow + j);
                    } else if (take) {
                        if (j < x.nj) x.p[q].x = prow[j];
                        if (j + 1 < x.nj) x.p[q].y = prow[j + 1];
                        if (j + 2 < x.nj) x.p[q].z = prow[j + 2];
                        if (j + 3 < x.nj) x.p[q].w = prow[j + 3];
                    }
                }
                const uint16_t *src = F + cur * P.F.ss + col * P.F.sc + j0 * P.F.sr;
                const int n = col < P.cols ? x.nj : 0;
                if (P.fvec) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint4 w = load8(src + 8 * h, n - 8 * h);
                        x.f[4 * h] = w.x, x.f[4 * h + 1] = w.y;
                        x.f[4 * h + 2] = w.z, x.f[4 * h + 3] = w.w;
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < kRankStep; ++e) x.f[e] = e < n ? __ldg(src + e * P.F.sr) : 0;
                }
            };
            auto send = [&](const Reads &x) {
                float p[kRankStep], lo[kRankStep], f[kRankStep];
                bool odd = false;
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    p[4 * q] = x.p[q].x, p[4 * q + 1] = x.p[q].y;
                    p[4 * q + 2] = x.p[q].z, p[4 * q + 3] = x.p[q].w;
                }
#pragma unroll
                for (int j = 0; j < kRankStep; ++j) {
                    const uint32_t w = P.fvec ? x.f[j >> 1] >> (16 * (j & 1)) : x.f[j];
                    const uint16_t h = static_cast<uint16_t>(w);
                    f[j] = to_float(*reinterpret_cast<const T *>(&h));
                    if (!finite(f[j])) {
                        odd = true;
                        f[j] = 0.0f;
                    }
                    if (!finite(p[j])) {
                        odd = true;
                        p[j] = 0.0f;
                    }
                    const float hi = __uint_as_float(__float_as_uint(p[j]) & 0xFFFFE000u);
                    lo[j] = p[j] - hi;  // exact
                    p[j] = hi;
                }
                // a wait that gave up is acted on at the barrier, by all loaders alike
                const uint32_t at = sent & 1;
                const bool gave_up = !mbar_wait(&lempty[at], ((sent >> 1) & 1) ^ 1, abort);
                if (gave_up) raise(P, abort, kErrTimeoutProducer);
                ++sent;
                uint8_t *sP = sLow + at * kLowBytes, *sF = sP + kHalf * 128;
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    *swizzled(sP, lt, c) =
                        make_float4(p[4 * c], p[4 * c + 1], p[4 * c + 2], p[4 * c + 3]);
                    *swizzled(sP, lt, 4 + c) =
                        make_float4(lo[4 * c], lo[4 * c + 1], lo[4 * c + 2], lo[4 * c + 3]);
                    *swizzled(sF, lt, c) =
                        make_float4(f[4 * c], f[4 * c + 1], f[4 * c + 2], f[4 * c + 3]);
                }
                if (odd)  // in both CTAs: a row of one meets columns of the other
                    for (uint32_t c = 0; c < 2; ++c)
                        store_flag(map_to_rank(smem_u32(const_cast<const int *>(&fix[slot])), c));
                if (lt == 0) message[at] = (x.nj + 7) / 8;
                fence_proxy_async_smem();
                if (loader_sync_or(gave_up)) return false;
                if (lt == 0) mbar_arrive_remote(map_to_rank(smem_u32(&lfull[at]), 0));
                return true;
            };
            // the next step's reads are on their way while one is written
            Reads now, next;
            bool have = advance();
            if (have) fetch(now);
            while (have) {
                have = advance();
                if (have) fetch(next);
                if (!send(now)) return false;
                now = next;
            }
            const uint32_t at = sent & 1;
            const bool gave_up = !mbar_wait(&lempty[at], ((sent >> 1) & 1) ^ 1, abort);
            if (gave_up) raise(P, abort, kErrTimeoutProducer);
            ++sent;
            if (loader_sync_or(gave_up)) return false;
            if (lt == 0) {
                message[at] = 0;
                mbar_arrive_remote(map_to_rank(smem_u32(&lfull[at]), 0));
            }
            return true;
        });
    }

    // Both CTAs leave their loops before either frees TMEM or exits: CTA 0's MMAs read CTA
    // 1's shared memory and CTA 1's epilogue and loaders arrive on CTA 0's barriers.
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();
    if (warp == 1) {
        __syncwarp();
        tc_fence_after();
        tmem_dealloc_pair(tmem_base, kTmemCols);
    }
}

// Instruction descriptors: D float32, A K-major, B K-major or N-major (bit 16).
constexpr uint32_t idesc(int type, int n, bool b_nmajor) {
    return (1u << 4) | (static_cast<uint32_t>(type) << 7) | (static_cast<uint32_t>(type) << 10) |
           (b_nmajor ? 1u << 16 : 0u) | (static_cast<uint32_t>(n >> 3) << 17) |
           (static_cast<uint32_t>(kBM >> 4) << 24);
}

template <typename T, bool kDrop>
cudaError_t launch(const CUtensorMap &tmM, const CUtensorMap &tmW, const Params &P,
                   cudaStream_t stream) {
    auto kernel = lr_gemm_kernel<T, kDrop>;
    static PerDevice<int> capacity;  // pairs that fit at once
    std::atomic<int> *known = capacity.here();
    if (!known) return cudaErrorInvalidDevice;
    int pairs = known->load(std::memory_order_acquire);
    if (pairs == 0) {
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             static_cast<int>(kSmem));
        if (e != cudaSuccess) return e;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(2 * 1024);
        cfg.blockDim = dim3(kThreads);
        cfg.dynamicSmemBytes = kSmem;
        cudaLaunchAttribute attr;
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim.x = 2;
        attr.val.clusterDim.y = 1;
        attr.val.clusterDim.z = 1;
        cfg.attrs = &attr;
        cfg.numAttrs = 1;
        e = cudaOccupancyMaxActiveClusters(&pairs, kernel, &cfg);
        if (e != cudaSuccess) return e;
        if (pairs < 1) return cudaErrorNotSupported;
        known->store(pairs, std::memory_order_release);
    }
    const int64_t grid = P.total < pairs ? P.total : pairs;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(2 * grid));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = kSmem;
    cfg.stream = stream;
    cudaLaunchAttribute attr;  // (the cluster's shape is the kernel's own)
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, tmM, tmW, P);
}

template <typename T>
cudaError_t expand(const ExpandOperands &o, int *err, cudaStream_t stream) {
    Params P;
    std::memset(&P, 0, sizeof(P));
    P.rows = o.rows;
    P.cols = o.cols;
    P.num_kb = static_cast<int>((o.inner + kBK - 1) / kBK);
    // one adapter's steps and the word that there are no more, spread over the product's steps
    P.every = P.num_kb / static_cast<int>((o.r + kRankStep - 1) / kRankStep + 1);
    P.every = P.every > 16 ? 16 : P.every < 2 ? 2 : P.every;
    P.tiles_m = static_cast<int>((o.rows + kBM - 1) / kBM);
    P.tiles_n = static_cast<int>((o.cols + kBN - 1) / kBN);
    P.total = int64_t(P.tiles_m) * P.tiles_n;
    P.w_nmajor = o.W.s0 != 1;
    const int type = std::is_same<T, __half>::value ? 0 : 1;
    P.idesc16 = idesc(type, kBN, P.w_nmajor);
    P.idesc32 = idesc(2, kBN, false);
    P.P = o.P;
    P.r = o.r;
    P.F = o.F;
    P.index = o.index;
    P.drop = o.drop;
    P.out = o.out;
    P.ldo = o.ldo;
    const uintptr_t bits = reinterpret_cast<uintptr_t>(o.out) | static_cast<uintptr_t>(2 * o.ldo) | 16;
    P.align = static_cast<int>(bits & (~bits + 1));
    P.stages = P.align == 16 ? kStages : kStages - 1;
    P.pvec = o.r % 4 == 0 && (reinterpret_cast<uintptr_t>(o.P) & 15) == 0;
    P.fvec = factor_mode(o.F) == kFR;
    P.err = err;
    CUtensorMap tmM, tmW;
    if (!make_map16(&tmM, o.M.p, o.inner, o.rows, o.M.s0, kBK, kHalf)) return cudaErrorInvalidValue;
    if (P.w_nmajor ? !make_map16(&tmW, o.W.p, o.cols, o.inner, o.W.s0, 64, kBK)
                   : !make_map16(&tmW, o.W.p, o.inner, o.cols, o.W.s1, kBK, kHalf))
        return cudaErrorInvalidValue;
    return o.drop.cut ? launch<T, true>(tmM, tmW, P, stream) : launch<T, false>(tmM, tmW, P, stream);
}

}  // namespace

bool make_map16(CUtensorMap *map, const void *base, int64_t inner, int64_t outer, int64_t ld,
                int box_inner, int box_outer) {
    EncodeTiledFn enc = get_encode_fn();
    if (!enc) return false;
    cuuint64_t dims[2] = {static_cast<cuuint64_t>(inner), static_cast<cuuint64_t>(outer)};
    cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld) * 2};
    cuuint32_t box[2] = {static_cast<cuuint32_t>(box_inner), static_cast<cuuint32_t>(box_outer)};
    cuuint32_t estr[2] = {1, 1};
    return enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, const_cast<void *>(base), dims, strides, box,
               estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

cudaError_t lr_expand_pairs(bool half, const ExpandOperands &o, int *err, cudaStream_t stream) {
    return half ? expand<__half>(o, err, stream) : expand<__nv_bfloat16>(o, err, stream);
}

}  // namespace ti
