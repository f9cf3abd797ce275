// ti_lr_wgrad.cu -- the gradients of the adapters: sums over each adapter's rows.
//
//   dA[s][c][j] = sum_{t: index[t] = s} m(t, c) X[t][c] dP[t][j]
//   dB[s][j][c] = sum_{t: index[t] = s} dY[t][c] P[t][j]
//
// Both are out[s] = M^T V with a wide 16-bit M (rows x cols) and a thin float32 V (rows x r); both
// run in one launch.  M's bytes bound them: each element is read once and meets r values of V.
// V keeps its 32 bits by entering mma.sync (tf32) in two parts, its upper 11 bits and the rest, while
// M's 16-bit values are exact in tf32; the legacy tensor path is enough for a product this thin.
// (An infinity in M meets both parts, so its column comes out infinite or NaN.)
//
//   lists  one CTA per adapter writes the positions of its rows, in order, so that an adapter's rows
//          are consecutive; no atomics, so the sums have one order.  A single adapter needs none.
//   wgrad  a CTA takes a chunk of that order and 512 columns, 64 per warp.  Each warp keeps its own
//          ring of asynchronous copies (16 rows x 128 bytes a step, four steps ahead) and waits for
//          no other warp; a thread reads 16 bytes of a row from it -- 8 columns that are the same
//          fragment position of 8 MMAs -- and applies the dropout mask there.  Where a chunk
//          crosses from one adapter to the next it writes its sums to another slot: chunk + adapter
//          numbers the (chunk, adapter) pairs that occur without gaps in either direction.
//   join   adds an adapter's slots in order and rounds once.  One chunk needs no join.
#include "ti_lr_dot.cuh"
#include "ti_lr_launch.cuh"

namespace ti {
namespace {

constexpr int kThreads = 256, kWarpCols = 64, kCtaCols = 8 * kWarpCols;
constexpr int kStage = 128;        // rows of V in shared memory at a time
constexpr int kStep = 16;          // rows of M per copy step
constexpr int kRing = 5;           // steps in a warp's ring: four on their way, one being read
constexpr int kStepBytes = kStep * 128;

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
    int64_t rows, r, s;
    RowIndex index;         // of a single adapter: rows of others are left out
    const int32_t *order;   // row numbers grouped by adapter, or null: all rows, adapter 0
    const int32_t *start;   // [s + 1] first position of each adapter, or null
};

template <typename T>
__device__ __forceinline__ float half_of(uint32_t w, int hi) {
    if constexpr (std::is_same<T, __nv_bfloat16>::value)
        return __uint_as_float(hi ? w & 0xFFFF0000u : w << 16);
    else
        return __half2float(__ushort_as_half(static_cast<unsigned short>(hi ? w >> 16 : w)));
}

__device__ __forceinline__ void mma_tf32(float (&d)[4], const float (&a)[4], float b0, float b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(__float_as_uint(a[0])), "r"(__float_as_uint(a[1])), "r"(__float_as_uint(a[2])),
          "r"(__float_as_uint(a[3])), "r"(__float_as_uint(b0)), "r"(__float_as_uint(b1)));
}

// 16 bytes to shared memory, of which the first `bytes` are read and the others become zero.
__device__ __forceinline__ void copy16(uint32_t dst, const void *src, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes)
                 : "memory");
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

// Accumulators of one warp: 16*kNJ ranks x 64 columns.  In MMA i, column n of the instruction is
// column 8n + i of the warp's 64, so a thread's two columns of a row are 16tq + i and 16tq + 8 + i.
template <typename T, int kNJ>
__device__ __forceinline__ void store_sums(const WgradParams &P, const Side &S,
                                           const float (&acc)[kNJ][8][4], int64_t slot, int64_t s,
                                           int64_t c0, int64_t j0, int g, int tq) {
    const int64_t ldc = (S.cols + 7) / 8 * 8;
#pragma unroll
    for (int nj = 0; nj < kNJ; ++nj)
#pragma unroll
        for (int h = 0; h < 2; ++h) {  // rank g or g + 8
            const int64_t j = j0 + 16 * nj + g + 8 * h;
            if (j >= P.r) continue;
#pragma unroll
            for (int k = 0; k < 2; ++k) {  // columns 16tq + 8k ..
                const int64_t c = c0 + 16 * tq + 8 * k;
                if (c >= S.cols) continue;
                if (S.part) {
                    float4 *dst = reinterpret_cast<float4 *>(S.part + (slot * P.r + j) * ldc + c);
                    dst[0] = make_float4(acc[nj][0][2 * h + k], acc[nj][1][2 * h + k],
                                         acc[nj][2][2 * h + k], acc[nj][3][2 * h + k]);
                    dst[1] = make_float4(acc[nj][4][2 * h + k], acc[nj][5][2 * h + k],
                                         acc[nj][6][2 * h + k], acc[nj][7][2 * h + k]);
                } else {
                    T *dst = static_cast<T *>(S.out) + s * S.ss + j * S.sr;
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (c + i < S.cols)
                            dst[(c + i) * S.sc] = from_float<T>(acc[nj][i][2 * h + k]);
                }
            }
        }
}

template <int kNJ>
constexpr size_t wgrad_smem() {
    return size_t(8) * kRing * kStepBytes + sizeof(float) * kStage * (16 * kNJ + 8) +
           sizeof(int32_t) * kStage;
}

template <typename T, int kNJ>
__global__ void __launch_bounds__(kThreads, 2) wgrad_kernel(const __grid_constant__ WgradParams P) {
    constexpr int kVStride = 16 * kNJ + 8;  // floats: the 4 x 8 fragment reads hit all 32 banks
    extern __shared__ __align__(128) uint8_t smem[];
    float(*sv)[kVStride] = reinterpret_cast<float(*)[kVStride]>(smem + 8 * kRing * kStepBytes);
    int32_t *srow = reinterpret_cast<int32_t *>(sv + kStage);
    const int64_t units_a = P.side[0].blocks * P.side[0].chunks;
    const int which = blockIdx.x < units_a ? 0 : 1;
    const Side &S = P.side[which];
    const int64_t unit = blockIdx.x - (which ? units_a : 0), chunk = unit / S.blocks;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, tq = lane & 3;
    const int64_t c0 = unit % S.blocks * kCtaCols + warp * kWarpCols;
    const int64_t j0 = int64_t(blockIdx.y) * 16 * kNJ;
    const int64_t total = P.start ? P.start[P.s] : P.rows;
    const bool direct = S.part == nullptr;
    int64_t pos = chunk * S.chunk;
    const int64_t stop = min(total, pos + S.chunk);
    const DropoutKeys key(S.drop.cut ? dropout_key(S.drop) : 0);

    // the first adapter whose rows reach past pos (from the first one, where every adapter's
    // gradient is written here)
    int64_t s = 0;
    if (P.start && !direct) {
        int64_t lo = 0, hi = P.s;
        while (lo < hi) {
            const int64_t mid = (lo + hi) / 2;
            if (P.start[mid + 1] > pos) hi = mid;
            else lo = mid + 1;
        }
        s = lo;
    }
    const int64_t col = c0 + 8 * g;
    const uint16_t *M = static_cast<const uint16_t *>(S.M);
    const uint8_t *ring_ptr = smem + warp * kRing * kStepBytes;
    const uint32_t ring = smem_u32(ring_ptr);
    for (; s < P.s && (direct || pos < stop); ++s) {
        const int64_t seg_end = P.start ? min(stop, int64_t(P.start[s + 1])) : stop;
        float acc[kNJ][8][4];
#pragma unroll
        for (int nj = 0; nj < kNJ; ++nj)
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[nj][i][e] = 0.0f;

        for (int64_t b = pos; b < seg_end; b += kStage) {
            const int n = static_cast<int>(min(int64_t(kStage), seg_end - b));
            __syncthreads();  // the previous stage has been read
            if (threadIdx.x < kStage) {
                int t = -1;
                if (static_cast<int>(threadIdx.x) < n) {
                    t = P.order ? P.order[b + threadIdx.x] : static_cast<int32_t>(b + threadIdx.x);
                    if (!P.order && P.index.at(t) != 0) t = -1;
                }
                srow[threadIdx.x] = t;
            }
            __syncthreads();
            const int steps = (n + kStep - 1) / kStep;
            // A lane copies chunk lane % 8 of four of a step's rows.  Chunk c of row q lies at
            // c ^ 2 (q % 4): the 16-byte reads below then hit all banks.
            auto issue = [&](int step) {
                if (step < steps) {
#pragma unroll
                    for (int h = 0; h < 4; ++h) {
                        const int q = (lane >> 3) + 4 * h, c = lane & 7;
                        const int t = srow[step * kStep + q];
                        const int64_t left = S.cols - (c0 + 8 * c);
                        const int bytes =
                            t < 0 || left <= 0 ? 0 : left >= 8 ? 16 : static_cast<int>(2 * left);
                        copy16(ring + (step % kRing) * kStepBytes + q * 128 +
                                   ((c ^ ((q & 3) << 1)) << 4),
                               M + (bytes ? t * S.ld + c0 + 8 * c : 0), bytes);
                    }
                }
                asm volatile("cp.async.commit_group;" ::: "memory");
            };
            for (int k = 0; k < kRing - 1; ++k) issue(k);
            for (int e = threadIdx.x; e < kStage * 16 * kNJ; e += kThreads) {
                const int q = e / (16 * kNJ), j = e % (16 * kNJ);
                const int t = srow[q];
                sv[q][j] = t >= 0 && j0 + j < P.r ? S.V[int64_t(t) * P.r + j0 + j] : 0.0f;
            }
            __syncthreads();
#pragma unroll 1
            for (int k = 0; k < steps; ++k) {
                asm volatile("cp.async.wait_group %0;" ::"n"(kRing - 2) : "memory");
                __syncwarp();
                const int q = k * kStep;
                const uint8_t *src = ring_ptr + (k % kRing) * kStepBytes;
                uint4 x[4];
#pragma unroll
                for (int h = 0; h < 4; ++h)
                    x[h] = *reinterpret_cast<const uint4 *>(src + (4 * h + tq) * 128 +
                                                            ((g ^ (tq << 1)) << 4));
                __syncwarp();
                issue(k + kRing - 1);  // into the slot read in the step before
                if (S.drop.cut) {
#pragma unroll
                    for (int h = 0; h < 4; ++h)
                        x[h] = masked(x[h], S.drop, key,
                                      static_cast<uint32_t>(srow[q + 4 * h + tq]),
                                      static_cast<uint32_t>(col >> 3));
                }
#pragma unroll
                for (int k8 = 0; k8 < 2; ++k8) {  // two steps of 8 rows
                    const int q0 = q + 8 * k8 + tq;
                    const uint4 &xa = x[2 * k8], &xb = x[2 * k8 + 1];
                    const uint32_t m0[4] = {xa.x, xa.y, xa.z, xa.w};
                    const uint32_t m1[4] = {xb.x, xb.y, xb.z, xb.w};
#pragma unroll
                    for (int nj = 0; nj < kNJ; ++nj) {
                        const int j = 16 * nj + g;
                        float hi[4] = {sv[q0][j], sv[q0][j + 8], sv[q0 + 4][j], sv[q0 + 4][j + 8]};
                        float lo[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            // infinities and NaN stay whole in the upper part
                            const uint32_t bits = __float_as_uint(hi[e]);
                            const bool odd = (bits & 0x7F800000u) == 0x7F800000u;
                            const float up = __uint_as_float(bits & 0xFFFFE000u);
                            lo[e] = odd ? 0.0f : hi[e] - up;
                            hi[e] = odd ? hi[e] : up;
                        }
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const float b0 = half_of<T>(m0[i >> 1], i & 1);
                            const float b1 = half_of<T>(m1[i >> 1], i & 1);
                            mma_tf32(acc[nj][i], hi, b0, b1);
                        }
                        // (apart from the first eight, which they would have to wait for)
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const float b0 = half_of<T>(m0[i >> 1], i & 1);
                            const float b1 = half_of<T>(m1[i >> 1], i & 1);
                            mma_tf32(acc[nj][i], lo, b0, b1);
                        }
                    }
                }
            }
            asm volatile("cp.async.wait_group 0;" ::: "memory");
        }
        if (seg_end > pos || direct)
            store_sums<T, kNJ>(P, S, acc, chunk + s, s, c0, j0, g, tq);
        pos = max(pos, seg_end);
    }
}

// out[s][c][j] = the sum of adapter s's slots, in order.
template <typename T>
__global__ void __launch_bounds__(256) join_kernel(const __grid_constant__ WgradParams P) {
    const Side &S = P.side[blockIdx.y];
    if (!S.part) return;
    const int64_t ldc = (S.cols + 7) / 8 * 8;
    const int64_t total = P.start ? P.start[P.s] : P.rows;
    const int64_t quads = (S.cols + 3) / 4;
    for (int64_t u = blockIdx.x * int64_t(blockDim.x) + threadIdx.x; u < P.s * P.r * quads;
         u += int64_t(gridDim.x) * blockDim.x) {
        const int64_t c = u % quads * 4, j = u / quads % P.r, s = u / (quads * P.r);
        const int64_t first = P.start ? P.start[s] : 0;
        const int64_t end = P.start ? P.start[s + 1] : s == 0 ? total : 0;
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (end > first)
            for (int64_t k = first / S.chunk; k <= (end - 1) / S.chunk; ++k) {
                const float4 a =
                    *reinterpret_cast<const float4 *>(S.part + ((k + s) * P.r + j) * ldc + c);
                v.x += a.x;
                v.y += a.y;
                v.z += a.z;
                v.w += a.w;
            }
        T *dst = static_cast<T *>(S.out) + s * S.ss + j * S.sr;
        const float w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (c + e < S.cols) dst[(c + e) * S.sc] = from_float<T>(w[e]);
    }
}

}  // namespace

// Chunks of rows: one wave of CTAs, two per SM, so that the partial sums, which are written and
// read once for each chunk, stay few.  The mask makes a row of dA cost about twice a row of dB
// (4096 x 4096, r = 16: 45 us against 30 us with equal chunks), so dA's chunks are half as long then.
WgradPlan lr_wgrad_plan(int64_t rows, int64_t r, int64_t s, int64_t cols_a, int64_t cols_b,
                        bool listed, bool dropped) {
    constexpr int64_t kCtas = 296;  // fixed: the workspace is sized without a device
    WgradPlan p{};
    const int64_t cols[2] = {cols_a, cols_b}, weight[2] = {dropped ? 2 : 1, 1};
    int64_t cost = 0;
    for (int w = 0; w < 2; ++w)
        cost += weight[w] * ((cols[w] + kCtaCols - 1) / kCtaCols) * (r <= 16 ? 1 : (r + 31) / 32);
    for (int w = 0; w < 2; ++w) {
        int64_t chunks = cost ? weight[w] * kCtas / cost : 1;
        const int64_t most = (rows + 63) / 64;  // 64 rows are worth a chunk
        if (chunks > most) chunks = most;
        if (chunks < 1) chunks = 1;
        p.chunk[w] = ((rows + chunks - 1) / chunks + 15) / 16 * 16;
        if (p.chunk[w] == 0) p.chunk[w] = 16;
        p.chunks[w] = rows ? (rows + p.chunk[w] - 1) / p.chunk[w] : 1;
        if (p.chunks[w] > 1)
            p.part[w] = sizeof(float) * static_cast<size_t>((p.chunks[w] + s - 1) * r *
                                                            ((cols[w] + 7) / 8 * 8));
    }
    p.list_bytes = listed ? sizeof(int32_t) * static_cast<size_t>(rows + s + 1) : 0;
    return p;
}

template <typename T>
static cudaError_t wgrad(const WgradParams &P, int num_sms, cudaStream_t stream) {
    const int nj = P.r <= 16 ? 1 : 2;
    const int64_t units = P.side[0].blocks * P.side[0].chunks + P.side[1].blocks * P.side[1].chunks;
    const dim3 grid(static_cast<unsigned>(units),
                    static_cast<unsigned>((P.r + 16 * nj - 1) / (16 * nj)));
    auto kernel = nj == 1 ? wgrad_kernel<T, 1> : wgrad_kernel<T, 2>;
    const size_t smem = nj == 1 ? wgrad_smem<1>() : wgrad_smem<2>();
    static PerDevice<int> ready[2];
    std::atomic<int> *set = ready[nj - 1].here();
    if (!set) return cudaErrorInvalidDevice;
    if (!set->load(std::memory_order_acquire)) {
        const cudaError_t e = cudaFuncSetAttribute(
            kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
        if (e != cudaSuccess) return e;
        set->store(1, std::memory_order_release);
    }
    kernel<<<grid, kThreads, smem, stream>>>(P);
    if (P.side[0].part || P.side[1].part) {
        const int64_t cols = P.side[0].cols > P.side[1].cols ? P.side[0].cols : P.side[1].cols;
        const int64_t want = (P.s * P.r * ((cols + 3) / 4) + 255) / 256, most = int64_t(num_sms) * 4;
        join_kernel<T><<<dim3(static_cast<unsigned>(want < most ? want : most), 2), 256, 0, stream>>>(P);
    }
    return cudaGetLastError();
}

cudaError_t lr_wgrad(bool half, const WgradOperand &a, const WgradOperand &b, int64_t rows,
                     int64_t r, const RowIndex &index, const WgradPlan &plan, void *lists,
                     int num_sms, cudaStream_t stream) {
    WgradParams P{};
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
