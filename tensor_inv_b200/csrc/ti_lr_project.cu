// ti_lr_project.cu -- the project form: P[t] = f * (m M)[t] F[i], i = index[t].
//
//   P[t][j] = alpha * scale[i] * sum_c m(t, c) M[t][c] F[i][c][j]        (float32, t x r)
//
// One pass over M: 2 r operations per element against 2 bytes, so M's bytes bound it for the
// ranks that adapters have, and the legacy tensor path (mma.sync, operands in registers) is fast
// enough -- what counts is that M goes from memory to registers once, with the mask applied on the
// way, and never through shared memory.  Two kernels:
//   tiles: 128 rows x a slice of the inner dimension per CTA; a cluster of up to 8 CTAs shares the
//          rows and adds its slices through distributed shared memory.  Every warp walks the distinct
//          adapters of its own 32 rows (one, for the runs of rows that prompts and training steps
//          have), reads their factor in fragment order straight from the caches and waits for
//          nobody; a row keeps the result of its own adapter.
//   rows:  one row per cluster, plain multiply-adds: for few rows each with an adapter of its own
//          F's bytes bound it, and no product is shared between rows.
#include "ti_lr_dot.cuh"
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
    int64_t slice;  // inner elements per CTA, a multiple of 128 (tiles) or 256 (rows)
    int mode;       // how F is read: kFC vectors along c, kFR vectors along j, kFScalar
};

template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&d)[4], uint32_t a0, uint32_t a1,
                                                        uint32_t a2, uint32_t a3, uint32_t b0,
                                                        uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__half>(float (&d)[4], uint32_t a0, uint32_t a1,
                                                 uint32_t a2, uint32_t a3, uint32_t b0,
                                                 uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void store_cluster(uint32_t addr, float v) {
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v));
}

constexpr int kTileRows = 128, kTileThreads = 256, kGroups = 2;  // two groups share the slice
constexpr int kChunk = 64;  // inner elements per warp and step

template <int kNT>
constexpr size_t tile_smem() {
    return sizeof(float) * kGroups * kTileRows * 8 * kNT;
}

// kNT 16-bit elements in one load (kNT = 1, 2 or 4).
template <int kNT>
__device__ __forceinline__ uint2 load_few(const uint16_t *p) {
    if constexpr (kNT == 4) return __ldg(reinterpret_cast<const uint2 *>(p));
    if constexpr (kNT == 2) return make_uint2(__ldg(reinterpret_cast<const uint32_t *>(p)), 0);
    return make_uint2(__ldg(p), 0);
}

// F's fragments for 32 inner elements: f[n] holds, for column tile n, the thread's elements
// c .. c + 7 of its column, in pairs.  Where F's vectors run along the rank (kFR), a thread reads
// kNT consecutive ranks of each element, so the columns of the tiles interleave: column `g` of
// tile n is rank kNT * g + n, else 8 * n + g.  kWhole: no element lies past the end (c + 8 <= end;
// for kFR, r is a multiple of kNT); the general form handles every edge and every stride.
template <int kNT, int kMode, bool kWhole>
__device__ __forceinline__ void load_fragments(const ProjectParams &P, const uint16_t *F, int64_t c,
                                               int64_t end, int64_t j0, int g, uint4 (&f)[kNT]) {
    const int r = static_cast<int>(P.r);
    if constexpr (kMode == kFR) {
        const int j = static_cast<int>(j0) + kNT * g;
        uint2 v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            v[e] = make_uint2(0, 0);
            const uint16_t *src = F + (c + e) * P.F.sc + j;
            if (kWhole) {
                if (j < r) v[e] = load_few<kNT>(src);
            } else if (c + e < end) {
#pragma unroll
                for (int n = 0; n < kNT; ++n)
                    if (j + n < r)
                        (n < 2 ? v[e].x : v[e].y) |= static_cast<uint32_t>(__ldg(src + n))
                                                     << (16 * (n & 1));
            }
        }
#pragma unroll
        for (int n = 0; n < kNT; ++n) {
            const uint32_t sel = n & 1 ? 0x7632u : 0x5410u;  // upper or lower halves of two words
            auto word = [&](int e) { return n < 2 ? v[e].x : v[e].y; };
            f[n] = make_uint4(__byte_perm(word(0), word(1), sel), __byte_perm(word(2), word(3), sel),
                              __byte_perm(word(4), word(5), sel), __byte_perm(word(6), word(7), sel));
        }
    } else {
#pragma unroll
        for (int n = 0; n < kNT; ++n) {
            const int j = static_cast<int>(j0) + 8 * n + g;
            f[n] = make_uint4(0, 0, 0, 0);
            if (kWhole) {
                if (j < r) f[n] = __ldg(reinterpret_cast<const uint4 *>(F + j * P.F.sr + c));
            } else if (j < r) {
                uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (c + e < end)
                        w[e >> 1] |= static_cast<uint32_t>(__ldg(F + (c + e) * P.F.sc + j * P.F.sr))
                                     << (16 * (e & 1));
                f[n] = make_uint4(w[0], w[1], w[2], w[3]);
            }
        }
    }
}

template <typename T, int kNT, bool kDrop, int kMode>
__global__ void __launch_bounds__(kTileThreads, 2)
    project_tiles_kernel(const __grid_constant__ ProjectParams P) {
    extern __shared__ __align__(16) uint8_t smem[];
    // what this CTA finishes: [sending CTA and group][row of its share][8*kNT]
    float *sum = reinterpret_cast<float *>(smem);
    __shared__ int sidx[kTileRows];
    cluster_arrive();  // awaited before anything is written to another CTA: it must have started

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, tq = lane & 3;
    const int group = warp >> 2;
    const uint32_t crank = cluster_rank(), csize = cluster_size();
    const int share = kTileRows / static_cast<int>(csize);  // rows that each CTA finishes
    const int64_t row0 = int64_t(blockIdx.x / csize) * kTileRows;
    const int64_t j0 = int64_t(blockIdx.y) * 8 * kNT;
    const int64_t begin = int64_t(crank) * P.slice;
    const int64_t end = min(P.cols, begin + P.slice);
    const uint64_t key = kDrop ? dropout_key(P.drop) : 0;

    const int wrow = (warp & 3) * 32;  // this warp's 32 rows; the thread's are wrow + g + 8*i
    const int64_t mine = row0 + wrow + lane;
    const int my = mine < P.rows ? P.index.at(mine) : -1;
    if (group == 0) sidx[wrow + lane] = my;
    int idx[4];
    const uint16_t *M[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        idx[i] = __shfl_sync(0xFFFFFFFFu, my, g + 8 * i);
        M[i] = static_cast<const uint16_t *>(P.M) + (row0 + wrow + g + 8 * i) * P.ld;
    }
    // F's vectors can be read whole (a factor in neither vector order runs as kFC, by elements)
    const bool vectors = P.mode == kMode && (kMode == kFC || P.r % kNT == 0);
    int cur = -1;
    bool started = false;
    while (true) {
        // the next adapter of the warp's rows in increasing order
        const unsigned next = __reduce_min_sync(
            0xFFFFFFFFu, my > cur ? static_cast<unsigned>(my) : 0x7FFFFFFFu);
        if (next == 0x7FFFFFFFu) break;
        cur = static_cast<int>(next);
        const uint16_t *F = static_cast<const uint16_t *>(P.F.p) + cur * P.F.ss;
        float acc[2][kNT][4];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int n = 0; n < kNT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[i][n][e] = 0.0f;

        auto step = [&](int64_t c0, auto whole) {
            constexpr bool kWhole = decltype(whole)::value;
            uint4 x[kChunk / 32][4], f[kChunk / 32][kNT];
#pragma unroll
            for (int s = 0; s < kChunk / 32; ++s) {
                const int64_t c = c0 + 32 * s + 8 * tq;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    x[s][i] = make_uint4(0, 0, 0, 0);
                    if (idx[i] == cur)
                        x[s][i] = kWhole ? __ldg(reinterpret_cast<const uint4 *>(M[i] + c))
                                         : load8(M[i] + c, end - c);
                }
            }
#pragma unroll
            for (int s = 0; s < kChunk / 32; ++s)
                load_fragments<kNT, kMode, kWhole>(P, F, c0 + 32 * s + 8 * tq, end, j0, g, f[s]);
#pragma unroll
            for (int s = 0; s < kChunk / 32; ++s) {
                if (kDrop) {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        x[s][i] = masked(x[s][i], P.drop, key,
                                         static_cast<uint32_t>(row0 + wrow + g + 8 * i),
                                         static_cast<uint32_t>((c0 + 32 * s + 8 * tq) >> 3));
                }
#pragma unroll
                for (int n = 0; n < kNT; ++n) {
                    // the order of the inner dimension is free: a thread's 8 consecutive
                    // elements fill the slots of two k16 steps, in M and F alike
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const uint4 &a = x[s][2 * i], &b = x[s][2 * i + 1];
                        mma16816<T>(acc[i][n], a.x, b.x, a.y, b.y, f[s][n].x, f[s][n].y);
                        mma16816<T>(acc[i][n], a.z, b.z, a.w, b.w, f[s][n].z, f[s][n].w);
                    }
                }
            }
        };
        int64_t c0 = begin + group * kChunk;
        if (vectors)
#pragma unroll 1
            for (; c0 + kChunk <= end; c0 += kGroups * kChunk) step(c0, std::true_type{});
#pragma unroll 1
        for (; c0 < end; c0 += kGroups * kChunk) step(c0, std::false_type{});
        // rows of this adapter keep its sums
        if (!started) {
            started = true;
            cluster_wait();
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (idx[i] == cur) {
                const int lr = wrow + g + 8 * i;
                float *dst = sum + ((crank * kGroups + group) * share + lr % share) * 8 * kNT;
                const uint32_t to = map_to_rank(smem_u32(dst), lr / share);
#pragma unroll
                for (int n = 0; n < kNT; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int col = 2 * tq + e;
                        store_cluster(to + 4 * (kMode == kFR ? kNT * col + n : 8 * n + col),
                                      acc[i >> 1][n][2 * (i & 1) + e]);
                    }
            }
    }
    if (!started) cluster_wait();
    // the kernel that reads P may prepare itself now; it waits for this grid before P
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    cluster_sync_all();  // every sum has arrived; no remote access follows
    // the cluster's slices, added in order
    for (int e = threadIdx.x; e < share * 8 * kNT; e += kTileThreads) {
        const int lr = static_cast<int>(crank) * share + e / (8 * kNT), j = e % (8 * kNT);
        const int64_t t = row0 + lr;
        if (t >= P.rows || j0 + j >= P.r) continue;
        const int i = sidx[lr];
        float v = 0.0f;
        if (i >= 0) {
            for (uint32_t q = 0; q < kGroups * csize; ++q) v += sum[q * share * 8 * kNT + e];
            v *= P.alpha * (P.scale ? P.scale[i] : 1.0f);
        }
        P.P[t * P.r + j0 + j] = v;
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
                                          uint64_t key, uint32_t row, int warp, int lane,
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
                            kDrop ? dropout_key(P.drop) : 0, static_cast<uint32_t>(t), warp, lane,
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

template <typename K>
cudaError_t launch_cluster(K kernel, int parts, dim3 grid, int threads, size_t smem,
                           const ProjectParams &P, cudaStream_t stream) {
    // (Repeated settings are cheap and keep no state per device.)  An SM whose shared memory is
    // carved out small would have to drain before the expanding kernel's CTAs fit beside this one.
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout,
                                         cudaSharedmemCarveoutMaxShared);
    if (e == cudaSuccess && smem > 48 * 1024)
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 static_cast<int>(smem));
    if (e != cudaSuccess) return e;
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
    return cudaLaunchKernelEx(&cfg, kernel, P);
}

template <typename T, int kNT>
cudaError_t tiles(const ProjectParams &P, int parts, dim3 grid, cudaStream_t stream) {
    const size_t smem = tile_smem<kNT>();
    if (P.mode == kFR)
        return P.drop.cut ? launch_cluster(project_tiles_kernel<T, kNT, true, kFR>, parts, grid,
                                           kTileThreads, smem, P, stream)
                          : launch_cluster(project_tiles_kernel<T, kNT, false, kFR>, parts, grid,
                                           kTileThreads, smem, P, stream);
    return P.drop.cut ? launch_cluster(project_tiles_kernel<T, kNT, true, kFC>, parts, grid,
                                       kTileThreads, smem, P, stream)
                      : launch_cluster(project_tiles_kernel<T, kNT, false, kFC>, parts, grid,
                                       kTileThreads, smem, P, stream);
}

template <typename T>
cudaError_t project(ProjectParams P, int num_sms, cudaStream_t stream) {
    int parts = 1;
    if (P.rows <= kProjectRowsLimit) {
        // slices of 1024 (8 elements for each of 128 lanes) until 8 CTAs share a row
        while (parts < 8 && P.cols > 1024 * parts) ++parts;
        P.slice = ((P.cols + parts - 1) / parts + 255) / 256 * 256;
        const dim3 grid(static_cast<unsigned>(parts * P.rows));
        return P.drop.cut ? launch_cluster(project_rows_kernel<T, true>, parts, grid, kRowThreads,
                                           0, P, stream)
                          : launch_cluster(project_rows_kernel<T, false>, parts, grid, kRowThreads,
                                           0, P, stream);
    }
    const int64_t tile_count = (P.rows + kTileRows - 1) / kTileRows;
    // 8, 16 or 32 ranks per CTA; more of them read M again, from L2
    const int nt = P.r <= 8 ? 1 : P.r <= 16 ? 2 : 4;
    const int64_t blocks = (P.r + 8 * nt - 1) / (8 * nt);
    // 1, 2, 4 or 8 CTAs share a tile's inner dimension, until two per SM have work
    constexpr int kStep = kGroups * kChunk;
    while (parts < 8 && tile_count * blocks * parts < 2 * num_sms && P.cols >= 2 * parts * kStep)
        parts *= 2;
    P.slice = ((P.cols + parts - 1) / parts + kStep - 1) / kStep * kStep;
    const dim3 grid(static_cast<unsigned>(parts * tile_count), static_cast<unsigned>(blocks));
    switch (nt) {
        case 1: return tiles<T, 1>(P, parts, grid, stream);
        case 2: return tiles<T, 2>(P, parts, grid, stream);
        default: return tiles<T, 4>(P, parts, grid, stream);
    }
}

}  // namespace

cudaError_t lr_project(bool half, const ProjectOperands &o, int num_sms, cudaStream_t stream) {
    const ProjectParams P{o.M.p,   o.M.s0,  o.rows, o.cols, o.F, o.r,
                          o.index, o.scale, o.alpha, o.drop, o.P, 0, factor_mode(o.F)};
    return half ? project<__half>(P, num_sms, stream) : project<__nv_bfloat16>(P, num_sms, stream);
}

}  // namespace ti
