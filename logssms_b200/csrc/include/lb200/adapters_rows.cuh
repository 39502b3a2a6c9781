// Adapters of decoding rows, bfloat16: one launch, a cluster of 4 or 8 CTAs for 1 to 8 rows.
//
// Bound by reading the adapters (a row's rank x (K + N) numbers) and by the chain of a call's steps.  So both products are in one
// kernel: a CTA multiplies its part of K, hands its sums to all CTAs of the cluster (which add them up in the CTAs' order), and adds
// its part of the features to y.  What does not hang on something before it is asked for early: the first features of B and y are on
// their way while the sums are handed over.  Rows are columns of m16n8k16 products whose rows are ranks (A) or features (B): the
// adapters are read as they lie in memory, 16 or 8 bytes a lane (the lanes' pieces are what the product takes as its k, in an order
// that both operands share).  Rows of a cluster that name the same adapter share its reading.  The warps share out the adapters that
// the cluster's rows name, and then the parts of K or the features, so that all of them are read at the same time; a warp's products
// count for the rows of its adapter alone, and nothing of one adapter reaches another's rows.
//
// One row, 1,024 -> 4,096, rank 16: 5.6 us a call; 64 rows of 64 adapters, 4,096 -> 4,096: 9.3 (16.8 MB of adapters, 1.8 TB/s).
//
// Sums are 32-bit.  The short sums go into the second product as two bfloat16 numbers (value and remainder, 2^-17 of it lost): one
// alone would be off by as much as the output's own rounding.
#pragma once
#include "lb200/adapters.cuh"
#include "lb200/adapters_order.cuh"
#include "lb200/common.cuh"

namespace lb200 {
namespace adapter_rows {
typedef __nv_bfloat16 bf16;
constexpr int kMostParts = 8, kWarps = 8, kThreads = 32 * kWarps, kRows = 8;
constexpr int kMostRanks = 256;

__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// n numbers of a row from column c on as pairs, zeros behind `end`; VEC: the row lies so that they are one load
template <bool VEC, int N>
__device__ __forceinline__ void load(uint32_t (&r)[N / 2], const bf16* row, int c, int end) {
    if (VEC) {
        if (c < end) {                                    // (end and c are multiples of N)
            if (N == 8) { const uint4 v = *reinterpret_cast<const uint4*>(row + c); r[0] = v.x; r[1] = v.y; r[2] = v.z; r[N / 2 - 1] = v.w; }
            else { const uint2 v = *reinterpret_cast<const uint2*>(row + c); r[0] = v.x; r[1] = v.y; }
        } else {
#pragma unroll
            for (int i = 0; i < N / 2; ++i) r[i] = 0u;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
            const uint32_t lo = c + 2 * i < end ? reinterpret_cast<const unsigned short*>(row)[c + 2 * i] : 0u;
            const uint32_t hi = c + 2 * i + 1 < end ? reinterpret_cast<const unsigned short*>(row)[c + 2 * i + 1] : 0u;
            r[i] = lo | hi << 16;
        }
    }
}
__device__ __forceinline__ uint32_t smem_at(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void hand(uint32_t at, uint32_t rank, float v) {
    asm volatile("{\n\t.reg .b32 p;\n\tmapa.shared::cluster.u32 p, %0, %1;\n\tst.shared::cluster.f32 [p], %2;\n\t}" ::"r"(at), "r"(rank), "f"(v) : "memory");
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// The rows at places t0 .. t0 + rows - 1.  MT: 16 MT ranks at a time.  XV: rows of x and A lie on 16 bytes and K is a multiple of 8;
// BV: rows of B on 8 bytes, R a multiple of 4.
template <int MT, bool XV, bool BV>
__device__ __forceinline__ void block_of_rows(const AdapterArgs& a, long t0, int rows, int parts) {
    constexpr int kRanks = 16 * MT;
    constexpr int kUnits = MT == 4 ? 1 : 2;                // units of K, or of features, on their way (twice as many features)
    __shared__ float part[kWarps][kRanks][kRows];         // the warps' sums of some ranks
    __shared__ __align__(16) uint32_t high[kRows][kMostRanks / 2 + 4], low[kRows][kMostRanks / 2 + 4];      // the sums times the scale
    extern __shared__ float handed[];                     // [parts][ranks][kRows]: the CTAs' sums
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n = lane >> 2, c = lane & 3;
    const int rank = (int)(blockIdx.x % (unsigned)parts), padded = (a.R + 15) / 16 * 16;
    const bf16* x = (const bf16*)a.x + row_at(a, t0 + min(n, rows - 1)) * a.ldx; // row n of the columns
    const bf16* y = (const bf16*)a.y;
    bf16* out = (bf16*)a.out;
    // this CTA's part of K, in units of 32, and of the features, in units of 16
    const int k_units = (a.K + 31) / 32, k_per = (k_units + parts - 1) / parts;
    const int k_from = min(rank * k_per, k_units), k_to = min(k_from + k_per, k_units);
    const int n_units = (a.N + 15) / 16, n_per = (n_units + parts - 1) / parts;
    const int n_from = min(rank * n_per, n_units), n_to = min(n_from + n_per, n_units);
    // the adapters that the rows name, in ascending order, and each row's place among them (0 for a row without one)
    const int own = lane < rows ? adapter_of(a, t0 + lane) : -1;                 // of row `lane`
    int adapters = 0, place = 0;
    for (int i = next_adapter(own, -1); i != kNoAdapter; i = next_adapter(own, i)) { if (own == i) place = adapters; ++adapters; }
    if (adapters == 0) {                                   // (the same in all warps and CTAs of the cluster)
        for (int i = n_from * 16 + threadIdx.x; i < min(n_to * 16, a.N); i += kThreads)
            for (int r = 0; r < rows; ++r) { const long t = row_at(a, t0 + r); out[t * a.ldo + i] = y[t * a.ldy + i]; }
        return;
    }
    cluster_arrive();                                      // this CTA is there
    // warps take turns at them: 8 / shares warps for each
    const int shares = adapters > 4 ? 8 : adapters > 2 ? 4 : adapters, ours = warp & (shares - 1), team = warp / shares, teams = kWarps / shares;
    const unsigned named = __ballot_sync(0xffffffffu, own >= 0 && place == ours);
    const int i = named != 0 ? __shfl_sync(0xffffffffu, own, __ffs(named) - 1) : -1;       // this warp's adapter
    const int ranks = i >= 0 ? rank_of(a, i) : 0;
    const int place_n = __shfl_sync(0xffffffffu, place, lane & 7);
    const bool ours_n = i >= 0 && __shfl_sync(0xffffffffu, own, n) == i;

    // ------------------------------------------------------------ ranks x rows: this warp's units of K
    // (all of A's ranks: each has a sum of its own, and those behind the adapter's own are left out later)
    for (int j0 = 0; j0 < a.R; j0 += kRanks) {
        const int tiles = min((a.R - j0 + 15) / 16, MT);   // of 16 ranks
        float sum[MT][4] = {};
        if (i >= 0) {
            const bf16* A = (const bf16*)a.A + (size_t)i * a.a_adapter + (size_t)j0 * a.a_row;
            for (int u = k_from + team; u < k_to; u += kUnits * teams) {
                uint32_t xv[kUnits][4], av[kUnits][MT][2][4];
#pragma unroll
                for (int h = 0; h < kUnits; ++h) {
                    const int k = 32 * (u + h * teams) + 8 * c, end = u + h * teams < k_to ? a.K : 0;
                    load<XV, 8>(xv[h], x, k, ours_n ? end : 0);
#pragma unroll
                    for (int m = 0; m < MT; ++m) {
                        const int r = 16 * m + n;
                        load<XV, 8>(av[h][m][0], A + (size_t)r * a.a_row, k, j0 + r < a.R ? end : 0);
                        load<XV, 8>(av[h][m][1], A + (size_t)(r + 8) * a.a_row, k, j0 + r + 8 < a.R ? end : 0);
                    }
                }
#pragma unroll
                for (int h = 0; h < kUnits; ++h)
#pragma unroll
                    for (int m = 0; m < MT; ++m) {
                        mma(sum[m], av[h][m][0][0], av[h][m][1][0], av[h][m][0][1], av[h][m][1][1], xv[h][0], xv[h][1]);
                        mma(sum[m], av[h][m][0][2], av[h][m][1][2], av[h][m][0][3], av[h][m][1][3], xv[h][2], xv[h][3]);
                    }
            }
        }
        if (j0 > 0) __syncthreads();                       // (the last ranks' sums have been read)
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            *reinterpret_cast<float2*>(&part[warp][16 * m + n][2 * c]) = make_float2(sum[m][0], sum[m][1]);
            *reinterpret_cast<float2*>(&part[warp][16 * m + n + 8][2 * c]) = make_float2(sum[m][2], sum[m][3]);
        }
        __syncthreads();
        if (j0 == 0) cluster_wait();                       // every CTA is there
        for (int e = threadIdx.x; e < 16 * tiles * kRows; e += kThreads) {       // (a thread's row is lane % 8)
            if ((lane & 7) >= rows) continue;
            float v = 0.f;
            for (int w = place_n; w < kWarps; w += shares) v += part[w][e / kRows][e % kRows];
            const uint32_t at = smem_at(handed + (rank * padded + j0) * kRows + e);
            for (int p = 0; p < parts; ++p) hand(at, p, v);
        }
    }
    if (a.R <= 0) cluster_wait();
    cluster_arrive();                                      // the sums are handed over
    // ------------------------------------------------------------ the first features and y's are on their way in the meantime
    // The rows that are this warp's to write: those of its adapter, and the first adapter's warps write rows without one.
    constexpr int kAhead = 2 * kUnits;
    const int own0 = __shfl_sync(0xffffffffu, own, 2 * c), own1 = __shfl_sync(0xffffffffu, own, 2 * c + 1);
    const bool write0 = 2 * c < rows && (own0 >= 0 ? own0 == i : ours == 0), write1 = 2 * c + 1 < rows && (own1 >= 0 ? own1 == i : ours == 0);
    const long row0 = row_at(a, t0 + min(2 * c, rows - 1)), row1 = row_at(a, t0 + min(2 * c + 1, rows - 1));
    const bf16* B = (const bf16*)a.B + (size_t)max(i, 0) * a.b_adapter;
    uint32_t bv[kAhead][MT][2][2];
    auto features = [&](int u, int j0) {                   // ranks j0 .. of the features of units u, u + teams, ...
        const int end = min(a.R - j0, kRanks);
#pragma unroll
        for (int h = 0; h < kAhead; ++h)
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                const int f = 16 * (u + h * teams) + n, j = 16 * m + 4 * c;
                const bool there = u + h * teams < n_to;
                load<BV, 4>(bv[h][m][0], B + (size_t)f * a.b_row + j0, j, there && f < a.N ? end : 0);
                load<BV, 4>(bv[h][m][1], B + (size_t)(f + 8) * a.b_row + j0, j, there && f + 8 < a.N ? end : 0);
            }
    };
    bf16 yv[kAhead][4];
    auto outputs = [&](int u) {
#pragma unroll
        for (int h = 0; h < kAhead; ++h)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int f = 16 * (u + h * teams) + n + (e >> 1) * 8;
                if ((e & 1 ? write1 : write0) && u + h * teams < n_to && f < a.N) yv[h][e] = y[(e & 1 ? row1 : row0) * a.ldy + f];
            }
    };
    const int u0 = n_from + team;
    if (i >= 0) { features(u0, 0); outputs(u0); }
    const int who = lane < 8 ? own : -1;                   // (a thread's row in the next loop is lane % 8 again)
    const int its = __shfl_sync(0xffffffffu, who >= 0 ? rank_of(a, who) : 0, lane & 7);
    const float scale = __shfl_sync(0xffffffffu, who >= 0 && a.scales ? a.scales[who] : 1.f, lane & 7);
    cluster_wait();
    for (int e = threadIdx.x; e < padded / 2 * kRows; e += kThreads) {           // two ranks of a row each
        const int r = e % kRows, j = 2 * (e / kRows);
        float v[2] = {0.f, 0.f};
        if (j < its) {                                     // (nothing for a row without an adapter)
            float got[2][kMostParts];
#pragma unroll
            for (int p = 0; p < kMostParts; ++p)
                if (p < parts) {
                    got[0][p] = handed[(p * padded + j) * kRows + r];
                    got[1][p] = handed[(p * padded + j + 1) * kRows + r];
                }
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                float total = 0.f;
#pragma unroll
                for (int p = 0; p < kMostParts; ++p) if (p < parts) total += got[q][p];
                v[q] = j + q < its ? total * scale : 0.f;
            }
        }
        const __nv_bfloat162 h = __floats2bfloat162_rn(v[0], v[1]);
        const float2 back = __bfloat1622float2(h);         // (an infinity has no remainder)
        const __nv_bfloat162 l = __floats2bfloat162_rn(isinf(back.x) ? 0.f : v[0] - back.x, isinf(back.y) ? 0.f : v[1] - back.y);
        high[r][j / 2] = *reinterpret_cast<const uint32_t*>(&h);
        low[r][j / 2] = *reinterpret_cast<const uint32_t*>(&l);
    }
    __syncthreads();
    // ------------------------------------------------------------ features x rows, 16 features to a product
    if (i < 0) return;
    for (int u = u0; u < n_to; u += kAhead * teams) {
        if (u != u0) outputs(u);
        float sum[kAhead][4] = {};
        for (int j0 = 0; j0 < ranks; j0 += kRanks) {
            if (u != u0 || j0 > 0) features(u, j0);
            if (ranks - j0 < kRanks && ranks < a.R) {      // columns behind the adapter's rank may hold anything
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        const int j = j0 + 16 * m + 4 * c + 2 * q;
                        const uint32_t keep = (j < ranks ? 0xffffu : 0u) | (j + 1 < ranks ? 0xffff0000u : 0u);
#pragma unroll
                        for (int h = 0; h < kAhead; ++h) { bv[h][m][0][q] &= keep; bv[h][m][1][q] &= keep; }
                    }
            }
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                const int at = j0 / 2 + 8 * m + 2 * c;
                if (16 * m < ranks - j0) {                 // (behind the rank nothing was written)
                    const uint2 h = ours_n ? *reinterpret_cast<const uint2*>(&high[n][at]) : make_uint2(0u, 0u);
                    const uint2 l = ours_n ? *reinterpret_cast<const uint2*>(&low[n][at]) : make_uint2(0u, 0u);
#pragma unroll
                    for (int w = 0; w < kAhead; ++w) {
                        mma(sum[w], bv[w][m][0][0], bv[w][m][1][0], bv[w][m][0][1], bv[w][m][1][1], h.x, h.y);
                        mma(sum[w], bv[w][m][0][0], bv[w][m][1][0], bv[w][m][0][1], bv[w][m][1][1], l.x, l.y);
                    }
                }
            }
        }
#pragma unroll
        for (int h = 0; h < kAhead; ++h)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int f = 16 * (u + h * teams) + n + (e >> 1) * 8;
                if ((e & 1 ? write1 : write0) && u + h * teams < n_to && f < a.N)
                    out[(e & 1 ? row1 : row0) * a.ldo + f] = (e & 1 ? own1 : own0) >= 0 ? __float2bfloat16_rn(__bfloat162float(yv[h][e]) + sum[h][e]) : yv[h][e];
            }
    }
}

// grid: clusters, each with rows_per rows, or with a tile of rows in order
template <int MT, bool XV, bool BV>
__global__ void __launch_bounds__(kThreads, MT == 1 ? 3 : 2) adapter_rows_kernel(AdapterArgs a, int rows_per, int parts) {
    pdl_wait();
    const long cluster = blockIdx.x / (unsigned)parts, t0 = cluster * rows_per;
    if (a.order == nullptr) {
        block_of_rows<MT, XV, BV>(a, t0, (int)min((long)rows_per, a.T - t0), parts);
    } else if (cluster < *a.n_tiles) {
        const int4 its = a.tiles[cluster];
        block_of_rows<MT, XV, BV>(a, its.y, its.z, parts);
    }
}

template <int MT, bool XV, bool BV>
inline int launch_as(const AdapterArgs& a, cudaStream_t stream) {
    // About 64 clusters while there are rows for them; of 8 CTAs where all of them are on an SM at once, else of 4.
    int rows_per = 1;
    while (rows_per < kRows && a.T > 64 * rows_per) rows_per *= 2;
    const long clusters = a.order == nullptr ? (a.T + rows_per - 1) / rows_per : adapter_order::most_tiles(a.T, a.adapters, kRows);
    const int parts = clusters <= 40 ? 8 : 4;
    if (clusters * parts > 0x7fffffffL) return kTooLarge;
    const size_t smem = (size_t)parts * ((a.R + 15) / 16 * 16) * kRows * sizeof(float);
    static SharedLimits limits;
    int rc = ensure_dynamic_smem(adapter_rows_kernel<MT, XV, BV>, smem + 25 * 1024, limits);        // (with what it has besides)
    if (rc != 0) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(clusters * parts)); cfg.blockDim = dim3(kThreads); cfg.dynamicSmemBytes = smem; cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)parts; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr; cfg.numAttrs = 2;
    return launched(cudaLaunchKernelEx(&cfg, adapter_rows_kernel<MT, XV, BV>, a, rows_per, parts));
}
template <bool XV, bool BV>
inline int launch_ranks(const AdapterArgs& a, cudaStream_t stream) {
    return a.R <= 16 ? launch_as<1, XV, BV>(a, stream) : a.R <= 32 ? launch_as<2, XV, BV>(a, stream) : launch_as<4, XV, BV>(a, stream);
}

inline int launch(const AdapterArgs& a, cudaStream_t stream) {
    const bool xv = ((uintptr_t)a.x & 15) == 0 && ((uintptr_t)a.A & 15) == 0 && a.ldx % 8 == 0 && a.a_row % 8 == 0 && a.a_adapter % 8 == 0 && a.K % 8 == 0;
    const bool bv = ((uintptr_t)a.B & 7) == 0 && a.b_row % 4 == 0 && a.b_adapter % 4 == 0 && a.R % 4 == 0;
    const int rc = xv ? bv ? launch_ranks<true, true>(a, stream) : launch_ranks<true, false>(a, stream)
                      : bv ? launch_ranks<false, true>(a, stream) : launch_ranks<false, false>(a, stream);
    return rc != 0 ? rc : launch_status();
}

}  // namespace adapter_rows
}  // namespace lb200
