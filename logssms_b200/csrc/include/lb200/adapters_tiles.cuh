// Adapters of prompts, bfloat16, on the 5th-generation tensor cores: tiles of 128 rows, one launch.
//
// Bound by reading x and y and writing the output once: the products are a tenth of that.  8,192 rows, 4,096 -> 12,288, 8 adapters of
// rank 64: 100 us, 4.9 TB/s (74 us at the copy rate).  A cluster of 1 to 8 CTAs (as many as make
// about as many CTAs as there are SMs) has a tile.  Each CTA multiplies its part of K (x and A by TMA, 64 columns a stage, one product
// for each adapter that the tile's rows name, at most four: their A tiles lie side by side as one B operand); the CTAs' sums meet in
// distributed shared memory, each CTA adding up a part of the rows and handing them, times the scale and as two bfloat16 numbers
// (value and remainder), to all; then each CTA goes through its part of the features, 128 at a time: y by TMA into shared memory, the
// product of the short sums with B beside it, and the rows of y that name the adapter get its product added in place, from where TMA
// stores them.  Rows of one adapter never see another's product: it is made for all 128 rows and kept by those that name it.
//
// 12 warps: TMA loads of x and y, products, loads of B (and zeros behind an adapter's rank: 0 x NaN would be NaN), TMA stores, and two
// groups of 128 threads, a thread per row, which take the tiles of features in turn.
//
// A tile whose rows name more adapters than that (decoding rows in front of a prompt, a batch in any order) is left to others: the
// rows of all such tiles are put in the order of their adapters (adapters_order.cuh), and the grid's last clusters take them by tiles of
// one adapter each, whose rows TMA gathers and scatters four at a time.  A tile's last four may hold its last row several times; the
// rows behind them hold anything, which nothing of the others' depends on.  8,000 rows in random order: 264 us with 8 adapters, 378 with
// 60 (row by row 2,892 and 3,407).
//
// PLAIN: the rows of y or of the output do not lie at multiples of 16 bytes (an odd number of features).  Every eighth row does, or lies
// as far behind one: eight tensors, 8 columns more than a tile's, hold all rows.  Gathered rows come one by one, by copies of the pieces
// of 16 bytes that have any of a row's columns.  The products, turned round in shared memory, are added by whole warps row by row and
// stored 2 bytes a lane.  8,000 x 12,001, rank 61: 220 us for the tiles; rows copied one by one, both ways 660 and in alone 333 (a copy costs about
// as much as sixteen rows of a tensor's box); y read 2 bytes a lane 860 (beside 227 KB of shared memory little of the L1 is left, and few
// such reads are on their way).  Such a tile has two adapters at most.  x, A and B that do not lie so are copied first (adapters_lay.cuh).
#pragma once
#include <type_traits>
#include "lb200/adapters.cuh"
#include "lb200/adapters_lay.cuh"
#include "lb200/adapters_order.cuh"
#include "lb200/common.cuh"
#include "lb200/tcgen05.cuh"

namespace lb200 {
namespace adapter_tiles {
using namespace tc;
typedef __nv_bfloat16 bf16;
constexpr int kRows = 128, kCols = 128, kMost = 4;        // rows and features of a tile, adapters
constexpr int kFirstAdder = 4, kThreads = 32 * (kFirstAdder + 8);
constexpr uint32_t kXTile = kRows * 128, kYTile = 2 * kRows * 128;
constexpr int kPlainY = 3;                                // PLAIN: tiles of y on their way or at work
constexpr uint32_t kPlainPitch = kCols * 2 + 16, kPlainTile = kRows * kPlainPitch;
constexpr int kTurned = 36;                               // numbers from row to row of the turned products (16 bytes at a time hit all banks once)
struct Eighths { CUtensorMap map[8]; };                   // rows e, e + 8, ... of y, from the 16-byte boundary at or in front of row e on
__device__ __forceinline__ int plain_slot(int row) { return (row & 7) * 16 + (row >> 3); }

// RB: blocks of 64 ranks
template <int RB> struct Shape {
    // Tiles of y and of B on their way or at work.  Three of y held 4.5 TB/s, five 5.4: a tile is on its way, at work, or being
    // stored for a microsecond or two each.
    static constexpr int kY = RB == 1 ? 5 : 3, kB = 2;
    static constexpr uint32_t kBTile = RB * kCols * 128, kH = RB * kRows * 128;  // bytes; of the short sums' values (remainders the same)
    static constexpr uint32_t kSums = kRows * (RB * 64 + 4) * 4;                 // this CTA's sums, float32
    // short sums | y ring | B ring; the first product's ring and this CTA's sums lie over both, which are filled afterwards
    static constexpr uint32_t kRings = kY * kYTile + kB * kBTile, kWork = 2 * kH + kRings;
    static_assert(kSums <= kRings, "sums over the rings");
    static constexpr uint32_t kSmem = kWork + 1024 + 640; // ... | barriers, the rows' scales, ranks and places
    static constexpr int kMostStages = 8;
    static_assert(kSmem <= 227 * 1024, "shared memory");
};

struct TileArgs {
    AdapterArgs a;
    int straight;                                         // tiles of rows as they come
    int parts, padded, limit;                             // CTAs of a cluster; ranks, filled up to a multiple of 16; adapters of such a tile
    int* error;
};

__device__ __forceinline__ void report(int* error, int role, int step) { atomicCAS(error, 0, (role << 24) | ((blockIdx.x & 0xFFF) << 12) | (step & 0xFFF) | 0x40000000); }
__device__ __forceinline__ void cluster_meet() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t at_rank(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ float4 remote4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void hand2(uint32_t addr, uint32_t x, uint32_t y) {
    asm volatile("st.shared::cluster.v2.b32 [%0], {%1, %2};" ::"r"(addr), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ void fence_async_all() { asm volatile("fence.proxy.async;" ::: "memory"); }
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, const void* src, int x, int y) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(map), "r"(x), "r"(y), "r"(smem_u32(src)) : "memory");
}

__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
                 ::"r"(smem_u32(dst)), "l"(map), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z) : "memory");
}

// four rows each
__device__ __forceinline__ void tma_gather4(void* dst, const CUtensorMap* map, uint64_t* bar, int x, const int4& rows) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6, %7}], [%2];"
                 ::"r"(smem_u32(dst)), "l"(map), "r"(smem_u32(bar)), "r"(x), "r"(rows.x), "r"(rows.y), "r"(rows.z), "r"(rows.w) : "memory");
}
__device__ __forceinline__ void tma_scatter4(const CUtensorMap* map, const void* src, int x, const int4& rows) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile::scatter4.bulk_group [%0, {%1, %2, %3, %4, %5}], [%6];"
                 ::"l"(map), "r"(x), "r"(rows.x), "r"(rows.y), "r"(rows.z), "r"(rows.w), "r"(smem_u32(src)) : "memory");
}

// grid: (tiles of rows as they come, then tiles of rows in order) x parts; a cluster: a tile's parts
template <int RB, bool PLAIN>
__global__ void __launch_bounds__(kThreads)
adapter_tiles_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                     const __grid_constant__ CUtensorMap map_y, const __grid_constant__ CUtensorMap map_out, const __grid_constant__ CUtensorMap map_x1,
                     const __grid_constant__ CUtensorMap map_y1, const __grid_constant__ CUtensorMap map_out1,
                     const __grid_constant__ Eighths eighths, TileArgs ta) {
    typedef Shape<RB> Sh;
    static_assert(!PLAIN || kPlainY * kPlainTile + 8 * 32 * kTurned * 4 <= Sh::kY * kYTile, "the tiles of y and the turned products");
    const AdapterArgs& a = ta.a;
    extern __shared__ __align__(1024) uint8_t base[];      // (the swizzle goes by the address)
    uint8_t* h_s = base;                                  // values: blocks of 64 ranks, [128][128 B]; then remainders
    uint8_t* y_s = h_s + 2 * Sh::kH;
    uint8_t* b_s = y_s + Sh::kY * kYTile;
    float* sums = reinterpret_cast<float*>(y_s);
    uint8_t* ring = y_s;                                  // the first product's: x tile, then the adapters' A tiles
    uint64_t* bars = reinterpret_cast<uint64_t*>(base + Sh::kWork);
    uint64_t* x_full = bars;                              // [kMostStages]
    uint64_t* x_empty = x_full + Sh::kMostStages;
    uint64_t* low_ready = x_empty + Sh::kMostStages;      // the first product is done
    uint64_t* b_full = low_ready + 1;
    uint64_t* b_clear = b_full + Sh::kB;                  // ... and has nothing behind its adapter's rank
    uint64_t* b_empty = b_clear + Sh::kB;
    uint64_t* y_full = b_empty + Sh::kB;
    uint64_t* y_empty = y_full + Sh::kY;
    uint64_t* y_done = y_empty + Sh::kY;                  // the sums are in y's place (128 arrivals)
    uint64_t* d_full = y_done + Sh::kY;                   // [4]: per group of adders two accumulators
    uint64_t* d_empty = d_full + 4;
    int* list = reinterpret_cast<int*>(d_empty + 4);      // the adapters, their ranks
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(list + 2 * kMost);
    volatile int* failed = reinterpret_cast<volatile int*>(tmem_slot + 1);
    float* row_scale = reinterpret_cast<float*>(tmem_slot + 2);        // [128]
    unsigned char* row_ranks = reinterpret_cast<unsigned char*>(row_scale + kRows);     // [128]: 0 without an adapter
    int4* fours = reinterpret_cast<int4*>(base + Sh::kWork + 1152);              // the rows of a tile in order, four by four
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = (int)(blockIdx.x % (unsigned)ta.parts), tile = (int)(blockIdx.x / (unsigned)ta.parts);
    const long t0 = (long)tile * kRows;

    // ------------------------------------------------------------ who is in the tile (all warps alike)
    int count = 0, who[kMost] = {}, n_fours = 0, n_rows = 0;           // n_fours > 0: the tile's rows are gathered
    // (the kernel in front, which puts rows in order, has waited for all others before this one began)
    auto straight_adapter = [&](long t) { const int i = t < a.T ? a.index[t] : -1; return i >= 0 && i < a.adapters ? i : -1; };
    if (a.order == nullptr || tile >= ta.straight) pdl_wait();
    if (tile >= ta.straight) {
        const int at = tile - ta.straight;
        if (at >= *a.n_tiles) return;                      // (the whole cluster)
        const int4 its = a.tiles[at];
        count = its.x >= 0 ? 1 : 0;
        who[0] = its.x;
        n_rows = its.z;
        n_fours = (n_rows + 3) / 4;
        if (threadIdx.x < 4 * n_fours) reinterpret_cast<int*>(fours)[threadIdx.x] = a.order[its.y + min((int)threadIdx.x, n_rows - 1)];
    } else {
        int own[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) own[q] = straight_adapter(t0 + 32 * q + lane);
        int prev = -1;
        while (true) {
            int best = kNoAdapter;
#pragma unroll
            for (int q = 0; q < 4; ++q) if (own[q] > prev) best = min(best, own[q]);
            best = __reduce_min_sync(0xffffffffu, best);
            if (best == kNoAdapter) break;
#pragma unroll
            for (int q = 0; q < kMost; ++q) if (q == count) who[q] = best;
            prev = best;
            if (++count > ta.limit) return;                // (the whole cluster: these rows are put in order)
        }
    }
    const int n_tiles = (a.N + kCols - 1) / kCols, mine = n_tiles > rank ? (n_tiles - rank + ta.parts - 1) / ta.parts : 0;      // tiles rank, rank + parts, ...
    const int k_tiles = count > 0 ? (a.K + 63) / 64 : 0, k_per = (k_tiles + ta.parts - 1) / ta.parts;
    const int k_from = min(rank * k_per, k_tiles), k_n = min(k_per, k_tiles - k_from);
    const uint32_t a_tile = ta.padded * 128, stage = kXTile + count * a_tile, x_bytes = n_fours > 0 ? n_fours * 512 : kXTile;    // (A tiles: multiples of 2,048 bytes)
    const int stages = min((int)((Sh::kWork - 2 * Sh::kH) / stage), Sh::kMostStages);

    if (threadIdx.x == 0) {
        for (int s = 0; s < Sh::kMostStages; ++s) { mbar_init(x_full + s, 1); mbar_init(x_empty + s, 1); }
        mbar_init(low_ready, 1);
        for (int s = 0; s < Sh::kB; ++s) { mbar_init(b_full + s, 1); mbar_init(b_clear + s, 1); mbar_init(b_empty + s, 1); }
        for (int s = 0; s < Sh::kY; ++s) { mbar_init(y_full + s, 1); mbar_init(y_empty + s, PLAIN ? 128 : 1); mbar_init(y_done + s, 128); }
        for (int s = 0; s < 4; ++s) { mbar_init(d_full + s, 1); mbar_init(d_empty + s, 128); }
        for (int q = 0; q < kMost; ++q) { list[q] = who[q]; list[kMost + q] = q < count ? rank_of(a, who[q]) : 0; }
        *failed = 0;
        mbar_fence_init();
    }
    if (warp == 1) tmem_alloc<512>(tmem_slot);
    fence_before_sync();
    __syncthreads();
    fence_after_sync();
    const uint32_t tmem = *tmem_slot;

    // a wait of a whole warp
    auto wait = [&](uint64_t* bar, uint32_t parity, int role, int step) -> bool {
        const bool ok = __all_sync(0xffffffffu, (mbar_test(bar, parity) || mbar_wait(bar, parity)) && !*failed);
        if (!ok) { if (lane == 0 && !*failed) report(ta.error, role, step); *failed = 1; }
        return ok;
    };

    // ------------------------------------------------------------ short sums: this CTA's part of K
    int issued = 0;
    if (warp == 0) {
        for (int i = 0; i < k_n; ++i) {
            const int s = i % stages;
            if (i >= stages && !wait(x_empty + s, ((i / stages) - 1) & 1, 1, i)) break;
            if (elect_one()) {
                uint8_t* at = ring + s * stage;
                mbar_expect_tx(x_full + s, x_bytes + count * a_tile);
                if (n_fours == 0) tma_load_2d(at, &map_x, x_full + s, (k_from + i) * 64, (int)t0);
                for (int f = 0; f < n_fours; ++f) tma_gather4(at + f * 512, &map_x1, x_full + s, (k_from + i) * 64, fours[f]);
                for (int q = 0; q < count; ++q) tma_load_3d(at + kXTile + q * a_tile, &map_a, x_full + s, (k_from + i) * 64, 0, list[q]);
            }
            __syncwarp();
            issued = i + 1;
        }
        if (*failed) for (int i = max(0, issued - stages); i < issued; ++i) mbar_wait(x_full + i % stages, (i / stages) & 1);
    } else if (warp == 1 && k_n > 0) {
        const uint32_t idesc = umma_idesc(kRows, ta.padded);
        const uint64_t desc0 = umma_desc(ring);
        bool ok = true;
        for (int i = 0; i < k_n && ok; ++i) {
            const int s = i % stages;
            ok = wait(x_full + s, (i / stages) & 1, 2, i);
            if (!ok) break;
            fence_after_sync();
            if (elect_one()) {
                const uint64_t xd = desc0 + (uint64_t)(s * (stage >> 4));
                for (int q = 0; q < count; ++q) {
                    const uint64_t ad = xd + ((kXTile + q * a_tile) >> 4);
#pragma unroll
                    for (int k = 0; k < 4; ++k) umma_bf16(tmem + q * ta.padded, xd + 2 * k, ad + 2 * k, idesc, (i > 0 || k > 0) ? 1u : 0u);
                }
                umma_commit(x_empty + s);
                if (i + 1 == k_n) umma_commit(low_ready);
            }
            __syncwarp();
        }
    }
    const int group = (warp - kFirstAdder) >> 2, r = (warp & 3) * 32 + lane;     // of an adder: its row is its lane of tensor memory
    const uint32_t lane_addr = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const int own = warp < kFirstAdder ? -1 : n_fours == 0 ? straight_adapter(t0 + r) : r < 4 * n_fours ? who[0] : -1;
    int place = -1;
    if (own >= 0)
        for (int q = 0; q < count; ++q) if (list[q] == own) place = q;
    if (warp >= kFirstAdder && group == 1) {
        row_scale[r] = own >= 0 && a.scales ? a.scales[own] : 1.f;
        row_ranks[r] = (unsigned char)(own >= 0 ? rank_of(a, own) : 0);
    }
    if (warp >= kFirstAdder && group == 0 && count > 0) {
        float* to = sums + r * (RB * 64 + 4);
        const bool ok = k_n <= 0 || wait(low_ready, 0, 5, 0);
        fence_after_sync();
        for (int j = 0; j < ta.padded; j += 16) {
            float keep[16] = {};
            if (ok && k_n > 0)
                for (int q = 0; q < count; ++q) {
                    uint32_t v[16];
                    tmem_get16(lane_addr + q * ta.padded + j, v);
                    if (place == q) {
#pragma unroll
                        for (int e = 0; e < 16; ++e) keep[e] = __uint_as_float(v[e]);
                    }
                }
#pragma unroll
            for (int e = 0; e < 16; e += 4) *reinterpret_cast<float4*>(to + j + e) = make_float4(keep[e], keep[e + 1], keep[e + 2], keep[e + 3]);
        }
        fence_before_sync();
    }
    __syncthreads();
    if (ta.parts > 1) cluster_meet();
    // ------------------------------------------------------------ this CTA's part of the rows: all CTAs' sums, handed to all
    if (warp >= kFirstAdder && count > 0) {
        const int pieces = ta.padded / 4;                  // four ranks
        const uint32_t from = smem_u32(sums), to = smem_u32(h_s);
        for (int i = threadIdx.x - 32 * kFirstAdder; i < kRows / ta.parts * pieces; i += 256) {
            const int row = rank * (kRows / ta.parts) + i / pieces, j = 4 * (i % pieces);
            const int ranks = row_ranks[row];
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            if (j < ranks) {
                const uint32_t at = from + 4 * (row * (RB * 64 + 4) + j);
                float4 got[8];
#pragma unroll
                for (int p = 0; p < 8; ++p) if (p < ta.parts) got[p] = remote4(ta.parts > 1 ? at_rank(at, p) : at);
#pragma unroll
                for (int p = 0; p < 8; ++p) if (p < ta.parts) { v.x += got[p].x; v.y += got[p].y; v.z += got[p].z; v.w += got[p].w; }
                const float scale = row_scale[row];
                v.x *= scale;
                v.y = j + 1 < ranks ? v.y * scale : 0.f;
                v.z = j + 2 < ranks ? v.z * scale : 0.f;
                v.w = j + 3 < ranks ? v.w * scale : 0.f;
            }
            const __nv_bfloat162 h0 = __floats2bfloat162_rn(v.x, v.y), h1 = __floats2bfloat162_rn(v.z, v.w);
            const float2 b0 = __bfloat1622float2(h0), b1 = __bfloat1622float2(h1);         // (an infinity has no remainder)
            const __nv_bfloat162 l0 = __floats2bfloat162_rn(isinf(b0.x) ? 0.f : v.x - b0.x, isinf(b0.y) ? 0.f : v.y - b0.y);
            const __nv_bfloat162 l1 = __floats2bfloat162_rn(isinf(b1.x) ? 0.f : v.z - b1.x, isinf(b1.y) ? 0.f : v.w - b1.y);
            // rank j of a row: block j / 64, piece (j % 64) / 8 at (that) ^ (row & 7)
            const uint32_t at = to + (j >> 6) * (kRows * 128) + row * 128 + ((((j & 63) >> 3) ^ (row & 7)) << 4) + (j & 7) * 2;
            for (int p = 0; p < ta.parts; ++p) {
                const uint32_t there = ta.parts > 1 ? at_rank(at, p) : at;
                hand2(there, *reinterpret_cast<const uint32_t*>(&h0), *reinterpret_cast<const uint32_t*>(&h1));
                hand2(there + Sh::kH, *reinterpret_cast<const uint32_t*>(&l0), *reinterpret_cast<const uint32_t*>(&l1));
            }
        }
        fence_async_all();
    }
    __syncthreads();
    if (ta.parts > 1) cluster_meet();
    fence_async_all();

    // ------------------------------------------------------------ this CTA's tiles of features
    const int steps = mine * max(count, 1);                // (tile, adapter) by (tile, adapter)
    if (PLAIN && warp == 0) {
        int y_asked = 0;
        for (int i = 0; i < mine && !*failed; ++i) {
            const int n0 = (rank + i * ta.parts) * kCols, s = i % kPlainY, bytes = 2 * min(kCols, a.N - n0);
            if (i >= kPlainY && !wait(y_empty + s, ((i / kPlainY) - 1) & 1, 6, i)) break;
            if (n_fours == 0) {                            // eight tensors of every eighth row, whose rows are 16 ldy bytes apart
                if (elect_one()) {
                    mbar_expect_tx(y_full + s, kPlainTile);
                    for (int e = 0; e < 8; ++e) tma_load_2d(y_s + s * kPlainTile + e * (16 * kPlainPitch), &eighths.map[e], y_full + s, n0, (int)(t0 >> 3));
                }
            } else {
                uintptr_t from[4];
                uint32_t length[4], all = 0;
#pragma unroll
                for (int q = 0; q < 4; ++q) {              // the pieces of 16 bytes that have any of the row's columns
                    const int r = 32 * q + lane;
                    const uintptr_t at = (uintptr_t)((const bf16*)a.y + (long)(r < n_rows ? reinterpret_cast<int*>(fours)[r] : 0) * a.ldy + n0);
                    from[q] = at & ~(uintptr_t)15;
                    length[q] = r < n_rows ? (uint32_t)(((at + bytes + 15) & ~(uintptr_t)15) - from[q]) : 0u;
                    all += length[q];
                }
                all = __reduce_add_sync(0xffffffffu, all);
                if (lane == 0) mbar_expect_tx(y_full + s, all);
                __syncwarp();
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    if (length[q] != 0)
                        asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                                     ::"r"(smem_u32(y_s + s * kPlainTile + plain_slot(32 * q + lane) * kPlainPitch)), "l"(from[q]), "r"(length[q]), "r"(smem_u32(y_full + s)) : "memory");
            }
            __syncwarp();
            y_asked = i + 1;
        }
        if (*failed) {
            for (int i = max(0, y_asked - kPlainY); i < y_asked; ++i) mbar_wait(y_full + i % kPlainY, (i / kPlainY) & 1);
        }
    } else if (PLAIN && warp == 3) {
        // (the adders store)
    } else if (warp == 0) {
        int y_asked = 0;
        for (int i = 0; i < mine && !*failed; ++i) {
            const int n0 = (rank + i * ta.parts) * kCols, s = i % Sh::kY;
            if (i >= Sh::kY && !wait(y_empty + s, ((i / Sh::kY) - 1) & 1, 6, i)) break;
            if (elect_one()) {
                const bool both = n_fours == 0 || n0 + 64 < a.N;
                mbar_expect_tx(y_full + s, both ? 2 * x_bytes : x_bytes);
                if (n_fours == 0) {
                    tma_load_2d(y_s + s * kYTile, &map_y, y_full + s, n0, (int)t0);
                    tma_load_2d(y_s + s * kYTile + kRows * 128, &map_y, y_full + s, n0 + 64, (int)t0);
                }
                for (int f = 0; f < n_fours; ++f) {
                    const int4 rows = fours[f];
                    tma_gather4(y_s + s * kYTile + f * 512, &map_y1, y_full + s, n0, rows);
                    if (both) tma_gather4(y_s + s * kYTile + kRows * 128 + f * 512, &map_y1, y_full + s, n0 + 64, rows);
                }
            }
            __syncwarp();
            y_asked = i + 1;
        }
        if (*failed) {                                     // let the copies already under way land before the CTA leaves
            for (int i = max(0, y_asked - Sh::kY); i < y_asked; ++i) mbar_wait(y_full + i % Sh::kY, (i / Sh::kY) & 1);
        }
    } else if (warp == 1 && count > 0) {
        constexpr uint32_t idesc = umma_idesc(kRows, kCols);
        const uint64_t hd = umma_desc(h_s), bd0 = umma_desc(b_s);
        for (int u = 0; u < steps; ++u) {
            const int i = u / count, q = u - i * count, sb = u % Sh::kB, grp = i & 1;
            const int v = (i >> 1) * count + q, d = 2 * grp + (v & 1);           // the group's step, its accumulator
            if (!wait(b_clear + sb, (u / Sh::kB) & 1, 8, u)) break;
            if (v >= 2 && !wait(d_empty + d, ((v >> 1) - 1) & 1, 9, u)) break;
            fence_after_sync();
            const int k_steps = (list[kMost + q] + 15) / 16;
            if (elect_one()) {
                const uint64_t bd = bd0 + (uint64_t)(sb * (Sh::kBTile >> 4));
                const uint32_t to = tmem + d * kCols;
                for (int k = 0; k < k_steps; ++k) {
                    const uint64_t off = (uint64_t)((k >> 2) * (kRows * 128 >> 4) + 2 * (k & 3));
                    umma_bf16(to, hd + off, bd + off, idesc, k > 0 ? 1u : 0u);
                    umma_bf16(to, hd + (Sh::kH >> 4) + off, bd + off, idesc, 1u);
                }
                umma_commit(b_empty + sb);
                umma_commit(d_full + d);
            }
            __syncwarp();
        }
    } else if (warp == 2 && count > 0) {
        int b_asked = 0;
        auto ask = [&](int u) -> bool {                    // B of step u
            const int i = u / count, q = u - i * count, sb = u % Sh::kB, n0 = (rank + i * ta.parts) * kCols;
            if (u >= Sh::kB && !wait(b_empty + sb, ((u / Sh::kB) - 1) & 1, 7, u)) return false;
            if (elect_one()) {
                mbar_expect_tx(b_full + sb, Sh::kBTile);
#pragma unroll
                for (int blk = 0; blk < RB; ++blk) tma_load_3d(b_s + sb * Sh::kBTile + blk * (kCols * 128), &map_b, b_full + sb, blk * 64, n0, list[q]);
            }
            __syncwarp();
            b_asked = u + 1;
            return true;
        };
        bool ok = steps == 0 || ask(0);
        for (int u = 0; u < steps && ok; ++u) {
            if (u + 1 < steps && !ask(u + 1)) break;
            const int q = u % count, sb = u % Sh::kB, ranks = list[kMost + q], end = (ranks + 15) / 16 * 16;
            ok = wait(b_full + sb, (u / Sh::kB) & 1, 10, u);
            if (!ok) break;
            if (ranks < a.R && ranks < end) {              // (columns behind R are zeros already)
                uint8_t* b = b_s + sb * Sh::kBTile + (ranks >> 6) * (kCols * 128);
                for (int f = lane; f < kCols; f += 32)
                    for (int j = ranks; j < end; ++j)
                        *reinterpret_cast<unsigned short*>(b + f * 128 + ((((j & 63) >> 3) ^ (f & 7)) << 4) + (j & 7) * 2) = 0;
                fence_async_smem();
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(b_clear + sb);
        }
        if (*failed) for (int u = max(0, b_asked - Sh::kB); u < b_asked; ++u) mbar_wait(b_full + u % Sh::kB, (u / Sh::kB) & 1);
    } else if (warp == 3) {
        // One store may still be reading its tile while the next one's sums are made; with two tiles in all it is waited for at once.
        constexpr int kBehind = Sh::kY > 2 ? 1 : 0;
        for (int i = 0; i < mine; ++i) {
            const int s = i % Sh::kY, n0 = (rank + i * ta.parts) * kCols;
            if (!wait(y_done + s, (i / Sh::kY) & 1, 13, i)) break;
            if (lane == 0) {                               // (the same thread every time: it waits for its own stores)
                if (n_fours == 0) {
                    tma_store_2d(&map_out, y_s + s * kYTile, n0, (int)t0);
                    if (n0 + 64 < a.N) tma_store_2d(&map_out, y_s + s * kYTile + kRows * 128, n0 + 64, (int)t0);
                }
                for (int f = 0; f < n_fours; ++f) {
                    const int4 rows = fours[f];
                    tma_scatter4(&map_out1, y_s + s * kYTile + f * 512, n0, rows);
                    if (n0 + 64 < a.N) tma_scatter4(&map_out1, y_s + s * kYTile + kRows * 128 + f * 512, n0 + 64, rows);
                }
                asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(kBehind) : "memory");
                if (i >= kBehind) mbar_arrive(y_empty + (i - kBehind) % Sh::kY);
            }
            __syncwarp();
        }
        if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    } else if (PLAIN && warp >= kFirstAdder) {
        float* turned = reinterpret_cast<float*>(y_s + kPlainY * kPlainTile) + (warp - kFirstAdder) * (32 * kTurned);      // of this warp: [32 rows][32 features]
        const long own_row = n_fours == 0 ? (t0 + r < a.T ? t0 + r : -1) : r < n_rows ? (long)reinterpret_cast<int*>(fours)[r] : -1;
        const unsigned named = __ballot_sync(0xffffffffu, place >= 0 && list[kMost + max(place, 0)] > 0);
        const int own_off = (int)((uintptr_t)((const bf16*)a.y + max(own_row, 0L) * a.ldy) & 15);        // (n0 is a multiple of 8)
        int off8[8];                                       // rows as they come: every eighth lies alike
#pragma unroll
        for (int k = 0; k < 8; ++k) off8[k] = __shfl_sync(0xffffffffu, own_off, k);
        const int first_there = (warp & 3) * 32, rows_there = (int)min(32L, a.T - t0 - first_there);
        // (shuffles and shared memory are what this loop is bound by)
        auto add = [&](auto straight, int col, const uint8_t* tile_s) {
            unsigned short* out = reinterpret_cast<unsigned short*>(a.out) + col + (straight.value ? (t0 + first_there) * a.ldo : 0L);
#pragma unroll 1
            for (int k0 = 0; k0 < 32; k0 += 16) {          // (all reads in front of the first store, which they may not pass)
                const uint8_t* from = tile_s + (first_there + k0) / 8 * kPlainPitch + 2 * (col & (kCols - 1));
                uint32_t w[16];
                float sum[16];
#pragma unroll
                for (int k = 0; k < 16; ++k) {
                    const int off = straight.value ? off8[k & 7] : __shfl_sync(0xffffffffu, own_off, k0 + k);
                    w[k] = *reinterpret_cast<const unsigned short*>(from + plain_slot(k) * kPlainPitch + off);
                    sum[k] = turned[(k0 + k) * kTurned + lane];
                }
#pragma unroll
                for (int k = 0; k < 16; ++k) {
                    const uint32_t added = __bfloat16_as_ushort(__float2bfloat16_rn(__uint_as_float(w[k] << 16) + sum[k]));
                    const long row = straight.value ? (k0 + k < rows_there ? k0 + k : -1) : (long)__shfl_sync(0xffffffffu, (int)own_row, k0 + k);
                    if (col < a.N && row >= 0) out[row * a.ldo] = (unsigned short)(named >> (k0 + k) & 1u ? added : w[k]);
                }
            }
        };
        bool ok = true;
        for (int i = group; i < mine && ok; i += 2) {
            const int n0 = (rank + i * ta.parts) * kCols, s = i % kPlainY;
            const int v = (i >> 1) * count, d = 2 * group + (v & 1);             // the first adapter's step and accumulator; a second one's: the other
            ok = wait(y_full + s, (i / kPlainY) & 1, 11, i) && (count == 0 || wait(d_full + d, (v >> 1) & 1, 12, i)) &&
                 (count <= 1 || wait(d_full + d + 1, (v >> 1) & 1, 12, i));
            if (!ok) break;
            fence_after_sync();
            const uint8_t* tile_s = y_s + s * kPlainTile;
#pragma unroll 1
            for (int piece = 0; piece < kCols / 32; ++piece) {
                if (named != 0) {
                    uint32_t acc[32];
                    tmem_ld32(lane_addr + d * kCols + piece * 32, acc);
                    if (count > 1) {
                        uint32_t other[32];
                        tmem_ld32(lane_addr + (d + 1) * kCols + piece * 32, other);
                        if (place == 1) {
#pragma unroll
                            for (int k = 0; k < 32; ++k) acc[k] = other[k];
                        }
                    }
#pragma unroll
                    for (int k = 0; k < 32; k += 4) *reinterpret_cast<uint4*>(turned + lane * kTurned + k) = make_uint4(acc[k], acc[k + 1], acc[k + 2], acc[k + 3]);
                    __syncwarp();
                }
                if (n_fours == 0) add(std::true_type(), n0 + piece * 32 + lane, tile_s);
                else add(std::false_type(), n0 + piece * 32 + lane, tile_s);
                __syncwarp();
            }
            if (count > 0) {
                fence_before_sync();
                mbar_arrive(d_empty + d);
                if (count > 1) mbar_arrive(d_empty + d + 1);
            }
            mbar_arrive(y_empty + s);
        }
    } else if (warp >= kFirstAdder) {
        bool ok = true;
        for (int i = group; i < mine && ok; i += 2) {
            const int s = i % Sh::kY;
            ok = wait(y_full + s, (i / Sh::kY) & 1, 11, i);
            if (!ok) break;
            uint8_t* row = y_s + s * kYTile + r * 128;
            for (int q = 0; q < count && ok; ++q) {
                const int v = (i >> 1) * count + q, d = 2 * group + (v & 1);
                ok = wait(d_full + d, (v >> 1) & 1, 12, i);
                if (!ok) break;
                fence_after_sync();
                const bool any = __any_sync(0xffffffffu, place == q) && list[kMost + q] > 0;
#pragma unroll
                for (int piece = 0; piece < kCols / 32; ++piece) {
                    if (!any) break;
                    uint32_t acc[32];
                    tmem_ld32(lane_addr + d * kCols + piece * 32, acc);
                    if (place == q) {
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            uint4* at = reinterpret_cast<uint4*>(row + (piece >> 1) * (kRows * 128) + ((((piece & 1) * 4 + c) ^ (r & 7)) << 4));
                            uint4 w = *at;
                            uint32_t* e = reinterpret_cast<uint32_t*>(&w);
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                const float lo = __uint_as_float(e[k] << 16) + __uint_as_float(acc[8 * c + 2 * k]);
                                const float hi = __uint_as_float(e[k] & 0xffff0000u) + __uint_as_float(acc[8 * c + 2 * k + 1]);
                                const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
                                e[k] = *reinterpret_cast<const uint32_t*>(&b);
                            }
                            *at = w;
                        }
                    }
                }
                fence_before_sync();
                mbar_arrive(d_empty + d);
            }
            fence_async_smem();
            if (ok) mbar_arrive(y_done + s);
        }
    }
    fence_before_sync();
    __syncthreads();
    if (warp == 1) tmem_free<512>(tmem);
}

// [layers][rows][width] bfloat16 with free strides (multiples of 8 elements, base on 16 bytes): boxes of 64 x box_rows x 1, 128-byte
// swizzle, zeros outside.
inline int make_tile_map_3d(CUtensorMap* map, const void* ptr, long layers, long rows, long width, long layer_stride, long row_stride, int box_rows) {
    thread_local KeyedCache<CUtensorMap, 7, 64, 8> kept;   // (weights come back step after step)
    const KeyedCache<CUtensorMap, 7, 64, 8>::Key key = {(int64_t)(uintptr_t)ptr, layers, rows, width, layer_stride, row_stride, box_rows};
    if (const CUtensorMap* known = kept.find(key)) {
        *map = *known;
        return 0;
    }
    EncodeTiled enc = tensor_map_encoder();
    if (enc == nullptr) return (int)cudaErrorNotSupported;
    const cuuint64_t dims[3] = {(cuuint64_t)width, (cuuint64_t)rows, (cuuint64_t)layers};
    const cuuint64_t strides[2] = {(cuuint64_t)row_stride * 2, (cuuint64_t)layer_stride * 2};
    const cuuint32_t box[3] = {64u, (cuuint32_t)box_rows, 1u};
    const cuuint32_t elem[3] = {1, 1, 1};
    const CUresult rc = enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(ptr), dims, strides, box, elem,
                            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (rc != CUDA_SUCCESS) return (int)cudaErrorInvalidValue;
    kept.put(key, *map);
    return 0;
}

// Rows of bfloat16 that lie alike within 16 bytes, from the boundary at or in front of the first one on: boxes of kCols + 8 columns x 16
// rows, as they lie.  (What comes with them from in front of a row is of the 16 bytes that hold its first column.)
inline int make_eighth(CUtensorMap* map, const void* ptr, long rows, long width, long row_stride) {
    EncodeTiled enc = tensor_map_encoder();
    if (enc == nullptr) return (int)cudaErrorNotSupported;
    const uintptr_t at = (uintptr_t)ptr, base = at & ~(uintptr_t)15;
    const cuuint64_t dims[2] = {(cuuint64_t)width + (at - base) / 2, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)row_stride * 2};
    const cuuint32_t box[2] = {(cuuint32_t)kCols + 8, 16u};
    const cuuint32_t elem[2] = {1, 1};
    const CUresult rc = enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, reinterpret_cast<void*>(base), dims, strides, box, elem,
                            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return rc == CUDA_SUCCESS ? 0 : (int)cudaErrorInvalidValue;
}

// What TMA can fetch and store as it lies.
struct Lying { bool x, A, B, y; };
inline Lying lying(const AdapterArgs& a) {
    auto lies = [](const void* p, long stride, long width) { return ((uintptr_t)p & 15) == 0 && stride % 8 == 0 && stride >= width; };
    auto layers = [&](long stride) { return a.adapters == 1 || (stride > 0 && stride % 8 == 0); };
    return {lies(a.x, a.ldx, a.K), lies(a.A, a.a_row, a.K) && layers(a.a_adapter), lies(a.B, a.b_row, a.R) && layers(a.b_adapter),
            lies(a.y, a.ldy, a.N) && lies(a.out, a.ldo, a.N)};
}
inline int pitch_of(int width) { return (width + 7) / 8 * 8; }
// Words of 4 bytes that the copies take.
inline long words_of_copies(const AdapterArgs& a, const Lying& l) {
    return ((l.x ? 0 : a.T * pitch_of(a.K)) + (l.A ? 0 : (long)a.adapters * a.R * pitch_of(a.K)) + (l.B ? 0 : (long)a.adapters * a.N * pitch_of(a.R))) / 2;
}
// Does the kernel take the call (apart from its number of rows)?  Adapters are not copied for a few rows each: the rows' kernel reads
// an adapter for every 8 rows of it, at about the same rate as a copy is read and written.
inline bool takes(const AdapterArgs& a) {
    if (!(a.R > 0 && a.R <= 128 && a.K > 0 && a.adapters > 0)) return false;
    const Lying l = lying(a);
    if (!l.y && !(a.R <= 64 && a.ldy >= a.N)) return false;                    // (PLAIN)
    const long most = 1L << 33;                            // (values of a copy: the copying kernel counts pieces of 16 bytes in 32 bits)
    return ((l.A && l.B) || a.T >= 16L * a.adapters) && a.T * pitch_of(a.K) < most && (long)a.adapters * a.R * pitch_of(a.K) < most &&
           (long)a.adapters * a.N * pitch_of(a.R) < most;
}

template <int RB, bool PLAIN>
inline int launch_as(const TileArgs& ta, long clusters, cudaStream_t stream) {
    const AdapterArgs& a = ta.a;
    CUtensorMap map_x, map_a, map_b, map_y, map_out, map_x1, map_y1, map_out1;
    int rc = make_tile_map(&map_x, a.x, a.T, a.K, a.ldx, kRows);
    if (rc == 0) rc = make_tile_map_3d(&map_a, a.A, a.adapters, a.R, a.K, a.adapters > 1 ? a.a_adapter : a.a_row * a.R, a.a_row, ta.padded);
    if (rc == 0) rc = make_tile_map_3d(&map_b, a.B, a.adapters, a.N, a.R, a.adapters > 1 ? a.b_adapter : a.b_row * a.N, a.b_row, kCols);
    if (rc == 0) rc = make_tile_map(&map_x1, a.x, a.T, a.K, a.ldx, 1);                     // (a row at a time, four by four)
    Eighths eighths{};
    if (PLAIN) {
        map_y = map_out = map_y1 = map_out1 = map_x;       // (not used)
        for (int e = 0; e < 8 && rc == 0; ++e) rc = make_eighth(&eighths.map[e], (const bf16*)a.y + e * a.ldy, (a.T - e + 7) / 8, a.N, 8 * a.ldy);
    } else {
        if (rc == 0) rc = make_tile_map(&map_y, a.y, a.T, a.N, a.ldy, kRows);
        if (rc == 0) rc = make_tile_map(&map_out, a.out, a.T, a.N, a.ldo, kRows);
        if (rc == 0) rc = make_tile_map(&map_y1, a.y, a.T, a.N, a.ldy, 1);
        if (rc == 0) rc = make_tile_map(&map_out1, a.out, a.T, a.N, a.ldo, 1);
    }
    static SharedLimits limits;
    if (rc == 0) rc = ensure_dynamic_smem(adapter_tiles_kernel<RB, PLAIN>, Shape<RB>::kSmem, limits);
    if (rc != 0) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(clusters * ta.parts)); cfg.blockDim = dim3(kThreads); cfg.dynamicSmemBytes = Shape<RB>::kSmem; cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)ta.parts; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr; cfg.numAttrs = 2;
    return launched(cudaLaunchKernelEx(&cfg, adapter_tiles_kernel<RB, PLAIN>, map_x, map_a, map_b, map_y, map_out, map_x1, map_y1, map_out1, eighths, ta));
}

// `copies`: scratch for what does not lie as TMA wants it; `plan` (null: there is one adapter): for the rows in order.
inline int launch(AdapterArgs a, bf16* copies, int* plan, int* error, cudaStream_t stream) {
    const long tiles = (a.T + kRows - 1) / kRows, most = plan != nullptr ? adapter_order::most_tiles(a.T, a.adapters, kRows) : 0;
    const int parts = tiles <= 18 ? 8 : tiles <= 37 ? 4 : tiles <= 74 ? 2 : 1, padded = (a.R + 15) / 16 * 16;
    const Lying l = lying(a);
    const int limit = !l.y ? 2 : 256 / padded < kMost ? 256 / padded : kMost;
    if ((tiles + most) * parts > 0x7fffffffL) return kTooLarge;
    int rc = 0;
    if (!l.x || !l.A || !l.B) {
        adapter_lay::Pieces pieces{};
        const int pk = pitch_of(a.K), pr = pitch_of(a.R);
        if (!l.x) {
            pieces.p[0] = {(const bf16*)a.x, copies, (unsigned)a.T, (unsigned)a.T, a.K, pk, 0, a.ldx};
            a.x = copies; a.ldx = pk;
            copies += a.T * pk;
        }
        if (!l.A) {
            pieces.p[1] = {(const bf16*)a.A, copies, (unsigned)a.R, (unsigned)a.R * a.adapters, a.K, pk, a.a_adapter, a.a_row};
            a.A = copies; a.a_row = pk; a.a_adapter = (long)a.R * pk;
            copies += (long)a.adapters * a.R * pk;
        }
        if (!l.B) {
            pieces.p[2] = {(const bf16*)a.B, copies, (unsigned)a.N, (unsigned)a.N * a.adapters, a.R, pr, a.b_adapter, a.b_row};
            a.B = copies; a.b_row = pr; a.b_adapter = (long)a.N * pr;
        }
        rc = adapter_lay::launch(pieces, stream);
    }
    if (rc == 0 && plan != nullptr) rc = adapter_order::launch(a, plan, kRows, limit, stream);
    if (rc != 0) return rc;
    const TileArgs ta{a, (int)tiles, parts, padded, limit, error};
    const long all = tiles + most;
    rc = !l.y ? launch_as<1, true>(ta, all, stream) : a.R <= 64 ? launch_as<1, false>(ta, all, stream) : launch_as<2, false>(ta, all, stream);
    return rc != 0 ? rc : launch_status();
}

}  // namespace adapter_tiles
}  // namespace lb200
