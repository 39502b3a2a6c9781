// The prefix's part of attention over a shared prefix on the 5th-generation tensor cores: bfloat16, heads of 64, 96 or 128, pages of a
// multiple of 16 keys.  The products, the softmax threads and the lazily followed maximum are those of the prompt kernel
// (attention_prefill_tc.cu); what differs is whose rows meet: the rows of a tile are (token, head) pairs of one group, gathered into
// shared memory by the threads (TMA has no box for them), and every row sees the same keys.
//
// 11 warps: one that asks TMA for tiles of 64 keys, K and V into rings of their own (K of a tile is done with as soon as its scores
// are there, V only behind the softmax), two that issue products (one per softmax group), two groups of 128 softmax threads, a
// thread per row.
//   TWO: a tile is 256 rows, 128 per softmax group, and both groups go through all keys: a K|V tile is fetched once for 256 rows.
//   else: a tile is 128 rows; group g takes the key tiles g, g + 2, ...
// The weights go into the product with the values as two bfloat16 numbers each (the prompt kernel's as one): rounded to one, they would
// leave an error as large as the output's own rounding, where `attention_decode` over the same keys leaves none.  It costs the products
// of PV once more and three instructions for two weights: 256 requests over 32,768 keys 117 us instead of 106, most calls 0 to 2 us.
// Ranges of keys that are the CTAs of one cluster join their results through distributed shared memory (each CTA adds up a part of
// the rows), so that few of them go through global memory: 16 ranges of 768 rows would be 6 MB written and read again.
//
// 120 registers a thread (three warps of this kernel and one of 152 registers have room on a quarter of an SM) and 177 KB of shared
// memory, so that a CTA of the own keys' kernel fits beside it: the
// tensor cores and the special-function units work here while that one waits for memory.
#pragma once
#include "lb200/attention_shared.h"
#include "lb200/common.cuh"
#include "lb200/tcgen05.cuh"

namespace lb200 {
namespace shared_tc {
using namespace tc;
typedef __nv_bfloat16 bf16;

constexpr int kQ = 128, kKV = 64;
constexpr int kFirstSoftmaxWarp = 3;
constexpr int kThreads = 32 * (kFirstSoftmaxWarp + 8);
constexpr float kTau = 8.f;                               // log2 of the growth of a row's maximum that O is rescaled for

constexpr int kMostRanks = 4;                             // CTAs of a cluster

template <int HD, bool TWO> struct Shape {
    static constexpr int kBlocks = (HD + 63) / 64;        // of 64 columns (heads of 96: the second one is half used)
    static constexpr int kPitch = HD == 64 ? 16 : 32;     // pieces of 16 bytes from row to row of a result
    // tiles of K and of V on their way or at work: a tile's copy takes about as long as the softmax of two
    static constexpr int kK = (TWO ? 3 : 4) * (HD == 64 ? 2 : 1), kV = kK + (HD == 64 ? 2 : 1);
    static constexpr int kRows = TWO ? 256 : 128;
    static constexpr uint32_t kQBlock = kQ * 128, kKVBlock = kKV * 128;
    static constexpr uint32_t kQBytes = kQBlock * kBlocks, kTileBytes = kKVBlock * kBlocks;
    static constexpr uint32_t kGroupCols = 128 + HD;      // per group: S (then the weights, in two parts) of even tiles, of odd tiles, O from 128
    static constexpr uint32_t kResult = 2 * kQ * kPitch * 16;   // both groups' O at the end, over Q and the rings
    static constexpr uint32_t kTiles = kQBytes * (TWO ? 2 : 1) + (kK + kV) * kTileBytes;
    // ... with their rows' (maximum, sum), and of this CTA's part of the rows the results' weights and where they go
    static constexpr int kSources = kMostRanks * (TWO ? 1 : 2);
    static constexpr uint32_t kEnd = kResult + 2 * kQ * 8 + kRows * (kSources * 4 + 8);
    static constexpr uint32_t kWork = kTiles > kEnd ? kTiles : kEnd;
    static constexpr uint32_t kSmem = kWork + 512;
    static_assert(2 * kGroupCols <= 512, "tensor memory");
};

__device__ __forceinline__ void report(int* error, int role, int tile) {
    atomicCAS(error, 0, (role << 24) | ((blockIdx.x & 0xFFF) << 12) | (tile & 0xFFF) | 0x40000000);
}

__device__ __forceinline__ uint32_t cluster_rank() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
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
__device__ __forceinline__ float2 remote2(uint32_t addr) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
    return v;
}

// grid: (tiles x kv heads) x ranges of keys; `ranks` ranges, which follow one another, are a cluster and one of a row's results
template <int HD, bool TWO>
__global__ void __maxnreg__(120)
shared_prefix_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, SharedArgs a, int ranks, int box) {
    pdl_wait();
    pdl_trigger();                                        // the own parts need nothing of this kernel's
    typedef Shape<HD, TWO> Sh;
    constexpr int kK = Sh::kK, kV = Sh::kV, kBlocks = Sh::kBlocks;
    constexpr uint32_t kTileBytes = Sh::kTileBytes, kGroupCols = Sh::kGroupCols;
    extern __shared__ __align__(1024) uint8_t base[];      // (the swizzle goes by the address)
    uint8_t* q_s = base;                                  // per group of rows: blocks of [128][128 B]
    uint8_t* k_s = q_s + Sh::kQBytes * (TWO ? 2 : 1);     // stages of K: blocks of [64][128 B]
    uint8_t* v_s = k_s + kK * kTileBytes;
    float2* ml_s = reinterpret_cast<float2*>(base + Sh::kResult);      // at the end: (maximum, sum) of both groups' rows
    constexpr int kMostSources = Sh::kSources;
    long* slots = reinterpret_cast<long*>(ml_s + 2 * kQ);
    float* weights = reinterpret_cast<float*>(slots + Sh::kRows);
    uint64_t* k_full = reinterpret_cast<uint64_t*>(base + Sh::kWork);
    uint64_t* k_empty = k_full + kK;
    uint64_t* v_full = k_empty + kK;
    uint64_t* v_empty = v_full + kV;
    uint64_t* s_ready = v_empty + kV;                     // per group and tile parity: S of the tile is in tensor memory
    uint64_t* p_ready = s_ready + 4;                      // ... P of the tile is in tensor memory (128 arrivals)
    uint64_t* o_ready = p_ready + 4;                      // ... PV of the tile is added to O
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(o_ready + 4);
    volatile int* failed = reinterpret_cast<volatile int*>(tmem_slot + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    const int ranges = a.prefix_splits * ranks;
    const int range = blockIdx.x % ranges, item = blockIdx.x / ranges, kvh = item % a.Hkv;
    const int G = a.Hq / a.Hkv;
    int first, n_tokens, longest;
    long row0;
    if (!find_tile(a, item / a.Hkv, G, Sh::kRows, &longest, &row0, &first, &n_tokens)) return;   // (the whole cluster)
    const int rows = (int)min((long)Sh::kRows, (long)n_tokens * G - row0);
    const int active = TWO ? (rows > kQ ? 2 : 1) : 2;     // softmax groups at work
    const int request = a.token_req[first];
    const bool known = request >= 0 && request < a.requests;
    const int prefix = known ? (int)min((long)longest, (long)a.bt_cols * a.page_size) : 0;
    const int all_kt = (prefix + kKV - 1) / kKV, per = (all_kt + ranges - 1) / ranges;
    const int kt_begin = min(range * per, all_kt), n_kt = min(per, all_kt - kt_begin);
    const int* bt = a.block_table + (long)(known ? request : 0) * a.bt_stride;

    if (warp == 1) tmem_alloc<512>(tmem_slot);
    bool bad = false;                                     // one of the range's pages is not there
    if (warp == 0) {
        if (lane == 0) {
            for (int s = 0; s < kK; ++s) { mbar_init(k_full + s, 1); mbar_init(k_empty + s, TWO ? active : 1); }
            for (int s = 0; s < kV; ++s) { mbar_init(v_full + s, 1); mbar_init(v_empty + s, TWO ? active : 1); }
            for (int i = 0; i < 4; ++i) { mbar_init(s_ready + i, 1); mbar_init(o_ready + i, 1); mbar_init(p_ready + i, 128); }
            *failed = 0;
            mbar_fence_init();
        }
    } else if (n_kt > 0) {
        for (int p = kt_begin * kKV / a.page_size + threadIdx.x - 32; p <= ((kt_begin + n_kt) * kKV - 1) / a.page_size && p < a.bt_cols; p += kThreads - 32)
            bad = bad || bt[p] < 0 || bt[p] >= a.pages;
        // the queries: rows of 64 dims are 128 bytes; piece c of row r lies at c ^ (r & 7)
        constexpr int kPieces = HD / 8, kOwn = (Sh::kRows * kPieces + kThreads - 33) / (kThreads - 32);
        const bf16* q = (const bf16*)a.q;
        uint4 v[kOwn];
#pragma unroll
        for (int n = 0; n < kOwn; ++n) {
            const int i = (int)threadIdx.x - 32 + n * (kThreads - 32), r = i / kPieces, c = i % kPieces;
            v[n] = make_uint4(0u, 0u, 0u, 0u);
            if (r < rows) {
                const int at = (int)row0 + r, token = at / G;
                v[n] = *reinterpret_cast<const uint4*>(q + (long)(first + token) * a.q_stride + (kvh * G + at - token * G) * HD + c * 8);
            }
        }
#pragma unroll
        for (int n = 0; n < kOwn; ++n) {
            const int i = (int)threadIdx.x - 32 + n * (kThreads - 32), r = i / kPieces, c = i % kPieces, grp = r >> 7, rr = r & 127;
            if (r < Sh::kRows)
                *reinterpret_cast<uint4*>(q_s + grp * Sh::kQBytes + (c >> 3) * Sh::kQBlock + rr * 128 + (((c & 7) ^ (rr & 7)) << 4)) = v[n];
        }
    }
    int k_issued = 0, v_issued = 0;
    // Where the keys of a tile lie, kept by the lanes: lane n has the row of its keys n * box .. (a box of keys lies within a page).  A
    // page that is not there: rows behind the pool, which read as zeros (its scores are left out below).  (Whole warps: see elect_one.)
    const int boxes = kKV / box;
    auto row_of = [&](int i) -> int {
        const int j = (kt_begin + i) * kKV + min(lane, boxes - 1) * box, page = j / a.page_size;
        const int id = page < a.bt_cols ? bt[page] : -1;
        return (int)((id >= 0 && id < a.pages ? (long)id : a.pages) * a.page_size + (j - page * a.page_size));
    };
    auto load = [&](int i, int row, int stages, uint8_t* ring, const CUtensorMap* map, uint64_t* full, uint64_t* empty, int role) -> bool {
        const int s = i % stages;
        if (i >= stages && !__all_sync(0xffffffffu, mbar_wait(empty + s, ((i / stages) - 1) & 1))) {
            if (lane == 0) report(a.error, role, i);
            *failed = 1;
            return false;
        }
        if (elect_one()) mbar_expect_tx(full + s, kTileBytes);
        __syncwarp();
        for (int n = 0; n < boxes; ++n) {
            const int y = __shfl_sync(0xffffffffu, row, n);
            if (elect_one()) {
#pragma unroll
                for (int blk = 0; blk < kBlocks; ++blk)
                    tma_load_2d(ring + s * kTileBytes + blk * Sh::kKVBlock + n * box * 128, map, full + s, kvh * HD + blk * 64, y);
            }
            __syncwarp();
        }
        return true;
    };
    int first_row = 0;
    if (warp == 0) {
        __syncwarp();
        if (n_kt > 0) {                                    // the first tile is on its way while the queries are gathered
            first_row = row_of(0);
            load(0, first_row, kK, k_s, &map_k, k_full, k_empty, 1);
            load(0, first_row, kV, v_s, &map_v, v_full, v_empty, 4);
            k_issued = v_issued = 1;
        }
    }
    fence_async_smem();
    fence_before_sync();
    const bool any_bad = __syncthreads_or(bad);
    fence_after_sync();
    const uint32_t tmem = *tmem_slot;

    if (warp == 0) {
        if (n_kt > 0) {
            // K runs a tile ahead of V: its stage is free as soon as the scores are there
            int row = first_row, k_row = n_kt > 1 ? row_of(1) : 0;
            bool ok = n_kt <= 1 || load(1, k_row, kK, k_s, &map_k, k_full, k_empty, 1);
            if (n_kt > 1 && ok) k_issued = 2;
            for (int i = 1; i < n_kt && ok && !*failed; ++i) {
                row = k_row;
                if (i + 1 < n_kt) {
                    k_row = row_of(i + 1);
                    if (!(ok = load(i + 1, k_row, kK, k_s, &map_k, k_full, k_empty, 1))) break;
                    k_issued = i + 2;
                }
                if (!(ok = load(i, row, kV, v_s, &map_v, v_full, v_empty, 4))) break;
                v_issued = i + 1;
            }
            if (*failed) {                                // let the copies already under way land before the CTA leaves
                for (int i = max(0, k_issued - kK); i < k_issued; ++i) mbar_wait(k_full + i % kK, (i / kK) & 1);
                for (int i = max(0, v_issued - kV); i < v_issued; ++i) mbar_wait(v_full + i % kV, (i / kV) & 1);
            }
        }
    } else if (warp < kFirstSoftmaxWarp) {
        const int g = warp - 1, step = TWO ? 1 : 2, from = TWO ? 0 : g;
        if (g < active) {                                  // (whole warps: see elect_one)
            constexpr uint32_t idesc_s = umma_idesc(kQ, kKV), idesc_o = umma_idesc(kQ, HD) | kBMnMajor;
            const uint64_t qdesc = umma_desc(q_s + (TWO ? g * Sh::kQBytes : 0)), kdesc0 = umma_desc(k_s), vdesc0 = umma_desc_mn(v_s, Sh::kKVBlock);
            const uint32_t cols = tmem + g * kGroupCols;
            bool ok = true;
            auto loaded = [&](uint64_t* full, int stages, int i) { return mbar_spin(full + i % stages, (i / stages) & 1); };
            auto issue_s = [&](int i, int t) {             // S of tile i, the group's tile number t, into its S buffer t & 1
                const uint64_t kdesc = kdesc0 + (uint64_t)((i % kK) * (kTileBytes >> 4));
                const uint32_t d = cols + (t & 1) * 64;
#pragma unroll
                for (int blk = 0; blk < kBlocks; ++blk)
#pragma unroll
                    for (int k = 0; k < (HD - 64 * blk >= 64 ? 4 : (HD - 64 * blk) / 16); ++k)
                        umma_bf16(d, qdesc + blk * (Sh::kQBlock >> 4) + 2 * k, kdesc + blk * (Sh::kKVBlock >> 4) + 2 * k, idesc_s, (blk | k) != 0);
                umma_commit(s_ready + 2 * g + (t & 1));
                umma_commit(k_empty + i % kK);
            };
            for (int t = 0; t < 2 && ok; ++t) {
                const int i = from + t * step;
                if (i >= n_kt) break;
                ok = __all_sync(0xffffffffu, loaded(k_full, kK, i));
                if (!ok) { if (lane == 0) report(a.error, 2, i); *failed = 1; break; }
                fence_after_sync();
                if (elect_one()) issue_s(i, t);
                __syncwarp();
            }
            for (int i = from, t = 0; i < n_kt && ok && !*failed; i += step, ++t) {
                // V of the tile is there, K of the tile after the next, and P, which is waited for last: then all of it goes out at once
                const int later = i + 2 * step;
                const bool fine = loaded(v_full, kV, i) && (later >= n_kt || loaded(k_full, kK, later)) && mbar_spin(p_ready + 2 * g + (t & 1), (t >> 1) & 1);
                if (!__all_sync(0xffffffffu, fine)) { if (lane == 0) report(a.error, 3, i); *failed = 1; break; }
                fence_after_sync();
                if (elect_one()) {
                    const uint64_t vdesc = vdesc0 + (uint64_t)((i % kV) * (kTileBytes >> 4));
                    const uint32_t p = cols + (t & 1) * 64;
#pragma unroll
                    for (int k = 0; k < 2 * kKV / 16; ++k) // all dims in one product: one of 64 columns takes as long as one of 128
                        umma_bf16_tmem_a(cols + 128, p + 8 * k, vdesc + (uint64_t)(2048 >> 4) * (k % (kKV / 16)), idesc_o, (t > 0 || k != 0) ? 1u : 0u);
                    umma_commit(o_ready + 2 * g + (t & 1));
                    umma_commit(v_empty + i % kV);
                    if (later < n_kt) issue_s(later, t + 2);
                }
                __syncwarp();
            }
        }
    } else {
        const int grp = (warp - kFirstSoftmaxWarp) / 4;
        const int lr = (warp & 3) * 32 + lane;             // this thread's lane of tensor memory
        const int r = (TWO ? grp * kQ : 0) + lr;           // and row of the tile
        const uint32_t lane_addr = tmem + ((uint32_t)((warp & 3) * 32) << 16) + grp * kGroupCols;
        // the keys that the row sees: those in front of the prefix's end, and of its own position's
        const int limit = r < rows ? min(prefix, keys_of(a, first + (int)((row0 + r) / G))) : prefix;
        const int step = TWO ? 1 : 2, from = TWO ? 0 : grp;
        float m_used = -INFINITY, l = 0.f;
        uint64_t* o_bar = o_ready + 2 * grp;
        bool ok = true;
        int done = 0;
        auto wait_pv = [&](int t_of, int code, int at) -> bool {
            bool good = mbar_test(o_bar + (t_of & 1), (t_of >> 1) & 1) || mbar_wait(o_bar + (t_of & 1), (t_of >> 1) & 1);
            if (!good && lane == 0) { report(a.error, code, at); *failed = 1; }
            return __all_sync(0xffffffffu, good && !*failed);
        };
        for (int i = from, t = 0; i < n_kt && grp < active; i += step, ++t) {
            const int j0 = (kt_begin + i) * kKV;
            ok = mbar_test(s_ready + 2 * grp + (t & 1), (t >> 1) & 1) || mbar_wait(s_ready + 2 * grp + (t & 1), (t >> 1) & 1);
            // keys of the last tile behind the prefix (another request's, or nobody's): their V rows become zeros, which either group
            // may do any number of times
            const bool mends = j0 + kKV > prefix;
            if (mends) ok = mbar_wait(v_full + i % kV, (i / kV) & 1) && ok;
            if (!ok && lane == 0) { report(a.error, 5, i); *failed = 1; }
            if (!__all_sync(0xffffffffu, ok && !*failed)) { ok = false; break; }
            fence_after_sync();
            if (mends) {
                uint8_t* v_tile = v_s + (i % kV) * kTileBytes;
                const int first_bad = prefix - j0;
                for (int x = lr; x < (kKV - first_bad) * 8 * kBlocks; x += 128) {
                    const int blk = x / ((kKV - first_bad) * 8), y = x - blk * (kKV - first_bad) * 8;
                    *reinterpret_cast<uint4*>(v_tile + blk * Sh::kKVBlock + (first_bad + y / 8) * 128 + (y % 8) * 16) = make_uint4(0u, 0u, 0u, 0u);
                }
            }
            const int seen = limit;                        // keys of the tile that the row sees: those in front of `seen` ...
            uint64_t lost = 0;                             // ... that are not on a page that is not there
            if (any_bad)
                for (int c = 0; c < kKV; c += 16) {
                    const int page = (j0 + c) / a.page_size, id = page < a.bt_cols ? bt[page] : -1;
                    if (id < 0 || id >= a.pages) lost |= (uint64_t)0xffff << c;
                }
            const bool whole = __all_sync(0xffffffffu, j0 + kKV <= seen && lost == 0);
            uint32_t sc[64], pk[32], rest[32];             // the row's scores, its weights and what is cut off them
            float mx4[4], sum[4];                          // (four chains each: two warps a scheduler hide no latency)
            // the weights relative to `ref`, and the scores' maximum on the way
            auto weigh = [&](float ref) {
#pragma unroll
                for (int e = 0; e < 4; ++e) { mx4[e] = -INFINITY; sum[e] = 0.f; }
#pragma unroll
                for (int c = 0; c < 64; c += 2) {
                    const float x0 = __uint_as_float(sc[c]), x1 = __uint_as_float(sc[c + 1]);
                    const float e0 = ex2_approx(fmaf(x0, a.scale_log2, -ref)), e1 = ex2_approx(fmaf(x1, a.scale_log2, -ref));
                    mx4[(c >> 1) & 3] = fmaxf(mx4[(c >> 1) & 3], fmaxf(x0, x1));
                    split_weights(e0, e1, pk[c >> 1], rest[c >> 1]);
                    sum[(c >> 1) & 1] += e0;
                    sum[2 + ((c >> 1) & 1)] += e1;
                }
            };
            auto top = [&] { return fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * a.scale_log2; };
            tmem_get64(lane_addr + (t & 1) * 64, sc);
            // Mostly no row's maximum grows by more than 2^kTau: the weights are made without waiting for it, and again where it does.
            bool again = !whole || __any_sync(0xffffffffu, m_used == -INFINITY);
            if (!again) {
                weigh(m_used);
                again = __any_sync(0xffffffffu, top() > m_used + kTau);
                if (again) tmem_get64(lane_addr + (t & 1) * 64, sc);
            }
            if (again) {
                if (!whole) {
#pragma unroll
                    for (int c = 0; c < 64; ++c) if (j0 + c >= seen || (lost >> c & 1u)) sc[c] = 0xff800000u;
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) mx4[e] = -INFINITY;
#pragma unroll
                for (int c = 0; c < 64; c += 8)
#pragma unroll
                    for (int e = 0; e < 4; ++e) mx4[e] = fmaxf(mx4[e], fmaxf(__uint_as_float(sc[c + e]), __uint_as_float(sc[c + 4 + e])));
                const float mx = top();
                const bool grow = mx > m_used + kTau;
                if (__any_sync(0xffffffffu, grow)) {
                    float factor = 1.f;
                    if (grow) { factor = exp2f(m_used - mx); m_used = mx; l *= factor; }
                    if (t > 0) {
                        if (!wait_pv(t - 1, 6, i)) { ok = false; break; }
                        fence_after_sync();
#pragma unroll 1
                        for (int piece = 0; piece < HD / 8; ++piece) {
                            uint32_t ov[8];
                            tmem_get8(lane_addr + 128 + piece * 8, ov);
#pragma unroll
                            for (int c = 0; c < 8; ++c) ov[c] = __float_as_uint(__uint_as_float(ov[c]) * factor);
                            tmem_st8(lane_addr + 128 + piece * 8, ov);
                        }
                        tmem_st_wait();
                    }
                }
                weigh(m_used == -INFINITY ? 0.f : m_used);
            }
            l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
            tmem_st32(lane_addr + (t & 1) * 64, pk);
            tmem_st32(lane_addr + (t & 1) * 64 + 32, rest);
            tmem_st_wait();
            if (mends) fence_async_smem();
            fence_before_sync();
            mbar_arrive(p_ready + 2 * grp + (t & 1));
            done = t + 1;
        }
        if (ok && done > 0) ok = wait_pv(done - 1, 8, from + (done - 1) * step);
        if (ok && done > 0) fence_after_sync();
        const bool have = ok && done > 0;
        if (l != l) m_used = 0.f;                          // (a NaN among the scores: the range counts, and makes the row NaN)
        asm volatile("bar.sync 1, 256;" ::: "memory");     // every product has read Q and the rings: the results lie over them
        // a row of O: pieces of 16 bytes, piece c at c ^ (row % kPitch)
        constexpr int kPitch = Sh::kPitch;
        float4* mine = reinterpret_cast<float4*>(base) + (size_t)(grp * kQ + lr) * kPitch;
        ml_s[grp * kQ + lr] = have ? make_float2(m_used, l) : make_float2(-INFINITY, 0.f);
        if (have) {
#pragma unroll 1
            for (int piece = 0; piece < HD / 32; ++piece) {
                uint32_t ov[32];
                tmem_ld32(lane_addr + 128 + piece * 32, ov);
#pragma unroll
                for (int c = 0; c < 8; ++c)
                    mine[(piece * 8 + c) ^ (lr & (kPitch - 1))] =
                        make_float4(__uint_as_float(ov[4 * c]), __uint_as_float(ov[4 * c + 1]), __uint_as_float(ov[4 * c + 2]), __uint_as_float(ov[4 * c + 3]));
            }
        }
    }
    fence_before_sync();
    __syncthreads();
    if (warp == 1) tmem_free<512>(tmem);
    if (ranks > 1) cluster_meet();
    // This CTA's part of the rows, rank, rank + ranks, ...: a thread per row puts together the results' weights, then a warp takes a row
    // at a time, 16 bytes a lane, with all results of two rows on their way.
    {
        constexpr int kPieces = HD / 4, kPitch = Sh::kPitch, kSources = TWO ? 1 : 2;
        const uint32_t here = smem_u32(base), ml_here = smem_u32(ml_s), rank = ranks > 1 ? cluster_rank() : 0u;
        const int splits = a.prefix_splits + a.own_splits, sources = ranks * kSources, ours = (rows - (int)rank + ranks - 1) / ranks;
        if ((int)threadIdx.x < ours) {
            const int r = (int)rank + ranks * (int)threadIdx.x, at = (int)row0 + r, token = at / G;
            float2 ml[kMostSources];
#pragma unroll
            for (int s = 0; s < kMostSources; ++s)
                if (s < sources) ml[s] = remote2(ranks > 1 ? at_rank(ml_here + 8 * (r + (s % kSources) * kQ), s / kSources) : ml_here + 8 * (r + (s % kSources) * kQ));
            float m = -INFINITY, l = 0.f;
#pragma unroll
            for (int s = 0; s < kMostSources; ++s) if (s < sources) m = fmaxf(m, ml[s].x);
            const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
            for (int s = 0; s < kMostSources; ++s)
                if (s < sources) {
                    const float f = exp2f(ml[s].x - ref);
                    l += ml[s].y * f;
                    weights[threadIdx.x * kMostSources + s] = f;
                }
            const long slot = ((long)(first + token) * a.Hq + kvh * G + at - token * G) * splits + range / ranks;
            slots[threadIdx.x] = slot;
            *reinterpret_cast<float2*>(a.part_ml + 2 * slot) = make_float2(m, l);
        }
        __syncthreads();
        for (int n0 = warp; n0 < ours; n0 += 2 * (kThreads / 32)) {
            float4 v[2][kMostSources];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int n = n0 + h * (kThreads / 32), r = (int)rank + ranks * n;
                const uint32_t piece = here + 16 * (uint32_t)(r * kPitch + (lane ^ (r & (kPitch - 1))));      // (128 rows on: the same place)
#pragma unroll
                for (int s = 0; s < kMostSources; ++s) {
                    v[h][s] = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (n < ours && s < sources && lane < kPieces && weights[n * kMostSources + s] != 0.f) {         // (a range without keys left nothing)
                        const uint32_t at = piece + (s % kSources) * (kQ * kPitch * 16);
                        v[h][s] = remote4(ranks > 1 ? at_rank(at, s / kSources) : at);
                    }
                }
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int n = n0 + h * (kThreads / 32);
                if (n >= ours || lane >= kPieces) continue;
                float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int s = 0; s < kMostSources; ++s)
                    if (s < sources) {
                        const float w = weights[n * kMostSources + s];
                        o.x = fmaf(v[h][s].x, w, o.x); o.y = fmaf(v[h][s].y, w, o.y); o.z = fmaf(v[h][s].z, w, o.z); o.w = fmaf(v[h][s].w, w, o.w);
                    }
                *reinterpret_cast<float4*>(a.part_o + slots[n] * HD + 4 * lane) = o;
            }
        }
    }
    if (ranks > 1) cluster_meet();                         // nobody leaves while another CTA reads its results
}

template <int HD, bool TWO>
inline int launch_prefix(const SharedArgs& a, int ranks, cudaStream_t stream) {
    typedef Shape<HD, TWO> Sh;
    const long rows = (long)a.tokens * (a.Hq / a.Hkv);
    const long tiles = most_tiles(rows, a.groups < a.tokens ? a.groups : a.tokens, Sh::kRows);
    const long grid = tiles * a.Hkv * a.prefix_splits * ranks;
    if (grid > 0x7fffffffL) return kTooLarge;
    CUtensorMap map_k, map_v;
    const int box = a.page_size % 64 == 0 ? 64 : a.page_size % 32 == 0 ? 32 : 16;          // keys that one copy brings
    int rc = make_tile_map(&map_k, a.k_cache, a.pages * a.page_size, (long)a.Hkv * HD, (long)a.Hkv * HD, box);
    if (rc == 0) rc = make_tile_map(&map_v, a.v_cache, a.pages * a.page_size, (long)a.Hkv * HD, (long)a.Hkv * HD, box);
    static SharedLimits limits;
    static DoneOnce carveout;
    if (rc == 0) rc = ensure_dynamic_smem(shared_prefix_kernel<HD, TWO>, Sh::kSmem, limits);
    if (rc == 0) rc = whole_carveout(shared_prefix_kernel<HD, TWO>, carveout);
    if (rc != 0) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid); cfg.blockDim = dim3(kThreads); cfg.dynamicSmemBytes = Sh::kSmem; cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)ranks; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr; cfg.numAttrs = 2;
    return launched(cudaLaunchKernelEx(&cfg, shared_prefix_kernel<HD, TWO>, map_k, map_v, a, ranks, box));
}

}  // namespace shared_tc
}  // namespace lb200
