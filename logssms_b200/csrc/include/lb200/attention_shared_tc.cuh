// The prefix's part of attention over a shared prefix on the 5th-generation tensor cores: bfloat16, heads of 64 or 128, pages of a
// multiple of 64 keys.  The products, the softmax threads and the lazily followed maximum are those of the prompt kernel
// (attention_prefill_tc.cu); what differs is whose rows meet: the rows of a tile are (token, head) pairs of one group, gathered into
// shared memory by the threads (TMA has no box for them), and every row sees the same keys.
//
// 11 warps: one that asks TMA for K|V tiles of 64 keys, two that issue products (one per softmax group), two groups of 128 softmax
// threads, a thread per row.
//   TWO: a tile is 256 rows, 128 per softmax group, and both groups go through all keys: a K|V tile is fetched once for 256 rows.
//   else: a tile is 128 rows; group g takes the key tiles g, g + 2, ..., and the groups' results meet in shared memory.
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

template <int HD, bool TWO> struct Shape {
    static constexpr int kBlocks = HD / 64;
    static constexpr int kStages = HD == 64 ? 6 : 4;
    static constexpr int kRows = TWO ? 256 : 128;
    static constexpr uint32_t kQBlock = kQ * 128, kKVBlock = kKV * 128;
    static constexpr uint32_t kQBytes = kQBlock * kBlocks, kTileBytes = kKVBlock * kBlocks;
    static constexpr uint32_t kGroupCols = 128 + HD;      // per group: S (then P) of even tiles, of odd tiles, O from 128
    static constexpr uint32_t kMergeBytes = (64 + 2) * kQ * 4;
    static constexpr uint32_t kSmem = kQBytes * (TWO ? 2 : 1) + kStages * 2 * kTileBytes + 256 + 1024;
    static_assert(2 * kGroupCols <= 512 && kMergeBytes <= kStages * 2 * kTileBytes, "tensor memory; the partial result lies over the ring");
};

__device__ __forceinline__ void report(int* error, int role, int tile) {
    atomicCAS(error, 0, (role << 24) | ((blockIdx.x & 0xFFF) << 12) | (tile & 0xFFF) | 0x40000000);
}

// grid: tiles x kv heads x ranges of keys
template <int HD, bool TWO>
__global__ void __launch_bounds__(kThreads)
shared_prefix_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, SharedArgs a, int tiles) {
    pdl_wait();
    pdl_trigger();                                        // the own parts need nothing of this kernel's
    typedef Shape<HD, TWO> Sh;
    constexpr int kStages = Sh::kStages, kBlocks = Sh::kBlocks;
    constexpr uint32_t kTileBytes = Sh::kTileBytes, kGroupCols = Sh::kGroupCols;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* base = reinterpret_cast<uint8_t*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint8_t* q_s = base;                                  // per group of rows: blocks of [128][128 B]
    uint8_t* kv_s = q_s + Sh::kQBytes * (TWO ? 2 : 1);    // stages of K (blocks of [64][128 B]) | V (the same)
    float* merge = reinterpret_cast<float*>(kv_s);
    uint64_t* kv_full = reinterpret_cast<uint64_t*>(kv_s + kStages * 2 * kTileBytes);
    uint64_t* kv_empty = kv_full + kStages;
    uint64_t* s_ready = kv_empty + kStages;               // per group and tile parity: S of the tile is in tensor memory
    uint64_t* p_ready = s_ready + 4;                      // ... P of the tile is in tensor memory (128 arrivals)
    uint64_t* o_ready = p_ready + 4;                      // ... PV of the tile is added to O
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(o_ready + 4);
    volatile int* failed = reinterpret_cast<volatile int*>(tmem_slot + 1);
    int* bad_pages = reinterpret_cast<int*>(tmem_slot + 2);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    const int tile = blockIdx.x % tiles, kvh = (blockIdx.x / tiles) % a.Hkv, split = blockIdx.x / (tiles * a.Hkv);
    const int G = a.Hq / a.Hkv;
    int g_no, first, n_tokens;
    long row0;
    if (!find_tile(a, tile, G, Sh::kRows, &g_no, &row0, &first, &n_tokens)) return;
    const int rows = (int)min((long)Sh::kRows, (long)n_tokens * G - row0);
    const int active = TWO ? (rows > kQ ? 2 : 1) : 2;     // softmax groups at work
    const int request = a.token_req[first];
    const bool known = request >= 0 && request < a.requests;
    const int prefix = known ? (int)min((long)a.prefix_lens[g_no], (long)a.bt_cols * a.page_size) : 0;
    const int all_kt = (prefix + kKV - 1) / kKV, per = (all_kt + a.prefix_splits - 1) / a.prefix_splits;
    const int kt_begin = min(split * per, all_kt), n_kt = min(per, all_kt - kt_begin);
    const int* bt = a.block_table + (long)(known ? request : 0) * a.bt_stride;
    const int splits = a.prefix_splits + a.own_splits;
    auto slot_of = [&](int r) -> size_t {                 // of row r of the tile
        const long at = row0 + r;
        return ((size_t)(first + at / G) * a.Hq + kvh * G + at % G) * splits + split;
    };
    if (n_kt <= 0) {                                      // a range without keys
        for (int r = threadIdx.x; r < rows; r += kThreads) {
            float* ml = a.part_ml + 2 * slot_of(r);
            ml[0] = -INFINITY; ml[1] = 0.f;
        }
        return;
    }

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) { mbar_init(kv_full + s, 1); mbar_init(kv_empty + s, TWO ? active : 1); }
        for (int i = 0; i < 4; ++i) { mbar_init(s_ready + i, 1); mbar_init(o_ready + i, 1); mbar_init(p_ready + i, 128); }
        *failed = 0;
        *bad_pages = 0;
        mbar_fence_init();
    }
    if (warp == 1) tmem_alloc<512>(tmem_slot);
    {
        // rows of 64 dims are 128 bytes; piece c of row r lies at c ^ (r & 7)
        constexpr int kPieces = HD / 8;
        const bf16* q = (const bf16*)a.q;
        for (int i = threadIdx.x; i < Sh::kRows * kPieces; i += kThreads) {
            const int r = i / kPieces, c = i % kPieces, grp = r >> 7, rr = r & 127;
            uint4 v = make_uint4(0u, 0u, 0u, 0u);
            if (r < rows) {
                const long at = row0 + r;
                v = *reinterpret_cast<const uint4*>(q + (first + at / G) * a.q_stride + (kvh * G + at % G) * HD + c * 8);
            }
            *reinterpret_cast<uint4*>(q_s + grp * Sh::kQBytes + (c >> 3) * Sh::kQBlock + rr * 128 + (((c & 7) ^ (rr & 7)) << 4)) = v;
        }
    }
    fence_async_smem();
    fence_before_sync();
    __syncthreads();
    fence_after_sync();
    for (int p = kt_begin * kKV / a.page_size + threadIdx.x; p <= ((kt_begin + n_kt) * kKV - 1) / a.page_size && p < a.bt_cols; p += kThreads)
        if (bt[p] < 0 || bt[p] >= a.pages) *bad_pages = 1;
    __syncthreads();
    const uint32_t tmem = *tmem_slot;
    const bool any_bad = *bad_pages != 0;

    if (warp == 0) {
        if (lane == 0) {
            int issued = 0;
            for (int i = 0; i < n_kt && !*failed; ++i, ++issued) {
                const int s = i % kStages;
                if (i >= kStages && !mbar_wait(kv_empty + s, ((i / kStages) - 1) & 1)) { report(a.error, 1, i); *failed = 1; break; }
                const int j0 = (kt_begin + i) * kKV, page = j0 / a.page_size, id = bt[page];
                // a page that is not there: rows behind the pool, which read as zeros (its scores are left out below)
                const int row = (int)((id >= 0 && id < a.pages ? (long)id : a.pages) * a.page_size + (j0 - page * a.page_size));
                uint8_t* k_tile = kv_s + (size_t)s * 2 * kTileBytes;
                mbar_expect_tx(kv_full + s, 2 * kTileBytes);
#pragma unroll
                for (int blk = 0; blk < kBlocks; ++blk) {
                    tma_load_2d(k_tile + blk * Sh::kKVBlock, &map_k, kv_full + s, kvh * HD + blk * 64, row);
                    tma_load_2d(k_tile + kTileBytes + blk * Sh::kKVBlock, &map_v, kv_full + s, kvh * HD + blk * 64, row);
                }
            }
            if (*failed)                                  // let the copies already under way land before the CTA leaves
                for (int i = max(0, issued - kStages); i < issued; ++i) mbar_wait(kv_full + i % kStages, (i / kStages) & 1);
        }
    } else if (warp < kFirstSoftmaxWarp) {
        const int g = warp - 1, step = TWO ? 1 : 2, from = TWO ? 0 : g;
        if (lane == 0 && g < active) {
            const uint32_t idesc_s = umma_idesc(kQ, kKV), idesc_o = idesc_s | kBMnMajor;
            uint64_t qdesc[kBlocks];
#pragma unroll
            for (int blk = 0; blk < kBlocks; ++blk) qdesc[blk] = umma_desc(q_s + (TWO ? g * Sh::kQBytes : 0) + blk * Sh::kQBlock);
            bool ok = true;
            auto issue_s = [&](int i, int t) -> bool {     // S of tile i, the group's tile number t, into its S buffer t & 1
                const int s = i % kStages;
                if (!mbar_wait(kv_full + s, (i / kStages) & 1)) { report(a.error, 2, i); *failed = 1; return false; }
                fence_after_sync();
#pragma unroll
                for (int blk = 0; blk < kBlocks; ++blk) {
                    const uint64_t kdesc = umma_desc(kv_s + (size_t)s * 2 * kTileBytes + blk * Sh::kKVBlock);
#pragma unroll
                    for (int k = 0; k < 4; ++k) umma_bf16(tmem + g * kGroupCols + (t & 1) * 64, qdesc[blk] + 2 * k, kdesc + 2 * k, idesc_s, (blk | k) != 0);
                }
                umma_commit(s_ready + 2 * g + (t & 1));
                return true;
            };
            if (from < n_kt) ok = issue_s(from, 0);
            if (ok && from + step < n_kt) ok = issue_s(from + step, 1);
            for (int i = from, t = 0; i < n_kt && ok && !*failed; i += step, ++t) {
                const int s = i % kStages;
                if (!mbar_wait(p_ready + 2 * g + (t & 1), (t >> 1) & 1)) { report(a.error, 3, i); *failed = 1; break; }
                fence_after_sync();
                const uint32_t p_tmem = tmem + g * kGroupCols + (t & 1) * 64;
#pragma unroll
                for (int blk = 0; blk < kBlocks; ++blk) {
                    const uint64_t vdesc = umma_desc(kv_s + (size_t)s * 2 * kTileBytes + kTileBytes + blk * Sh::kKVBlock);
#pragma unroll
                    for (int k = 0; k < kKV / 16; ++k)
                        umma_bf16_tmem_a(tmem + g * kGroupCols + 128 + blk * 64, p_tmem + 8 * k, vdesc + (uint64_t)(2048 >> 4) * k, idesc_o,
                                         (t > 0 || k != 0) ? 1u : 0u);
                }
                umma_commit(o_ready + 2 * g + (t & 1));
                umma_commit(kv_empty + s);
                if (i + 2 * step < n_kt) ok = issue_s(i + 2 * step, t + 2);
            }
        }
    } else {
        const int grp = (warp - kFirstSoftmaxWarp) / 4;
        const int lr = (warp & 3) * 32 + lane;             // this thread's lane of tensor memory
        const int r = (TWO ? grp * kQ : 0) + lr;           // and row of the tile
        const uint32_t lane_addr = tmem + ((uint32_t)((warp & 3) * 32) << 16) + grp * kGroupCols;
        // the keys that the row sees: those in front of the prefix's end, and of its own position's
        const int limit = r < rows ? min(prefix, a.positions[first + (int)((row0 + r) / G)] + 1) : prefix;
        const int step = TWO ? 1 : 2, from = TWO ? 0 : grp;
        float m_used = -INFINITY, l = 0.f;
        uint64_t* o_bar = o_ready + 2 * grp;
        bool ok = true;
        int done = 0;
        auto wait_pv = [&](int t_of, int code, int at) -> bool {
            bool good = mbar_wait(o_bar + (t_of & 1), (t_of >> 1) & 1);
            if (!good && lane == 0) { report(a.error, code, at); *failed = 1; }
            return __all_sync(0xffffffffu, good && !*failed);
        };
        for (int i = from, t = 0; i < n_kt && grp < active; i += step, ++t) {
            const int j0 = (kt_begin + i) * kKV;
            ok = mbar_wait(s_ready + 2 * grp + (t & 1), (t >> 1) & 1);
            if (!ok && lane == 0) { report(a.error, 5, i); *failed = 1; }
            if (!__all_sync(0xffffffffu, ok && !*failed)) { ok = false; break; }
            fence_after_sync();
            // keys of the last tile behind the prefix (another request's, or nobody's): zero their V rows, which any group may do
            // any number of times
            if (j0 + kKV > prefix) {
                uint8_t* v_tile = kv_s + (size_t)(i % kStages) * 2 * kTileBytes + kTileBytes;
                const int first_bad = prefix - j0;
                for (int x = lr; x < (kKV - first_bad) * 8 * kBlocks; x += 128) {
                    const int blk = x / ((kKV - first_bad) * 8), y = x - blk * (kKV - first_bad) * 8;
                    *reinterpret_cast<uint4*>(v_tile + blk * Sh::kKVBlock + (size_t)(first_bad + y / 8) * 128 + (y % 8) * 16) = make_uint4(0u, 0u, 0u, 0u);
                }
            }
            int seen = limit;                              // keys of the tile that the row sees: those in front of `seen`
            if (any_bad) {
                const int id = bt[j0 / a.page_size];
                if (id < 0 || id >= a.pages) seen = 0;
            }
            const bool whole = __all_sync(0xffffffffu, j0 + kKV <= seen);
            uint32_t pk[32];
            {
                uint32_t s0[32], s1[32];
                tmem_ld32(lane_addr + (t & 1) * 64, s0);
                tmem_ld32(lane_addr + (t & 1) * 64 + 32, s1);
                float mx = -INFINITY;
                if (whole) {
#pragma unroll
                    for (int c = 0; c < 32; ++c) mx = fmaxf(mx, fmaxf(__uint_as_float(s0[c]), __uint_as_float(s1[c])));
                } else {
#pragma unroll
                    for (int c = 0; c < 32; ++c) {
                        float v0 = __uint_as_float(s0[c]), v1 = __uint_as_float(s1[c]);
                        if (j0 + c >= seen) v0 = -INFINITY;
                        if (j0 + 32 + c >= seen) v1 = -INFINITY;
                        s0[c] = __float_as_uint(v0); s1[c] = __float_as_uint(v1);
                        mx = fmaxf(mx, fmaxf(v0, v1));
                    }
                }
                mx *= a.scale_log2;
                const bool grow = mx > m_used + kTau;
                float factor = 1.f;
                if (grow) { factor = exp2f(m_used - mx); m_used = mx; l *= factor; }
                if (t > 0 && __any_sync(0xffffffffu, grow)) {
                    if (!wait_pv(t - 1, 6, i)) { ok = false; break; }
                    fence_after_sync();
#pragma unroll
                    for (int piece = 0; piece < HD / 32; ++piece) {
                        uint32_t ov[32];
                        tmem_ld32(lane_addr + 128 + piece * 32, ov);
#pragma unroll
                        for (int c = 0; c < 32; ++c) ov[c] = __float_as_uint(__uint_as_float(ov[c]) * factor);
                        tmem_st32(lane_addr + 128 + piece * 32, ov);
                    }
                    tmem_st_wait();
                }
                const float ref = m_used == -INFINITY ? 0.f : m_used;
                float sum = 0.f;
#pragma unroll
                for (int c = 0; c < 64; c += 2) {
                    const float x0 = __uint_as_float(c < 32 ? s0[c] : s1[c - 32]);
                    const float x1 = __uint_as_float(c + 1 < 32 ? s0[c + 1] : s1[c + 1 - 32]);
                    const float e0 = ex2_approx(fmaf(x0, a.scale_log2, -ref)), e1 = ex2_approx(fmaf(x1, a.scale_log2, -ref));
                    __nv_bfloat162 pr = __floats2bfloat162_rn(e0, e1);
                    pk[c >> 1] = *reinterpret_cast<uint32_t*>(&pr);
                    const float2 as_used = __bfloat1622float2(pr);     // the row sum takes the weights as the product will see them
                    sum += as_used.x + as_used.y;
                }
                l += sum;
            }
            tmem_st32(lane_addr + (t & 1) * 64, pk);
            tmem_st_wait();
            if (j0 + kKV > prefix) fence_async_smem();
            fence_before_sync();
            mbar_arrive(p_ready + 2 * grp + (t & 1));
            done = t + 1;
        }
        if (ok && done > 0) ok = wait_pv(done - 1, 8, from + (done - 1) * step);
        if (ok && done > 0) fence_after_sync();
        if (TWO) {
            if (grp < active && r < rows) {
                const size_t slot = slot_of(r);
                if (l != l) m_used = 0.f;                  // (a NaN among the scores: the range counts, and makes the row NaN)
                a.part_ml[2 * slot] = ok ? m_used : -INFINITY;
                a.part_ml[2 * slot + 1] = ok ? l : 0.f;
            }
#pragma unroll 1
            for (int piece = 0; piece < HD / 32 && ok && done > 0; ++piece) {
                uint32_t ov[32];
                tmem_ld32(lane_addr + 128 + piece * 32, ov);
                if (r < rows) {
                    float4* po = reinterpret_cast<float4*>(a.part_o + slot_of(r) * HD + piece * 32);
#pragma unroll
                    for (int c = 0; c < 8; ++c)
                        po[c] = make_float4(__uint_as_float(ov[4 * c]), __uint_as_float(ov[4 * c + 1]), __uint_as_float(ov[4 * c + 2]), __uint_as_float(ov[4 * c + 3]));
                }
            }
        } else {
            float f0 = 1.f, f1 = 0.f;
#pragma unroll 1
            for (int piece = 0; piece < HD / 64; ++piece) {
                float o[64];
#pragma unroll
                for (int d = 0; d < 64; ++d) o[d] = 0.f;
                if (ok && done > 0) {
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        uint32_t ov[32];
                        tmem_ld32(lane_addr + 128 + piece * 64 + half * 32, ov);
#pragma unroll
                        for (int c = 0; c < 32; ++c) o[half * 32 + c] = __uint_as_float(ov[c]);
                    }
                }
                asm volatile("bar.sync 1, 256;" ::: "memory");         // the ring (or the piece before) is done with
                if (grp > 0) {
#pragma unroll
                    for (int d = 0; d < 64; ++d) merge[d * kQ + lr] = o[d];
                    merge[64 * kQ + lr] = l != l ? 0.f : m_used;
                    merge[65 * kQ + lr] = l;
                }
                asm volatile("bar.sync 1, 256;" ::: "memory");
                if (grp == 0 && r < rows) {
                    if (l != l) m_used = 0.f;
                    const float m1 = merge[64 * kQ + lr], mt = fmaxf(m_used, m1), ref = mt == -INFINITY ? 0.f : mt;
                    f0 = exp2f(m_used - ref);
                    f1 = exp2f(m1 - ref);
                    const size_t slot = slot_of(r);
                    if (piece == 0) {
                        a.part_ml[2 * slot] = ok ? mt : -INFINITY;
                        a.part_ml[2 * slot + 1] = ok ? l * f0 + merge[65 * kQ + lr] * f1 : 0.f;
                    }
                    float4* po = reinterpret_cast<float4*>(a.part_o + slot * HD + piece * 64);
#pragma unroll
                    for (int c = 0; c < 16; ++c) {
                        float v[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) v[e] = o[4 * c + e] * f0 + merge[(4 * c + e) * kQ + lr] * f1;
                        po[c] = make_float4(v[0], v[1], v[2], v[3]);
                    }
                }
            }
        }
    }
    fence_before_sync();
    __syncthreads();
    __syncwarp();
    if (warp == 1) tmem_free<512>(tmem);
}

template <int HD, bool TWO>
inline int launch_prefix(const SharedArgs& a, cudaStream_t stream) {
    typedef Shape<HD, TWO> Sh;
    const long rows = (long)a.tokens * (a.Hq / a.Hkv);
    const long tiles = rows / Sh::kRows + (a.groups < a.tokens ? a.groups : a.tokens);
    const long grid = tiles * a.Hkv * a.prefix_splits;
    if (grid > 0x7fffffffL) return kTooLarge;
    CUtensorMap map_k, map_v;
    int rc = make_tile_map(&map_k, a.k_cache, a.pages * a.page_size, (long)a.Hkv * HD, (long)a.Hkv * HD, kKV);
    if (rc == 0) rc = make_tile_map(&map_v, a.v_cache, a.pages * a.page_size, (long)a.Hkv * HD, (long)a.Hkv * HD, kKV);
    static SharedLimits limits;
    if (rc == 0) rc = ensure_dynamic_smem(shared_prefix_kernel<HD, TWO>, Sh::kSmem, limits);
    if (rc == 0) rc = launch_pdl(shared_prefix_kernel<HD, TWO>, dim3((unsigned)grid), dim3(kThreads), Sh::kSmem, stream, map_k, map_v, a, (int)tiles);
    return rc;
}

}  // namespace shared_tc
}  // namespace lb200
