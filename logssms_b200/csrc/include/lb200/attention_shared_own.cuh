// A token's own keys (behind the shared prefix): bfloat16, heads of 64, 96 or 128, pages of a multiple of 16 keys.
//
// Bound by reading the keys and values once: 16 query heads of a key/value head are the rows of m16n8k16 products, which is all the
// arithmetic needs (the tile of 128 rows that tcgen05 wants would be an eighth full, and its scores would go through tensor memory).
// Each of a CTA's two warps has a ring of its own, tiles of 16 keys that TMA brings (tiles lie at multiples of 16 keys, so none
// crosses a page); no warp waits for another before the end, where the results meet in shared memory.  What a tile costs a warp is
// latency, so the scores are summed in four chains, and the loads of a CTA's beginning go out together.  Weights are two bfloat16 numbers
// each, as in the prefix's kernel (64 requests with 8,192 keys of their own: 69 us instead of 67).
#pragma once
#include "lb200/attention_shared.h"
#include "lb200/common.cuh"
#include "lb200/tcgen05.cuh"

namespace lb200 {
namespace shared_own {
using namespace tc;
typedef __nv_bfloat16 bf16;
constexpr int kWarps = 2, kThreads = 32 * kWarps, kKeys = 16, kStages = 3, kRows = 16, kLeast = 256;
constexpr float kTau = 8.f;                               // log2 of the growth of a row's maximum that sums are scaled for

// A tile: blocks of 64 columns, [16 keys][128 bytes]; 16-byte piece c of key r lies at c ^ (r & 7).
template <int HD> struct Shape {
    static constexpr int kBlocks = (HD + 63) / 64;
    static constexpr uint32_t kBlock = kKeys * 128, kTile = kBlocks * kBlock, kStage = 2 * kTile, kRing = kStages * kStage;
    static constexpr uint32_t kResult = kWarps * kRows * (HD + 2) * 4;         // at the end, over the rings
    static constexpr uint32_t kSmem = kWarps * kRing + 64;
    static_assert(kResult <= kWarps * kRing, "results over the rings");
};

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// role 9: a warp's wait for a tile
__device__ __forceinline__ void report(int* error, int tile) { atomicCAS(error, 0, (9 << 24) | ((blockIdx.x & 0xFFF) << 12) | (tile & 0xFFF) | 0x40000000); }

// grid: (tokens x tiles of 16 of a token's heads, kv heads, ranges)
template <int HD>
__global__ void __maxnreg__(152)
shared_own_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, SharedArgs a, int head_tiles) {
    typedef Shape<HD> Sh;
    constexpr int kK = HD / 16;                           // steps of 16 columns
    extern __shared__ __align__(1024) uint8_t smem[];      // (the swizzle goes by the address)
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int G = a.Hq / a.Hkv, kvh = blockIdx.y, split = blockIdx.z;
    const int t = blockIdx.x / head_tiles, h0 = (blockIdx.x % head_tiles) * kRows;
    const int rows = min(kRows, G - h0);
    // The grid's last CTA waits for the prefix's kernel at its end, so that this kernel ends behind it, and the merge, which waits
    // for this one, behind both.  (If all waited, they would keep their places on the SMs until then.)
    const bool last = blockIdx.x == gridDim.x - 1 && blockIdx.y == gridDim.y - 1 && blockIdx.z == gridDim.z - 1;

    const int request = a.token_req[t], position = a.positions[t];
    int begin = 0, first_token;
    const bool grouped = prefix_of(a, t, &begin, &first_token);
    // (behind the loads on whose answers the first tile waits) the queries as A operands: rows lane / 4 and + 8, columns 2 (lane % 4) and + 8 of each step
    uint32_t qa[kK][4];
    {
        const bf16* q = (const bf16*)a.q + (size_t)t * a.q_stride + (size_t)(kvh * G + h0) * HD + 2 * (lane & 3);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int row = (lane >> 2) + 8 * e;
#pragma unroll
            for (int k = 0; k < kK; ++k) {
                qa[k][e] = row < rows ? *reinterpret_cast<const uint32_t*>(q + (size_t)row * HD + 16 * k) : 0u;
                qa[k][2 + e] = row < rows ? *reinterpret_cast<const uint32_t*>(q + (size_t)row * HD + 16 * k + 8) : 0u;
            }
        }
    }
    const bool known = request >= 0 && request < a.requests;
    const int end = known ? (int)min((long)position + 1, (long)a.bt_cols * a.page_size) : 0;
    int from = 0, to = 0;                                 // from: a multiple of 16; keys below `begin` are left out
    if (grouped && end > begin) {
        const int first = begin / kKeys * kKeys;
        // (no range is shorter than kLeast: a CTA's beginning and end take as long as 200 keys)
        const int per = max(((end - first + a.own_splits - 1) / a.own_splits + kKeys * kWarps - 1) / (kKeys * kWarps) * (kKeys * kWarps), kLeast);
        from = (int)min((long)first + (long)split * per, (long)end);
        to = (int)min((long)from + per, (long)end);
    }
    const int splits = a.prefix_splits + a.own_splits;
    const size_t slot0 = ((size_t)t * a.Hq + kvh * G + h0) * splits + a.prefix_splits + split;      // of row r: + r * splits
    if (from >= to) {                                     // no keys: nothing to merge (a token of no group has no merge either)
        if (grouped && threadIdx.x < rows) {
            float* ml = a.part_ml + 2 * (slot0 + (size_t)threadIdx.x * splits);
            ml[0] = -INFINITY; ml[1] = 0.f;
        }
        if (last) pdl_wait();
        return;
    }
    const int* bt = a.block_table + (long)request * a.bt_stride;
    const int n_tiles = (to - from + kKeys - 1) / kKeys;
    const int mine = (n_tiles + kWarps - 1 - warp) / kWarps;               // of this warp: tiles warp, warp + kWarps, ...
    auto tile_at = [&](int i) { return from + (i * kWarps + warp) * kKeys; };
    // where the next tile that is asked for lies: its place in the table and within the page
    int entry = tile_at(0) / a.page_size, offset = tile_at(0) - entry * a.page_size;
    int next = mine > 0 ? bt[entry] : -1;

    uint64_t* full = reinterpret_cast<uint64_t*>(smem + kWarps * Sh::kRing) + warp * kStages;
    uint8_t* ring = smem + warp * Sh::kRing;
    if (lane == 0) {
        for (int s = 0; s < kStages; ++s) mbar_init(full + s, 1);
        mbar_fence_init();
    }
    __syncwarp();
    uint32_t there = 0;                                   // a bit per tile on its way: its page is there
    // tile i into stage s (a page that is not there: rows behind the pool, which read as zeros).  Whole warps: see elect_one.
    auto fetch = [&](int i, int s, int ahead) {
        if (i >= mine) return;
        const bool ok = next >= 0 && next < a.pages;
        there |= (uint32_t)ok << ahead;
        const int row = (ok ? next : (int)a.pages) * a.page_size + offset;
        if (elect_one()) {
            mbar_expect_tx(full + s, Sh::kStage);
#pragma unroll
            for (int b = 0; b < Sh::kBlocks; ++b) {
                tma_load_2d(ring + s * Sh::kStage + b * Sh::kBlock, &map_k, full + s, kvh * HD + b * 64, row);
                tma_load_2d(ring + s * Sh::kStage + Sh::kTile + b * Sh::kBlock, &map_v, full + s, kvh * HD + b * 64, row);
            }
        }
        __syncwarp();
        offset += kKeys * kWarps;
        while (offset >= a.page_size) { offset -= a.page_size; ++entry; }
        next = i + 1 < mine ? bt[entry] : -1;
    };
#pragma unroll
    for (int s = 0; s < kStages - 1; ++s) fetch(s, s, s);

    float acc[2 * kK][4];                                 // 8 columns each
#pragma unroll
    for (int i = 0; i < 2 * kK; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][e] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    int s = 0, i = 0;
    uint32_t phase = 0;
    bool good = true;
    for (; i < mine; ++i) {
        fetch(i + kStages - 1, s == 0 ? kStages - 1 : s - 1, kStages - 1);
        good = mbar_test(full + s, phase) || mbar_wait(full + s, phase);
        good = __all_sync(0xffffffffu, good);
        if (!good) break;
        const uint32_t k_at = smem_u32(ring) + s * Sh::kStage, v_at = k_at + Sh::kTile;
        float sc4[2][2][4] = {};                          // [keys 0..7 / 8..15][even and odd steps]
#pragma unroll
        for (int k = 0; k < kK; ++k) {
            // matrices: keys 0..7 / 8..15 (lane / 16) x columns 0..7 / 8..15 of the step (lane / 8 % 2)
            uint32_t b[4];
            const int key = (lane & 7) + ((lane >> 4) << 3), c = 2 * (k & 3) + ((lane >> 3) & 1);
            ldsm4(b, k_at + (k >> 2) * Sh::kBlock + key * 128 + ((c ^ (key & 7)) << 4));
            mma(sc4[0][k & 1], qa[k], b[0], b[1]);
            mma(sc4[1][k & 1], qa[k], b[2], b[3]);
        }
        const int j0 = tile_at(i);
        const bool page_ok = there & 1u;
        there >>= 1;
        // keys of the tile that count: lo .. hi - 1; the values of the others become zeros
        const int lo = page_ok ? max(begin - j0, 0) : kKeys, hi = min(to - j0, kKeys);
        const bool whole = lo == 0 && hi == kKeys;
        if (!whole) {
            for (int x = lane; x < kKeys * 8 * Sh::kBlocks; x += 32) {
                const int key = (x >> 3) % kKeys, b = (x >> 3) / kKeys;
                if (key < lo || key >= hi)
                    *reinterpret_cast<uint4*>(ring + s * Sh::kStage + Sh::kTile + b * Sh::kBlock + key * 128 + (x & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
            }
            fence_async_smem();                           // (the stage's next tile comes by TMA)
            __syncwarp();
        }
        float sc[2][4], mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int key = 8 * n + 2 * (lane & 3) + (e & 1);
                const float v = (sc4[n][0][e] + sc4[n][1][e]) * a.scale_log2;
                sc[n][e] = whole || (key >= lo && key < hi) ? v : -INFINITY;
                mx[e >> 1] = fmaxf(mx[e >> 1], sc[n][e]);
            }
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) {
            mx[0] = fmaxf(mx[0], __shfl_xor_sync(0xffffffffu, mx[0], o));
            mx[1] = fmaxf(mx[1], __shfl_xor_sync(0xffffffffu, mx[1], o));
        }
        // the maximum is followed lazily: sums are scaled only where it has grown by more than 2^8
        const bool grow0 = mx[0] > m[0] + kTau, grow1 = mx[1] > m[1] + kTau;
        if (__any_sync(0xffffffffu, grow0 || grow1)) {
            const float f0 = grow0 ? exp2f(m[0] - mx[0]) : 1.f, f1 = grow1 ? exp2f(m[1] - mx[1]) : 1.f;
            if (grow0) m[0] = mx[0];
            if (grow1) m[1] = mx[1];
            l[0] *= f0; l[1] *= f1;
#pragma unroll
            for (int c = 0; c < 2 * kK; ++c) { acc[c][0] *= f0; acc[c][1] *= f0; acc[c][2] *= f1; acc[c][3] *= f1; }
        }
        const float r0 = m[0] == -INFINITY ? 0.f : m[0], r1 = m[1] == -INFINITY ? 0.f : m[1];
        uint32_t p[4], rest[4];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            float w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = ex2_approx(sc[n][e] - (e < 2 ? r0 : r1));
            split_weights(w[0], w[1], p[2 * n], rest[2 * n]);
            split_weights(w[2], w[3], p[2 * n + 1], rest[2 * n + 1]);
            l[0] += w[0] + w[1];
            l[1] += w[2] + w[3];
        }
#pragma unroll
        for (int k = 0; k < kK; ++k) {
            // matrices: keys 0..7 / 8..15 (lane / 8 % 2) x columns 0..7 / 8..15 of the step (lane / 16), transposed
            uint32_t b[4];
            const int key = (lane & 7) + (((lane >> 3) & 1) << 3), c = 2 * (k & 3) + (lane >> 4);
            ldsm4_t(b, v_at + (k >> 2) * Sh::kBlock + key * 128 + ((c ^ (key & 7)) << 4));
            mma(acc[2 * k], p, b[0], b[1]);
            mma(acc[2 * k + 1], p, b[2], b[3]);
            mma(acc[2 * k], rest, b[0], b[1]);
            mma(acc[2 * k + 1], rest, b[2], b[3]);
        }
        __syncwarp();                                     // the stage may be filled again
        if (++s == kStages) { s = 0; phase ^= 1u; }
    }
    if (!good) {                                          // a copy that did not land: the row's result means nothing
        if (lane == 0) report(a.error, i);
        for (int x = i; x < min(i + kStages, mine); ++x) mbar_wait(full + x % kStages, (x / kStages) & 1);
        m[0] = m[1] = -INFINITY;
        l[0] = l[1] = 0.f;
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
        l[0] += __shfl_xor_sync(0xffffffffu, l[0], o);
        l[1] += __shfl_xor_sync(0xffffffffu, l[1], o);
    }
    __syncthreads();                                      // every ring is done with
    float* res = reinterpret_cast<float*>(smem);
    constexpr int kLd = HD + 2;
    {
        const int c = 2 * (lane & 3);
        float* w0 = res + (warp * kRows + (lane >> 2)) * kLd;
        float* w1 = w0 + 8 * kLd;
#pragma unroll
        for (int n = 0; n < 2 * kK; ++n) {
            *reinterpret_cast<float2*>(w0 + 8 * n + c) = make_float2(acc[n][0], acc[n][1]);
            *reinterpret_cast<float2*>(w1 + 8 * n + c) = make_float2(acc[n][2], acc[n][3]);
        }
        if ((lane & 3) == 0) {
            w0[HD] = l[0] != l[0] ? 0.f : m[0]; w0[HD + 1] = l[0];          // (NaN among the scores: the range counts)
            w1[HD] = l[1] != l[1] ? 0.f : m[1]; w1[HD + 1] = l[1];
        }
    }
    __syncthreads();
    // a thread: row threadIdx / 8 and 8 on, columns 4 (threadIdx % 8) and 32 further on
    for (int r = threadIdx.x >> 3; r < rows; r += kThreads / 8) {
        float mt = -INFINITY, f[kWarps], lt = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) mt = fmaxf(mt, res[(w * kRows + r) * kLd + HD]);
        const float ref = mt == -INFINITY ? 0.f : mt;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            f[w] = exp2f(res[(w * kRows + r) * kLd + HD] - ref);
            lt += res[(w * kRows + r) * kLd + HD + 1] * f[w];
        }
        const size_t slot = slot0 + (size_t)r * splits;
        if ((threadIdx.x & 7) == 0) { a.part_ml[2 * slot] = mt; a.part_ml[2 * slot + 1] = lt; }
#pragma unroll
        for (int d = 4 * (threadIdx.x & 7); d < HD; d += 32) {
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float2 u = *reinterpret_cast<const float2*>(res + (w * kRows + r) * kLd + d), v = *reinterpret_cast<const float2*>(res + (w * kRows + r) * kLd + d + 2);
                o.x = fmaf(u.x, f[w], o.x); o.y = fmaf(u.y, f[w], o.y); o.z = fmaf(v.x, f[w], o.z); o.w = fmaf(v.y, f[w], o.w);
            }
            *reinterpret_cast<float4*>(a.part_o + slot * HD + d) = o;
        }
    }
    if (last) pdl_wait();
}

template <int HD>
inline int launch_own(const SharedArgs& a, cudaStream_t stream) {
    const int head_tiles = (a.Hq / a.Hkv + kRows - 1) / kRows;
    static SharedLimits limits;
    static DoneOnce carveout;
    CUtensorMap map_k, map_v;
    int rc = make_tile_map(&map_k, a.k_cache, a.pages * a.page_size, (long)a.Hkv * HD, (long)a.Hkv * HD, kKeys);
    if (rc == 0) rc = make_tile_map(&map_v, a.v_cache, a.pages * a.page_size, (long)a.Hkv * HD, (long)a.Hkv * HD, kKeys);
    if (rc == 0) rc = ensure_dynamic_smem(shared_own_kernel<HD>, Shape<HD>::kSmem, limits);
    if (rc == 0) rc = whole_carveout(shared_own_kernel<HD>, carveout);
    if (rc == 0) rc = launch_pdl(shared_own_kernel<HD>, dim3((unsigned)(a.tokens * head_tiles), a.Hkv, a.own_splits), dim3(kThreads), Shape<HD>::kSmem, stream, map_k, map_v, a, head_tiles);
    return rc;
}

}  // namespace shared_own
}  // namespace lb200
