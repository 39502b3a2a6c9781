// A token's own keys (behind the shared prefix) in bfloat16, heads in steps of 16 up to 128.
//
// Bound by reading the keys and values once: 16 query heads of a key/value head are the rows of m16n8k16 products, which is all the
// arithmetic needs.  Each of the four warps has a ring of its own: tiles of 16 keys, brought by 16-byte asynchronous copies and read
// with ldmatrix; no warp waits for another before the end, where the four results meet in shared memory.
#pragma once
#include "lb200/attention_shared.h"
#include "lb200/common.cuh"

namespace lb200 {
namespace shared_own {
typedef __nv_bfloat16 bf16;
constexpr int kWarps = 4, kThreads = 32 * kWarps, kKeys = 16, kStages = 3, kRows = 16;
constexpr float kTau = 8.f;

// Rows of HDP columns (64 or 128); 16-byte piece c of row r lies at c ^ (r & 7), so that eight rows' pieces are in eight banks.
template <int HDP> struct Shape {
    static constexpr uint32_t kPitch = HDP * 2, kTile = kKeys * kPitch, kStage = 2 * kTile, kRing = kStages * kStage;
    static constexpr uint32_t kSmem = kWarps * kRing;     // (the results at the end, [warp][16][HDP + 2] float32, lie over the rings)
    static_assert(kWarps * kRows * (HDP + 2) * 4 <= kSmem, "results over the rings");
};

__device__ __forceinline__ uint32_t smem_at(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool there) {         // zeros where nothing is there
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack(float x, float y) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&v);
}

// grid: (tokens x tiles of 16 of a token's heads, kv heads, ranges)
template <int HDP>
__global__ void __launch_bounds__(kThreads) shared_own_kernel(SharedArgs a, int head_tiles) {
    typedef Shape<HDP> Sh;
    constexpr int kK = HDP / 16;                          // steps of 16 columns
    extern __shared__ __align__(128) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, hd = a.hd, steps = hd >> 4;
    const int G = a.Hq / a.Hkv, kvh = blockIdx.y, split = blockIdx.z;
    const int t = blockIdx.x / head_tiles, h0 = (blockIdx.x % head_tiles) * kRows;
    const int rows = min(kRows, G - h0);
    const int g = group_of(a, t);
    int from = 0, to = 0;
    const int request = a.token_req[t];
    const bool known = request >= 0 && request < a.requests;
    if (g >= 0) {
        const int begin = max(a.prefix_lens[g], 0);
        const int end = known ? (int)min((long)a.positions[t] + 1, (long)a.bt_cols * a.page_size) : 0;
        if (end > begin) {
            const int per = ((end - begin + a.own_splits - 1) / a.own_splits + kKeys * kWarps - 1) / (kKeys * kWarps) * (kKeys * kWarps);
            from = (int)min((long)begin + (long)split * per, (long)end);
            to = (int)min((long)from + per, (long)end);
        }
    }
    const int splits = a.prefix_splits + a.own_splits;
    const size_t slot0 = ((size_t)t * a.Hq + kvh * G + h0) * splits + a.prefix_splits + split;      // of row r: + r * splits
    if (from >= to) {                                     // no keys: nothing to merge (a token of no group has no merge either)
        if (g >= 0 && threadIdx.x < rows) {
            float* ml = a.part_ml + 2 * (slot0 + (size_t)threadIdx.x * splits);
            ml[0] = -INFINITY; ml[1] = 0.f;
        }
        pdl_wait();
        return;
    }
    const int* bt = a.block_table + (long)request * a.bt_stride;
    const bf16* kc = (const bf16*)a.k_cache + (size_t)kvh * hd;
    const bf16* vc = (const bf16*)a.v_cache + (size_t)kvh * hd;
    const size_t key_stride = (size_t)a.Hkv * hd;

    // the queries as A operands: rows lane / 4 and + 8, columns 2 (lane % 4) and + 8 of each step
    uint32_t qa[kK][4];
    {
        const bf16* q = (const bf16*)a.q + (size_t)t * a.q_stride + (size_t)(kvh * G + h0) * hd;
        const int r = lane >> 2, c = 2 * (lane & 3);
#pragma unroll
        for (int k = 0; k < kK; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int row = r + (e & 1) * 8, col = 16 * k + c + (e >> 1) * 8;
                qa[k][e] = row < rows && col < hd ? *reinterpret_cast<const uint32_t*>(q + (size_t)row * hd + col) : 0u;
            }
    }
    const uint32_t ring = smem_at(smem) + warp * Sh::kRing;
    const int n_tiles = (to - from + kKeys * kWarps - 1) / (kKeys * kWarps);        // of this warp: i-th begins at from + (4 i + warp) 16
    // the place of key j (lanes 0 .. 15 ask for one each): its row in the pool, or -1
    auto place = [&](int i) -> long {
        const int j = from + (i * kWarps + warp) * kKeys + (lane & 15);
        if (i >= n_tiles || j >= to) return -1;
        const int page = bt[j / a.page_size];
        return page >= 0 && page < a.pages ? (long)page * a.page_size + j % a.page_size : -1;
    };
    uint64_t there = 0;                                   // 16 bits a tile: which of its keys there are; the tile at work in the lowest
    static_assert(16 * kStages <= 64, "tiles on their way");
    constexpr int kPieces = HDP / 8;
    auto fetch = [&](int s, int ahead, long row) {
        there |= (uint64_t)(__ballot_sync(0xffffffffu, row >= 0) & 0xffffu) << (16 * ahead);
        const uint32_t k_at = ring + s * Sh::kStage, v_at = k_at + Sh::kTile;
#pragma unroll
        for (int n = 0; n < kKeys * kPieces / 32; ++n) {
            const int key = (n * 32 + lane) / kPieces, c = (n * 32 + lane) % kPieces;
            const long at = __shfl_sync(0xffffffffu, row, key);
            const bool ok = at >= 0 && c * 8 < hd;
            const size_t off = ok ? (size_t)at * key_stride + c * 8 : 0;
            const uint32_t d = key * Sh::kPitch + ((c ^ (key & 7)) << 4);
            copy16(k_at + d, kc + off, ok);
            copy16(v_at + d, vc + off, ok);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    long next = place(0);
#pragma unroll
    for (int s = 0; s < kStages - 1; ++s) {
        const long row = next;
        next = place(s + 1);
        fetch(s, s, row);
    }

    float acc[2 * kK][4];                                 // 8 columns each
#pragma unroll
    for (int i = 0; i < 2 * kK; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][e] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    int s = 0;
#pragma unroll kStages
    for (int i = 0; i < n_tiles; ++i) {
        {
            const long row = next;
            next = place(i + kStages);
            fetch((s + kStages - 1) % kStages, kStages - 1, row);
        }
        asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
        __syncwarp();
        const uint32_t k_at = ring + s * Sh::kStage, v_at = k_at + Sh::kTile;
        float sc[2][4] = {};
#pragma unroll
        for (int k = 0; k < kK; ++k) {
            if (k < steps) {
                // matrices: keys 0..7 / 8..15 (lane / 16) x columns 0..7 / 8..15 of the step (lane / 8 % 2)
                uint32_t b[4];
                const int key = (lane & 7) + ((lane >> 4) << 3), c = 2 * k + ((lane >> 3) & 1);
                ldsm4(b, k_at + key * Sh::kPitch + ((c ^ (key & 7)) << 4));
                mma(sc[0], qa[k], b[0], b[1]);
                mma(sc[1], qa[k], b[2], b[3]);
            }
        }
        const uint32_t ok = (uint32_t)there & 0xffffu;
        there >>= 16;
        float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int key = 8 * n + 2 * (lane & 3) + (e & 1);
                sc[n][e] = ok >> key & 1u ? sc[n][e] * a.scale_log2 : -INFINITY;
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
        uint32_t p[4];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            p[2 * n] = pack(exp2f(sc[n][0] - r0), exp2f(sc[n][1] - r0));
            p[2 * n + 1] = pack(exp2f(sc[n][2] - r1), exp2f(sc[n][3] - r1));
            // the sums take the weights as the product sees them, rounded
            const float2 u = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&p[2 * n]));
            const float2 v = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&p[2 * n + 1]));
            l[0] += u.x + u.y;
            l[1] += v.x + v.y;
        }
#pragma unroll
        for (int k = 0; k < kK; ++k) {
            if (k < steps) {
                // matrices: keys 0..7 / 8..15 (lane / 8 % 2) x columns 0..7 / 8..15 of the step (lane / 16), transposed
                uint32_t b[4];
                const int key = (lane & 7) + (((lane >> 3) & 1) << 3), c = 2 * k + (lane >> 4);
                ldsm4_t(b, v_at + key * Sh::kPitch + ((c ^ (key & 7)) << 4));
                mma(acc[2 * k], p, b[0], b[1]);
                mma(acc[2 * k + 1], p, b[2], b[3]);
            }
        }
        __syncwarp();                                     // the stage may be filled again
        s = s + 1 == kStages ? 0 : s + 1;
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
        l[0] += __shfl_xor_sync(0xffffffffu, l[0], o);
        l[1] += __shfl_xor_sync(0xffffffffu, l[1], o);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();                                      // every ring is done with
    float* res = reinterpret_cast<float*>(smem);
    constexpr int kLd = HDP + 2;
    {
        const int r = lane >> 2, c = 2 * (lane & 3);
        float* w0 = res + (warp * kRows + r) * kLd;
        float* w1 = w0 + 8 * kLd;
#pragma unroll
        for (int i = 0; i < 2 * kK; ++i) {
            *reinterpret_cast<float2*>(w0 + 8 * i + c) = make_float2(acc[i][0], acc[i][1]);
            *reinterpret_cast<float2*>(w1 + 8 * i + c) = make_float2(acc[i][2], acc[i][3]);
        }
        if ((lane & 3) == 0) {
            w0[HDP] = l[0] != l[0] ? 0.f : m[0]; w0[HDP + 1] = l[0];
            w1[HDP] = l[1] != l[1] ? 0.f : m[1]; w1[HDP + 1] = l[1];
        }
    }
    __syncthreads();
    // a thread: row threadIdx / 8, columns 4 (threadIdx % 8) and 32 further on
    const int r = threadIdx.x >> 3;
    if (r < rows) {
        float mt = -INFINITY, f[kWarps], lt = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) mt = fmaxf(mt, res[(w * kRows + r) * kLd + HDP]);
        const float ref = mt == -INFINITY ? 0.f : mt;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            f[w] = exp2f(res[(w * kRows + r) * kLd + HDP] - ref);
            lt += res[(w * kRows + r) * kLd + HDP + 1] * f[w];
        }
        const size_t slot = slot0 + (size_t)r * splits;
        if ((threadIdx.x & 7) == 0) { a.part_ml[2 * slot] = mt; a.part_ml[2 * slot + 1] = lt; }
        for (int d = 4 * (threadIdx.x & 7); d < hd; d += 32) {
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float2 u = *reinterpret_cast<const float2*>(res + (w * kRows + r) * kLd + d), v = *reinterpret_cast<const float2*>(res + (w * kRows + r) * kLd + d + 2);
                o.x = fmaf(u.x, f[w], o.x); o.y = fmaf(u.y, f[w], o.y); o.z = fmaf(v.x, f[w], o.z); o.w = fmaf(v.y, f[w], o.w);
            }
            *reinterpret_cast<float4*>(a.part_o + slot * hd + d) = o;
        }
    }
    pdl_wait();                                           // the prefix's kernel has ended when this one has
}

template <int HDP>
inline int launch_own(const SharedArgs& a, cudaStream_t stream) {
    const int head_tiles = (a.Hq / a.Hkv + kRows - 1) / kRows;
    static SharedLimits limits;
    int rc = ensure_dynamic_smem(shared_own_kernel<HDP>, Shape<HDP>::kSmem, limits);
    if (rc == 0) rc = launch_pdl(shared_own_kernel<HDP>, dim3((unsigned)(a.tokens * head_tiles), a.Hkv, a.own_splits), dim3(kThreads), Shape<HDP>::kSmem, stream, a, head_tiles);
    return rc;
}

}  // namespace shared_own
}  // namespace lb200
