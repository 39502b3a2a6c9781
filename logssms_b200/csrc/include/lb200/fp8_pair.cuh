// 8-bit products of many rows: a pair of CTAs works on a tile of 256 rows x 256 features of W (SwiGLU: 128 gate and 128 up
// features) with the two-CTA form of tcgen05.mma.  Each CTA loads half of the rows and half of the features of a block, so that
// an SM fetches 32 KB per block of 128 columns where a tile of 128 x 256 of its own would take 48: at the 8-bit rate of the
// tensor cores (512 cycles a block) that is 64 bytes a cycle and SM instead of 96.  A pair stays and takes tile after tile.
//
//   warp 0      one thread issues this CTA's TMA loads; their bytes are counted at the first CTA's barrier
//   warp 1      first CTA: one thread issues the products for both, into one of two accumulators of 256 columns each; both
//               CTAs: allocates tensor memory
//   warps 4-11  two warpgroups: a thread is a row of its CTA's 128 and takes 128 columns of the accumulator: it reads a block's
//               sums, multiplies them by the block's scales and adds them to its 128 sums, while the tensor cores work on the
//               next block.  Warps 0-3 give up registers for that.
// SwiGLU: the features are laid out so that a thread has gate and up of the same 64 features (columns 0-63 and 64-127 of its
// half); only a row's largest magnitude is exchanged between the two warpgroups.
//
// Every wait on an mbarrier is bounded; one that gives up records itself in `error`, the roles run out of their own bounded
// waits, both CTAs still meet the last cluster barrier, tensor memory is freed and the kernel returns.
#pragma once
#include "lb200/fp8_linear.cuh"

namespace lb200 {
namespace fp8 {

constexpr int kPairThreads = 384, kPairStages = 6;
constexpr uint32_t kPairStage = 256 * kBK;                // this CTA's 128 rows of x and 128 features of W
constexpr int kPairRows = 256;
constexpr size_t kPairSmem = 1024 + (size_t)kPairStages * kPairStage;

__device__ __forceinline__ void tma_load_2d_pair(void* dst, const CUtensorMap* map, uint32_t bar, int x, int y) {
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
                 ::"r"(smem_u32(dst)), "l"(map), "r"(bar), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ void umma_f8_pair(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
}
// the barrier of both CTAs gets one arrival when every product issued by this thread so far has completed
__device__ __forceinline__ void umma_commit_pair(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                 ::"r"(smem_u32(bar)), "h"((unsigned short)3) : "memory");
}
__device__ __forceinline__ void mbar_arrive_at(uint32_t bar) {
    // (not a release at cluster scope, which waits for every load of the thread that is under way: 1,900 cycles a block.  What is
    // handed over is tensor memory, ordered by tcgen05's own wait and fences)
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tmem_ld32_async(uint32_t addr, uint32_t (&r)[32]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
                 "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
                 "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
                   "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
                   "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(addr));
}

// tile number -> place: bands of 8 tiles of rows, all features of a band before the next, the rows fastest, so that the pairs
// at work at one time share their rows and their features in L2
struct Tile { int m, n; };
__device__ __forceinline__ Tile tile_at(int t, int tiles_m, int tiles_n) {
    constexpr int kBand = 8;
    const int band = t / (kBand * tiles_n), in = t - band * kBand * tiles_n;
    const int high = min(kBand, tiles_m - band * kBand);
    return {band * kBand + in % high, in / high};
}

template <bool kSwiglu>
__global__ void __launch_bounds__(kPairThreads, 1)
fp8_pair_kernel(const __grid_constant__ CUtensorMap map_w0, const __grid_constant__ CUtensorMap map_w1,
                const __grid_constant__ CUtensorMap map_x, Args a) {
    constexpr int kFeat = kSwiglu ? 128 : 256;            // output features of a tile
    extern __shared__ uint8_t smem_raw[];
    uint8_t* base = reinterpret_cast<uint8_t*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    __shared__ __align__(8) uint64_t full[kPairStages], empty[kPairStages], acc_full[2], acc_empty[2];
    __shared__ uint32_t tops[2][128];                     // SwiGLU: a row's largest magnitude in either half of the features
    __shared__ uint32_t tmem_slot;
    __shared__ volatile int failed;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = (int)cluster_rank();
    const int tiles_m = (a.M + kPairRows - 1) / kPairRows, tiles_n = (a.N + kFeat - 1) / kFeat, tiles = tiles_m * tiles_n;
    const int pairs = gridDim.x / 2, pair = blockIdx.x / 2;
    const int kbn = (a.K + kBK - 1) / kBK;
    if (threadIdx.x == 0) {
        for (int s = 0; s < kPairStages; ++s) { mbar_init(full + s, 1); mbar_init(empty + s, 1); }
        for (int s = 0; s < 2; ++s) { mbar_init(acc_full + s, 1); mbar_init(acc_empty + s, 16); }
        failed = 0;
        mbar_fence_init();
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&tmem_slot)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    fence_before_sync();
    __syncthreads();
    cluster_arrive();                                      // both CTAs' barriers are ready
    cluster_wait();
    fence_after_sync();
    const uint32_t tmem = tmem_slot;
    pdl_trigger();
    pdl_wait();
    int issued = 0;
    const uint32_t full0 = peer_addr(smem_u32(full), 0);
    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
        // (whole warps: see elect_one; the next block's barrier is asked for before the current block is worked on, since a wait
        // takes some 200 cycles even when the phase is long over)
        if (warp == 0) {
            int s = 0, parity = 1;
            bool ready = true, going = true;
            for (int t = pair; t < tiles && going; t += pairs) {
                const Tile at = tile_at(t, tiles_m, tiles_n);
                const int row = at.m * kPairRows + rank * 128, feat = at.n * kFeat;
                for (int kb = 0; kb < kbn; ++kb, ++issued) {
                    if (!ready) ready = mbar_wait(empty + s, parity);
                    if (!__all_sync(0xffffffffu, ready)) { if (lane == 0) report(a.error, 1, kb); failed = 1; going = false; break; }
                    const int s1 = s + 1 == kPairStages ? 0 : s + 1, parity1 = s1 == 0 ? parity ^ 1 : parity;
                    ready = issued + 1 < kPairStages || mbar_test(empty + s1, parity1);
                    if (elect_one()) {
                        uint8_t* x = base + (size_t)s * kPairStage;
                        uint8_t* w = x + 128 * kBK;
                        if (rank == 0) mbar_expect_tx(full + s, 2 * kPairStage);
                        const uint32_t bar = full0 + s * 8;
                        tma_load_2d_pair(x, &map_x, bar, kb * kBK, row);
                        if (kSwiglu) {                     // gate and up of this CTA's 64 features
                            tma_load_2d_pair(w, &map_w0, bar, kb * kBK, feat + rank * 64);
                            tma_load_2d_pair(w + 64 * kBK, &map_w1, bar, kb * kBK, feat + rank * 64);
                        } else {
                            tma_load_2d_pair(w, &map_w0, bar, kb * kBK, feat + rank * 128);
                        }
                    }
                    s = s1; parity = parity1;
                }
            }
        } else if (warp == 1 && rank == 0) {
            constexpr uint32_t idesc = f8_idesc(256, 256);
            const uint64_t desc0 = umma_desc(base);
            const int total = ((tiles - pair + pairs - 1) / pairs) * kbn;      // blocks of all tiles of this pair
            int s = 0, parity = 0;
            bool ready = false, room = true;
            for (int n = 0; n < total; ++n) {
                const int acc = n & 1;
                if (!ready) ready = mbar_wait(full + s, parity);
                if (!room) room = mbar_wait(acc_empty + acc, ((n >> 1) - 1) & 1);
                if (!__all_sync(0xffffffffu, ready && room)) { if (lane == 0) report(a.error, ready ? 3 : 2, n); failed = 1; break; }
                fence_after_sync();
                const int s1 = s + 1 == kPairStages ? 0 : s + 1, parity1 = s1 == 0 ? parity ^ 1 : parity;
                if (elect_one()) {
                    const uint64_t xdesc = desc0 + (uint64_t)(s * (kPairStage >> 4)), wdesc = xdesc + (128 * kBK >> 4);
#pragma unroll
                    for (int k = 0; k < kBK / 32; ++k) umma_f8_pair(tmem + acc * 256, xdesc + 2 * k, wdesc + 2 * k, idesc, k != 0);
                    umma_commit_pair(empty + s);
                    umma_commit_pair(acc_full + acc);
                }
                __syncwarp();
                ready = n + 1 < total && mbar_test(full + s1, parity1);
                room = n == 0 || (n + 1 < total && mbar_test(acc_empty + (acc ^ 1), (((n + 1) >> 1) - 1) & 1));
                s = s1; parity = parity1;
            }
        }
        __syncwarp();
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
        const int group = (warp - 4) >> 2, quarter = warp & 3, in_tile = quarter * 32 + lane;
        const uint32_t from = tmem + ((uint32_t)(quarter * 32) << 16) + group * 128;
        const uint32_t release0 = peer_addr(smem_u32(acc_empty), 0);
        const int last_block = (a.N + kBK - 1) / kBK - 1;
        int n = 0;
        bool ok = true;
        // A block's scales are asked for two blocks ahead, into one of two sets of registers
        struct Scales { float x, w, u; };
        Scales even, odd;
        const float *sx = nullptr, *sw = nullptr, *su = nullptr;
        auto fetch = [&](Scales& f, int kb) {
            kb = min(kb, kbn - 1);
            f.x = sx[kb * a.sx_block];
            f.w = sw[kb * a.sw_block];
            f.u = kSwiglu ? su[kb * a.sw_block] : 0.f;
        };
        auto open = [&](int t) {                           // the scales' places of a tile, and its first two blocks' on their way
            const Tile at = tile_at(t, tiles_m, tiles_n);
            sx = a.sx + (long)min(at.m * kPairRows + rank * 128 + in_tile, a.M - 1) * a.sx_row;
            const int block = kSwiglu ? at.n : min(2 * at.n + group, last_block);
            sw = a.sw0 + block * a.sw_row;
            if (kSwiglu) su = a.sw1 + block * a.sw_row;
            fetch(even, 0);
            fetch(odd, 1);
        };
        if (pair < tiles) open(pair);
        for (int t = pair; t < tiles && ok; t += pairs) {
            const Tile at = tile_at(t, tiles_m, tiles_n);
            uint64_t sum2[64];
#pragma unroll
            for (int j = 0; j < 64; ++j) sum2[j] = 0;
            // 32 columns at a time, the next 32 on their way meanwhile, also from one block to the next: the wait for a block's
            // accumulator is asked for early and its first columns are fetched before the last ones of the block before are added
            uint32_t d[2][32];
            auto arrived = [&](int at, bool known) {       // this warp may read accumulator number `at`
                bool yes = known || mbar_wait(acc_full + (at & 1), (at >> 1) & 1);
                yes = __all_sync(0xffffffffu, yes && !failed);
                if (!yes && lane == 0 && !failed) { report(a.error, 4, at); failed = 1; }
                fence_after_sync();
                return yes;
            };
            auto block = [&](int kb, Scales& f) {
                const float s = join(f.x, f.w), v = kSwiglu ? join(f.x, f.u) : s;
                fetch(f, kb + 2);
                const uint64_t low = pair_of(s, s), high = pair_of(v, v);
                const uint32_t at = from + (n & 1) * 256;
                bool ready = false;
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    tmem_ld_wait();
                    if (c < 3) {
                        tmem_ld32_async(at + 32 * (c + 1), d[(c + 1) & 1]);
                        if (c == 1) ready = mbar_test(acc_full + ((n + 1) & 1), ((n + 1) >> 1) & 1);
                    } else {
                        fence_before_sync();
                        __syncwarp();
                        if (lane == 0) mbar_arrive_at(release0 + (n & 1) * 8);
                        if (kb + 1 < kbn) {
                            ok = arrived(n + 1, ready);
                            if (ok) tmem_ld32_async(from + ((n + 1) & 1) * 256, d[0]);
                        }
                    }
#pragma unroll
                    for (int j = 0; j < 16; ++j) fma2(sum2[16 * c + j], d[c & 1][2 * j], d[c & 1][2 * j + 1], c < 2 ? low : high);
                }
                ++n;
            };
            ok = arrived(n, false);
            if (ok) tmem_ld32_async(from + (n & 1) * 256, d[0]);
            for (int kb = 0; kb < kbn && ok; kb += 2) {
                block(kb, even);
                if (ok && kb + 1 < kbn) block(kb + 1, odd);
            }
            if (!ok) break;
            if (t + pairs < tiles) open(t + pairs);
            float sum[128];
#pragma unroll
            for (int j = 0; j < 64; ++j) { sum[2 * j] = low_of(sum2[j]); sum[2 * j + 1] = high_of(sum2[j]); }
            const long m = (long)at.m * kPairRows + rank * 128 + in_tile;
            if constexpr (kSwiglu) {
                const int f0 = at.n * 128 + group * 64;    // this thread's features
                uint32_t top = 0;
#pragma unroll
                for (int j = 0; j < 64; ++j) {
                    sum[j] = f0 + j < a.N ? silu_f(sum[j] * a.act_scale) * sum[64 + j] : 0.f;
                    top = max(top, magnitude(sum[j]));
                }
                tops[group][in_tile] = top;
                asm volatile("bar.sync 1, 256;" ::: "memory");
                const float scale = fp8_scale(max(top, tops[group ^ 1][in_tile])), back = 1.f / scale;
                asm volatile("bar.sync 1, 256;" ::: "memory");
                if (m < a.M) {
                    uint8_t* q = a.q + m * a.ldq + f0;
#pragma unroll
                    for (int j = 0; j < 64; j += 16) {
                        uint32_t w[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            w[e] = fp8_quad(sum[j + 4 * e] * back, sum[j + 4 * e + 1] * back, sum[j + 4 * e + 2] * back, sum[j + 4 * e + 3] * back);
                        // rows are filled up to 16 bytes
                        if (f0 + j < a.N) *reinterpret_cast<uint4*>(q + j) = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                    if (group == 0) a.qs[m * a.qs_row + at.n * a.qs_block] = scale;
                }
            } else if (m < a.M) {
                const int n0 = at.n * 256 + group * 128;
                const int size = a.out_f32 ? 4 : 2;
                uint8_t* out = (uint8_t*)a.out + ((size_t)m * a.ldo + n0) * size;
                const bool whole = ((uintptr_t)out & 15) == 0;
#pragma unroll
                for (int j = 0; j < 128; j += 8) {
                    float o[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float b = a.bias != nullptr && n0 + j + e < a.N ? a.bias[n0 + j + e] : 0.f;
                        o[e] = (sum[j + e] + b) * a.out_scale;
                    }
                    if (whole && n0 + j + 8 <= a.N) {
                        if (a.out_f32) {
                            reinterpret_cast<float4*>(out + 4 * j)[0] = make_float4(o[0], o[1], o[2], o[3]);
                            reinterpret_cast<float4*>(out + 4 * j)[1] = make_float4(o[4], o[5], o[6], o[7]);
                        } else {
                            uint4 w;
                            __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&w);
#pragma unroll
                            for (int e = 0; e < 4; ++e) h[e] = __floats2bfloat162_rn(o[2 * e], o[2 * e + 1]);
                            *reinterpret_cast<uint4*>(out + 2 * j) = w;
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            if (n0 + j + e < a.N) {
                                if (a.out_f32) reinterpret_cast<float*>(out)[j + e] = o[e];
                                else reinterpret_cast<__nv_bfloat16*>(out)[j + e] = __float2bfloat16_rn(o[e]);
                            }
                    }
                }
            }
        }
    }
    // nobody leaves while the other CTA may still signal here, read these tiles or write to this accumulator
    if (failed && warp == 0 && lane == 0 && rank == 0)     // copies still under way land first
        for (int i = max(0, issued - kPairStages); i < issued; ++i) mbar_wait(full + i % kPairStages, (i / kPairStages) & 1);
    fence_before_sync();
    __syncthreads();
    cluster_arrive();
    cluster_wait();
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

}  // namespace fp8
}  // namespace lb200
