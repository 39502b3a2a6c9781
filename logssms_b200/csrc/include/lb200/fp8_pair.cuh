// 8-bit products of many rows: a pair of CTAs works on a tile of 256 rows x 256 features of W (SwiGLU: 128 gate and 128 up
// features) with the two-CTA form of tcgen05.mma.  Each CTA loads half of the rows and half of the features of a block, so that
// an SM fetches 32 KB per block of 128 columns where a tile of 128 x 256 of its own would take 48: at the 8-bit rate of the
// tensor cores (512 cycles a block) that is 64 bytes a cycle and SM instead of 96.  A pair stays and takes tile after tile.
//
//   warp 0      issues this CTA's TMA loads; their bytes are counted at the first CTA's barrier
//   warps 1, 3  first CTA: issue the products for both, one warp for either half of 128 columns; two accumulators of 256 columns.
//               Warp 1 also allocates tensor memory (both CTAs)
//   warp 2      watches the accumulators, hands stages back, wakes the warps that add
//   warps 4-19  four warpgroups: a thread is a row of its CTA's 128 and takes 64 columns of the accumulator: it reads a block's
//               sums, multiplies them by the block's scales and adds them to its 64 sums, while the tensor cores work on the next
//               block.  Warps 0-3 give up registers for that.
// What bounds it: the adding (256 cycles of multiply-adds and two waits for tensor memory per block), the products (512 cycles) and
// the hand-over of an accumulator between them lie within a quarter of each other; left out one at a time, down 8,192 x 3,072 x 12,288
// took 264 us without the multiply-adds, 277 with a quarter of the products, 285 without loads, 314 with all.  Now it takes 303 us in
// bursts (2.04 PFLOP/s), 347 in a long row of calls on random data, when the power limit sets the clock (1,447 MHz), and 249 on zeros.
// SwiGLU: the features are laid out so that a thread has gate and up of the same 32 features; only a row's largest magnitude is
// exchanged between the four warpgroups.
//
// Fewer tiles than pairs, and those left over from whole rounds: a cluster of two or four pairs shares a tile's blocks (kParts; see
// `launch_pair` for what it brings).
//
// Every wait on an mbarrier is bounded; one that gives up records itself in `error`, the roles run out of their own bounded
// waits, both CTAs still meet the last cluster barrier, tensor memory is freed and the kernel returns.
#pragma once
#include "lb200/fp8_linear.cuh"
#include <type_traits>

namespace lb200 {
namespace fp8 {

constexpr int kPairRows = 256;
constexpr int kPairGroups = 4, kAdders = 128 * kPairGroups, kPairThreads = 128 + kAdders;
constexpr int kCols = 64 * kPairGroups, kHalf = kCols / 2;                // accumulator columns of a block, and of one of its halves
constexpr int kHalfAdders = kAdders / 2;
constexpr uint32_t kPairStage = (128 + kCols / 2) * kBK;            // a CTA's 128 rows of x and half of the features
constexpr int kPairStages = 6;                            // even: each of the two warps that issue meets every use of its stages
constexpr size_t kPairTurn = 4 * kPairGroups * 32 * 16 * 4;            // 32 rows x 16 features for each warp that adds
constexpr size_t pair_smem(bool ragged) { return 1024 + (size_t)kPairStages * kPairStage + (ragged ? kPairTurn : 0); }

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
__device__ __forceinline__ void umma_commit_pair(uint64_t* bar, int ctas) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                 ::"r"(smem_u32(bar)), "h"((unsigned short)ctas) : "memory");
}
__device__ __forceinline__ void mbar_arrive_at(uint32_t bar) {
    // (not a release at cluster scope, which waits for every load of the thread that is under way: 1,900 cycles a block.  What is
    // handed over is tensor memory, ordered by tcgen05's own wait and fences)
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// the same where `mine` is set, without a branch
__device__ __forceinline__ void mbar_arrive_at_if(uint32_t bar, uint32_t mine) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %1, 0;\n\t@p mbarrier.arrive.shared::cluster.b64 _, [%0];\n\t}" ::"r"(bar), "r"(mine) : "memory");
}
__device__ __forceinline__ bool mbar_test_at(uint32_t bar, uint32_t parity) {
    uint32_t done;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(done) : "r"(bar), "r"(parity) : "memory");
    return done != 0;
}
// barriers of the CTA among `kCount` threads: some only arrive, the others sleep until all have
constexpr int kWakeAdders = 2;                             // one for each accumulator, up to four
template <int kCount>
__device__ __forceinline__ void wake(int id) { asm volatile("bar.arrive %0, %1;" ::"r"(id), "n"(kCount) : "memory"); }
template <int kCount>
__device__ __forceinline__ void sleep_until_woken(int id) { asm volatile("bar.sync %0, %1;" ::"r"(id), "n"(kCount) : "memory"); }
__device__ __forceinline__ void store32(void* p, const uint32_t (&w)[8]) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
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

// kRagged: rows of `out` that do not lie on 32 bytes, or features that do not fill 32 bytes
// kParts > 1: a cluster of so many pairs shares the blocks of a tile; for tiles that do not fill a round of all pairs.  Once every
// pair's ring is empty, each thread hands the other pairs their share of its 64 sums, over the ring, and finishes its own share: the
// sums of all pairs are added in the order of their blocks.
template <bool kSwiglu, bool kRagged, int kParts>
__global__ void __launch_bounds__(kPairThreads, 1)
fp8_pair_kernel(const __grid_constant__ CUtensorMap map_w0, const __grid_constant__ CUtensorMap map_w1,
                const __grid_constant__ CUtensorMap map_x, Args a) {
    constexpr int kFeat = kSwiglu ? 128 : 256;            // output features of a tile
    constexpr int kMine = 64 / kParts;                    // columns that a thread finishes
    static_assert(!kSwiglu || kParts == 1, "a row's largest magnitude is taken in one CTA");
    extern __shared__ uint8_t smem_raw[];
    uint8_t* base = reinterpret_cast<uint8_t*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    __shared__ __align__(16) uint64_t acc_full[4], acc_empty[4], full[kPairStages], empty[kPairStages];
    __shared__ uint32_t tops[kSwiglu ? kPairGroups : 1][128];       // SwiGLU: a row's largest magnitude among a group's features
    __shared__ uint32_t tmem_slot;
    __shared__ volatile int failed;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int in_cluster = (int)cluster_rank(), rank = kParts > 1 ? in_cluster & 1 : in_cluster;
    const int leader = kParts > 1 ? in_cluster & ~1 : 0, part = kParts > 1 ? in_cluster >> 1 : 0;
    const int tiles_m = (a.M + kPairRows - 1) / kPairRows, tiles_n = (a.N + kFeat - 1) / kFeat;
    const int pairs = gridDim.x / 2, pair = blockIdx.x / 2;
    // this pair's tiles, and the blocks of K that it takes of each
    const int first = kParts > 1 ? a.tile0 + pair / kParts : pair, end = kParts > 1 ? first + 1 : a.tiles;
    const int all = (a.K + kBK - 1) / kBK;
    const int kb0 = kParts > 1 ? all * part / kParts : 0, kbn = kParts > 1 ? all * (part + 1) / kParts - kb0 : all;
    if (threadIdx.x == 0) {
        for (int s = 0; s < kPairStages; ++s) { mbar_init(full + s, 1); mbar_init(empty + s, 2); }
        for (int s = 0; s < 4; ++s) { mbar_init(acc_full + s, 1); mbar_init(acc_empty + s, 2 * kHalfAdders / 32); }
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
    const int total = (kParts > 1 ? 1 : (end - first + pairs - 1) / pairs) * kbn;       // blocks of all tiles of this pair
    const uint32_t full0 = peer_addr(smem_u32(full), leader);
    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 32;");              // 640 threads x 96 registers at launch: 128 x 32 + 512 x 112
        // (whole warps: see elect_one; the next block's barrier is asked for before the current block is worked on, since a wait
        // takes some 200 cycles even when the phase is long over)
        if (warp == 0) {
            int s = 0, parity = 1;
            bool ready = true, going = true;
            for (int t = first; t < end && going; t += pairs) {
                const Tile at = tile_at(t, tiles_m, tiles_n);
                const int row = at.m * kPairRows + rank * 128;
                const int feat = at.n * kFeat + rank * (kSwiglu ? 32 : 64);
                for (int kb = 0; kb < kbn; ++kb, ++issued) {
                    if (!ready) ready = mbar_spin(empty + s, parity);
                    if (!__all_sync(0xffffffffu, ready)) { if (lane == 0) report(a.error, 1, kb); failed = 1; going = false; break; }
                    const int s1 = s + 1 == kPairStages ? 0 : s + 1, parity1 = s1 == 0 ? parity ^ 1 : parity;
                    ready = issued + 1 < kPairStages || mbar_test(empty + s1, parity1);
                    if (elect_one()) {
                        uint8_t* x = base + (size_t)s * kPairStage;
                        uint8_t* w = x + 128 * kBK;
                        if (rank == 0) mbar_expect_tx(full + s, 2 * kPairStage);
                        const uint32_t bar = full0 + s * 8;
                        const int k = (kb0 + kb) * kBK;
                        tma_load_2d_pair(x, &map_x, bar, k, row);
#pragma unroll
                        for (int h = 0; h < 2; ++h) {      // the features of this CTA in either half of the columns
                            if (kSwiglu) {
                                tma_load_2d_pair(w + 64 * h * kBK, &map_w0, bar, k, feat + 64 * h);
                                tma_load_2d_pair(w + (64 * h + 32) * kBK, &map_w1, bar, k, feat + 64 * h);
                            } else {
                                tma_load_2d_pair(w + 64 * h * kBK, &map_w0, bar, k, feat + 128 * h);
                            }
                        }
                    }
                    s = s1; parity = parity1;
                }
            }
        } else if (warp != 2 && rank == 0) {
            // Two warps issue the products, one for either half of the columns: what a warp has to do for a block besides (two barriers,
            // a fence, descriptors, the commit) takes it some 400 cycles.
            const int half = warp >> 1;
            constexpr uint32_t idesc = f8_idesc(256, kHalf);
            const uint64_t desc0 = umma_desc(base);
            int s = 0, parity = 0;
#pragma unroll 1
            for (int n = 0; n < total; ++n) {
                const int acc = (n & 1) * 2 + half;
                bool fine = mbar_spin(full + s, parity);
                if (n >= 2) fine = mbar_spin(acc_empty + acc, ((n >> 1) - 1) & 1) && fine;
                if (!__all_sync(0xffffffffu, fine)) { if (lane == 0) report(a.error, 2, n); failed = 1; break; }
                const uint64_t xdesc = desc0 + (uint64_t)(s * (kPairStage >> 4)), wdesc = xdesc + ((128 + 64 * half) * kBK >> 4);
                const uint32_t d = tmem + (n & 1) * kCols + half * kHalf;
                fence_after_sync();
                if (elect_one()) {
#pragma unroll
                    for (int k = 0; k < kBK / 32; ++k) umma_f8_pair(d, xdesc + 2 * k, wdesc + 2 * k, idesc, k != 0);
                    umma_commit_pair(acc_full + acc, 3 << leader);
                }
                __syncwarp();
                if (++s == kPairStages) { s = 0; parity ^= 1; }
            }
        } else if (warp == 2) {
            // Watches the accumulators: hands the block's stage back to the producer of its CTA and wakes the warps that add, by a
            // barrier that costs them nothing while they wait: a dozen warps that ask the same mbarrier make each answer, also the one
            // to the warp that issues the products, some 300 cycles late.  (It is never more than
            // the accumulators ahead of them.)  After a wait that gave up it meets them at that barrier instead, block by block, until
            // their loops have ended by count.
            bool fine = true;
            for (int n = 0, s = 0; n < total; ++n) {
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const int acc = (n & 1) * 2 + half;
                    if (fine) {
                        fine = __all_sync(0xffffffffu, mbar_spin(acc_full + acc, (n >> 1) & 1));
                        if (!fine) { if (lane == 0) report(a.error, 4, n); failed = 1; }
                    }
                    fence_after_sync();
                    fence_before_sync();
                    if (fine) wake<kHalfAdders + 32>(kWakeAdders + acc); else sleep_until_woken<kHalfAdders + 32>(kWakeAdders + acc);
                    if (lane == 0) mbar_arrive(empty + s);
                }
                s = s + 1 == kPairStages ? 0 : s + 1;
            }
        }
        __syncwarp();
        if constexpr (kParts > 1) { cluster_arrive(); cluster_wait(); cluster_arrive(); cluster_wait(); }      // as the warps that add
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 112;");
        const int group = (warp - 4) >> 2, quarter = warp & 3, in_tile = quarter * 32 + lane;
        const uint32_t from = tmem + ((uint32_t)(quarter * 32) << 16) + group * 64;
        const uint32_t release0 = peer_addr(smem_u32(acc_empty + (group >> 1)), leader);
        int n = 0;                                         // blocks so far
        // A block's scales are asked for two blocks ahead, into one of two sets of registers
        struct Scales { float x, w, u; };
        Scales even, odd;
        const float *sx = nullptr, *sw = nullptr, *su = nullptr;          // of the block that is asked for next
        auto fetch = [&](Scales& f) {
            f.x = *sx;
            f.w = *sw;
            sx += a.sx_block;
            sw += a.sw_block;
            if (kSwiglu) { f.u = *su; su += a.sw_block; }
        };
        auto open = [&](int t) {                           // the scales' places of a tile, and its first two blocks' on their way
            const Tile at = tile_at(t, tiles_m, tiles_n);
            sx = a.sx + (long)min(at.m * kPairRows + rank * 128 + in_tile, a.M - 1) * a.sx_row + kb0 * a.sx_block;
            sw = a.sw0 + (kSwiglu ? at.n : min(2 * at.n + (group >> 1), (a.N - 1) / kBK)) * a.sw_row + kb0 * a.sw_block;
            if (kSwiglu) su = a.sw1 + at.n * a.sw_row + kb0 * a.sw_block;
            fetch(even);
            if (kbn > 1) fetch(odd);
        };
        open(first);
        for (int t = first; t < end; t += pairs) {
            float sum[64];
#pragma unroll
            for (int j = 0; j < 64; ++j) sum[j] = 0.f;
            // a block's accumulator, times its scales, joins this thread's sums, 32 columns at a time
            auto add = [&](Scales& f, bool more, auto plain_scales) {
                const uint32_t col = from + (n & 1) * kCols;
                if constexpr (plain_scales.value) {
                    uint32_t d[32];
                    const float s = f.x * f.w, v = kSwiglu ? f.x * f.u : s;
                    if (more) fetch(f);
                    sleep_until_woken<kHalfAdders + 32>(kWakeAdders + (n & 1) * 2 + (group >> 1));
                    fence_after_sync();
                    tmem_ld32(col, d);
#pragma unroll
                    for (int j = 0; j < 32; ++j) sum[j] = fmaf(__uint_as_float(d[j]), s, sum[j]);
                    tmem_ld32(col + 32, d);
                    fence_before_sync();
                    mbar_arrive_at_if(release0 + (n & 1) * 16, lane == 0);
#pragma unroll
                    for (int j = 0; j < 32; ++j) sum[32 + j] = fmaf(__uint_as_float(d[j]), v, sum[32 + j]);
                } else {                                   // one scale after the other, so many columns at a time as cost the other form no registers
                    constexpr int kStep = kSwiglu ? 8 : 32;
                    sleep_until_woken<kHalfAdders + 32>(kWakeAdders + (n & 1) * 2 + (group >> 1));
                    fence_after_sync();
#pragma unroll
                    for (int c = 0; c < 64; c += kStep) {
                        float factor, then;
                        Apart(kSwiglu && c >= 32 ? f.u : f.w).of(f.x, factor, then);
                        uint32_t d[kStep];
                        if constexpr (kStep == 32) tmem_ld32(col + c, d);
                        else { tmem_ld8(col + c, d); tmem_ld_wait(); }
#pragma unroll
                        for (int j = 0; j < kStep; ++j) sum[c + j] = fmaf(__uint_as_float(d[j]) * factor, then, sum[c + j]);
                    }
                    fence_before_sync();
                    mbar_arrive_at_if(release0 + (n & 1) * 16, lane == 0);
                    if (more) fetch(f);
                }
                ++n;
            };
            auto block = [&](Scales& f, bool more) {
                if (__builtin_expect(__all_sync(0xffffffffu, plain(f.x * f.w) && (!kSwiglu || plain(f.x * f.u))), 1)) add(f, more, std::true_type{});
                else add(f, more, std::false_type{});
            };
#pragma unroll 1
            for (int kb = 0; kb < kbn; kb += 2) {
                block(even, kb + 2 < kbn);
                if (kb + 1 < kbn) block(odd, kb + 3 < kbn);
            }
            if (t + pairs < end) open(t + pairs);
            if constexpr (kParts > 1) {
                cluster_arrive();                          // everybody's products are done
                cluster_wait();
                const uint32_t mine = smem_u32(base) + (threadIdx.x - 128) * 16;
#pragma unroll
                for (int p = 0; p < kParts; ++p) {
                    const uint32_t to = peer_addr(mine, 2 * p + rank) + part * (kMine / 4 * kAdders * 16);
#pragma unroll
                    for (int j = 0; j < kMine; j += 4)
                        store_peer4(to + j * (kAdders * 4), sum[p * kMine + j], sum[p * kMine + j + 1], sum[p * kMine + j + 2], sum[p * kMine + j + 3]);
                }
                cluster_arrive();                          // everybody's sums are here
                cluster_wait();
#pragma unroll
                for (int j = 0; j < kMine; ++j) sum[j] = 0.f;
#pragma unroll
                for (int p = 0; p < kParts; ++p)
#pragma unroll
                    for (int j = 0; j < kMine; j += 4) {
                        float v[4];
                        load_shared4(mine + (p * kMine + j) * (kAdders * 4), v);
#pragma unroll
                        for (int e = 0; e < 4; ++e) sum[j + e] += v[e];
                    }
            }
            const Tile at = tile_at(t, tiles_m, tiles_n);
            const long m = (long)at.m * kPairRows + rank * 128 + in_tile;
            if constexpr (kSwiglu) {
                const int f0 = at.n * kFeat + group * 32;  // this thread's features
                uint32_t top = 0;
#pragma unroll
                for (int j = 0; j < 32; ++j) {
                    sum[j] = f0 + j < a.N ? silu_of(sum[j], 0.125f * a.act_scale) * sum[32 + j] : 0.f;
                    top = max(top, magnitude(sum[j]));
                }
                tops[group][in_tile] = top;
                asm volatile("bar.sync 1, 512;" ::: "memory");
#pragma unroll
                for (int g = 0; g < kPairGroups; ++g) top = max(top, tops[g][in_tile]);
                const float scale = fp8_scale(top);
                const Fp8Divide by(scale);
                asm volatile("bar.sync 1, 512;" ::: "memory");
                if (m < a.M) {
                    uint8_t* q = a.q + m * a.ldq + f0;
                    uint32_t w[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) w[e] = fp8_quad(by(sum[4 * e]), by(sum[4 * e + 1]), by(sum[4 * e + 2]), by(sum[4 * e + 3]));
                    if (f0 + 32 <= a.N && ((uintptr_t)q & 31) == 0) {
                        store32(q, w);
                    } else {                               // rows are filled up to 16 bytes
                        if (f0 < a.N) *reinterpret_cast<uint4*>(q) = make_uint4(w[0], w[1], w[2], w[3]);
                        if (f0 + 16 < a.N) *reinterpret_cast<uint4*>(q + 16) = make_uint4(w[4], w[5], w[6], w[7]);
                    }
                    if (group == 0) a.qs[m * a.qs_row + at.n * a.qs_block] = scale;
                }
            } else {
                const int n0 = at.n * kFeat + group * 64 + (kParts > 1 ? part * kMine : 0), live = a.N - n0;
                if (a.bias != nullptr) {
                    const float* bias = a.bias + n0;
#pragma unroll
                    for (int j = 0; j < kMine; ++j) sum[j] += bias[min(j, live - 1)];
                }
#pragma unroll
                for (int j = 0; j < kMine; ++j) sum[j] *= a.out_scale;
                const int size = a.out_f32 ? 4 : 2;
                uint8_t* out = (uint8_t*)a.out + ((size_t)m * a.ldo + n0) * size;
                if constexpr (!kRagged) {
                    // whole sectors of 32 bytes: a lane is a row, and every store of a warp touches 32 lines
                    if (m < a.M) {
                        if (a.out_f32) {
#pragma unroll
                            for (int j = 0; j < kMine; j += 8) {
                                uint32_t w[8];
#pragma unroll
                                for (int e = 0; e < 8; ++e) w[e] = __float_as_uint(sum[j + e]);
                                if (j < live) store32(out + 4 * j, w);
                            }
                        } else {
#pragma unroll
                            for (int j = 0; j < kMine; j += 16) {
                                uint32_t w[8];
                                __nv_bfloat162* b = reinterpret_cast<__nv_bfloat162*>(w);
#pragma unroll
                                for (int e = 0; e < 8; ++e) b[e] = __floats2bfloat162_rn(sum[j + 2 * e], sum[j + 2 * e + 1]);
                                if (j < live) store32(out + 2 * j, w);
                            }
                        }
                    }
                } else {
                    // 16 features of a warp's 32 rows at a time change places in shared memory, so that a store takes neighbours of two rows (one value of 32 rows each: 42 us instead of 12 for 512 rows
                    // of 1,003).
                    float* turn = reinterpret_cast<float*>(base + (size_t)kPairStages * kPairStage) + (warp - 4) * 512;
                    const int j = lane & 15, first = lane >> 4, rows = (int)min(32L, a.M - (m - lane));
#pragma unroll
                    for (int c = 0; c < kMine; c += 16) {
                        __syncwarp();
#pragma unroll
                        for (int e = 0; e < 16; ++e) turn[lane * 16 + (e ^ j)] = sum[c + e];
                        __syncwarp();
                        if (c + j < live) {
                            uint8_t* to = out + ((long)(first - lane) * a.ldo + c + j) * size;
#pragma unroll 1
                            for (int r = first; r < rows; r += 2, to += 2 * a.ldo * size) {
                                const float v = turn[r * 16 + (j ^ (r & 15))];
                                if (a.out_f32) *reinterpret_cast<float*>(to) = v;
                                else *reinterpret_cast<__nv_bfloat16*>(to) = __float2bfloat16_rn(v);
                            }
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
