// Products of 8-bit rows with an 8-bit weight on the 5th-generation tensor cores (e4m3 operands, a float32 scale per row and
// 128 columns of x and per 128 features and 128 columns of W; lb200/fp8.cuh):
//
//   y[m, n] = sum_b  sx[m, b] sw[n / 128, b]  sum_{k in block b} qx[m, k] qw[n, k]
//   plain   : out = round((y + bias) * out_scale)                      bfloat16 or float32
//   swiglu  : h = silu(act_scale * y_gate) * y_up, then 8-bit rows of h: a scale per row and 128 features
//
// The inner sums run on the tensor core, one block of 128 columns at a time into a fresh accumulator in tensor memory; the
// scales differ from block to block, so each block's accumulator is read back and joined into 32-bit registers, times its
// scales, while the tensor core works on the next block.
//
//   warp 0    one thread issues the TMA loads (128-byte swizzle, zeros outside the matrices) into a ring of stages: a block
//             of 128 columns of 128 features of W (swiglu: of 128 gate and 128 up features) and of the tile's rows of x
//   warps 1, 10  issue tcgen05.mma (one thread; kind::f8f6f4, K 32: four per block), block by block in turn, since what a warp has
//             to do for a block besides takes some 400 cycles; warp 1 allocates tensor memory
//   warps 2-9 two warpgroups: read a block's accumulator, multiply and add; for swiglu one holds the gate, one the up
//             features, otherwise each half of the columns
// Two ways round:
//   few rows (kSwap): 128 features are the M side of the instruction, up to 64 rows, padded to 16, 32 or 64, its N side:
//             bound by reading W once.  A thread is a feature; the scales of the rows lie ready in shared memory.
//   tiles     128 rows are the M side, 128 features (swiglu: 256) the N side.  A thread is a row.
// K split: where there are few tiles, up to 8 CTAs of a cluster take a range of blocks each and the sums meet in distributed
// shared memory: each CTA owns an equal share of the tile's rows, gets every CTA's sums for them by remote stores, and adds
// them in rank order, so that the result does not depend on timing.  There a warp takes a row, a lane 4 neighbouring features:
// stores are whole, and the largest magnitude of a row's 128 features takes one reduction (few rows without SwiGLU: a thread takes a feature and four rows).
//
// Every wait on an mbarrier is bounded; one that gives up records itself in `error`, all roles run out of their own bounded
// waits, every thread still meets the cluster barriers, tensor memory is freed and the kernel returns.
#include "lb200/fp8_linear.cuh"
#include "lb200/fp8_pair.cuh"
using namespace lb200;
using namespace lb200::fp8;

namespace {
constexpr int kFeat = 128;
constexpr uint32_t kWBytes = kFeat * kBK;
constexpr int kSumThreads = 256;                          // warps 2-9
constexpr int kThreads = 96 + kSumThreads;
constexpr int kMaxStages = 8, kMaxSplit = 8;

// kSwap: NR rows on the N side; else 128 rows on the M side (NR = 128).
template <bool kSwap, int NR, bool kSwiglu>
struct Form {
    static constexpr int kXRows = kSwap ? NR : 128;
    static constexpr uint32_t kXBytes = kXRows * kBK;
    static constexpr uint32_t kStage = (kSwiglu ? 2 : 1) * kWBytes + kXBytes;
    static constexpr int kCols = kSwap ? (kSwiglu ? 2 * NR : NR) : (kSwiglu ? 256 : 128);   // accumulator columns of a block
    static constexpr bool kTwoPerSm = kSwap && NR <= 32;   // CTAs on an SM: where 80 registers hold sums, columns and scales
    static constexpr int kAccs = kCols <= (kTwoPerSm ? 64 : 128) ? 4 : 2;      // accumulators in tensor memory
    static constexpr uint32_t kTmem = kCols * kAccs < 32 ? 32 : kCols * kAccs;
    static constexpr int kOutCols = kSwiglu ? 256 : 128;                       // features of a tile, gate and up counted
    static constexpr bool kQuads = kSwap && !kSwiglu;                          // the sums of four rows and a feature lie together
    static constexpr int kPitch = kOutCols + (kQuads ? 0 : 4);                 // floats of a row of sums (else rows start in different banks)
    static constexpr int kShareOf = kQuads ? 4 : 1;                            // a CTA owns a multiple of so many rows
    static constexpr int kMine = kSwap ? (kSwiglu ? NR : NR / 2) : (kSwiglu ? 128 : 64);   // sums of a thread
    static constexpr bool kOver = !kSwap || (NR == 64 && kSwiglu);             // the sums land over the ring
};

template <bool kSwap, int NR, bool kSwiglu>
__global__ void __launch_bounds__(kThreads, Form<kSwap, NR, kSwiglu>::kTwoPerSm ? 2 : 1)
fp8_linear_kernel(const __grid_constant__ CUtensorMap map_w0, const __grid_constant__ CUtensorMap map_w1,
                  const __grid_constant__ CUtensorMap map_x, Args a) {
    typedef Form<kSwap, NR, kSwiglu> F;
    constexpr uint32_t kStage = F::kStage;
    constexpr int kAccs = F::kAccs, kMine = F::kMine;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* base = reinterpret_cast<uint8_t*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    __shared__ __align__(8) uint64_t full[kMaxStages], empty[kMaxStages], acc_full[kAccs], acc_empty[kAccs];
    __shared__ uint32_t tmem_slot;
    __shared__ volatile int failed, odd;                  // odd: some of this CTA's pairs of scales have no normal product
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int split = a.split, rank = split > 1 ? (int)cluster_rank() : 0;
    const int tile = blockIdx.x / split, tile_m = tile / a.tiles_n, tile_n = tile - tile_m * a.tiles_n;
    const int m0 = tile_m * F::kXRows, n0 = tile_n * kFeat, rows = min(F::kXRows, a.M - m0);
    const int blocks = (a.K + kBK - 1) / kBK;
    const int kb0 = (int)((long)blocks * rank / split), kbn = (int)((long)blocks * (rank + 1) / split) - kb0;
    const int stages = a.stages, first = min(stages, kbn);
    const int share = ((rows + split - 1) / split + F::kShareOf - 1) / F::kShareOf * F::kShareOf;      // rows that a CTA of the cluster owns
    // The sums land here: [source CTA][row of the share][feature] (kQuads: [source CTA][four rows][feature][row]).  Few sums: behind
    // the ring (a peer may be done while this CTA still loads); many: over it, once the whole cluster has left it.  Few rows: then the
    // scales, [block][gate, up][row].
    float* recv = reinterpret_cast<float*>(F::kOver ? base : base + (size_t)stages * kStage);
    float* table = reinterpret_cast<float*>(base + (size_t)stages * kStage) + (F::kOver ? 0 : (size_t)(kSwiglu && split == 1 ? NR : split * share) * F::kPitch);
    const uint32_t table_at = smem_u32(table);
    auto load_w = [&](int s, int i) {
        uint8_t* w = base + (size_t)s * kStage;
        mbar_expect_tx(full + s, kStage);
        tma_load_2d(w, &map_w0, full + s, (kb0 + i) * kBK, n0);
        if (kSwiglu) tma_load_2d(w + kWBytes, &map_w1, full + s, (kb0 + i) * kBK, n0);
    };
    auto load_x = [&](int s, int i) {
        tma_load_2d(base + (size_t)s * kStage + (kSwiglu ? 2 : 1) * kWBytes, &map_x, full + s, (kb0 + i) * kBK, m0);
    };
    if (threadIdx.x == 0) {
        for (int s = 0; s < stages; ++s) { mbar_init(full + s, 1); mbar_init(empty + s, 1); }
        for (int s = 0; s < kAccs; ++s) { mbar_init(acc_full + s, 1); mbar_init(acc_empty + s, kSumThreads / 32); }
        failed = odd = 0;
        mbar_fence_init();
        if (a.early) for (int i = 0; i < first; ++i) load_w(i, i);     // its own barriers are ready
    }
    if (threadIdx.x == 64) asm volatile("prefetch.tensormap [%0];" ::"l"(&map_x) : "memory");
    if (warp == 1) tmem_alloc<F::kTmem>(&tmem_slot);
    fence_before_sync();
    __syncthreads();
    fence_after_sync();
    const uint32_t tmem = tmem_slot;
    pdl_trigger();
    if (split > 1) cluster_arrive();                       // "this CTA runs": its shared memory may be written to
    pdl_wait();

    int issued = 0;
    float sum[kMine];
#pragma unroll
    for (int j = 0; j < kMine; ++j) sum[j] = 0.f;
    const int group = (warp - 2) >> 2, quarter = warp & 3;             // warpgroup; the lanes of tensor memory a warp may read
    // (whole warps: see elect_one; the next block's barrier is asked for before the current block is worked on, since a wait takes
    // some 200 cycles even when the phase is long over)
    if (warp == 0) {
        if (elect_one())
            for (int i = 0; i < first; ++i) { if (!a.early) load_w(i, i); load_x(i, i); }
        issued = first;
        int s = 0, parity = 0;
        bool ready = false;
        for (; issued < kbn; ++issued) {
            if (!ready) ready = mbar_spin(empty + s, parity);
            if (!__all_sync(0xffffffffu, ready)) { if (lane == 0) report(a.error, 1, issued); failed = 1; break; }
            const int s1 = s + 1 == stages ? 0 : s + 1, parity1 = s1 == 0 ? parity ^ 1 : parity;
            ready = mbar_test(empty + s1, parity1);
            if (elect_one()) {
                load_w(s, issued);
                load_x(s, issued);
            }
            s = s1; parity = parity1;
        }
    } else if (warp == 1 || warp == 10) {
        constexpr uint32_t idesc = kSwap ? f8_idesc(128, NR) : f8_idesc(128, F::kCols);
        constexpr uint32_t kXAt = ((kSwiglu ? 2 : 1) * kWBytes) >> 4;
        const uint64_t desc0 = umma_desc(base);
        int s = warp == 1 ? 0 : 1, parity = 0;             // (see `launch` on the number of stages)
#pragma unroll 1
        for (int i = s; i < kbn; i += 2, s += 2) {
            while (s >= stages) { s -= stages; parity ^= 1; }
            const int acc = i % kAccs;
            bool fine = mbar_spin(full + s, parity);
            if (i >= kAccs) fine = mbar_spin(acc_empty + acc, (i / kAccs - 1) & 1) && fine;
            if (!__all_sync(0xffffffffu, fine)) { if (lane == 0) report(a.error, 2, i); failed = 1; break; }
            const uint64_t wdesc = desc0 + (uint64_t)(s * (kStage >> 4)), xdesc = wdesc + kXAt;
            const uint32_t d = tmem + acc * F::kCols;
            fence_after_sync();
            if (elect_one()) {
#pragma unroll
                for (int k = 0; k < kBK / 32; ++k) {       // 32 bytes along K: + 2 in the 16-byte address field
                    if (kSwap) {
                        umma_f8(d, wdesc + 2 * k, xdesc + 2 * k, idesc, k != 0);
                        if (kSwiglu) umma_f8(d + NR, wdesc + (kWBytes >> 4) + 2 * k, xdesc + 2 * k, idesc, k != 0);
                    } else {
                        umma_f8(d, xdesc + 2 * k, wdesc + 2 * k, idesc, k != 0);
                    }
                }
                umma_commit(acc_full + acc);
            }
            __syncwarp();
        }
    } else {
        const int t = threadIdx.x - 64;
        const uint32_t from = tmem + ((uint32_t)(quarter * 32) << 16) + group * kMine;
        const float* sw = kSwiglu && group ? a.sw1 : a.sw0;
        const int row = m0 + quarter * 32 + lane;          // tiles: this thread's row
        const float* sx = a.sx + (long)min(row, a.M - 1) * a.sx_row + kb0 * a.sx_block;
        sw += (long)tile_n * a.sw_row + kb0 * a.sw_block;
        float s_next = 0.f;
        if (kSwap) {
            // a thread has one row and every kEvery-th block, four at a time, their loads first.  (Short code: what runs once per CTA
            // comes from memory itself, instruction by instruction.)
            constexpr int kEvery = kSumThreads / NR, kBatch = 4;
            const int m = t % NR;
            const float* px = a.sx + (long)(m0 + min(m, rows - 1)) * a.sx_row;
            const float *p0 = a.sw0 + (long)tile_n * a.sw_row, *p1 = kSwiglu ? a.sw1 + (long)tile_n * a.sw_row : nullptr;
#pragma unroll 1
            for (int i0 = t / NR; i0 < kbn; i0 += kBatch * kEvery) {
                float x[kBatch], w0[kBatch], w1[kBatch];
#pragma unroll
                for (int q = 0; q < kBatch; ++q) {
                    const long kb = kb0 + min(i0 + q * kEvery, kbn - 1);
                    x[q] = px[kb * a.sx_block];
                    w0[q] = p0[kb * a.sw_block];
                    if (kSwiglu) w1[q] = p1[kb * a.sw_block];
                }
#pragma unroll
                for (int q = 0; q < kBatch; ++q) {
                    const int i = min(i0 + q * kEvery, kbn - 1);           // (the last one may be written several times, alike)
                    const float v0 = x[q] * w0[q], v1 = kSwiglu ? x[q] * w1[q] : 1.f;
                    if (!plain(v0) || !plain(v1)) odd = 1;
                    table[(kSwiglu ? 2 : 1) * i * NR + m] = v0;
                    if (kSwiglu) table[(2 * i + 1) * NR + m] = v1;
                }
            }
            asm volatile("bar.sync 1, 256;" ::: "memory");
        } else if (kbn > 0) {
            s_next = sx[0] * sw[0];
        }
        // (a loop of its own where some scales have no normal product: in one loop the rare part costs the other one registers)
        auto add_blocks = [&](auto rows_odd) {
            bool fine = true;
            int slot = 0;
            for (int i = 0; i < kbn; ++i) {
                const int acc = i % kAccs;
                [[maybe_unused]] const float s = s_next;
                if (!kSwap && i + 1 < kbn) s_next = sx[(i + 1) * a.sx_block] * sw[(i + 1) * a.sw_block];
                // one warp asks for the accumulator, the others sleep at the barrier: eight warps that ask make every answer late
                if (warp == 2 && fine) {
                    fine = __all_sync(0xffffffffu, mbar_spin(acc_full + acc, (i / kAccs) & 1));
                    if (!fine) { if (lane == 0) report(a.error, 4, i); failed = 1; }
                }
                asm volatile("bar.sync 1, 256;" ::: "memory");
                if (threadIdx.x == 64) mbar_arrive(empty + slot);             // the block's products have read its stage
                slot = slot + 1 == stages ? 0 : slot + 1;
                fence_after_sync();
                const uint32_t at = from + acc * F::kCols;
                if constexpr (!kSwap) {
                    constexpr int kStep = kMine > 64 ? 16 : 32;        // what the registers hold beside the sums
                    auto add = [&](auto to) {              // `to`: a sum and a block's share of it -> the new sum
#pragma unroll
                        for (int c = 0; c < kMine; c += kStep) {
                            uint32_t d[kStep];
                            if constexpr (kStep == 32) tmem_ld32(at + c, d);
                            else { tmem_ld16(at + c, d); tmem_ld_wait(); }
                            if (c + kStep == kMine) {
                                fence_before_sync();
                                if (lane == 0) mbar_arrive(acc_empty + acc);
                            }
#pragma unroll
                            for (int j = 0; j < kStep; ++j) sum[c + j] = to(d[j], sum[c + j]);
                        }
                    };
                    if (__builtin_expect(__all_sync(0xffffffffu, plain(s)), 1)) {
                        add([&](uint32_t d, float sum) { return fmaf(__uint_as_float(d), s, sum); });
                    } else {
                        float factor, then;
                        Apart(sw[i * a.sw_block]).of(sx[i * a.sx_block], factor, then);
                        add([&](uint32_t d, float sum) { return fmaf(__uint_as_float(d) * factor, then, sum); });
                    }
                } else if constexpr (rows_odd.value) {
                    const uint32_t tab = table_at + (kSwiglu ? (2 * i + group) * NR : i * NR + group * kMine) * 4;
                    const int r0 = m0 + (kSwiglu ? 0 : group * kMine);
#pragma unroll
                    for (int c = 0; c < kMine; c += 8) {
                        uint32_t d[8];
                        float f[8];
                        tmem_ld8(at + c, d);
                        load_shared4(tab + 4 * c, f);
                        load_shared4(tab + 4 * c + 16, f + 4);
                        tmem_ld_wait();
                        bool joined = true;                // (the same for the whole warp)
#pragma unroll
                        for (int j = 0; j < 8; ++j) joined = joined && plain(f[j]);
                        if (!joined) {                     // (sums of a block of zeros are zero, whatever the scales)
                            bool zero = true;
#pragma unroll
                            for (int j = 0; j < 8; ++j) zero = zero && (plain(f[j]) || (d[j] << 1 == 0 && magnitude(f[j]) < 0x7f800000u));
                            joined = __all_sync(0xffffffffu, zero);
                        }
                        if (joined) {
#pragma unroll
                            for (int j = 0; j < 8; ++j) sum[c + j] = fmaf(__uint_as_float(d[j]), f[j], sum[c + j]);
                        } else {
                            const Apart by(sw[i * a.sw_block]);
#pragma unroll
                            for (int j = 0; j < 8; ++j) {
                                float factor;
                                by.of(a.sx[(long)min(r0 + c + j, a.M - 1) * a.sx_row + (kb0 + i) * a.sx_block], factor, f[j]);
                                sum[c + j] = fmaf(__uint_as_float(d[j]) * factor, f[j], sum[c + j]);
                            }
                        }
                    }
                    fence_before_sync();
                    if (lane == 0) mbar_arrive(acc_empty + acc);
                } else {                                   // all columns at once: one wait for tensor memory a block
                    uint32_t d[kMine];
                    if constexpr (kMine == 8) tmem_ld8(at, d);
                    else if constexpr (kMine == 16) tmem_ld16(at, d);
                    else if constexpr (kMine == 32) tmem_ld32_async(at, d);
                    else tmem_ld64(at, d);
                    // the rows' scales, where there are registers for them while the columns are on their way
                    const uint32_t tab = table_at + (kSwiglu ? (2 * i + group) * NR : i * NR + group * kMine) * 4;
                    constexpr int kAhead = kMine <= 16 ? kMine : F::kTwoPerSm ? 8 : kMine == 32 ? 32 : 16;
                    float f[kAhead];
#pragma unroll
                    for (int j = 0; j < kAhead; j += 4) load_shared4(tab + 4 * j, f + j);
                    tmem_ld_wait();
                    fence_before_sync();
                    if (lane == 0) mbar_arrive(acc_empty + acc);
#pragma unroll
                    for (int c = 0; c < kMine; c += kAhead) {
#pragma unroll
                        for (int j = 0; j < kAhead; ++j) sum[c + j] = fmaf(__uint_as_float(d[c + j]), f[j], sum[c + j]);
                        if (c + kAhead < kMine) {
#pragma unroll
                            for (int j = 0; j < kAhead; j += 4) load_shared4(tab + 4 * (c + kAhead + j), f + j);
                        }
                    }
                }
            }
        };
        if (kSwap && __builtin_expect(odd, 0)) add_blocks(std::true_type{}); else add_blocks(std::false_type{});
    }
    // ---- the sums meet at the rows' owners
    fence_before_sync();
    if (split > 1) {
        cluster_wait();
        if (F::kOver) { cluster_arrive(); cluster_wait(); }    // every CTA of the cluster has left its ring
    } else if (F::kOver) {
        __syncthreads();
    }
    if (warp >= 2 && warp < 10) {
        const int feat = quarter * 32 + lane;
        if constexpr (kSwap && kSwiglu) {
            uint32_t at = smem_u32(recv) + (uint32_t)(rank * share * F::kPitch + group * 128 + feat) * 4;
            if (split == 1) {                              // there is room for all NR rows
#pragma unroll
                for (int j = 0; j < kMine; ++j) asm volatile("st.shared.f32 [%0], %1;" ::"r"(at + j * F::kPitch * 4), "f"(sum[j]) : "memory");
            } else {
                int owner = 0, r = 0;
                uint32_t to = peer_addr(at, 0);
#pragma unroll
                for (int j = 0; j < kMine; ++j) {
                    if (j < rows) store_peer(to, sum[j]);
                    to += F::kPitch * 4;
                    if (++r == share) { r = 0; to = peer_addr(at, min(++owner, split - 1)); }
                }
            }
        } else if constexpr (kSwap) {
            const int j0 = group * kMine, col = feat;
            int owner = j0 / share, r = j0 - owner * share;
#pragma unroll
            for (int j = 0; j < kMine; j += 4) {
                if (j0 + j < rows) {
                    const uint32_t at = smem_u32(recv) + (uint32_t)((rank * share + r) * F::kPitch + 4 * col) * 4;
                    store_peer4(split > 1 ? peer_addr(at, owner) : at, sum[j], sum[j + 1], sum[j + 2], sum[j + 3]);
                }
                r += 4;
                if (r == share) { r = 0; ++owner; }
            }
        } else if (feat < rows) {
            const int owner = feat / share, r = feat - owner * share;
            const uint32_t at = peer_addr(smem_u32(recv) + (uint32_t)((rank * share + r) * F::kPitch + group * kMine) * 4, owner);
#pragma unroll
            for (int j = 0; j < kMine; j += 4) store_peer4(at + 4 * j, sum[j], sum[j + 1], sum[j + 2], sum[j + 3]);
        }
    }
    if (split > 1) { cluster_arrive(); cluster_wait(); }
    else __syncthreads();
    if (F::kQuads && warp >= 2 && warp < 10) {
        // a thread takes a feature and four rows: the sums in rank order; a warp's stores lie side by side
        const int f = (threadIdx.x - 64) & 127, half = (threadIdx.x - 64) >> 7, n = n0 + f, r1 = min(share, rows - rank * share);
        const float bias = a.bias != nullptr && n < a.N ? a.bias[n] : 0.f;
#pragma unroll 1
        for (int r = 4 * half; r < r1; r += 8) {           // the same for all 128 threads of a half
            float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int src = 0; src < kMaxSplit; ++src)
                if (src < split) {
                    const float4 w = *reinterpret_cast<const float4*>(recv + (size_t)(src * share + r) * F::kPitch + 4 * f);
                    v[0] += w.x; v[1] += w.y; v[2] += w.z; v[3] += w.w;
                }
            const long m = m0 + rank * share + r;
            const int live = r1 - r;
            if (n < a.N) {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (j < live) {
                        const float o = (v[j] + bias) * a.out_scale;
                        if (a.out_f32) ((float*)a.out)[(m + j) * a.ldo + n] = o;
                        else ((__nv_bfloat16*)a.out)[(m + j) * a.ldo + n] = __float2bfloat16_rn(o);
                    }
            }
        }
    }
    if (!F::kQuads && warp >= 2 && warp < 10) {
        const int col = lane * 4, n = n0 + col;
        float b[4] = {0.f, 0.f, 0.f, 0.f};
        if (!kSwiglu && a.bias != nullptr) {
#pragma unroll
            for (int e = 0; e < 4; ++e) if (n + e < a.N) b[e] = a.bias[n + e];
        }
        const int r1 = min(share, rows - rank * share);
        // A row at a time in a short loop: its instructions stay where they are fetched from.  (Four rows at a time, twice as many
        // instructions in flight, took 1,250 cycles a row.)
#pragma unroll 1
        for (int r = warp - 2; r < r1; r += kSumThreads / 32) {
            float v[4] = {0.f, 0.f, 0.f, 0.f}, u[4] = {0.f, 0.f, 0.f, 0.f};
            uint32_t at = smem_u32(recv) + (uint32_t)(r * F::kPitch + col) * 4;
#pragma unroll 1
            for (int src = 0; src < split; ++src, at += share * F::kPitch * 4) {
                float w[4];
                load_shared4(at, w);
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] += w[e];
                if constexpr (kSwiglu) {
                    load_shared4(at + 512, w);
#pragma unroll
                    for (int e = 0; e < 4; ++e) u[e] += w[e];
                }
            }
            const long m = m0 + rank * share + r;
            if constexpr (kSwiglu) {
                uint32_t top = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    v[e] = n + e < a.N ? silu_of(v[e], 0.125f * a.act_scale) * u[e] : 0.f;
                    top = max(top, magnitude(v[e]));
                }
                const float scale = fp8_scale(__reduce_max_sync(0xffffffffu, top));
                const Fp8Divide by(scale);
                // rows are filled up to 16 bytes: four bytes that begin inside the row end inside its storage
                if (n < a.N) *reinterpret_cast<uint32_t*>(a.q + m * a.ldq + n) = fp8_quad(by(v[0]), by(v[1]), by(v[2]), by(v[3]));
                if (lane == 0) a.qs[m * a.qs_row + tile_n * a.qs_block] = scale;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = (v[e] + b[e]) * a.out_scale;
                const long to = m * a.ldo + n;
                if (a.out_f32) {
                    float* p = (float*)a.out + to;
                    if (n + 4 <= a.N && ((uintptr_t)p & 15) == 0) *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
                    else for (int e = 0; e < 4; ++e) if (n + e < a.N) p[e] = v[e];
                } else {
                    __nv_bfloat16* p = (__nv_bfloat16*)a.out + to;
                    if (n + 4 <= a.N && ((uintptr_t)p & 7) == 0) {
                        uint2 w;
                        reinterpret_cast<__nv_bfloat162*>(&w)[0] = __floats2bfloat162_rn(v[0], v[1]);
                        reinterpret_cast<__nv_bfloat162*>(&w)[1] = __floats2bfloat162_rn(v[2], v[3]);
                        *reinterpret_cast<uint2*>(p) = w;
                    } else for (int e = 0; e < 4; ++e) if (n + e < a.N) p[e] = __float2bfloat16_rn(v[e]);
                }
            }
        }
    }
    __syncthreads();
    if (failed && threadIdx.x == 0)                        // copies still under way land before the CTA leaves
        for (int i = max(0, issued - stages); i < issued; ++i) mbar_wait(full + i % stages, (i / stages) & 1);
    if (warp == 1) tmem_free<F::kTmem>(tmem);
}

struct Operands {
    const void *x, *w0, *w1;
    long ldx, ldw;                                        // row strides, bytes
};

template <bool kSwap, int NR, bool kSwiglu>
int launch(const Operands& o, Args a, int sms, cudaStream_t s) {
    typedef Form<kSwap, NR, kSwiglu> F;
    const int blocks = (a.K + kBK - 1) / kBK, per = (blocks + a.split - 1) / a.split;
    a.tiles_n = (a.N + kFeat - 1) / kFeat;
    const long tiles = (long)((a.M + F::kXRows - 1) / F::kXRows) * a.tiles_n;
    if (tiles * a.split > 0x7fffffffL) return kTooLarge;
    // Shared memory: a ring as deep as the CTA's share of an SM allows; few rows: beside it the sums that land and the scales
    const int rows = kSwap && a.M < NR ? a.M : F::kXRows, share = ((rows + a.split - 1) / a.split + F::kShareOf - 1) / F::kShareOf * F::kShareOf;
    const size_t side = kSwap ? ((F::kOver ? 0 : (size_t)(kSwiglu && a.split == 1 ? NR : a.split * share) * F::kPitch) + (size_t)per * NR * (kSwiglu ? 2 : 1)) * 4 : 0;
    const size_t sums = (size_t)(kSwap && kSwiglu && a.split == 1 ? NR : a.split * share) * F::kPitch * 4;
    const size_t budget = (F::kTwoPerSm && tiles * a.split > sms ? 112 : 224) * 1024;
    if (side + 1024 + F::kStage > budget) return kTooLarge;
    int stages = (int)((budget - 1024 - side) / F::kStage);
    stages = stages < kMaxStages ? stages : kMaxStages;
    // A ring that goes round has an even number of stages: each of the two warps that issue then meets every use of its stages.
    // (A warp that met every second use only could ask for a phase while the one before is not over: the answer would be yes.)
    stages = stages >= per ? per : stages & ~1;
    if (stages < 1) return kTooLarge;
    a.stages = stages;
    size_t smem = 1024 + a.stages * (size_t)F::kStage + side;
    if (F::kOver && smem < 1024 + sums + side) smem = 1024 + sums + side;
    CUtensorMap map_w0, map_w1, map_x;
    int rc = make_byte_map(&map_w0, o.w0, a.N, a.K, o.ldw, kFeat);
    if (rc == 0) { if (kSwiglu) rc = make_byte_map(&map_w1, o.w1, a.N, a.K, o.ldw, kFeat); else map_w1 = map_w0; }
    if (rc == 0) rc = make_byte_map(&map_x, o.x, a.M, a.K, o.ldx, F::kXRows);
    if (rc != 0) return rc;
    static SharedLimits limits;
    rc = ensure_dynamic_smem(fp8_linear_kernel<kSwap, NR, kSwiglu>, smem, limits);
    if (rc != 0) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(tiles * a.split)); cfg.blockDim = dim3(kThreads); cfg.dynamicSmemBytes = smem; cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)a.split; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr; cfg.numAttrs = a.split > 1 ? 2 : 1;
    rc = (int)cudaLaunchKernelEx(&cfg, fp8_linear_kernel<kSwap, NR, kSwiglu>, map_w0, map_w1, map_x, a);
    return rc != 0 ? rc : launch_status();
}

// CTAs that share a tile's blocks of K: doubled as long as the GPU holds them at once, `per_sm` on an SM, and `left` blocks remain
// to each.  Few rows, us for a split of 1 / 2 / 4 / 8: down 3,072 x 12,288 (24 tiles, 96 blocks) at 1 row 22 / 13 / 11 / 10, at 64 rows
// 33 / 19 / 13 / 19 (one CTA on an SM); gate|up 12,288 x 3,072 (96 tiles, 24 blocks) at 64 rows 22 / 30 / 37 / 81, 3,072 x 1,280 (24
// tiles, 10 blocks) at 1 row 5.5 / 4.5 / 4.7 / 5.2.  With one CTA on an SM not every SM can be in a larger cluster (tiles of 128 rows,
// 1,024 x 2,048: 8 tiles x 8 7.8 us, x 4 8.2; 16 tiles x 8 12.6, x 4 8.2; 32 tiles x 4 9.4, x 2 10.1; 64 tiles x 2 11.4, x 1 13.4).
int default_split(long tiles, int blocks, int sms, int per_sm, int left) {
    int split = 1;
    while (split < kMaxSplit) {
        // with one CTA on an SM five follow four: three clusters of five in a GPC of 16 to 20 SMs, two of eight (down 3,072 x 12,288,
        // 64 rows: 4 12.9, 5 12.1, 8 18.0; 1,280 x 3,072: 4 5.5, 5 5.2, 8 5.6)
        const int next = per_sm == 1 && split == 4 ? 5 : 2 * split;
        const long held = per_sm > 1 ? (long)sms * per_sm : split == 1 ? sms : split == 2 ? sms * 13 / 15 : sms * 5 / 6;
        if (blocks / next < left || tiles * next > held || split == 5) break;
        split = next;
    }
    return split;
}

enum : int { kAuto = 0, kRows = 1, kTiles = 2, kPair = 3 };

template <bool kSwiglu, bool kRagged, int kParts>
struct PairLaunch {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2] = {};
    int rc;
    PairLaunch(int pairs, cudaStream_t s) {
        constexpr size_t smem = pair_smem(kRagged);
        static SharedLimits limits;
        rc = ensure_dynamic_smem(fp8_pair_kernel<kSwiglu, kRagged, kParts>, smem, limits);
        cfg.gridDim = dim3((unsigned)(2 * pairs)); cfg.blockDim = dim3(kPairThreads); cfg.dynamicSmemBytes = smem; cfg.stream = s;
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        attr[1].id = cudaLaunchAttributeClusterDimension;
        attr[1].val.clusterDim.x = 2 * kParts; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
        cfg.attrs = attr; cfg.numAttrs = 2;
    }
    // (one pair for a tile: tile0 is 0)
    int run(const CUtensorMap& map_w0, const CUtensorMap& map_w1, const CUtensorMap& map_x, Args a, int tile0, int tiles) {
        a.tile0 = tile0; a.tiles = tiles;
        if (rc == 0) rc = (int)cudaLaunchKernelEx(&cfg, fp8_pair_kernel<kSwiglu, kRagged, kParts>, map_w0, map_w1, map_x, a);
        return rc != 0 ? rc : launch_status();
    }
    // clusters that are at work at one time (a group of neighbouring SMs holds whole clusters only: 15 of eight CTAs, 33 of four)
    static int at_once() {
        static AskedOnce asked;
        int device = 0;
        if (cudaGetDevice(&device) != cudaSuccess) device = -1;
        return asked.get(device, [] {
            PairLaunch l(kParts, nullptr);
            int n = 0;
            l.cfg.attrs = l.attr + 1; l.cfg.numAttrs = 1;
            if (l.rc == 0 && cudaOccupancyMaxActiveClusters(&n, fp8_pair_kernel<kSwiglu, kRagged, kParts>, &l.cfg) == cudaSuccess) return n;
            (void)cudaGetLastError();
            return 0;
        });
    }
};

// Tiles left over from whole rounds of all pairs (all tiles, where there are fewer) go to clusters of four or of two pairs, whichever
// are all at work at once, and where enough of a tile's blocks are saved: behind whole rounds the second launch and the sums that
// change places cost what 16 blocks take, on their own some 6.  us with one pair / two / four for a tile: 3,072 x 12,288 256 rows (12
// tiles) 48.8 / 30.5 / 21.2, 512 rows (24) 48.9 / 31.2 / 41.7, 2,048 rows (22 left) 97 / 83 / 93; 2,048 x 8,192 5,000 rows (12 left)
// 101 / 96 / 90; 1,280 x 3,072 512 rows (10) 16.4 / 12.7 / 11.8, 4,096 rows (6 left) 30.6 / 30.8 / 29.7; 1,024 x 2,048 5,000 rows (6
// left) 24.1 / 26.0 / 25.7; 8,192 x 1,024 200 rows (32) 10.1 / 10.5 / 29.  A SwiGLU's tiles are not shared: a row's largest magnitude
// would cross the cluster once more, and gate | up have the most tiles.
template <bool kSwiglu, bool kRagged>
int launch_pair(const Operands& o, const Args& a, int parts, int sms, cudaStream_t s) {
    const long all = (a.M + kPairRows - 1L) / kPairRows * ((a.N + (kSwiglu ? 127L : 255L)) / (kSwiglu ? 128 : 256));
    if (all > 0x3fffffffL) return kTooLarge;
    CUtensorMap map_w0, map_w1, map_x;
    int rc = make_byte_map(&map_w0, o.w0, a.N, a.K, o.ldw, kSwiglu ? 32 : 64);
    if (rc == 0) { if (kSwiglu) rc = make_byte_map(&map_w1, o.w1, a.N, a.K, o.ldw, 32); else map_w1 = map_w0; }
    if (rc == 0) rc = make_byte_map(&map_x, o.x, a.M, a.K, o.ldx, 128);
    if (rc != 0) return rc;
    const int tiles = (int)all, pairs = sms / 2, left = tiles % pairs;
    if constexpr (!kSwiglu) {
        typedef PairLaunch<false, kRagged, 2> Two;
        typedef PairLaunch<false, kRagged, 4> Four;
        const int blocks = (a.K + kBK - 1) / kBK;
        if (left == 0) parts = 1;
        else if (parts == 0) {
            parts = left <= Four::at_once() ? 4 : left <= Two::at_once() ? 2 : 1;
            if (blocks * (parts - 1) / parts < (tiles > pairs ? 16 : 6)) parts = 1;
        }
        if (parts > 1) {
            if (tiles > left) rc = PairLaunch<false, kRagged, 1>(pairs, s).run(map_w0, map_w1, map_x, a, 0, tiles - left);
            if (rc != 0) return rc;
            return parts == 4 ? Four(left * 4, s).run(map_w0, map_w1, map_x, a, tiles - left, tiles)
                              : Two(left * 2, s).run(map_w0, map_w1, map_x, a, tiles - left, tiles);
        }
    }
    return PairLaunch<kSwiglu, kRagged, 1>(tiles < pairs ? tiles : pairs, s).run(map_w0, map_w1, map_x, a, 0, tiles);
}

// Few rows, in tiles of 64 where there are more: as long as all of a product's tiles are at work at once.  us against tiles of 128
// rows and pairs: 1,024 x 2,048 512 rows (64 tiles) 8.0 / 9.7 / 10.7, 1,024 rows (128) 10.0 / 11.4 / 11.2; 1,280 x 3,072 400 rows (70)
// 9.1 / 12.1 / 11.7, 640 rows (100) 12.2 / 13.1 / 12.4; 4,096 x 4,096 256 rows (128) 14.7 / 15.8 / 15.6; 1,280 x 5,120 400 rows (70)
// 11.3 / 16.3 / 13.8, 512 rows (80) 16.9 / 17.0 / 13.8; 3,072 x 12,288 128 rows (48) 19.2 / 19.1 / 21.1, 256 rows (96) 34 / 33 / 21;
// gate|up 3,072 x 1,280 128 rows (48) 9.2 / 13.2 / 10.2, 256 rows (96) 9.9 / 13.8 / 10.2; 12,288 x 3,072 128 rows (192) 36 / 28 / 32.
bool in_rows(long M, long tiles_n, int blocks, bool swiglu, int sms) {
    const long tiles = (M + 63) / 64 * tiles_n;
    return M <= 64 || (swiglu ? tiles <= sms : tiles <= sms / 2 || (tiles <= sms && blocks <= 32));
}
// Pairs, us against tiles of 128 rows: 3,072 x 12,288 200 rows (48 tiles) 21 / 32, 512 rows (96) 31 / 67; 1,280 x 3,072 1,024 rows
// (80) 13.6 / 17.5, 2,048 rows (160) 18 / 34; 1,024 x 2,048 1,536 rows (96) 11.8 / 13.3; 12,288 x 3,072 128 rows (96) 18.5 / 18.3, 256
// rows (192) 19 / 36; 1,003 x 1,431 1,536 rows (96) 12.3 / 11.6; 8,192 x 1,024 256 rows (128) 10.1 / 9.6, 400 rows (256) 11 / 18;
// gate|up 12,288 x 3,072 65 rows 32 / 25, 128 rows 32 / 28, 203 rows 32 / 48.
bool in_pairs(long M, long tiles_n, int blocks, bool swiglu, int sms) {
    if (in_rows(M, tiles_n, blocks, swiglu, sms)) return false;
    const long tiles = (M + 127) / 128 * tiles_n;
    return swiglu ? M > 128 : tiles > sms || blocks >= 16;
}
int sm_count() {
    int device = 0, sms = 148;
    if (cudaGetDevice(&device) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
    return sms;
}

// `form`: kAuto, or the form that is asked for (its low byte) with so many CTAs per tile (pairs: so many pairs; the next byte; 0: by the rule)
template <bool kSwiglu>
int launch_any(const Operands& o, Args a, int form, cudaStream_t s) {
    const int sms = sm_count(), blocks = (a.K + kBK - 1) / kBK;
    const long tiles_n = (a.N + kFeat - 1) / kFeat;
    int split = (form >> 8) & 255;
    if (split > blocks) split = blocks;
    if (split > kMaxSplit) return kBadSize;
    form &= 255;
    const long rows_tiles = (a.M + 63L) / 64 * tiles_n;
    if (form == kRows || (form == kAuto && in_rows(a.M, tiles_n, blocks, kSwiglu, sms))) {
        a.split = split ? split : default_split(rows_tiles, blocks, sms, !kSwiglu && a.M <= 32 ? 2 : 1, kSwiglu ? 4 : 2);
        const int rc = a.M <= 16 ? launch<true, 16, kSwiglu>(o, a, sms, s) : a.M <= 32 ? launch<true, 32, kSwiglu>(o, a, sms, s)
                                                                                     : launch<true, 64, kSwiglu>(o, a, sms, s);
        if (rc != kTooLarge || form != kAuto) return rc;   // a K whose table of scales does not fit goes in tiles
    }
    const long tiles = (a.M + 127L) / 128 * tiles_n;
    if (form == kPair || (form == kAuto && in_pairs(a.M, tiles_n, blocks, kSwiglu, sms))) {
        if constexpr (kSwiglu) return launch_pair<true, false>(o, a, 1, sms, s);
        else {
            const int size = a.out_f32 ? 4 : 2, parts = split;
            const bool ragged = ((uintptr_t)a.out & 31) != 0 || a.ldo * size % 32 != 0 || a.N * (long)size % 32 != 0;
            return ragged ? launch_pair<false, true>(o, a, parts, sms, s) : launch_pair<false, false>(o, a, parts, sms, s);
        }
    }
    a.split = split ? split : default_split(tiles, blocks, sms, 1, 2);
    return launch<false, 128, kSwiglu>(o, a, sms, s);
}
}  // namespace

// x: [M, K] e4m3 bytes, row stride ldx; w: [N, K], row stride ldw (strides multiples of 16, bases on 16 bytes); sx: float32
// scales of x with a stride per row and per block of 128 columns, sw: of w with a stride per 128 features and per block.
// bias: float32 [N] or null.  out: bfloat16 or (out_f32) float32, row stride ldo elements.  early: w and sw are complete and
// stay as they are, whatever the kernels in front on the stream do.  `error`: a device int that is 0 before the call;
// non-zero afterwards: a wait gave up.  form: 0, or a form of the kernel (kRows, kTiles, kPair).
extern "C" int lb_linear_fp8(const void* x, long ldx, const float* sx, long sx_row, long sx_block, const void* w, long ldw,
                             const float* sw, long sw_row, long sw_block, const float* bias, void* out, long ldo, int M, int N,
                             int K, float out_scale, int out_f32, int early, int form, int* error, void* stream) {
    if (M <= 0 || N <= 0) return kOk;
    if (K <= 0 || ldx % 16 || ldw % 16 || (((uintptr_t)x | (uintptr_t)w) & 15)) return kBadSize;
    if (M > kFp8Most || N > kFp8Most || K > kFp8Most) return kTooLarge;
    Args a{};
    a.sx = sx; a.sx_row = sx_row; a.sx_block = sx_block; a.sw0 = sw; a.sw_row = sw_row; a.sw_block = sw_block;
    a.bias = bias; a.out = out; a.ldo = ldo; a.M = M; a.N = N; a.K = K; a.out_scale = out_scale; a.out_f32 = out_f32;
    a.early = early; a.error = error;
    return launch_any<false>(Operands{x, w, nullptr, ldx, ldw}, a, form, (cudaStream_t)stream);
}

// gate and up: [N, K] each, the same row stride, their scales with the same strides.  q: [M, N] bytes, row stride ldq (a
// multiple of 16), qs: its scales with a stride per row and per block.
extern "C" int lb_linear_swiglu_fp8(const void* x, long ldx, const float* sx, long sx_row, long sx_block, const void* gate,
                                    const void* up, long ldw, const float* sgate, const float* sup, long sw_row, long sw_block,
                                    void* q, long ldq, float* qs, long qs_row, long qs_block, int M, int N, int K,
                                    float act_scale, int early, int form, int* error, void* stream) {
    if (M <= 0 || N <= 0) return kOk;
    if (K <= 0 || ldx % 16 || ldw % 16 || ldq % 16 || (((uintptr_t)x | (uintptr_t)gate | (uintptr_t)up | (uintptr_t)q) & 15)) return kBadSize;
    if (M > kFp8Most || N > kFp8Most || K > kFp8Most) return kTooLarge;
    Args a{};
    a.sx = sx; a.sx_row = sx_row; a.sx_block = sx_block; a.sw0 = sgate; a.sw1 = sup; a.sw_row = sw_row; a.sw_block = sw_block;
    a.q = (uint8_t*)q; a.ldq = ldq; a.qs = qs; a.qs_row = qs_row; a.qs_block = qs_block; a.M = M; a.N = N; a.K = K;
    a.act_scale = act_scale; a.early = early; a.error = error;
    return launch_any<true>(Operands{x, gate, up, ldx, ldw}, a, form, (cudaStream_t)stream);
}
