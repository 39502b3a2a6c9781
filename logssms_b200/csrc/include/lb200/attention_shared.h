// Operands of the kernels for attention over a shared prefix (attention_shared.cu), and who belongs to which group.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include "lb200/per_device.h"

namespace lb200 {

struct SharedArgs {
    const void* q; long q_stride;                        // [tokens, Hq, hd], row stride
    const void* k_cache; const void* v_cache;            // [pages, page_size, Hkv, hd]
    void* out;                                           // [tokens, Hq, hd]
    const int* block_table; long bt_stride; int bt_cols; int requests;
    const int* token_req; const int* positions;
    const int* group_start; const int* prefix_lens; int groups;
    float* part_o; float* part_ml;                       // [tokens * Hq][splits][hd] and [..][2] (maximum in log2 units, sum)
    long pages;
    int tokens, Hq, Hkv, hd, page_size;
    int prefix_splits, own_splits;
    float scale_log2;
    int* error;
};

// An SM on which the kernel runs has all of its shared memory as such (and CTAs of another kernel find room beside it), on each
// device by itself.  `carveout` is a static of the calling launcher, one per kernel instantiation.
template <typename Kernel>
inline int whole_carveout(Kernel kernel, DoneOnce& carveout) {
    int device = 0;
    int rc = (int)cudaGetDevice(&device);
    if (rc == 0) rc = carveout.run(device, [&] { return (int)cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared); });
    if (rc != 0) (void)cudaGetLastError();
    return rc;
}

// Two weights of the softmax as bfloat16 operands: their first 8 bits, and what is cut off them, rounded; 2^-16 of a weight is lost.  What
// is cut off is above zero wherever the weight is (2^-20 of the weight is added, which the rounding would hide): an infinite value must
// not meet a zero or a number of the other sign.
__device__ __forceinline__ void split_weights(float x, float y, uint32_t& high, uint32_t& low) {
    const uint32_t a = __float_as_uint(x), b = __float_as_uint(y);
    constexpr float kMore = 1.f + 0x1p-20f;
    high = __byte_perm(a, b, 0x7632);
    const __nv_bfloat162 rest = __floats2bfloat162_rn(fmaf(x, kMore, -__uint_as_float(a & 0xffff0000u)), fmaf(y, kMore, -__uint_as_float(b & 0xffff0000u)));
    low = *reinterpret_cast<const uint32_t*>(&rest);
}

// At most so many tiles of `per_tile` rows hold `rows` rows of `groups` groups, none of them empty.  (No more: a CTA that finds no tile
// to do still has to find room on an SM before the kernel behind may start.)
inline long most_tiles(long rows, long groups, long per_tile) { return (rows + groups * (per_tile - 1)) / per_tile; }

// The tile `target` of the tiles of `per_tile` (token, head) rows that each group's tokens make, group by group: its group's prefix
// and tokens, its first row within the group.  Called by whole warps; false: there is no such tile.
__device__ __forceinline__ bool find_tile(const SharedArgs& a, long target, int rows_per_token, int per_tile, int* prefix, long* row0,
                                          int* first, int* tokens) {
    const int lane = threadIdx.x & 31;
    long before = 0;
    for (int base = 0; base < a.groups; base += 32) {
        const int g = base + lane;
        int t0 = 0, n = 0, p = 0;
        if (g < a.groups) {
            p = a.prefix_lens[g];
            t0 = min(max(a.group_start[g], 0), a.tokens);
            n = max(min(max(a.group_start[g + 1], 0), a.tokens) - t0, 0);
            if (p <= 0) n = 0;
        }
        const long mine = ((long)n * rows_per_token + per_tile - 1) / per_tile;
        long upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long v = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += v;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, before + upto > target);
        if (hit != 0) {
            const int who = __ffs(hit) - 1;
            *prefix = __shfl_sync(0xffffffffu, p, who);
            *row0 = (target - before - __shfl_sync(0xffffffffu, upto - mine, who)) * per_tile;
            *first = __shfl_sync(0xffffffffu, t0, who);
            *tokens = __shfl_sync(0xffffffffu, n, who);
            return true;
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
    }
    return false;
}

// How many keys a token sees: those up to its position.
__device__ __forceinline__ int keys_of(const SharedArgs& a, int t) { return min(a.positions[t], 0x7ffffffe) + 1; }

// The shared prefix of a token's group and the group's first token; false: the token is of no group.  Called by whole warps: up to 32
// groups are looked through at once, more by halves.
__device__ __forceinline__ bool prefix_of(const SharedArgs& a, int t, int* prefix, int* first) {
    if (a.groups <= 32) {
        const int lane = threadIdx.x & 31;
        int from = 0, to = 0, p = 0;
        if (lane < a.groups) { from = a.group_start[lane]; to = a.group_start[lane + 1]; p = a.prefix_lens[lane]; }
        const unsigned hit = __ballot_sync(0xffffffffu, t >= from && t < to);
        if (hit == 0) return false;
        *prefix = max(__shfl_sync(0xffffffffu, p, __ffs(hit) - 1), 0);
        *first = max(__shfl_sync(0xffffffffu, from, __ffs(hit) - 1), 0);
        return true;
    }
    int lo = 0, hi = a.groups;                           // the last group that starts at or in front of t
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (a.group_start[mid] <= t) lo = mid + 1; else hi = mid;
    }
    if (lo == 0 || t >= a.group_start[lo]) return false;
    *prefix = max(a.prefix_lens[lo - 1], 0);
    *first = max(a.group_start[lo - 1], 0);
    return true;
}

}  // namespace lb200
