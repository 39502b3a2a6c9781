// Operands of the kernels for attention over a shared prefix (attention_shared.cu), and who belongs to which group.
#pragma once
#include <cuda_runtime.h>

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

// The tile `target` of the tiles of `per_tile` (token, head) rows that each group's tokens make, group by group: its group, its
// first row within the group, the group's tokens.  Called by whole warps; false: there is no such tile.
__device__ __forceinline__ bool find_tile(const SharedArgs& a, long target, int rows_per_token, int per_tile, int* group, long* row0,
                                          int* first, int* tokens) {
    const int lane = threadIdx.x & 31;
    long before = 0;
    for (int base = 0; base < a.groups; base += 32) {
        const int g = base + lane;
        int t0 = 0, n = 0;
        if (g < a.groups) {
            t0 = min(max(a.group_start[g], 0), a.tokens);
            n = max(min(max(a.group_start[g + 1], 0), a.tokens) - t0, 0);
            if (a.prefix_lens[g] <= 0) n = 0;
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
            *group = base + who;
            *row0 = (target - before - __shfl_sync(0xffffffffu, upto - mine, who)) * per_tile;
            *first = __shfl_sync(0xffffffffu, t0, who);
            *tokens = __shfl_sync(0xffffffffu, n, who);
            return true;
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
    }
    return false;
}

// The group of a token, or -1.
__device__ __forceinline__ int group_of(const SharedArgs& a, int t) {
    int lo = 0, hi = a.groups;                           // the last group that starts at or in front of t
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (a.group_start[mid] <= t) lo = mid + 1; else hi = mid;
    }
    return lo > 0 && t < a.group_start[lo] ? lo - 1 : -1;
}

}  // namespace lb200
