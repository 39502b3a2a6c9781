// Operands of the adapters' kernels (adapters.cu).
#pragma once
#include <cuda_runtime.h>

namespace lb200 {

struct AdapterArgs {
    const void* y; long ldy;                            // [T, N]
    const void* x; long ldx;                            // [T, K]
    const void* A; long a_adapter, a_row;               // [adapters, R, K]
    const void* B; long b_adapter, b_row;               // [adapters, N, R]
    const int* index;                                   // a row's adapter; outside of [0, adapters): none
    const float* scales; const int* ranks;              // per adapter; null: 1, R
    void* out; long ldo;
    float* h;                                           // [T, R], by the places of the rows
    // the rows in the order of their adapters, by tiles of one adapter each (null: as they come): see adapters_order.cuh
    const int* order; const int4* tiles; const int* n_tiles;
    long T;
    int K, N, R, adapters, parts, part_k, slots;
};

// The smallest adapter behind `prev` that any of the warp's rows names (INT_MAX: none).
constexpr int kNoAdapter = 0x7fffffff;
__device__ __forceinline__ int next_adapter(int mine, int prev) { return __reduce_min_sync(0xffffffffu, mine > prev ? mine : kNoAdapter); }

// The row at place t.
__device__ __forceinline__ long row_at(const AdapterArgs& a, long t) { return a.order != nullptr ? a.order[t] : t; }
__device__ __forceinline__ int adapter_of(const AdapterArgs& a, long t) {
    if (t >= a.T) return -1;
    const int i = a.index[row_at(a, t)];
    return i >= 0 && i < a.adapters ? i : -1;
}
__device__ __forceinline__ int rank_of(const AdapterArgs& a, int i) { return a.ranks ? min(max(a.ranks[i], 0), a.R) : a.R; }

}  // namespace lb200
