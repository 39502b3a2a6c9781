// Operands of the adapters' kernels (adapters.cu).
#pragma once

namespace lb200 {

struct AdapterArgs {
    const void* y; long ldy;                            // [T, N]
    const void* x; long ldx;                            // [T, K]
    const void* A; long a_adapter, a_row;               // [adapters, R, K]
    const void* B; long b_adapter, b_row;               // [adapters, N, R]
    const int* index;                                   // a row's adapter; outside of [0, adapters): none
    const float* scales; const int* ranks;              // per adapter; null: 1, R
    void* out; long ldo;
    float* h;                                           // [parts, T, R]
    long T;
    int K, N, R, adapters, parts, part_k;
};

}  // namespace lb200
