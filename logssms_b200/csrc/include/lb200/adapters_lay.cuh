// Operands of the adapters' tile kernel whose rows do not lie at multiples of 16 bytes, which TMA cannot fetch, copied to where they
// do, zeros behind their ends.  Bound by memory: 4 bytes read and written a value; x, the longest, is small beside y and the output
// (8,000 rows, 4,001 -> 12,001: 37 us of 295).
#pragma once
#include "lb200/adapters.cuh"
#include "lb200/common.cuh"

namespace lb200 {
namespace adapter_lay {
typedef __nv_bfloat16 bf16;
constexpr int kThreads = 256, kMost = 3;

struct Piece {                                            // [layers x rows][width], rows `pitch` apart afterwards; null: nothing to do
    const bf16* from; bf16* to;
    unsigned rows, all; int width, pitch;                 // rows of a layer, of all layers
    long layer_stride, row_stride;
};
struct Pieces { Piece p[kMost]; };

// grid: (CTAs that share out a piece, pieces); a thread: 16 bytes at a time
__global__ void __launch_bounds__(kThreads) adapter_lay_kernel(const __grid_constant__ Pieces pieces) {
    pdl_wait();
    pdl_trigger();
    const Piece& p = pieces.p[blockIdx.y];
    if (p.to == nullptr) return;
    const unsigned chunks = (unsigned)p.pitch / 8, n = p.all * chunks, step = gridDim.x * kThreads;
    for (unsigned i = blockIdx.x * kThreads + threadIdx.x; i < n; i += step) {
        const unsigned row = i / chunks, c = (i - row * chunks) * 8, layer = row / p.rows;
        const unsigned short* from = reinterpret_cast<const unsigned short*>(p.from) + layer * p.layer_stride + (long)(row - layer * p.rows) * p.row_stride + c;
        uint32_t v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = (int)c + e < p.width ? from[e] : 0u;
        *reinterpret_cast<uint4*>(p.to + (size_t)row * p.pitch + c) = make_uint4(v[0] | v[1] << 16, v[2] | v[3] << 16, v[4] | v[5] << 16, v[6] | v[7] << 16);
        if (n - i <= step) break;                         // (i + step may pass 32 bits)
    }
}

inline int launch(const Pieces& pieces, cudaStream_t stream) { return launch_pdl(adapter_lay_kernel, dim3(148 * 8, kMost), dim3(kThreads), 0, stream, pieces); }

}  // namespace adapter_lay
}  // namespace lb200
