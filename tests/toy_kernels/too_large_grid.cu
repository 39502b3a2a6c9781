// A launch that CUDA refuses on the host: more blocks along z than a grid has.
#include "lb200/common.cuh"

namespace {
__global__ void nothing_kernel() { lb200::pdl_wait(); }
}  // namespace

extern "C" int lb_too_large_grid(int z, void* stream) {
    return lb200::launch_pdl(nothing_kernel, dim3(1, 1, (unsigned)z), dim3(32), 0, (cudaStream_t)stream);
}
extern "C" int lb_left_behind() { return lb200::launch_status(); }
