// What the kernels of 8-bit products share: their arguments, the pieces of inline PTX beyond lb200/tcgen05.cuh, the scales.
#pragma once
#include "lb200/common.cuh"
#include "lb200/fp8.cuh"
#include "lb200/tcgen05.cuh"

namespace lb200 {
namespace fp8 {
using namespace lb200::tc;

constexpr int kBK = kFp8Block;                            // columns of a block = bytes of a swizzled row

struct Args {
    const float* sx; long sx_row, sx_block;               // scales of x: strides per row and per block
    const float *sw0, *sw1; long sw_row, sw_block;        // scales of W (swiglu: gate, up): strides per 128 features and per block
    const float* bias; void* out; long ldo;
    uint8_t* q; long ldq; float* qs; long qs_row, qs_block;    // swiglu: the 8-bit rows
    int M, N, K;
    int split, stages, tiles_n;
    int early;                                            // W may be read before the kernels in front have ended
    int out_f32;
    float out_scale, act_scale;
    int* error;
};

__device__ __forceinline__ void report(int* error, int role, int step) {
    if (error != nullptr) atomicCAS(error, 0, 0x20000000 | (role << 24) | ((blockIdx.x & 0xFFF) << 12) | (step & 0xFFF));
}
__device__ __forceinline__ uint32_t cluster_rank() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t peer_addr(uint32_t local, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(local), "r"(rank));
    return r;
}
__device__ __forceinline__ void store_peer(uint32_t addr, float a) {
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(a) : "memory");
}
__device__ __forceinline__ void store_peer4(uint32_t addr, float a, float b, float c, float d) {
    asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "f"(a), "f"(b), "f"(c), "f"(d) : "memory");
}
// e4m3 operands, both K-major, float32 accumulator: formats 0 and 0
__host__ __device__ constexpr uint32_t f8_idesc(int M, int N) { return (1u << 4) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24); }
__device__ __forceinline__ void umma_f8(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
}
// 16 consecutive float32 columns of this thread's lane of tensor memory; complete after tmem_ld_wait()
__device__ __forceinline__ void tmem_ld16(uint32_t addr, uint32_t* r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
                   "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]) : "r"(addr));
}
__device__ __forceinline__ void tmem_ld8(uint32_t addr, uint32_t* r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]) : "r"(addr));
}
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
// Two float32 sums side by side in 64 bits, so that both are joined in one instruction: acc += (d0, d1) * scale
__device__ __forceinline__ uint64_t pair_of(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void fma2(uint64_t& acc, uint32_t d0, uint32_t d1, uint64_t scale) {
    asm("{\n\t.reg .b64 d;\n\tmov.b64 d, {%1, %2};\n\tfma.rn.f32x2 %0, d, %3, %0;\n\t}" : "+l"(acc) : "r"(d0), "r"(d1), "l"(scale));
}
__device__ __forceinline__ float low_of(uint64_t p) { return __uint_as_float((uint32_t)p); }
__device__ __forceinline__ float high_of(uint64_t p) { return __uint_as_float((uint32_t)(p >> 32)); }
// One thread of a whole warp.  The loops that feed the tensor core run on the whole warp, with this around the instructions that
// one thread issues, so that addresses and descriptors stay in the warp's own registers: as a branch for lane 0, the four
// products of a block and their two commits took 480 cycles to issue, nearly as long as they run.
__device__ __forceinline__ bool elect_one() {
    uint32_t yes;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(yes));
    return yes != 0;
}
// has the phase with this parity completed?  (No waiting: asked for ahead of the work that precedes its use.)
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
    uint32_t done;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(done) : "r"(smem_u32(bar)), "r"(parity) : "memory");
    return done != 0;
}
// Wait by asking again and again: mbarrier.try_wait takes some 300 cycles even when the phase is long over, a test 50, and the
// loops here hand an accumulator to and fro every 500.  false: the phase did not complete within about a second.
__device__ __forceinline__ bool mbar_spin(uint64_t* bar, uint32_t parity) {
    for (uint32_t spin = 0; spin < (kSpinLimit << 3); ++spin)
        if (mbar_test(bar, parity)) return true;
    return false;
}
// v / (1 + e^-v) by the special-function unit's exponential and reciprocal: off by (|v| + 6) 2^-24 of itself at most.  The
// accurate division and exponential made the end of a tile half as long as its products.
__device__ __forceinline__ float silu_of(float v) {
    float e = ex2_approx(-1.44269504f * v), r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
    return v * r;
}
// the product of two scales, finite where both are: a zero sum stays zero
__device__ __forceinline__ float join(float a, float b) {
    float s = a * b;
    if (magnitude(s) == 0x7f800000u) {
        if (magnitude(a) < 0x7f800000u && magnitude(b) < 0x7f800000u) s = copysignf(3.402823466e38f, s);
    }
    return s;
}

// A rows x width matrix of bytes whose rows lie `stride` bytes apart (a multiple of 16; base on a 16-byte boundary); box =
// box_rows x 128, 128-byte swizzle, zeros outside.  0 or a cudaError.
inline int make_byte_map(CUtensorMap* map, const void* ptr, long rows, long width, long stride, int box_rows) {
    EncodeTiled enc = tensor_map_encoder();
    if (enc == nullptr) return (int)cudaErrorNotSupported;
    const cuuint64_t dims[2] = {(cuuint64_t)width, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)stride};
    const cuuint32_t box[2] = {(cuuint32_t)kBK, (cuuint32_t)box_rows};
    const cuuint32_t elem[2] = {1, 1};
    const CUresult rc = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(ptr), dims, strides, box, elem,
                            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return rc == CUDA_SUCCESS ? 0 : (int)cudaErrorInvalidValue;
}

}  // namespace fp8
}  // namespace lb200
