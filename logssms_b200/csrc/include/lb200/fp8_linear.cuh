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
    int tile0, tiles;                                      // pairs: the tiles of this launch are tile0 up to here
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
__device__ __forceinline__ void load_shared4(uint32_t addr, float* r) {
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]) : "r"(addr));
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
__device__ __forceinline__ void tmem_ld32_async(uint32_t addr, uint32_t* r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
                 "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
                 "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), 
                   "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), 
                   "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(addr));
}
__device__ __forceinline__ void tmem_ld64(uint32_t addr, uint32_t* r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x64.b32 "
                 "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, "
                 "%32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, %48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [%64];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), 
                   "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), 
                   "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]), "=r"(r[32]), 
                   "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]), "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), 
                   "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]), "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), 
                   "=r"(r[55]), "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63])
                 : "r"(addr));
}
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
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
// v / (1 + e^-v) of v = sum * act_scale, by the special-function unit's exponential and reciprocal; `eighth`: act_scale / 8 (exact from
// 2^-123 up).  Off by (1.25 |v| + 8) 2^-24 of itself at most, and by what the sum and v are: the exponent's constant and its rounding
// (1.25 |v|), the exponential (4), the denominator (1), the reciprocal (2), the product (1).  v and the denominator are scaled by an
// eighth, else the reciprocal would be flushed to zero from -87.3 down; from -88.7 down e^-v is infinite and the result zero, as in
// any 32-bit form.  The accurate division and exponential made the end of a tile half as long as its products.
__device__ __forceinline__ float silu_of(float sum, float eighth) {
    const float v8 = sum * eighth, e = ex2_approx(-8.f * 1.44269504f * v8);
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(fmaf(e, 0.125f, 0.125f)));
    return v8 * r;
}
// A block's sums d (0, or 2^-18 to 2^25 in size) are multiplied by the product of its two scales where that is `plain`, a normal
// number.  Below 2^-126 or beyond 2^128 the product would lose its bits or be infinite, although its multiple of d may well be a number:
// there d is multiplied by one scale first, then by the other.  With `w` between 2^-100 and 2^100, d w is a normal number and the second
// product is rounded in its sum only; a `w` outside goes 2^64 nearer to 1 and x as far the other way: what x loses there lies below
// 2^-160, and past the largest number the result is infinite anyhow.  An infinite or NaN scale stays what it is; a zero sum stays zero
// under any two finite scales.  A row's sums do not hang on its neighbours' scales.  Blocks of zeros come here too, since they have the
// smallest scale.  us without / with a block of zeros in x / with a row of zeros (the weight in L2): 3,072 x 12,288 1 row 7.4 / 8.8 /
// 11.8, 64 rows 11.4 / 20.0 / 21.6, 512 rows 29.8 / 29.8 / 35.1, 8,192 rows 291 / 307 / 336.
__device__ __forceinline__ bool plain(float product) { return magnitude(product) - 0x00800000u < 0x7f000000u; }
constexpr float k2p64 = 18446744073709551616.f, k2m64 = 1.f / k2p64;
struct Apart {
    float w, first, more;                                  // the weight's scale; what d is multiplied by first, x's share besides
    __device__ __forceinline__ explicit Apart(float w_) : w(w_) {
        const uint32_t m = magnitude(w);
        const bool high = m > 0x71800000u && m < 0x7f800000u, low = m < 0x0d800000u && m != 0;
        first = w * (high ? k2m64 : low ? k2p64 : 1.f);
        more = high ? k2p64 : low ? k2m64 : 1.f;
    }
    // sum + d x w = (d * factor) * then + sum
    __device__ __forceinline__ void of(float x, float& factor, float& then) const {
        const float p = x * w;
        const bool joined = plain(p);
        then = x * more;
        if (more > 1.f && magnitude(then) == 0x7f800000u && magnitude(x) < 0x7f800000u) then = copysignf(3.402823466e38f, x);
        then = joined ? p : then;
        factor = joined ? 1.f : first;
    }
};

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
