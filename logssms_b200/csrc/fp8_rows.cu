// Rows and matrices in 8-bit floating point (lb200/fp8.cuh): RMSNorm with the residual's addition and an 8-bit output,
// quantisation of rows (a scale per row and 128 columns) and of a weight (a scale per 128 rows and 128 columns).
//
// All three read their input once, in 16-byte pieces that stay in registers between the passes over them, and are bound by
// those bytes.  16 neighbouring threads hold the 8 values each of a block of 128, so a block's maximum takes four shuffles.
// Widths that are no multiple of 8, and rows that do not lie on 16 bytes, go value by value (`*_any_kernel`).
#include "lb200/common.cuh"
#include "lb200/fp8.cuh"
using namespace lb200;

namespace {
constexpr int kLanes = kFp8Block / 8;                     // threads that hold a block of 128 in pieces of 8

__device__ __forceinline__ uint32_t block_top(uint32_t top) {       // over the 16 threads of a block
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    return top;
}
template <typename T> __device__ __forceinline__ void load8(const T* p, float (&v)[8]);
template <> __device__ __forceinline__ void load8<float>(const float* p, float (&v)[8]) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
template <> __device__ __forceinline__ void load8<__nv_bfloat16>(const __nv_bfloat16* p, float (&v)[8]) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { v[2 * i] = __uint_as_float(w[i] << 16); v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
}
template <typename T> __device__ __forceinline__ void store8(T* p, const float (&v)[8]);
template <> __device__ __forceinline__ void store8<float>(float* p, const float (&v)[8]) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}
template <> __device__ __forceinline__ void store8<__nv_bfloat16>(__nv_bfloat16* p, const float (&v)[8]) {
    uint4 u;
    __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&u);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
    *reinterpret_cast<uint4*>(p) = u;
}
__device__ __forceinline__ uint2 pack8(const float (&v)[8], float inv) {
    return make_uint2(fp8_quad(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv), fp8_quad(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv));
}

struct NormArgs {
    const void *x, *other, *residual; void* residual_out;
    const float* weight; uint8_t* q; float* scales;
    long ldx, ldo, ldr, ldres, ldq;                       // row strides, elements
    long scale_row, scale_block;                          // strides of `scales`
    int width; float eps, in0, in1, out_scale;
};

// r = x in0 + other in1 + residual;  residual_out = round(r);  n = r rsqrt(mean r^2 + eps) w out_scale, in 32 bits up to the
// 8-bit rounding.  A CTA per row, up to kPieces pieces of 8 values per thread.
template <typename T, int kPieces>
__global__ void __launch_bounds__(512) add_rmsnorm_fp8_kernel(NormArgs a) {
    pdl_trigger();
    pdl_wait();
    __shared__ float red[32];
    const long row = blockIdx.x;
    const T* x = (const T*)a.x + row * a.ldx;
    const T* other = a.other == nullptr ? nullptr : (const T*)a.other + row * a.ldo;
    const T* residual = a.residual == nullptr ? nullptr : (const T*)a.residual + row * a.ldr;
    const int pieces = a.width >> 3;
    float v[kPieces][8], o[kPieces][8], r[kPieces][8];
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
        const int at = (threadIdx.x + i * blockDim.x) * 8;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[i][e] = o[i][e] = r[i][e] = 0.f;
        if (at < a.width) {
            load8(x + at, v[i]);
            if (other != nullptr) load8(other + at, o[i]);
            if (residual != nullptr) load8(residual + at, r[i]);
        }
    }
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
        const int at = (threadIdx.x + i * blockDim.x) * 8;
        if (at < a.width) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                float s = v[i][e] * a.in0;
                if (other != nullptr) s += o[i][e] * a.in1;
                if (residual != nullptr) s += r[i][e];
                v[i][e] = s;
                ss += s * s;
            }
            if (a.residual_out != nullptr) store8((T*)a.residual_out + row * a.ldres + at, v[i]);
        }
    }
    ss = block_sum(ss, red);
    const float inv = rsqrtf(ss / (float)a.width + a.eps) * a.out_scale;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
        const int pc = threadIdx.x + i * blockDim.x, at = pc * 8;
        if (i * (int)blockDim.x >= pieces) break;          // the same for the whole CTA: every thread takes part in the shuffles
        uint32_t top = 0;
        if (at < a.width) {
            float w[8];
            load8(a.weight + at, w);
#pragma unroll
            for (int e = 0; e < 8; ++e) { v[i][e] = v[i][e] * inv * w[e]; top = max(top, magnitude(v[i][e])); }
        }
        const float scale = fp8_scale(block_top(top));
        if (at < a.width) {
            *reinterpret_cast<uint2*>(a.q + row * a.ldq + at) = pack8(v[i], 1.f / scale);
            if ((pc & (kLanes - 1)) == 0) a.scales[row * a.scale_row + (pc / kLanes) * a.scale_block] = scale;
        }
    }
}

// the same for any width and alignment: value by value, the row kept in shared memory, a warp per block of 128
template <typename T>
__global__ void __launch_bounds__(256) add_rmsnorm_fp8_any_kernel(NormArgs a) {
    pdl_trigger();
    pdl_wait();
    extern __shared__ float kept[];
    __shared__ float red[32];
    const long row = blockIdx.x;
    const T* x = (const T*)a.x + row * a.ldx;
    const T* other = a.other == nullptr ? nullptr : (const T*)a.other + row * a.ldo;
    const T* residual = a.residual == nullptr ? nullptr : (const T*)a.residual + row * a.ldr;
    float ss = 0.f;
    for (int c = threadIdx.x; c < a.width; c += blockDim.x) {
        float s = to_f32(x[c]) * a.in0;
        if (other != nullptr) s += to_f32(other[c]) * a.in1;
        if (residual != nullptr) s += to_f32(residual[c]);
        kept[c] = s;
        ss += s * s;
        if (a.residual_out != nullptr) ((T*)a.residual_out)[row * a.ldres + c] = from_f32<T>(s);
    }
    ss = block_sum(ss, red);                               // (two barriers: the row is complete)
    const float inv = rsqrtf(ss / (float)a.width + a.eps) * a.out_scale;
    const int lane = threadIdx.x & 31, blocks = (a.width + kFp8Block - 1) / kFp8Block;
    for (int b = threadIdx.x >> 5; b < blocks; b += blockDim.x >> 5) {
        float v[4];
        uint32_t top = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int c = b * kFp8Block + e * 32 + lane;
            v[e] = c < a.width ? kept[c] * inv * a.weight[c] : 0.f;
            top = max(top, magnitude(v[e]));
        }
        const float scale = fp8_scale(__reduce_max_sync(0xffffffffu, top)), back = 1.f / scale;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int c = b * kFp8Block + e * 32 + lane;
            if (c < a.width) a.q[row * a.ldq + c] = (uint8_t)fp8_pair(v[e] * back, 0.f);
        }
        if (lane == 0) a.scales[row * a.scale_row + b * a.scale_block] = scale;
    }
}

struct QuantArgs {
    const void* x; uint8_t* q; float* scales;
    long ldx, ldq, scale_row, scale_block;
    long rows; int width, blocks;                         // blocks of 128 columns
};

// 16 threads per row and block of 128
template <typename T>
__global__ void __launch_bounds__(256) quantize_rows_kernel(QuantArgs a) {
    pdl_trigger();
    pdl_wait();
    const long item = ((long)blockIdx.x * 256 + threadIdx.x) / kLanes;
    const long row = item / a.blocks;
    const int b = (int)(item - row * a.blocks), sub = threadIdx.x & (kLanes - 1), at = b * kFp8Block + sub * 8;
    const bool live = row < a.rows && at < a.width;
    float v[8];
    uint32_t top = 0;
    if (live) {
        load8((const T*)a.x + row * a.ldx + at, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) top = max(top, magnitude(v[e]));
    }
    const float scale = fp8_scale(block_top(top));
    if (live) {
        *reinterpret_cast<uint2*>(a.q + row * a.ldq + at) = pack8(v, 1.f / scale);
        if (sub == 0) a.scales[row * a.scale_row + b * a.scale_block] = scale;
    }
}
// a warp per row and block of 128, value by value
template <typename T>
__global__ void __launch_bounds__(256) quantize_rows_any_kernel(QuantArgs a) {
    pdl_trigger();
    pdl_wait();
    const long item = ((long)blockIdx.x * 256 + threadIdx.x) >> 5;
    const long row = item / a.blocks;
    if (row >= a.rows) return;                             // whole warps
    const int b = (int)(item - row * a.blocks), lane = threadIdx.x & 31;
    const T* x = (const T*)a.x + row * a.ldx;
    float v[4];
    uint32_t top = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int c = b * kFp8Block + e * 32 + lane;
        v[e] = c < a.width ? to_f32(x[c]) : 0.f;
        top = max(top, magnitude(v[e]));
    }
    const float scale = fp8_scale(__reduce_max_sync(0xffffffffu, top)), back = 1.f / scale;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int c = b * kFp8Block + e * 32 + lane;
        if (c < a.width) a.q[row * a.ldq + c] = (uint8_t)fp8_pair(v[e] * back, 0.f);
    }
    if (lane == 0) a.scales[row * a.scale_row + b * a.scale_block] = scale;
}

// A CTA per block of 128 x 128: 16 threads per row of the block, 16 rows at a time, all of it in registers
template <typename T>
__global__ void __launch_bounds__(256) quantize_weight_kernel(QuantArgs a) {
    __shared__ uint32_t tops[8];
    const int b = blockIdx.x % a.blocks;
    const long row0 = (long)(blockIdx.x / a.blocks) * kFp8Block + threadIdx.x / kLanes;
    const int at = b * kFp8Block + (threadIdx.x & (kLanes - 1)) * 8;
    float v[8][8];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const long row = row0 + 16 * i;
        if (row < a.rows && at < a.width) load8((const T*)a.x + row * a.ldx + at, v[i]);
        else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[i][e] = 0.f;
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) top = max(top, magnitude(v[i][e]));
    top = __reduce_max_sync(0xffffffffu, top);
    if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
    __syncthreads();
    top = tops[0];
#pragma unroll
    for (int w = 1; w < 8; ++w) top = max(top, tops[w]);
    const float scale = fp8_scale(top), back = 1.f / scale;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const long row = row0 + 16 * i;
        if (row < a.rows && at < a.width) *reinterpret_cast<uint2*>(a.q + row * a.ldq + at) = pack8(v[i], back);
    }
    if (threadIdx.x == 0) a.scales[(blockIdx.x / a.blocks) * a.scale_row + b * a.scale_block] = scale;
}
template <typename T>
__global__ void __launch_bounds__(256) quantize_weight_any_kernel(QuantArgs a) {
    __shared__ uint32_t tops[8];
    const int b = blockIdx.x % a.blocks;
    const long row0 = (long)(blockIdx.x / a.blocks) * kFp8Block;
    const int c = b * kFp8Block + (threadIdx.x & 127), step = 2;
    const int rows = (int)min((long)kFp8Block, a.rows - row0);
    uint32_t top = 0;
    if (c < a.width)
        for (int r = threadIdx.x >> 7; r < rows; r += step) top = max(top, magnitude(to_f32(((const T*)a.x)[(row0 + r) * a.ldx + c])));
    top = __reduce_max_sync(0xffffffffu, top);
    if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
    __syncthreads();
    top = tops[0];
#pragma unroll
    for (int w = 1; w < 8; ++w) top = max(top, tops[w]);
    const float scale = fp8_scale(top), back = 1.f / scale;
    if (c < a.width)
        for (int r = threadIdx.x >> 7; r < rows; r += step)
            a.q[(row0 + r) * a.ldq + c] = (uint8_t)fp8_pair(to_f32(((const T*)a.x)[(row0 + r) * a.ldx + c]) * back, 0.f);
    if (threadIdx.x == 0) a.scales[(blockIdx.x / a.blocks) * a.scale_row + b * a.scale_block] = scale;
}

inline bool on16(const void* p, long stride, int size) { return p == nullptr || (((uintptr_t)p & 15) == 0 && (stride * size) % 16 == 0); }
}  // namespace

// x, other, residual (the last two may be null) and residual_out (may be null; may be `residual`): rows of `width` values
// with row strides in elements; q: bytes, row stride ldq, rows on 8 bytes; scales: float32 with a stride per row and per block.
extern "C" int lb_add_rmsnorm_fp8(const void* x, long ldx, const void* other, long ldo, const void* residual, long ldr,
                                  void* residual_out, long ldres, const float* weight, void* q, long ldq, float* scales,
                                  long scale_row, long scale_block, int rows, int width, float eps, float in0, float in1,
                                  float out_scale, int dtype, void* stream) {
    if (dtype != kF32 && dtype != kBF16) return kBadDType;
    if (rows <= 0) return kOk;
    if (width <= 0 || ldq % 8 || ((uintptr_t)q & 7)) return kBadSize;
    const int size = dtype == kF32 ? 4 : 2;
    NormArgs a{x, other, residual, residual_out, weight, (uint8_t*)q, scales, ldx, ldo, ldr, ldres, ldq, scale_row, scale_block,
               width, eps, in0, in1, out_scale};
    cudaStream_t s = (cudaStream_t)stream;
    const int pieces = width / 8;
    if (width % 8 == 0 && pieces <= 1024 && on16(x, ldx, size) && on16(other, ldo, size) && on16(residual, ldr, size)
        && on16(residual_out, ldres, size) && on16(weight, 0, 4)) {
        const int per = pieces <= 512 ? 1 : 2, threads = ((pieces + per - 1) / per + 31) / 32 * 32;
        LB_DISPATCH_DTYPE(dtype, {
            const int rc = per == 1 ? launch_pdl(add_rmsnorm_fp8_kernel<T, 1>, dim3(rows), dim3(threads), 0, s, a)
                                    : launch_pdl(add_rmsnorm_fp8_kernel<T, 2>, dim3(rows), dim3(threads), 0, s, a);
            if (rc != 0) return rc;
        })
    } else {
        const size_t smem = (size_t)width * 4;
        if (smem > 200 * 1024) return kTooLarge;
        LB_DISPATCH_DTYPE(dtype, {
            static size_t have = 0;
            ensure_dynamic_smem(add_rmsnorm_fp8_any_kernel<T>, smem, have);
            const int rc = launch_pdl(add_rmsnorm_fp8_any_kernel<T>, dim3(rows), dim3(256), smem, s, a);
            if (rc != 0) return rc;
        })
    }
    return launch_status();
}

// block_rows 1: a scale per row and 128 columns; 128: a scale per 128 rows and 128 columns.
extern "C" int lb_quantize_fp8(const void* x, long ldx, void* q, long ldq, float* scales, long scale_row, long scale_block,
                               long rows, int width, int block_rows, int dtype, void* stream) {
    if (dtype != kF32 && dtype != kBF16) return kBadDType;
    if (rows <= 0) return kOk;
    if (width <= 0 || ldq % 8 || ((uintptr_t)q & 7) || (block_rows != 1 && block_rows != kFp8Block)) return kBadSize;
    const int size = dtype == kF32 ? 4 : 2, blocks = (width + kFp8Block - 1) / kFp8Block;
    QuantArgs a{x, (uint8_t*)q, scales, ldx, ldq, scale_row, scale_block, rows, width, blocks};
    cudaStream_t s = (cudaStream_t)stream;
    const bool vec = width % 8 == 0 && on16(x, ldx, size);
    const long items = (block_rows == 1 ? rows : (rows + kFp8Block - 1) / kFp8Block) * (long)blocks;
    const long grid = block_rows == 1 ? (items * (vec ? kLanes : 32) + 255) / 256 : items;
    if (grid > 0x7fffffffL) return kTooLarge;
    LB_DISPATCH_DTYPE(dtype, {
        int rc = 0;
        if (block_rows == 1) rc = launch_pdl(vec ? quantize_rows_kernel<T> : quantize_rows_any_kernel<T>, dim3((unsigned)grid), dim3(256), 0, s, a);
        else if (vec) quantize_weight_kernel<T><<<(unsigned)grid, 256, 0, s>>>(a);
        else quantize_weight_any_kernel<T><<<(unsigned)grid, 256, 0, s>>>(a);
        if (rc != 0) return rc;
    })
    return launch_status();
}
