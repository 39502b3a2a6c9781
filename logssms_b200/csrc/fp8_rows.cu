// Rows and matrices in 8-bit floating point (lb200/fp8.cuh): RMSNorm with the residual's addition and an 8-bit output,
// quantisation of rows (a scale per row and 128 columns) and of a weight (a scale per 128 rows and 128 columns).
//
// All three read their input once, in 16-byte pieces that stay in registers between the passes over them, and are bound by
// those bytes and by their instructions (8,192 x 3,072 bfloat16: issue slots 75 % busy in the norm, 78 % in the rows'
// quantisation).  16 neighbouring threads hold the 8 values each of a block of 128, so a block's maximum takes four shuffles.
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
// eight values as they lie in memory, and as numbers
template <typename T> struct Raw8 { uint4 a[sizeof(T) / 2]; };
template <typename T> __device__ __forceinline__ Raw8<T> raw8(const T* p) {
    Raw8<T> r;
#pragma unroll
    for (int i = 0; i < (int)(sizeof(T) / 2); ++i) r.a[i] = reinterpret_cast<const uint4*>(p)[i];
    return r;
}
__device__ __forceinline__ void numbers(const Raw8<float>& r, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        v[4 * i] = __uint_as_float(r.a[i].x); v[4 * i + 1] = __uint_as_float(r.a[i].y);
        v[4 * i + 2] = __uint_as_float(r.a[i].z); v[4 * i + 3] = __uint_as_float(r.a[i].w);
    }
}
__device__ __forceinline__ void numbers(const Raw8<__nv_bfloat16>& r, float (&v)[8]) {
    const uint32_t w[4] = {r.a[0].x, r.a[0].y, r.a[0].z, r.a[0].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { v[2 * i] = __uint_as_float(w[i] << 16); v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
}
template <typename T> __device__ __forceinline__ void load8(const T* p, float (&v)[8]) { numbers(raw8(p), v); }
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
// eight values over their block's scale
__device__ __forceinline__ uint2 pack8(const float (&v)[8], const Fp8Divide& by) {
    return make_uint2(fp8_quad(by(v[0]), by(v[1]), by(v[2]), by(v[3])), fp8_quad(by(v[4]), by(v[5]), by(v[6]), by(v[7])));
}

struct NormArgs {
    const void *x, *other, *residual; void* residual_out;
    const float* weight; uint8_t* q; float* scales;
    long ldx, ldo, ldr, ldres, ldq;                       // row strides, elements
    long scale_row, scale_block;                          // strides of `scales`
    long rows; int width; float eps, in0, in1, out_scale;
};

// r = x in0 + other in1 + residual;  residual_out = round(r);  n = r rsqrt(mean r^2 + eps) w out_scale, in 32 bits up to the
// 8-bit rounding.  A CTA stays and takes row after row: the norm's weights, which are half as many bytes as a row of everything
// else, are read once, and the next row is on its way while this one is summed, divided and stored.  A thread has kPieces pieces of
// 8 values of each row.  One barrier a row: the partial sums of neighbouring rows have places of their own.
template <typename T, int kPieces> struct NormForm {        // threads of a CTA at most, and CTAs on an SM
    static constexpr int kThreads = kPieces == 1 ? 384 : 512, kCtas = kPieces == 1 ? (sizeof(T) == 2 ? 3 : 2) : (sizeof(T) == 2 ? 2 : 1);
};
template <typename T, int kPieces>
__global__ void __launch_bounds__(NormForm<T, kPieces>::kThreads, NormForm<T, kPieces>::kCtas) add_rmsnorm_fp8_kernel(NormArgs a) {
    pdl_trigger();
    pdl_wait();
    __shared__ float red[2][16];
    const int pieces = a.width >> 3, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    constexpr bool kKeep = kPieces == 1;                   // the norm's weights in registers (else from L1 for every row)
    float w[kPieces][8];
    Raw8<T> x[kPieces], o[kPieces], r[kPieces];
    auto fetch = [&](long row) {
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            const int at = (threadIdx.x + i * blockDim.x) * 8;
            if (at < a.width) {
                x[i] = raw8((const T*)a.x + row * a.ldx + at);
                if (a.other != nullptr) o[i] = raw8((const T*)a.other + row * a.ldo + at);
                if (a.residual != nullptr) r[i] = raw8((const T*)a.residual + row * a.ldr + at);
            }
        }
    };
    long row = blockIdx.x;
    fetch(row);
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
        const int at = (threadIdx.x + i * blockDim.x) * 8;
        if (kKeep && at < a.width) load8(a.weight + at, w[i]);
    }
    for (int turn = 0; row < a.rows; turn ^= 1) {
        float v[kPieces][8];
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            const int at = (threadIdx.x + i * blockDim.x) * 8;
            if (at < a.width) {
                float t[8];
                numbers(x[i], v[i]);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[i][e] *= a.in0;
                if (a.other != nullptr) {
                    numbers(o[i], t);
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[i][e] += t[e] * a.in1;
                }
                if (a.residual != nullptr) {
                    numbers(r[i], t);
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[i][e] += t[e];
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) ss += v[i][e] * v[i][e];
            }
        }
        const long next = row + gridDim.x;
        if (next < a.rows) fetch(next);
        if (a.residual_out != nullptr) {
#pragma unroll
            for (int i = 0; i < kPieces; ++i) {
                const int at = (threadIdx.x + i * blockDim.x) * 8;
                if (at < a.width) store8((T*)a.residual_out + row * a.ldres + at, v[i]);
            }
        }
        ss = warp_sum(ss);
        if (lane == 0) red[turn][threadIdx.x >> 5] = ss;
        __syncthreads();
        ss = warp_sum(lane < warps ? red[turn][lane] : 0.f);
        const float inv = rsqrtf(ss / (float)a.width + a.eps) * a.out_scale;
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            const int pc = threadIdx.x + i * blockDim.x, at = pc * 8;
            if (i * (int)blockDim.x >= pieces) break;      // the same for the whole CTA: every thread takes part in the shuffles
            uint32_t top = 0;
            if (at < a.width) {
                if (!kKeep) load8(a.weight + at, w[i]);
#pragma unroll
                for (int e = 0; e < 8; ++e) { v[i][e] = v[i][e] * inv * w[i][e]; top = max(top, magnitude(v[i][e])); }
            }
            const float scale = fp8_scale(block_top(top));
            if (at < a.width) {
                *reinterpret_cast<uint2*>(a.q + row * a.ldq + at) = pack8(v[i], Fp8Divide(scale));
                if ((pc & (kLanes - 1)) == 0) a.scales[row * a.scale_row + (pc / kLanes) * a.scale_block] = scale;
            }
        }
        row = next;
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
        const float scale = fp8_scale(__reduce_max_sync(0xffffffffu, top));
        const Fp8Divide by(scale);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int c = b * kFp8Block + e * 32 + lane;
            if (c < a.width) a.q[row * a.ldq + c] = (uint8_t)fp8_pair(by(v[e]), 0.f);
        }
        if (lane == 0) a.scales[row * a.scale_row + b * a.scale_block] = scale;
    }
}

struct QuantArgs {
    const void* x; uint8_t* q; float* scales;
    long ldx, ldq, scale_row, scale_block;
    long rows; int width, blocks;                         // blocks of 128 columns
};

// 16 threads per row and block of 128, kAtOnce of them after one another whose loads go out together
template <typename T, int kAtOnce>
__global__ void __launch_bounds__(256) quantize_rows_kernel(QuantArgs a) {
    pdl_trigger();
    pdl_wait();
    const uint32_t blocks = a.blocks, first = blockIdx.x * (256 / kLanes * kAtOnce) + threadIdx.x / kLanes;      // (64-bit division takes three times as long)
    const int sub = threadIdx.x & (kLanes - 1);
    Raw8<T> raw[kAtOnce];
    uint32_t rows[kAtOnce], b[kAtOnce];
    bool live[kAtOnce];
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
        const uint32_t item = first + k * (256 / kLanes);
        rows[k] = item / blocks;
        b[k] = item - rows[k] * blocks;
        live[k] = rows[k] < a.rows && (int)b[k] * kFp8Block + sub * 8 < a.width;
        raw[k] = live[k] ? raw8((const T*)a.x + rows[k] * a.ldx + b[k] * kFp8Block + sub * 8) : Raw8<T>{};
    }
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
        float v[8];
        uint32_t top = 0;
        numbers(raw[k], v);
#pragma unroll
        for (int e = 0; e < 8; ++e) top = max(top, magnitude(v[e]));
        const float scale = fp8_scale(block_top(top));
        if (live[k]) {
            *reinterpret_cast<uint2*>(a.q + rows[k] * a.ldq + b[k] * kFp8Block + sub * 8) = pack8(v, Fp8Divide(scale));
            if (sub == 0) a.scales[rows[k] * a.scale_row + b[k] * a.scale_block] = scale;
        }
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
    const float scale = fp8_scale(__reduce_max_sync(0xffffffffu, top));
    const Fp8Divide by(scale);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int c = b * kFp8Block + e * 32 + lane;
        if (c < a.width) a.q[row * a.ldq + c] = (uint8_t)fp8_pair(by(v[e]), 0.f);
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
    Raw8<T> raw[8];                                        // as they lie in memory: 32 registers of bfloat16, not 64
    float v[8];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const long row = row0 + 16 * i;
        if (row < a.rows && at < a.width) raw[i] = raw8((const T*)a.x + row * a.ldx + at);
        else raw[i] = Raw8<T>{};
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        numbers(raw[i], v);
#pragma unroll
        for (int e = 0; e < 8; ++e) top = max(top, magnitude(v[e]));
    }
    top = __reduce_max_sync(0xffffffffu, top);
    if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
    __syncthreads();
    top = tops[0];
#pragma unroll
    for (int w = 1; w < 8; ++w) top = max(top, tops[w]);
    const float scale = fp8_scale(top);
    const Fp8Divide by(scale);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const long row = row0 + 16 * i;
        numbers(raw[i], v);
        if (row < a.rows && at < a.width) *reinterpret_cast<uint2*>(a.q + row * a.ldq + at) = pack8(v, by);
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
    const float scale = fp8_scale(top);
    const Fp8Divide by(scale);
    if (c < a.width)
        for (int r = threadIdx.x >> 7; r < rows; r += step)
            a.q[(row0 + r) * a.ldq + c] = (uint8_t)fp8_pair(by(to_f32(((const T*)a.x)[(row0 + r) * a.ldx + c])), 0.f);
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
    if (width > kFp8Most) return kTooLarge;
    const int size = dtype == kF32 ? 4 : 2;
    NormArgs a{x, other, residual, residual_out, weight, (uint8_t*)q, scales, ldx, ldo, ldr, ldres, ldq, scale_row, scale_block,
               rows, width, eps, in0, in1, out_scale};
    cudaStream_t s = (cudaStream_t)stream;
    const int pieces = width / 8;
    if (width % 8 == 0 && pieces <= 1024 && on16(x, ldx, size) && on16(other, ldo, size) && on16(residual, ldr, size)
        && on16(residual_out, ldres, size) && on16(weight, 0, 4)) {
        const int per = pieces <= 384 ? 1 : 2, threads = ((pieces + per - 1) / per + 31) / 32 * 32;
        int device = 0, sms = 148;
        if (cudaGetDevice(&device) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
        LB_DISPATCH_DTYPE(dtype, {
            const int held = per == 1 ? NormForm<T, 1>::kThreads * NormForm<T, 1>::kCtas : NormForm<T, 2>::kThreads * NormForm<T, 2>::kCtas;
            const dim3 grid(min(rows, sms * max(1, held / threads)));
            const int rc = per == 1 ? launch_pdl(add_rmsnorm_fp8_kernel<T, 1>, grid, dim3(threads), 0, s, a)
                                    : launch_pdl(add_rmsnorm_fp8_kernel<T, 2>, grid, dim3(threads), 0, s, a);
            if (rc != 0) return rc;
        })
    } else {
        const size_t smem = (size_t)width * 4;
        if (smem > 200 * 1024) return kTooLarge;
        LB_DISPATCH_DTYPE(dtype, {
            static SharedLimits limits;
            int rc = ensure_dynamic_smem(add_rmsnorm_fp8_any_kernel<T>, smem, limits);
            if (rc == 0) rc = launch_pdl(add_rmsnorm_fp8_any_kernel<T>, dim3(rows), dim3(256), smem, s, a);
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
    if (width > kFp8Most) return kTooLarge;
    const int size = dtype == kF32 ? 4 : 2, blocks = (width + kFp8Block - 1) / kFp8Block;
    QuantArgs a{x, (uint8_t*)q, scales, ldx, ldq, scale_row, scale_block, rows, width, blocks};
    cudaStream_t s = (cudaStream_t)stream;
    const bool vec = width % 8 == 0 && on16(x, ldx, size);
    const long items = (block_rows == 1 ? rows : (rows + kFp8Block - 1) / kFp8Block) * (long)blocks;
    if (items > 0x7fffffffL / 2) return kTooLarge;         // (numbers of blocks are 32-bit: 137 GB of values)
    int device = 0, sms = 148;
    if (cudaGetDevice(&device) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
    long grid = block_rows == 1 ? (items * (vec ? kLanes : 32) + 255) / 256 : items;
    // many rows: four blocks a thread (8,192 x 3,072 bfloat16: 16.7 us, with one 19.2); few: one, as many CTAs as there are (2,048 x 1,536: 3.2)
    const bool many = block_rows == 1 && vec && grid > 32L * sms;
    if (many) grid = (grid + 3) / 4;
    LB_DISPATCH_DTYPE(dtype, {
        int rc = 0;
        if (block_rows == 1) rc = launch_pdl(many ? quantize_rows_kernel<T, 4> : vec ? quantize_rows_kernel<T, 1> : quantize_rows_any_kernel<T>, dim3((unsigned)grid), dim3(256), 0, s, a);
        else if (vec) quantize_weight_kernel<T><<<(unsigned)grid, 256, 0, s>>>(a);
        else quantize_weight_any_kernel<T><<<(unsigned)grid, 256, 0, s>>>(a);
        if (rc != 0) return rc;
    })
    return launch_status();
}
