// 8-bit floating point (e4m3) with a float32 scale per block of 128: the arithmetic that every kernel of it shares.
//
//   scale(block) = max(max |v| / 448, 2^-126)      448: the largest e4m3 number
//   q            = e4m3(v / scale), round to nearest even
//
// The floor keeps 1 / scale finite; a block of zeros has the floor as its scale and zeros as values.  A NaN in a block makes
// the scale and the block's values NaN; an infinity makes the scale infinite, itself NaN and the others zero: neither is
// lost on the way to the product.
#pragma once
#include <cuda_fp8.h>
#include <stdint.h>

namespace lb200 {

constexpr int kFp8Block = 128;
constexpr int kFp8Most = 0x7fff0000;                      // rows, features and columns at most: sums of a place and a tile's size stay whole numbers of 32 bits

// |v| as bits: their order as whole numbers is the order of magnitudes, infinity above every number and NaN above infinity
__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }

__device__ __forceinline__ float fp8_scale(uint32_t top) {
    const float s = __uint_as_float(top) / 448.f;
    return s < 1.17549435e-38f ? 1.17549435e-38f : s;      // a NaN stays
}
// v / scale, rounded as a division is (up to its last bit, where the quotient is tiny): the product with the reciprocal and one
// correction by what is left over.  A product alone lies on the wrong side of a rounding boundary where a quotient of bfloat16 values
// lies on it, which is not rare.
struct Fp8Divide {
    float scale, back;
    __device__ __forceinline__ explicit Fp8Divide(float s) : scale(magnitude(s) == 0x7f800000u ? 0.f : s), back(1.f / s) {}     // x / inf: 0, NaN for inf
    __device__ __forceinline__ float operator()(float v) const {
        const float q = v * back;
        return fmaf(fmaf(-q, scale, v), back, q);
    }
};
// two values, already divided by their scale, as two bytes (the first one in the low byte)
__device__ __forceinline__ uint32_t fp8_pair(float a, float b) {
    return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ uint32_t fp8_quad(float a, float b, float c, float d) { return fp8_pair(a, b) | (fp8_pair(c, d) << 16); }

}  // namespace lb200
