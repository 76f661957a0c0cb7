// Microscaling forms: 32 values that lie together along a row share a scale that is a power of two.
//   rows of activations: e4m3 values, a byte each;  rows of weights: e2m1 values, two in a byte, the lower half first.
// A row is padded to a multiple of 128 values with zeros of scale 1.  A scale is a byte s that stands for 2^(s - 127), 255 for NaN.
// The scales of 128 rows x 128 values are one block of 512 bytes, [row % 32][row / 32][group of 32], which is how the tensor
// cores take them (a lane of tensor memory holds the four groups of rows r, r + 32, r + 64, r + 96); the blocks of a matrix
// are [row / 128][value / 128].  Scales of rows past the end are there and mean nothing.
#pragma once

#include <cuda_fp4.h>
#include <cuda_fp8.h>

#include "common.cuh"

namespace janis {
namespace mx {

constexpr int GROUP = 32;          // values of a scale
constexpr int BLOCK = 128;         // rows and values of a block of scales
constexpr int BLOCK_BYTES = 512;

__host__ __device__ __forceinline__ int padded(int k) { return (k + BLOCK - 1) / BLOCK * BLOCK; }

// where the four scales of row r in value block kb of a matrix of `blocks` value blocks stand
__host__ __device__ __forceinline__ size_t scale_at(int r, int kb, int blocks) {
    return ((size_t)(r / BLOCK) * blocks + kb) * BLOCK_BYTES + (size_t)(r % 32) * 16 + (size_t)(r % BLOCK / 32) * 4;
}

// The byte of the smallest power of two 2^s with big <= 1.M * 2^(P + s), where 1.M * 2^P is the largest value of the type.  Taken
// from the bits of `big`, so exact: its exponent less P, and one more where its mantissa is over M.  Nothing in the group: scale 1.
// An infinity or a NaN in the group: 255, and the whole group stands for NaN.
template <int P, uint32_t MANTISSA>
__device__ __forceinline__ uint32_t scale_byte(float big) {
    const uint32_t b = __float_as_uint(big);
    if (b == 0u) return 127u;
    if (b >= 0x7f800000u) return 255u;
    const int e = (int)(b >> 23) - P + ((b & 0x7fffffu) > MANTISSA ? 1 : 0);
    return (uint32_t)(e > 0 ? e : 0);
}
__device__ __forceinline__ uint32_t scale_byte_e4m3(float big) { return scale_byte<8, 0x600000u>(big); }      // 448 = 1.75 * 2^8
__device__ __forceinline__ uint32_t scale_byte_e2m1(float big) { return scale_byte<2, 0x400000u>(big); }      // 6 = 1.5 * 2^2

// 2^-s for the byte of s, by which a group's values are multiplied before they are rounded; 0 for a group of NaN
__device__ __forceinline__ float inverse_scale(uint32_t byte) {
    return byte == 255u ? 0.f : byte == 254u ? __uint_as_float(0x00400000u) : __uint_as_float((254u - byte) << 23);
}
// 2^s (a NaN for 255, a subnormal for 0)
__device__ __forceinline__ float scale_value(uint32_t byte) {
    return byte == 0u ? __uint_as_float(0x00400000u) : byte == 255u ? __uint_as_float(0x7fc00000u) : __uint_as_float(byte << 23);
}

// two values as e4m3 (the first in the lower byte), or as e2m1 (the first in the lower half); ties go to the even code
__device__ __forceinline__ uint32_t two_e4m3(float a, float b) { return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3); }
__device__ __forceinline__ uint32_t two_e2m1(float a, float b) { return __nv_cvt_float2_to_fp4x2(make_float2(a, b), __NV_E2M1, cudaRoundNearest); }

__device__ __forceinline__ float value_e4m3(uint32_t code) {
    return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)code, __NV_E4M3)));
}
__device__ __forceinline__ float value_e2m1(uint32_t code) {
    return __half2float(__half(__nv_cvt_fp4_to_halfraw((__nv_fp4_storage_t)code, __NV_E2M1)));
}

// largest magnitude that tells of a NaN too (fmaxf would drop it): magnitudes compare as their bits do
__device__ __forceinline__ float larger(float a, float b) {
    return __uint_as_float(max(__float_as_uint(a) & 0x7fffffffu, __float_as_uint(b) & 0x7fffffffu));
}

}  // namespace mx
}  // namespace janis
