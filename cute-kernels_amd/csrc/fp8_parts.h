// The 8-bit block format: e4m3 values and one power-of-two scale (an e8m0 byte b, 2^(b - 127)) per block of 128 elements along a row, or
// per 128 x 128 elements of a weight. What it costs to convert, and the arithmetic that every kernel of the format shares.
//
//   scale = the smallest power of two that brings the block's largest magnitude to 448 (the largest e4m3 value) or less, 2^-126 at the least
//   value = x / scale, rounded to nearest even (the division is exact: only the exponent changes)
//
// A block with an infinity or a NaN has the scale byte 255 (NaN) and NaN values: e4m3 has no infinity, and a value that overflowed must
// not come back as a number. Powers of two because the matrix instruction v_mfma_scale_f32_16x16x128_f8f6f4 applies them to its operands
// at no cost, and because value * scale is then exact in bf16 and fp32 (in fp16 as far as its exponents reach; numbers of 248 * 2^120 and more round up to 2^128).
//
// A row of K elements has ceil(K / 128) scale bytes, filled up with 127 (one) to whole dwords: kernels fetch four at a time.
#pragma once

#include "common.h"

namespace fmahip {
namespace fp8 {

constexpr int kBlock = 128;

constexpr int64_t kMostWorkgroups = (1 << 24) - 1;  // of 256 threads: a launch has fewer than 2^32 threads

__host__ __device__ constexpr int64_t scale_pitch(int64_t K) { return (K + 511) / 512 * 4; }

typedef __attribute__((ext_vector_type(2))) float f32x2;

// the scale byte of a block whose largest magnitude has these bits (the sign bit clear)
__device__ __forceinline__ uint32_t scale_byte(uint32_t amax_bits) {
    if (amax_bits >= 0x7f800000u) return 255u;
    // 448 = 1.75 * 2^8: adding what is missing from 1.75 to 2 carries into the exponent where the mantissa is above 1.75
    const int b = (int)((amax_bits + 0x1fffffu) >> 23) - 8;
    return (uint32_t)(b < 1 ? 1 : b);
}
// what x is multiplied by: 1 / scale, or NaN
__device__ __forceinline__ float scale_inverse(uint32_t byte) {
    return __uint_as_float(byte == 255u ? 0x7fc00000u : (254u - byte) << 23);
}
__device__ __forceinline__ float scale_value(uint32_t byte) {
    return __uint_as_float(byte == 255u ? 0x7fc00000u : byte << 23);
}
// For arithmetic on the values: 2^128, the 8-bit form of the largest numbers, has to stay one, so a scale of 2^120 is one step less (2^-24 of it)
__device__ __forceinline__ float finite_scale_value(uint32_t byte) { return byte == 247u ? __uint_as_float(0x7b7fffffu) : scale_value(byte); }
__device__ __forceinline__ uint32_t magnitude_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }
__device__ __forceinline__ uint32_t max_u32(uint32_t a, uint32_t b) { return a > b ? a : b; }

// four floats of magnitude 448 or less (or NaN) -> four e4m3 bytes, round to nearest even
__device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d) {
    int v = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, v, true);
}
__device__ __forceinline__ void unpack4(uint32_t q, float (&f)[4]) {
    const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)q, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)q, true);
    f[0] = lo[0];
    f[1] = lo[1];
    f[2] = hi[0];
    f[3] = hi[1];
}

// Rows [R, K] in blocks of 1 x 128 as float16, 2^-shift[r] of row r. K a multiple of eight, values aligned to 8 bytes, out to 16.
int dequantize_shifted(const uint8_t* values, const uint8_t* scales, const uint8_t* shift, void* out, int64_t R, int64_t K, hipStream_t st);

// largest of v over a group of LANES neighbouring lanes
template <int LANES>
__device__ __forceinline__ uint32_t group_max(uint32_t v) {
#pragma unroll
    for (int d = 1; d < LANES; d <<= 1) v = max_u32(v, (uint32_t)__shfl_xor((int)v, d, kWave));
    return v;
}

}  // namespace fp8
}  // namespace fmahip
