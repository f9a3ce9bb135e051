// Rows packed in 8 bits: e4m3 codes with one power-of-two scale for each
// block of 128 columns.
//
//   block b of a row, m = its largest finite magnitude:
//     e     = the smallest integer in [-126, 127] with m <= 448 * 2^e
//     code  = x * 2^-e rounded to the nearest e4m3 value, ties to even
//             (a non-finite x: the NaN code)
//     scale = e + 127, one byte
//
// The scale is a power of two so that x * 2^-e is exact (the only rounding is
// to the code's three fraction bits; one as fine as the block's values allow
// would save nothing, for e4m3's step follows each value's binade), so that a
// decoded value is exact in bf16 (magnitudes from 1.9375 2^127 on round to 2^128,
// which decodes as infinity), and because gfx950's matrix cores multiply
// by scales of this form themselves.
//
// Layout: codes row-major, rows BLOCK8_BLOCK * ceil(cols / 128) bytes apart,
// zero past the columns; scale bytes row-major, rows 4 * ceil(blocks / 4)
// bytes apart, 127 past the blocks. Rows of codes are whole 128-byte lines,
// and four blocks' scales are one aligned word.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace pxg {

constexpr int BLOCK8_BLOCK = 128;
constexpr float BLOCK8_MAX = 448.0f;  // e4m3's largest value

__host__ __device__ inline uint64_t block8_blocks(uint64_t cols) { return (cols + 127) / 128; }
__host__ __device__ inline uint64_t block8_code_stride(uint64_t cols) { return block8_blocks(cols) * 128; }
__host__ __device__ inline uint64_t block8_scale_stride(uint64_t cols) { return (block8_blocks(cols) + 3) / 4 * 4; }

// e + 127 of a block whose largest finite magnitude is m: m is f * 2^x with f
// in [1, 2), and 448 is 1.75 * 2^8, so e is x - 8, or x - 7 when f > 1.75.
// The bounds keep 2^e and 2^-e normal; zero and subnormal m take the lower.
__device__ __forceinline__ uint32_t block8_scale_byte(float m) {
  const uint32_t b = __builtin_bit_cast(uint32_t, m);
  const int s = (int)(b >> 23) - 8 + ((b & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  return (uint32_t)(s < 1 ? 1 : s);
}
// 2^e and 2^-e from a byte that packing writes, 1 to 247.
__device__ __forceinline__ float block8_scale(uint32_t byte) { return __builtin_bit_cast(float, byte << 23); }
__device__ __forceinline__ float block8_inverse(uint32_t byte) {
  return __builtin_bit_cast(float, (254u - byte) << 23);
}

// The values of 8 codes of one block.
__device__ __forceinline__ void block8_decode(const uint32_t (&code)[2], float scale, float (&x)[8]) {
  typedef float f2v __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const f2v a = __builtin_amdgcn_cvt_pk_f32_fp8((int)code[i], false);
    const f2v b = __builtin_amdgcn_cvt_pk_f32_fp8((int)code[i], true);
    x[4 * i] = a[0] * scale;
    x[4 * i + 1] = a[1] * scale;
    x[4 * i + 2] = b[0] * scale;
    x[4 * i + 3] = b[1] * scale;
  }
}

}  // namespace pxg
