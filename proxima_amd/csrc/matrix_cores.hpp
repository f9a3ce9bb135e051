// Fragments of the matrix cores, and reads of operands that end at their tile.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

namespace pxg {

typedef uint32_t u4w __attribute__((ext_vector_type(4)));
typedef int i8v __attribute__((ext_vector_type(8)));
typedef float f4v __attribute__((ext_vector_type(4)));
typedef __bf16 bf8v __attribute__((ext_vector_type(8)));
typedef _Float16 hf8v __attribute__((ext_vector_type(8)));

template <class T>
__device__ __forceinline__ f4v mfma16(uint4 a, uint4 b, f4v c) {
  if constexpr (std::is_same_v<T, __bf16>)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8v, a), __builtin_bit_cast(bf8v, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(hf8v, a), __builtin_bit_cast(hf8v, b), c, 0, 0, 0);
}

#if defined(__HIP_DEVICE_COMPILE__)
// A raw buffer resource over [p, p + bytes), from wave-uniform scalars;
// accesses at offsets outside it read zeros.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t tile_rsrc(const void* p, uint64_t bytes) {
  const uint64_t a = (uint64_t)(uintptr_t)p;
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)a);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(a >> 32));
  const int n = __builtin_amdgcn_readfirstlane((int)(uint32_t)(bytes < 0x7FFFFFFF ? bytes : 0x7FFFFFFF));
  return __builtin_amdgcn_make_buffer_rsrc((void*)(uintptr_t)(((uint64_t)hi << 32) | lo), 0, n, 0x00020000);
}

constexpr uint32_t NOWHERE = 0xFFFFFF00u;  // an offset outside every resource

// 8 codes times their scale, in bf16.
__device__ __forceinline__ uint4 decode_bf16(uint32_t x, uint32_t y, float s) {
  typedef __bf16 bf2v __attribute__((ext_vector_type(2)));
  const bf2v a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, s, false);
  const bf2v b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, s, true);
  const bf2v c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(y, s, false);
  const bf2v d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(y, s, true);
  return make_uint4(__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b), __builtin_bit_cast(uint32_t, c),
                    __builtin_bit_cast(uint32_t, d));
}

// 8 16-bit elements of a row that a resource covers, from byte `at` of it on.
// ANY: rows begin at any multiple of two bytes; the words that hold them are
// read and shifted.
template <bool ANY>
struct Piece {
  uint4 v;
  [[maybe_unused]] uint32_t last;
};
template <bool ANY>
__device__ __forceinline__ Piece<ANY> load_piece(__amdgpu_buffer_rsrc_t rs, uint32_t at, bool in) {
  Piece<ANY> x;
  x.v = __builtin_bit_cast(uint4, (u4w)__builtin_amdgcn_raw_buffer_load_b128(rs, (int)(in ? at & ~3u : NOWHERE), 0, 0));
  if constexpr (ANY) x.last = __builtin_amdgcn_raw_buffer_load_b32(rs, (int)(in ? (at & ~3u) + 16 : NOWHERE), 0, 0);
  return x;
}
// The elements, zeros from the `valid`-th on (without ANY all of them or none are).
template <bool ANY>
__device__ __forceinline__ uint4 elements(const Piece<ANY>& x, uint32_t at, int valid) {
  if constexpr (!ANY) {
    return x.v;
  } else {
    const uint32_t w[5] = {x.v.x, x.v.y, x.v.z, x.v.w, x.last}, shift = (at & 2) * 8;
    uint32_t v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t both = __builtin_amdgcn_alignbit(w[e + 1], w[e], shift);
      v[e] = valid > 2 * e + 1 ? both : valid > 2 * e ? both & 0xFFFF : 0;
    }
    return make_uint4(v[0], v[1], v[2], v[3]);
  }
}
// A resource over rows of 16-bit elements whose last ends `bytes` from p on, and
// what an offset of it begins at.
template <bool ANY>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_rsrc(const char* p, uint64_t bytes, uint32_t& odd) {
  odd = ANY ? (uint32_t)(uintptr_t)p & 2 : 0;
  return tile_rsrc(p - odd, ANY ? (bytes + odd + 3) & ~3ull : bytes);
}
#endif

}  // namespace pxg
