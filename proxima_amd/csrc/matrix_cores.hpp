// Fragments of the matrix cores, and reads of operands that end at their tile.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

namespace pxg {

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
#endif

}  // namespace pxg
