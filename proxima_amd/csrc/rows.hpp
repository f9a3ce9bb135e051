// Rows of f32, f16 or bf16 read and written 8 columns a thread.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "../../include/proxima_hip.h"

namespace pxg {

template <class T>
__device__ __forceinline__ float to_float(T x) {
  return (float)x;
}

// 8 columns of a row from column c: one or two 16-byte loads where VEC (the
// row 16-byte aligned) and all eight exist, else one by one, zero past cols.
template <class T, bool VEC>
__device__ __forceinline__ void load8(const T* __restrict__ row, uint64_t c, uint64_t cols, float (&x)[8]) {
  if (VEC && c + 8 <= cols) {
    T v[8];
    const uint4* p = reinterpret_cast<const uint4*>(row + c);
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4*>(v)[i] = p[i];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_float(v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = c + i < cols ? to_float(row[c + i]) : 0.0f;
  }
}

// 16 bytes that are read or written once: the caches keep others.
typedef uint32_t u4v __attribute__((ext_vector_type(4)));
__device__ __forceinline__ uint4 load_once(const void* p) {
  return __builtin_bit_cast(uint4, __builtin_nontemporal_load((const u4v*)p));
}
__device__ __forceinline__ void store_once(void* p, uint4 x) {
  __builtin_nontemporal_store(__builtin_bit_cast(u4v, x), (u4v*)p);
}

// The same, left packed in T and read once.
template <class T>
struct Eight {
  uint4 q[sizeof(T) / 2];
  __device__ __forceinline__ void unpack(float (&x)[8]) const {
    T v[8];
    __builtin_memcpy(v, q, sizeof(v));
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_float(v[i]);
  }
};
template <class T, bool VEC>
__device__ __forceinline__ Eight<T> raw8(const T* __restrict__ row, uint64_t c, uint64_t cols) {
  Eight<T> x;
  if (VEC && c + 8 <= cols) {
    const uint4* p = reinterpret_cast<const uint4*>(row + c);
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) x.q[i] = load_once(p + i);
  } else {
    T v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c + i < cols ? row[c + i] : (T)0.0f;
    __builtin_memcpy(x.q, v, sizeof(v));
  }
  return x;
}

// One rounding of the f32 value: kept apart from the product before it, which
// the compiler may otherwise fuse into the conversion to f16 in some variants
// of a kernel and not in others.
template <class T>
__device__ __forceinline__ T rounded(float x) {
  if constexpr (std::is_same_v<T, _Float16>) asm("" : "+v"(x));
  return (T)x;
}

template <class T, bool VEC>
__device__ __forceinline__ void store8(T* __restrict__ row, uint64_t c, uint64_t cols, const float (&x)[8]) {
  if (VEC && c + 8 <= cols) {
    T v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = rounded<T>(x[i]);
    uint4* p = reinterpret_cast<uint4*>(row + c);
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) p[i] = reinterpret_cast<uint4*>(v)[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < cols) row[c + i] = rounded<T>(x[i]);
  }
}

// Calls f with a value of the element type and whether 16-byte accesses are
// aligned in every row.
template <class F>
inline void by_type(int type, bool vec, F f) {
  auto g = [&](auto t) {
    if (vec) f(t, std::true_type{});
    else f(t, std::false_type{});
  };
  if (type == PXG_F32) g(float{});
  else if (type == PXG_F16) g((_Float16)0);
  else g((__bf16)0.0f);
}

}  // namespace pxg
