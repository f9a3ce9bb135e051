// The activations of expert layers and their slopes.
#pragma once

#include <hip/hip_runtime.h>

#include "common.hpp"

namespace pxg {

// f(h) and f'(h) of the activations:
//   silu: h s, s = 1 / (1 + exp(-h));  s (1 + h (1 - s))
//   gelu: h P, P = (1 + erf(h / sqrt 2)) / 2;  P + h exp(-h^2 / 2) / sqrt(2 pi)
//
// f32 takes the math library's functions. For 16-bit types these would cost
// more than the memory (gelu's backward pass, 16384 x 4096 in bf16: 90 us with
// them), so they take the hardware's exp2 and reciprocal, and for gelu one
// polynomial: 1 - P(|h|) = exp(-h^2 / 2) t R(t), t = 1 / (1 + 0.28 |h|), with R
// the polynomial of degree 8 of least largest relative error over all h
// (1.7e-7). Evaluated in f32 the tail is off by 6e-7 of itself up to |h| = 3,
// 2e-6 to 6 and 7.4e-6 at 13, from the rounding of h^2 in the exponent; half of
// f16's last place is 2^-11, 4.9e-4. SiLU's exp is off by 5e-6 where it is
// largest. The tail's exp is the slope's second term's too.
template <class T>
constexpr bool fast_activation = sizeof(T) == 2;

__device__ __forceinline__ float fast_exp(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504f); }

// 1 - P(|h|), and exp(-h^2 / 2).
__device__ __forceinline__ float gelu_tail(float h, float& e) {
  const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.28f, fabsf(h), 1.0f));
  float r = 0.0247248504f;
  r = __builtin_fmaf(r, t, -0.0936122835f);
  r = __builtin_fmaf(r, t, 0.0924588069f);
  r = __builtin_fmaf(r, t, -0.00647497689f);
  r = __builtin_fmaf(r, t, 0.0727872029f);
  r = __builtin_fmaf(r, t, 0.0836275741f);
  r = __builtin_fmaf(r, t, 0.103085108f);
  r = __builtin_fmaf(r, t, 0.111699775f);
  r = __builtin_fmaf(r, t, 0.111703858f);
  e = __builtin_amdgcn_exp2f(h * h * -0.72134752f);
  return e * (t * r);
}

template <class T, int ACT>
__device__ __forceinline__ float act_value(float h) {
  if constexpr (ACT == PXG_SILU) {
    if constexpr (fast_activation<T>) return h * __builtin_amdgcn_rcpf(1.0f + fast_exp(-h));
    return h / (1.0f + expf(-h));
  }
  if constexpr (fast_activation<T>) {
    float e;
    const float q = gelu_tail(h, e);
    return h * (h < 0.0f ? q : 1.0f - q);
  }
  return h * (0.5f * (1.0f + erff(h * 0.70710678f)));
}
template <class T, int ACT>
__device__ __forceinline__ float act_slope(float h) {
  if constexpr (ACT == PXG_SILU) {
    float s;
    if constexpr (fast_activation<T>) s = __builtin_amdgcn_rcpf(1.0f + fast_exp(-h));
    else s = 1.0f / (1.0f + expf(-h));
    return s * (1.0f + h * (1.0f - s));
  }
  if constexpr (fast_activation<T>) {
    float e;
    const float q = gelu_tail(h, e);
    return __builtin_fmaf(h * 0.39894228f, e, h < 0.0f ? q : 1.0f - q);
  }
  const float p = 0.5f * (1.0f + erff(h * 0.70710678f));
  return p + h * (0.39894228f * expf(-0.5f * h * h));
}

// f(v) in place, evaluated as precisely as a result of type O shows.
template <class O, int N>
__device__ __forceinline__ void activate(float (&v)[N], int activation) {
  if (activation == PXG_GELU) {
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = act_value<O, PXG_GELU>(v[e]);
  } else if (activation == PXG_SILU) {
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = act_value<O, PXG_SILU>(v[e]);
  }
}

constexpr int NO_ACTIVATION = -1;

inline void check_activation(int64_t kind) {
  if (kind != PXG_SILU && kind != PXG_GELU) config_error("activation", (uint64_t)kind, "must be SiLU or GELU");
}
inline void check_optional_activation(int64_t kind) {
  if (kind != NO_ACTIVATION) check_activation(kind);
}

}  // namespace pxg
