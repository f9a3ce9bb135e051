// Packing rows in 8 bits (block8.hpp), and the activations whose input is
// kept that way for their backward pass. All of these read and write each
// element once, and memory bounds them; a thread takes 8 columns, one access of
// 16 bytes, so the 16 threads of a block of 128 columns exchange its largest
// magnitude in registers. 16384 x 4096 in bf16 takes 58 (SiLU) and 65 us (GELU)
// with the packed input, its gradient 60 and 63 (a copy of as many bytes: 65).
// Results are rounded to their type once, from f32; what is packed is the
// rounded input itself.
#include <algorithm>
#include <cmath>

#include "block8.hpp"
#include "common.hpp"
#include "device.hpp"
#include "products.hpp"

namespace pxg {
namespace {

constexpr int ROW_THREADS = 256;

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

// The codes of 8 columns and their block's scale byte; all 16 threads of a
// block call it together. The maximum passes NaN over, and NaN times a scale
// becomes the NaN code by itself; infinities, which neither does, take the
// branch.
__device__ __forceinline__ uint32_t pack8(const float (&x)[8], uint32_t (&code)[2]) {
  constexpr float INF = __builtin_inff();
  float y[8];
  float m = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    y[i] = x[i];
    m = fmaxf(m, fabsf(x[i]));
  }
  if (m == INF) {
    m = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (fabsf(y[i]) == INF) y[i] = __builtin_nanf("");
      m = fmaxf(m, fabsf(y[i]));
    }
  }
  auto other = [&](uint32_t o) { m = fmaxf(m, __builtin_bit_cast(float, o)); };
  other(xor_lane<1>(__builtin_bit_cast(uint32_t, m)));
  other(xor_lane<2>(__builtin_bit_cast(uint32_t, m)));
  other(xor_lane<4>(__builtin_bit_cast(uint32_t, m)));
  other(xor_lane<8>(__builtin_bit_cast(uint32_t, m)));
  const uint32_t byte = block8_scale_byte(m);
  const float inv = block8_inverse(byte);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * i] * inv, y[4 * i + 1] * inv, 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * i + 2] * inv, y[4 * i + 3] * inv, w, true);
    code[i] = (uint32_t)w;
  }
  return byte;
}

// Where a thread begins: threads of a workgroup are blockDim.x / 16 blocks of
// 128 columns by blockDim.y rows. The rows are the grid's x; its y are column
// parts.
struct Place {
  uint64_t row;
  uint32_t col, step;
  __device__ Place() {
    row = (uint64_t)blockIdx.x * blockDim.y + threadIdx.y;
    col = (blockIdx.y * blockDim.x + threadIdx.x) * 8;
    step = gridDim.y * blockDim.x * 8;
  }
};

// The scale byte of a block, and 127 in the bytes past the row's last block.
__device__ __forceinline__ void store_scale(uint8_t* __restrict__ scales, const Place& at, uint32_t wide,
                                            uint32_t sstride, uint32_t col, uint32_t byte) {
  if (col % 128) return;
  uint8_t* s = scales + at.row * sstride;
  const uint32_t b = col / 128;
  s[b] = (uint8_t)byte;
  if (b == wide / 128 - 1)
    for (uint32_t i = b + 1; i < sstride; ++i) s[i] = 127;
}

template <class T, bool VEC>
__global__ void __launch_bounds__(ROW_THREADS)
block8_pack_rows(const T* __restrict__ x, uint64_t xs, uint32_t rows, uint32_t cols, uint32_t wide, uint32_t sstride,
                 uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
  const Place at;
  if (at.row >= rows) return;
  for (uint32_t col = at.col; col < wide; col += at.step) {
    float v[8];
    load8<T, VEC>(x + at.row * xs, col, cols, v);
    uint32_t code[2];
    const uint32_t byte = pack8(v, code);
    *reinterpret_cast<uint2*>(codes + at.row * wide + col) = make_uint2(code[0], code[1]);
    store_scale(scales, at, wide, sstride, col, byte);
  }
}

template <class T, bool VEC>
__global__ void __launch_bounds__(ROW_THREADS)
block8_unpack_rows(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, uint32_t rows, uint32_t cols,
                   uint32_t wide, uint32_t sstride, T* __restrict__ out, uint64_t os) {
  const Place at;
  if (at.row >= rows) return;
  for (uint32_t col = at.col; col < wide; col += at.step) {
    const uint2 w = *reinterpret_cast<const uint2*>(codes + at.row * wide + col);
    const uint32_t code[2] = {w.x, w.y};
    float v[8];
    block8_decode(code, block8_scale(scales[at.row * sstride + col / 128]), v);
    store8<T, VEC>(out + at.row * os, col, cols, v);
  }
}

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

template <class T, bool VEC, int ACT>
__global__ void __launch_bounds__(ROW_THREADS)
activation_pack_rows(const T* __restrict__ h, uint64_t hs, uint32_t rows, uint32_t cols, uint32_t wide,
                     uint32_t sstride, T* __restrict__ a, uint64_t as, uint8_t* __restrict__ codes,
                     uint8_t* __restrict__ scales) {
  const Place at;
  if (at.row >= rows) return;
  for (uint32_t col = at.col; col < wide; col += at.step) {
    float v[8], f[8];
    load8<T, VEC>(h + at.row * hs, col, cols, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = act_value<T, ACT>(v[i]);
    store8<T, VEC>(a + at.row * as, col, cols, f);
    uint32_t code[2];
    const uint32_t byte = pack8(v, code);
    *reinterpret_cast<uint2*>(codes + at.row * wide + col) = make_uint2(code[0], code[1]);
    store_scale(scales, at, wide, sstride, col, byte);
  }
}

template <class T, bool VEC, int ACT>
__global__ void __launch_bounds__(ROW_THREADS)
activation_grad_rows(const T* __restrict__ g, uint64_t gs, uint32_t rows, uint32_t cols, uint32_t wide,
                     uint32_t sstride, const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                     T* __restrict__ out, uint64_t os) {
  const Place at;
  if (at.row >= rows) return;
  for (uint32_t col = at.col; col < wide; col += at.step) {
    float v[8], d[8];
    load8<T, VEC>(g + at.row * gs, col, cols, d);
    const uint2 w = *reinterpret_cast<const uint2*>(codes + at.row * wide + col);
    const uint32_t code[2] = {w.x, w.y};
    block8_decode(code, block8_scale(scales[at.row * sstride + col / 128]), v);
#pragma unroll
    for (int i = 0; i < 8; ++i) d[i] *= act_slope<T, ACT>(v[i]);
    store8<T, VEC>(out + at.row * os, col, cols, d);
  }
}

// Calls launch(grid, block, first, count) for rows first to first + count, with
// a thread for 8 columns: workgroups of one row's 2048 columns, or of several
// rows of fewer. A launch has less than 2^32 work-items along x, so more rows
// take several (the rest along z instead, and a row's index from both, cost all
// calls 4 to 8%: GELU's gradient, 16384 x 4096 in bf16, 61 us, 65).
template <class F>
void by_rows(uint64_t rows, uint64_t wide, F launch) {
  uint64_t x = 16;
  while (x < ROW_THREADS && x * 8 < wide) x *= 2;
  const uint64_t y = ROW_THREADS / x, parts = (wide / 8 + x - 1) / x;
  by_launches((rows + y - 1) / y, [&](uint64_t a, uint64_t m) {
    launch(dim3((unsigned)m, (unsigned)(parts < 1024 ? parts : 1024)), dim3((unsigned)x, (unsigned)y), a * y,
           std::min(rows - a * y, m * y));
    PXG_HIP(hipGetLastError());
  });
}

// Calls f with a value of the element type and whether 16-byte accesses are
// aligned in every row.
template <class F>
void by_type(int type, bool vec, F f) {
  auto g = [&](auto t) {
    if (vec) f(t, std::true_type{});
    else f(t, std::false_type{});
  };
  if (type == PXG_F32) g(float{});
  else if (type == PXG_F16) g((_Float16)0);
  else g((__bf16)0.0f);
}

void check_packed(uint64_t rows, uint64_t cols, const void* codes, const void* scales) {
  check_size("cols", cols);
  check_packed_rows("codes", codes, "scales", scales, rows);
}

void check_activation(int kind) {
  if (kind != PXG_SILU && kind != PXG_GELU) config_error("activation", (uint64_t)kind, "must be SiLU or GELU");
}

}  // namespace
}  // namespace pxg

using namespace pxg;

extern "C" {

uint64_t pxg_block8_code_stride(uint64_t cols) { return block8_code_stride(cols); }
uint64_t pxg_block8_scale_stride(uint64_t cols) { return block8_scale_stride(cols); }

int pxg_block8_pack_device(int type, const void* d_x, uint64_t rows, uint64_t cols, uint64_t x_stride, void* d_codes,
                           void* d_scales, void* stream) {
  return guard([&] {
    check_type(type, true);
    check_packed(rows, cols, d_codes, d_scales);
    check_rows(type, "x", d_x, rows, cols, x_stride);
    if (rows == 0) return;
    const uint64_t wide = block8_code_stride(cols), ss = block8_scale_stride(cols);
    by_type(type, rows_aligned(type, d_x, x_stride), [&](auto t, auto vec) {
      using T = decltype(t);
      by_rows(rows, wide, [&](dim3 grid, dim3 block, uint64_t at, uint64_t count) {
        hipLaunchKernelGGL((block8_pack_rows<T, decltype(vec)::value>), grid, block, 0,
                           (hipStream_t)stream, (const T*)d_x + at * x_stride, x_stride, (uint32_t)count,
                           (uint32_t)cols, (uint32_t)wide, (uint32_t)ss, (uint8_t*)d_codes + at * wide,
                           (uint8_t*)d_scales + at * ss);
      });
    });
  });
}

int pxg_block8_unpack_device(int type, const void* d_codes, const void* d_scales, uint64_t rows, uint64_t cols,
                             void* d_out, uint64_t out_stride, void* stream) {
  return guard([&] {
    check_type(type, true);
    check_packed(rows, cols, d_codes, d_scales);
    check_rows(type, "out", d_out, rows, cols, out_stride);
    if (rows == 0) return;
    const uint64_t wide = block8_code_stride(cols), ss = block8_scale_stride(cols);
    by_type(type, rows_aligned(type, d_out, out_stride), [&](auto t, auto vec) {
      using T = decltype(t);
      by_rows(rows, wide, [&](dim3 grid, dim3 block, uint64_t at, uint64_t count) {
        hipLaunchKernelGGL((block8_unpack_rows<T, decltype(vec)::value>), grid, block, 0,
                           (hipStream_t)stream, (const uint8_t*)d_codes + at * wide,
                           (const uint8_t*)d_scales + at * ss, (uint32_t)count, (uint32_t)cols, (uint32_t)wide,
                           (uint32_t)ss, (T*)d_out + at * out_stride, out_stride);
      });
    });
  });
}

int pxg_activation_pack_device(int activation, int type, const void* d_h, uint64_t rows, uint64_t cols,
                               uint64_t h_stride, void* d_a, uint64_t a_stride, void* d_codes, void* d_scales,
                               void* stream) {
  return guard([&] {
    check_activation(activation);
    check_type(type, true);
    check_packed(rows, cols, d_codes, d_scales);
    check_rows(type, "h", d_h, rows, cols, h_stride);
    check_rows(type, "a", d_a, rows, cols, a_stride);
    if (rows == 0) return;
    const uint64_t wide = block8_code_stride(cols), ss = block8_scale_stride(cols);
    const bool vec = rows_aligned(type, d_h, h_stride) && rows_aligned(type, d_a, a_stride);
    by_type(type, vec, [&](auto t, auto v) {
      using T = decltype(t);
      constexpr bool V = decltype(v)::value;
      by_rows(rows, wide, [&](dim3 grid, dim3 block, uint64_t at, uint64_t count) {
        auto kernel = activation == PXG_SILU ? activation_pack_rows<T, V, PXG_SILU>
                                             : activation_pack_rows<T, V, PXG_GELU>;
        hipLaunchKernelGGL(kernel, grid, block, 0, (hipStream_t)stream, (const T*)d_h + at * h_stride,
                           h_stride, (uint32_t)count, (uint32_t)cols, (uint32_t)wide, (uint32_t)ss,
                           (T*)d_a + at * a_stride, a_stride, (uint8_t*)d_codes + at * wide,
                           (uint8_t*)d_scales + at * ss);
      });
    });
  });
}

int pxg_activation_grad_device(int activation, int type, const void* d_grad, uint64_t rows, uint64_t cols,
                               uint64_t grad_stride, const void* d_codes, const void* d_scales, void* d_out,
                               uint64_t out_stride, void* stream) {
  return guard([&] {
    check_activation(activation);
    check_type(type, true);
    check_packed(rows, cols, d_codes, d_scales);
    check_rows(type, "grad", d_grad, rows, cols, grad_stride);
    check_rows(type, "out", d_out, rows, cols, out_stride);
    if (rows == 0) return;
    const uint64_t wide = block8_code_stride(cols), ss = block8_scale_stride(cols);
    const bool vec = rows_aligned(type, d_grad, grad_stride) && rows_aligned(type, d_out, out_stride);
    by_type(type, vec, [&](auto t, auto v) {
      using T = decltype(t);
      constexpr bool V = decltype(v)::value;
      by_rows(rows, wide, [&](dim3 grid, dim3 block, uint64_t at, uint64_t count) {
        auto kernel = activation == PXG_SILU ? activation_grad_rows<T, V, PXG_SILU>
                                             : activation_grad_rows<T, V, PXG_GELU>;
        hipLaunchKernelGGL(kernel, grid, block, 0, (hipStream_t)stream,
                           (const T*)d_grad + at * grad_stride, grad_stride, (uint32_t)count, (uint32_t)cols,
                           (uint32_t)wide, (uint32_t)ss, (const uint8_t*)d_codes + at * wide,
                           (const uint8_t*)d_scales + at * ss, (T*)d_out + at * out_stride, out_stride);
      });
    });
  });
}

}  // extern "C"
