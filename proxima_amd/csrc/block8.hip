// Packing rows in 8 bits (block8.hpp), and the activations whose input is
// kept that way for their backward pass. All of these read and write each
// element once; a thread takes 8 columns, so the 16 threads of a block of 128
// columns exchange its largest magnitude in registers.
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
// block call it together.
__device__ __forceinline__ uint32_t pack8(const float (&x)[8], uint32_t (&code)[2]) {
  uint32_t m = 0;  // magnitudes order as their bits; infinities and NaN are left out
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x[i]) & 0x7FFFFFFFu;
    const uint32_t f = b < 0x7F800000u ? b : 0u;
    m = f > m ? f : m;
  }
  uint32_t o;
  o = xor_lane<1>(m), m = o > m ? o : m;
  o = xor_lane<2>(m), m = o > m ? o : m;
  o = xor_lane<4>(m), m = o > m ? o : m;
  o = xor_lane<8>(m), m = o > m ? o : m;
  const uint32_t byte = block8_scale_byte(__builtin_bit_cast(float, m));
  const float inv = block8_inverse(byte);
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x[i]) & 0x7FFFFFFFu;
    y[i] = b < 0x7F800000u ? x[i] * inv : __builtin_bit_cast(float, 0x7FC00000u);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * i], y[4 * i + 1], 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * i + 2], y[4 * i + 3], w, true);
    code[i] = (uint32_t)w;
  }
  return byte;
}

// Where thread `item` of a launch over rows of `wide` (a multiple of 128)
// columns is.
struct Place {
  uint64_t row;
  uint32_t col;
  bool live;
  __device__ Place(uint32_t rows, uint32_t wide) {
    const uint32_t item = blockIdx.x * ROW_THREADS + threadIdx.x, per = wide / 8;
    const uint32_t r = item / per;
    row = r;
    col = (item - r * per) * 8;
    live = r < rows;  // uniform over the 16 threads of a block: per is a multiple of 16
  }
};

// The scale byte of a block, and 127 in the bytes past the row's last block.
__device__ __forceinline__ void store_scale(uint8_t* __restrict__ scales, const Place& at, uint32_t wide,
                                            uint32_t sstride, uint32_t byte) {
  if (at.col % 128) return;
  uint8_t* s = scales + at.row * sstride;
  const uint32_t b = at.col / 128;
  s[b] = (uint8_t)byte;
  if (b == wide / 128 - 1)
    for (uint32_t i = b + 1; i < sstride; ++i) s[i] = 127;
}

template <class T, bool VEC>
__global__ void __launch_bounds__(ROW_THREADS)
block8_pack_rows(const T* __restrict__ x, uint64_t xs, uint32_t rows, uint32_t cols, uint32_t wide, uint32_t sstride,
                 uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
  const Place at(rows, wide);
  if (!at.live) return;
  float v[8];
  load8<T, VEC>(x + at.row * xs, at.col, cols, v);
  uint32_t code[2];
  const uint32_t byte = pack8(v, code);
  *reinterpret_cast<uint2*>(codes + at.row * wide + at.col) = make_uint2(code[0], code[1]);
  store_scale(scales, at, wide, sstride, byte);
}

template <class T, bool VEC>
__global__ void __launch_bounds__(ROW_THREADS)
block8_unpack_rows(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, uint32_t rows, uint32_t cols,
                   uint32_t wide, uint32_t sstride, T* __restrict__ out, uint64_t os) {
  const Place at(rows, wide);
  if (!at.live) return;
  const uint2 w = *reinterpret_cast<const uint2*>(codes + at.row * wide + at.col);
  const uint32_t code[2] = {w.x, w.y};
  float v[8];
  block8_decode(code, block8_scale(scales[at.row * sstride + at.col / 128]), v);
  store8<T, VEC>(out + at.row * os, at.col, cols, v);
}

// f(h) and f'(h) of the activations:
//   silu: h s, s = 1 / (1 + exp(-h));  s (1 + h (1 - s))
//   gelu: h P, P = (1 + erf(h / sqrt 2)) / 2;  P + h exp(-h^2 / 2) / sqrt(2 pi)
template <int ACT>
__device__ __forceinline__ float act_value(float h) {
  if constexpr (ACT == PXG_SILU) return h / (1.0f + expf(-h));
  return h * (0.5f * (1.0f + erff(h * 0.70710678f)));
}
template <int ACT>
__device__ __forceinline__ float act_slope(float h) {
  if constexpr (ACT == PXG_SILU) {
    const float s = 1.0f / (1.0f + expf(-h));
    return s * (1.0f + h * (1.0f - s));
  }
  const float p = 0.5f * (1.0f + erff(h * 0.70710678f));
  return p + h * (0.39894228f * expf(-0.5f * h * h));
}

template <class T, bool VEC, int ACT>
__global__ void __launch_bounds__(ROW_THREADS)
activation_pack_rows(const T* __restrict__ h, uint64_t hs, uint32_t rows, uint32_t cols, uint32_t wide,
                     uint32_t sstride, T* __restrict__ a, uint64_t as, uint8_t* __restrict__ codes,
                     uint8_t* __restrict__ scales) {
  const Place at(rows, wide);
  if (!at.live) return;
  float v[8], f[8];
  load8<T, VEC>(h + at.row * hs, at.col, cols, v);
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = act_value<ACT>(v[i]);
  store8<T, VEC>(a + at.row * as, at.col, cols, f);
  uint32_t code[2];
  const uint32_t byte = pack8(v, code);
  *reinterpret_cast<uint2*>(codes + at.row * wide + at.col) = make_uint2(code[0], code[1]);
  store_scale(scales, at, wide, sstride, byte);
}

template <class T, bool VEC, int ACT>
__global__ void __launch_bounds__(ROW_THREADS)
activation_grad_rows(const T* __restrict__ g, uint64_t gs, uint32_t rows, uint32_t cols, uint32_t wide,
                     uint32_t sstride, const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                     T* __restrict__ out, uint64_t os) {
  const Place at(rows, wide);
  if (!at.live) return;
  float v[8], d[8];
  load8<T, VEC>(g + at.row * gs, at.col, cols, d);
  const uint2 w = *reinterpret_cast<const uint2*>(codes + at.row * wide + at.col);
  const uint32_t code[2] = {w.x, w.y};
  block8_decode(code, block8_scale(scales[at.row * sstride + at.col / 128]), v);
#pragma unroll
  for (int i = 0; i < 8; ++i) d[i] *= act_slope<ACT>(v[i]);
  store8<T, VEC>(out + at.row * os, at.col, cols, d);
}

// A launch's rows are bounded so that its threads count in 31 bits.
template <class F>
void by_rows(uint64_t rows, uint64_t wide, F launch) {
  const uint64_t per = wide / 8, most = ((1ull << 31) - 1) / per;
  for (uint64_t r = 0; r < rows; r += most) {
    const uint64_t m = rows - r < most ? rows - r : most;
    launch(r, (uint32_t)m, dim3((unsigned)((m * per + ROW_THREADS - 1) / ROW_THREADS)));
    PXG_HIP(hipGetLastError());
  }
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
      by_rows(rows, wide, [&](uint64_t r, uint32_t m, dim3 grid) {
        hipLaunchKernelGGL((block8_pack_rows<T, decltype(vec)::value>), grid, dim3(ROW_THREADS), 0,
                           (hipStream_t)stream, (const T*)d_x + r * x_stride, x_stride, m, (uint32_t)cols,
                           (uint32_t)wide, (uint32_t)ss, (uint8_t*)d_codes + r * wide, (uint8_t*)d_scales + r * ss);
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
      by_rows(rows, wide, [&](uint64_t r, uint32_t m, dim3 grid) {
        hipLaunchKernelGGL((block8_unpack_rows<T, decltype(vec)::value>), grid, dim3(ROW_THREADS), 0,
                           (hipStream_t)stream, (const uint8_t*)d_codes + r * wide,
                           (const uint8_t*)d_scales + r * ss, m, (uint32_t)cols, (uint32_t)wide, (uint32_t)ss,
                           (T*)d_out + r * out_stride, out_stride);
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
      by_rows(rows, wide, [&](uint64_t r, uint32_t m, dim3 grid) {
        auto kernel = activation == PXG_SILU ? activation_pack_rows<T, V, PXG_SILU>
                                             : activation_pack_rows<T, V, PXG_GELU>;
        hipLaunchKernelGGL(kernel, grid, dim3(ROW_THREADS), 0, (hipStream_t)stream, (const T*)d_h + r * h_stride,
                           h_stride, m, (uint32_t)cols, (uint32_t)wide, (uint32_t)ss, (T*)d_a + r * a_stride,
                           a_stride, (uint8_t*)d_codes + r * wide, (uint8_t*)d_scales + r * ss);
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
      by_rows(rows, wide, [&](uint64_t r, uint32_t m, dim3 grid) {
        auto kernel = activation == PXG_SILU ? activation_grad_rows<T, V, PXG_SILU>
                                             : activation_grad_rows<T, V, PXG_GELU>;
        hipLaunchKernelGGL(kernel, grid, dim3(ROW_THREADS), 0, (hipStream_t)stream,
                           (const T*)d_grad + r * grad_stride, grad_stride, m, (uint32_t)cols, (uint32_t)wide,
                           (uint32_t)ss, (const uint8_t*)d_codes + r * wide, (const uint8_t*)d_scales + r * ss,
                           (T*)d_out + r * out_stride, out_stride);
      });
    });
  });
}

}  // extern "C"
