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

#include "activation.hpp"
#include "block8.hpp"
#include "common.hpp"
#include "device.hpp"
#include "products.hpp"
#include "rows.hpp"

namespace pxg {
namespace {

constexpr int ROW_THREADS = 256;

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

void check_packed(uint64_t rows, uint64_t cols, const void* codes, const void* scales) {
  check_size("cols", cols);
  check_packed_rows("codes", codes, "scales", scales, rows);
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
