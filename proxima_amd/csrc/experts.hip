// Matrix products of rows in ragged groups, each group with a matrix of its
// own (expert layers), their gradients, and the same product over packed
// 8-bit rows (block8.hpp).
//
//   forward      y[t, :]  = x[t, :] w_g^T        t in group g, w_g n x k
//   grad input   dx[t, :] = dy[t, :] w_g
//   grad weight  dw_g     = sum over t in g of dy[t, :]^T x[t, :]
//
// Every sum is held in f32 on the matrix cores and rounded once, to the
// output's type.
#include <type_traits>

#include "block8.hpp"
#include "common.hpp"
#include "device.hpp"
#include "groups.hpp"
#include "products.hpp"

namespace pxg {
namespace {

typedef float f4v __attribute__((ext_vector_type(4)));
typedef __bf16 bf8v __attribute__((ext_vector_type(8)));
typedef _Float16 hf8v __attribute__((ext_vector_type(8)));

enum Form { FORWARD, GRAD_INPUT, GRAD_WEIGHT };

// One call. Row-major operands, strides in elements: A is x or dy, B is w
// (forward, grad input) or x (grad weight), C the result. m, n, k are the
// product's own: C is m x n (per group for grad weight) and k is summed.
struct Product {
  const void* a;
  const void* b;
  void* c;
  const int64_t* offsets;
  uint64_t as, bs, cs;  // row strides
  uint64_t bg, cg;      // strides of a group's matrix in B and C
  // packed operands (a and b hold codes): their scale bytes, rows ss apart
  const uint8_t *a_scales, *b_scales;
  uint64_t ss;
  int rows, groups;     // rows of x and dy
  int m, n, k;
};

template <class T>
__device__ __forceinline__ f4v mfma16(uint4 a, uint4 b, f4v c) {
  if constexpr (std::is_same_v<T, __bf16>)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8v, a), __builtin_bit_cast(bf8v, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(hf8v, a), __builtin_bit_cast(hf8v, b), c, 0, 0, 0);
}

// ---------------------------------------------------------------------------
// Any stride and alignment: 64 x 64 tiles, 32 summed at a time, staged in LDS
// element by element with zeros outside the operands.
// ---------------------------------------------------------------------------
constexpr int ANY_TILE = 64, ANY_K = 32;
constexpr int ANY_LD = ANY_K + 8;  // LDS rows of 80 bytes: 16-byte aligned, and 8 rows meet every bank

// 64 rows of an operand whose summed index runs along its rows: row r, then
// elements k0 .. k0 + 31 of it.
template <class T>
__device__ __forceinline__ void any_stage_rows(T* lds, const T* __restrict__ p, uint64_t stride, int rows, int k0,
                                               int k) {
  const int r = threadIdx.x >> 2, c = (threadIdx.x & 3) * 8;
  T v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = r < rows && k0 + c + i < k ? p[(uint64_t)r * stride + (k0 + c + i)] : (T)0.0f;
  *reinterpret_cast<uint4*>(&lds[r * ANY_LD + c]) = *reinterpret_cast<uint4*>(v);
}
// The same of one whose summed index runs across its rows.
template <class T>
__device__ __forceinline__ void any_stage_cols(T* lds, const T* __restrict__ p, uint64_t stride, int cols, int k0,
                                               int k) {
  const int r = threadIdx.x >> 3, c = (threadIdx.x & 7) * 8;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    lds[(c + i) * ANY_LD + r] = k0 + r < k && c + i < cols ? p[(uint64_t)(k0 + r) * stride + (c + i)] : (T)0.0f;
}

// Rows, and columns, of packed operands: codes times scales, exact in bf16.
__device__ __forceinline__ void any_stage_packed_rows(__bf16* lds, const uint8_t* __restrict__ codes,
                                                      const uint8_t* __restrict__ scales, uint64_t stride,
                                                      uint64_t sstride, int rows, int k0) {
  const int r = threadIdx.x >> 2, c = (threadIdx.x & 3) * 8;
  float v[8] = {};
  if (r < rows) {  // k0 + c is inside the codes' row, whose columns are a multiple of 128
    const uint2 w = *reinterpret_cast<const uint2*>(codes + (uint64_t)r * stride + k0 + c);
    const uint32_t code[2] = {w.x, w.y};
    block8_decode(code, block8_scale(scales[(uint64_t)r * sstride + k0 / 128]), v);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) lds[r * ANY_LD + c + i] = (__bf16)v[i];
}
__device__ __forceinline__ void any_stage_packed_cols(__bf16* lds, const uint8_t* __restrict__ codes,
                                                 const uint8_t* __restrict__ scales, uint64_t stride, uint64_t sstride,
                                                 int n0, int cols, int k0, int k) {
  const int r = threadIdx.x >> 3, c = (threadIdx.x & 7) * 8;
  float v[8] = {};
  if (k0 + r < k && c < cols) {  // whole columns past `cols` stay zero, and codes past a row's columns are
    const uint2 w = *reinterpret_cast<const uint2*>(codes + (uint64_t)(k0 + r) * stride + n0 + c);
    const uint32_t code[2] = {w.x, w.y};
    block8_decode(code, block8_scale(scales[(uint64_t)(k0 + r) * sstride + n0 / 128]), v);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) lds[(c + i) * ANY_LD + r] = (__bf16)v[i];
}

template <class T, class O, int FORM, bool PACKED>
__global__ void __launch_bounds__(256) product_any(Product p) {
  __shared__ __align__(16) T as[ANY_TILE * ANY_LD], bs[ANY_TILE * ANY_LD];
  const int tiles_n = (p.n + ANY_TILE - 1) / ANY_TILE;
  const int n0 = (int)(blockIdx.x % tiles_n) * ANY_TILE;
  int index = (int)(blockIdx.x / tiles_n);
  int m0, m_end, k_end, group;
  [[maybe_unused]] uint64_t lo = 0;  // B's first row (grad weight, packed)
  const T *a, *b;
  O* c;
  if constexpr (FORM == GRAD_WEIGHT) {
    const int tiles_m = (p.m + ANY_TILE - 1) / ANY_TILE;
    group = index / tiles_m;
    m0 = (index - group * tiles_m) * ANY_TILE;
    m_end = p.m;
    int first, end;
    group_range(p.offsets, group, p.rows, first, end);
    lo = first;
    k_end = end - first;
    a = (const T*)p.a + lo * p.as + m0;
    b = (const T*)p.b + lo * p.bs + n0;
    c = (O*)p.c + group * p.cg;
  } else {
    RowTile t;
    if (!find_row_tile(p.offsets, p.groups, p.rows, ANY_TILE, index, t)) return;
    m0 = t.row;
    m_end = t.end;
    k_end = t.group < 0 ? 0 : p.k;
    group = t.group < 0 ? 0 : t.group;
    lo = (uint64_t)group * p.n + n0;
    a = (const T*)p.a + (uint64_t)m0 * p.as;
    b = (const T*)p.b + group * p.bg + (FORM == FORWARD ? (uint64_t)n0 * p.bs : (uint64_t)n0);
    c = (O*)p.c;
  }
  const int rows = m_end - m0 < ANY_TILE ? m_end - m0 : ANY_TILE;
  const int cols = p.n - n0 < ANY_TILE ? p.n - n0 : ANY_TILE;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wm = (wave & 1) * 32, wn = (wave >> 1) * 32;
  f4v acc[2][2] = {};
  for (int k0 = 0; k0 < k_end; k0 += ANY_K) {
    __syncthreads();
    if constexpr (FORM == GRAD_WEIGHT) any_stage_cols(as, a, p.as, rows, k0, k_end);
    else if constexpr (PACKED)
      any_stage_packed_rows(as, (const uint8_t*)p.a + (uint64_t)m0 * p.as, p.a_scales + (uint64_t)m0 * p.ss, p.as, p.ss, rows, k0);
    else any_stage_rows(as, a, p.as, rows, k0, k_end);
    if constexpr (FORM == GRAD_WEIGHT && PACKED)
      any_stage_packed_cols(bs, (const uint8_t*)p.b + lo * p.bs, p.b_scales + lo * p.ss, p.bs, p.ss, n0, cols, k0,
                            k_end);
    else if constexpr (PACKED)
      any_stage_packed_rows(bs, (const uint8_t*)p.b + lo * p.bs, p.b_scales + lo * p.ss, p.bs, p.ss, cols, k0);
    else if constexpr (FORM == FORWARD) any_stage_rows(bs, b, p.bs, cols, k0, k_end);
    else any_stage_cols(bs, b, p.bs, cols, k0, k_end);
    __syncthreads();
    uint4 fa[2], fb[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      fa[i] = *reinterpret_cast<const uint4*>(&as[(wm + 16 * i + (lane & 15)) * ANY_LD + (lane >> 4) * 8]);
      fb[i] = *reinterpret_cast<const uint4*>(&bs[(wn + 16 * i + (lane & 15)) * ANY_LD + (lane >> 4) * 8]);
    }
    // B first: a lane then holds four adjacent columns of one row of C
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) acc[i][j] = mfma16<T>(fb[j], fa[i], acc[i][j]);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int r = wm + 16 * i + (lane & 15), q = wn + 16 * j + (lane >> 4) * 4;
      if (r >= rows) continue;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (q + e < cols) c[(uint64_t)(m0 + r) * p.cs + (n0 + q + e)] = (O)acc[i][j][e];
    }
}

// ---------------------------------------------------------------------------
template <class F>
void by_types(int type, int out_type, F f) {
  auto g = [&](auto t) {
    if (out_type == PXG_F32) f(t, float{});
    else f(t, t);
  };
  if (type == PXG_F16) g((_Float16)0);
  else g((__bf16)0.0f);
}

unsigned grid_size(uint64_t tiles) {
  if (tiles > PRODUCT_SIZE_MAX) config_error("rows", tiles, "gives more tiles than a launch has workgroups");
  return (unsigned)tiles;
}

void check_groups(uint64_t groups, const int64_t* offsets) {
  if (groups == 0 || groups > (1u << 20)) config_error("groups", groups, "must be between 1 and 1048576");
  if (!offsets && groups != 1) config_error("groups", groups, "must be 1 without offsets");
  check_aligned("offsets", offsets, 8);
}
void check_out_type(int type, int out_type) {
  if (out_type != type && out_type != PXG_F32)
    config_error("out_type", (uint64_t)out_type, "must be the operands' type or f32");
}

template <int FORM, class T, class O, bool PACKED>
void launch_product(const Product& p, hipStream_t s) {
  const uint64_t tm = FORM == GRAD_WEIGHT ? (uint64_t)p.groups * ((p.m + ANY_TILE - 1) / ANY_TILE)
                                          : row_tiles_max(p.rows, p.groups, ANY_TILE, p.offsets != nullptr);
  const uint64_t tn = (p.n + ANY_TILE - 1) / ANY_TILE;
  hipLaunchKernelGGL((product_any<T, O, FORM, PACKED>), dim3(grid_size(tm * tn)), dim3(256), 0, s, p);
  PXG_HIP(hipGetLastError());
}

template <int FORM>
void run_product(int type, int out_type, const Product& p, hipStream_t s) {
  by_types(type, out_type, [&](auto t, auto o) {
    using T = decltype(t);
    using O = decltype(o);
    if constexpr (FORM == GRAD_WEIGHT && std::is_same_v<T, __bf16>) {
      if (p.b_scales) return launch_product<FORM, T, O, true>(p, s);
    }
    launch_product<FORM, T, O, false>(p, s);
  });
}

}  // namespace
}  // namespace pxg

using namespace pxg;

extern "C" {

int pxg_grouped_matmul_device(int type, const void* d_x, uint64_t rows, uint64_t k, uint64_t x_stride, const void* d_w,
                              uint64_t groups, uint64_t n, uint64_t w_stride, uint64_t w_group_stride,
                              const int64_t* d_offsets, int out_type, void* d_y, uint64_t y_stride, void* stream) {
  return guard([&] {
    check_type(type, false);
    check_out_type(type, out_type);
    check_size("k", k);
    check_size("n", n);
    check_groups(groups, d_offsets);
    check_rows(type, "x", d_x, rows, k, x_stride);
    check_rows(type, "w", d_w, n, k, w_stride);
    check_rows(out_type, "y", d_y, rows, n, y_stride);
    if (rows == 0) return;
    Product p{d_x, d_w, d_y, d_offsets, x_stride, w_stride, y_stride, w_group_stride, 0, nullptr, nullptr, 0, (int)rows, (int)groups,
              (int)rows, (int)n, (int)k};
    run_product<FORWARD>(type, out_type, p, (hipStream_t)stream);
  });
}

int pxg_grouped_matmul_grad_input_device(int type, const void* d_grad, uint64_t rows, uint64_t n, uint64_t grad_stride,
                                         const void* d_w, uint64_t groups, uint64_t k, uint64_t w_stride,
                                         uint64_t w_group_stride, const int64_t* d_offsets, int out_type, void* d_dx,
                                         uint64_t dx_stride, void* stream) {
  return guard([&] {
    check_type(type, false);
    check_out_type(type, out_type);
    check_size("k", k);
    check_size("n", n);
    check_groups(groups, d_offsets);
    check_rows(type, "grad", d_grad, rows, n, grad_stride);
    check_rows(type, "w", d_w, n, k, w_stride);
    check_rows(out_type, "dx", d_dx, rows, k, dx_stride);
    if (rows == 0) return;
    Product p{d_grad, d_w, d_dx, d_offsets, grad_stride, w_stride, dx_stride, w_group_stride, 0, nullptr, nullptr, 0, (int)rows,
              (int)groups, (int)rows, (int)k, (int)n};
    run_product<GRAD_INPUT>(type, out_type, p, (hipStream_t)stream);
  });
}

int pxg_grouped_matmul_grad_weight_device(int type, const void* d_grad, uint64_t rows, uint64_t n,
                                          uint64_t grad_stride, const void* d_x, uint64_t k, uint64_t x_stride,
                                          const int64_t* d_offsets, uint64_t groups, int out_type, void* d_dw,
                                          uint64_t dw_stride, uint64_t dw_group_stride, void* stream) {
  return guard([&] {
    check_type(type, false);
    check_out_type(type, out_type);
    check_size("k", k);
    check_size("n", n);
    if (!d_offsets) config_error("offsets", 0, "must not be null");
    check_groups(groups, d_offsets);
    check_rows(type, "grad", d_grad, rows, n, grad_stride);
    check_rows(type, "x", d_x, rows, k, x_stride);
    check_rows(out_type, "dw", d_dw, n, k, dw_stride);
    Product p{d_grad, d_x, d_dw, d_offsets, grad_stride, x_stride, dw_stride, 0, dw_group_stride, nullptr, nullptr, 0, (int)rows,
              (int)groups, (int)n, (int)k, 0};
    run_product<GRAD_WEIGHT>(type, out_type, p, (hipStream_t)stream);
  });
}

int pxg_grouped_matmul_grad_weight_block8_device(const void* d_grad, uint64_t rows, uint64_t n, uint64_t grad_stride,
                                                 const void* d_codes, const void* d_scales, uint64_t k,
                                                 const int64_t* d_offsets, uint64_t groups, int out_type, void* d_dw,
                                                 uint64_t dw_stride, uint64_t dw_group_stride, void* stream) {
  return guard([&] {
    check_out_type(PXG_BF16, out_type);
    check_size("k", k);
    check_size("n", n);
    if (!d_offsets) config_error("offsets", 0, "must not be null");
    check_groups(groups, d_offsets);
    check_rows(PXG_BF16, "grad", d_grad, rows, n, grad_stride);
    check_packed_rows("codes", d_codes, "scales", d_scales, rows);
    check_rows(out_type, "dw", d_dw, n, k, dw_stride);
    Product p{d_grad, d_codes, d_dw, d_offsets, grad_stride, block8_code_stride(k), dw_stride, 0, dw_group_stride,
              nullptr, (const uint8_t*)d_scales, block8_scale_stride(k), (int)rows, (int)groups, (int)n, (int)k, 0};
    run_product<GRAD_WEIGHT>(PXG_BF16, out_type, p, (hipStream_t)stream);
  });
}

int pxg_block8_matmul_device(const void* d_codes, const void* d_scales, uint64_t rows, uint64_t k,
                             const void* d_w_codes, const void* d_w_scales, uint64_t groups, uint64_t n,
                             const int64_t* d_offsets, int out_type, void* d_y, uint64_t y_stride, void* stream) {
  return guard([&] {
    check_type(out_type, true);
    check_size("k", k);
    check_size("n", n);
    check_groups(groups, d_offsets);
    check_packed_rows("codes", d_codes, "scales", d_scales, rows);
    check_packed_rows("w_codes", d_w_codes, "w_scales", d_w_scales, n);
    check_rows(out_type, "y", d_y, rows, n, y_stride);
    if (rows == 0) return;
    const uint64_t wide = block8_code_stride(k);
    Product p{d_codes, d_w_codes, d_y, d_offsets, wide, wide, y_stride, 0, 0, (const uint8_t*)d_scales,
              (const uint8_t*)d_w_scales, block8_scale_stride(k), (int)rows, (int)groups, (int)rows, (int)n,
              (int)wide};
    const hipStream_t s = (hipStream_t)stream;
    if (out_type == PXG_F32) launch_product<FORWARD, __bf16, float, true>(p, s);
    else if (out_type == PXG_F16) launch_product<FORWARD, __bf16, _Float16, true>(p, s);
    else launch_product<FORWARD, __bf16, __bf16, true>(p, s);
  });
}

}  // extern "C"
