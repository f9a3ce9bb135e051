// Argument checks shared by the packed rows' and the products' entry points.
#pragma once

#include "common.hpp"

namespace pxg {

// Columns and rows of one matrix count in 31 bits; offsets inside tensors are
// 64-bit throughout.
constexpr uint64_t PRODUCT_SIZE_MAX = (1ull << 31) - 1024;

inline uint64_t type_bytes(int type) { return type == PXG_F32 ? 4 : 2; }

inline void check_type(int type, bool f32) {
  if (type != PXG_F16 && type != PXG_BF16 && !(f32 && type == PXG_F32))
    config_error("type", (uint64_t)type, f32 ? "must be f32, f16 or bf16" : "must be f16 or bf16");
}
// `name` must be a string literal.
inline void check_size(const char* name, uint64_t size) {
  if (size == 0 || size > PRODUCT_SIZE_MAX) config_error(name, size, "must be between 1 and 2147482624");
}
inline void check_aligned(const char* name, const void* p, uint64_t bytes) {
  if ((uint64_t)(uintptr_t)p % bytes) config_error(name, (uint64_t)(uintptr_t)p, "must be aligned: codes and workspace to 16 bytes, offsets to 8, scales to 4");
}
// A product's operand: a tile's offsets count in 31 bits. The distance of a
// single row to the next means nothing and is the columns.
inline uint64_t check_stride(uint64_t rows, uint64_t cols, uint64_t stride) {
  if (rows <= 1) stride = cols;
  if (stride > (1ull << 22)) config_error("stride", stride, "must be at most 4194304 elements");
  return stride;
}
// A row-major matrix: rows may be 0 (the pointer is then not looked at).
inline void check_rows(int type, const char* name, const void* p, uint64_t rows, uint64_t cols, uint64_t stride) {
  if (rows > PRODUCT_SIZE_MAX) config_error("rows", rows, "must be at most 2147482624");
  if (rows > 1 && stride < cols) config_error("stride", stride, "must be at least the columns");
  if (rows && !p) config_error(name, 0, "must not be null");
  if (rows && (uint64_t)(uintptr_t)p % type_bytes(type))
    config_error(name, (uint64_t)(uintptr_t)p, "must be aligned to its type");
}
// The groups' matrices of a result, each of n rows of `cols`: one after the
// other or, row by row, between one another. Overlapping ones would be written
// by several groups at once.
inline void check_matrices_apart(const char* name, uint64_t groups, uint64_t n, uint64_t cols, uint64_t stride,
                                 uint64_t group_stride) {
  using u128 = unsigned __int128;
  if (groups <= 1) return;
  const bool after = group_stride >= (u128)(n - 1) * stride + cols;
  const bool between = group_stride >= cols && stride >= (u128)(groups - 1) * group_stride + cols;
  if (!after && !between) config_error(name, group_stride, "must keep the groups' matrices apart");
}
// Packed rows (block8.hpp), laid out as the packing entry point does.
inline void check_packed_rows(const char* codes_name, const void* codes, const char* scales_name, const void* scales,
                              uint64_t rows) {
  if (rows > PRODUCT_SIZE_MAX) config_error("rows", rows, "must be at most 2147482624");
  if (rows && !codes) config_error(codes_name, 0, "must not be null");
  if (rows && !scales) config_error(scales_name, 0, "must not be null");
  check_aligned(codes_name, codes, 16);
  check_aligned(scales_name, scales, 4);
}
// Whether every row starts on a 16-byte boundary.
inline bool rows_aligned(int type, const void* p, uint64_t stride) {
  return ((uint64_t)(uintptr_t)p | (stride * type_bytes(type))) % 16 == 0;
}

}  // namespace pxg
