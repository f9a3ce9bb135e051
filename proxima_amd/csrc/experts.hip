// Matrix products of rows in ragged groups, each group with a matrix of its
// own (expert layers), their gradients, and the same product over packed
// 8-bit rows (block8.hpp). The kernels are in product_kernels.hpp.
#include "product_kernels.hpp"

using namespace pxg;

extern "C" {

int pxg_grouped_matmul_set_kernel(int rows) {
  return guard([&] {
    if (rows != 0 && rows != 16 && rows != 64 && rows != 128 && rows != 256)
      config_error("rows", (uint64_t)rows, "must be 0, 16, 64, 128 or 256");
    g_kernel = rows;
  });
}
uint32_t pxg_grouped_matmul_last_kernel(void) { return g_last_kernel; }

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
    x_stride = check_stride(rows, k, x_stride);
    w_stride = check_stride(n, k, w_stride);
    if (rows == 0) return;
    Product p{d_x, d_w, d_y, d_offsets, x_stride, w_stride, y_stride, w_group_stride, 0, nullptr, nullptr, 0, (int)rows, (int)groups,
              (int)rows, (int)n, (int)k, false};
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
    grad_stride = check_stride(rows, n, grad_stride);
    w_stride = check_stride(n, k, w_stride);
    if (rows == 0) return;
    Product p{d_grad, d_w, d_dx, d_offsets, grad_stride, w_stride, dx_stride, w_group_stride, 0, nullptr, nullptr, 0, (int)rows,
              (int)groups, (int)rows, (int)k, (int)n, false};
    run_product<GRAD_INPUT>(type, out_type, p, (hipStream_t)stream);
  });
}

uint64_t pxg_grouped_matmul_grad_weight_workspace(uint64_t rows, uint64_t n, uint64_t k, uint64_t groups) {
  if (rows > PRODUCT_SIZE_MAX || n == 0 || n > PRODUCT_SIZE_MAX || k == 0 || k > PRODUCT_SIZE_MAX || groups == 0 ||
      groups > (1u << 20))
    return 0;
  Product p{};
  p.rows = (int)rows;
  p.groups = (int)groups;
  p.m = (int)n;
  p.n = (int)k;
  const Cost cost = product_cost(GRAD_WEIGHT, p, false, UINT64_MAX, asked_tile(false));
  return 4 * group_slots_max(rows, groups, cost.limit) * n * k;
}

int pxg_grouped_matmul_grad_weight_device(int type, const void* d_grad, uint64_t rows, uint64_t n,
                                          uint64_t grad_stride, const void* d_x, uint64_t k, uint64_t x_stride,
                                          const int64_t* d_offsets, uint64_t groups, int out_type, void* d_dw,
                                          uint64_t dw_stride, uint64_t dw_group_stride, void* d_workspace,
                                          uint64_t workspace_bytes, void* stream) {
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
    check_matrices_apart("dw_group_stride", groups, n, k, dw_stride, dw_group_stride);
    check_aligned("workspace", d_workspace, 16);
    grad_stride = check_stride(rows, n, grad_stride);
    x_stride = check_stride(rows, k, x_stride);
    Product p{d_grad, d_x, d_dw, d_offsets, grad_stride, x_stride, dw_stride, 0, dw_group_stride, nullptr, nullptr, 0, (int)rows,
              (int)groups, (int)n, (int)k, 0, false};
    p.workspace = (float*)d_workspace;
    run_product<GRAD_WEIGHT>(type, out_type, p, (hipStream_t)stream, d_workspace ? workspace_bytes : 0);
  });
}

int pxg_grouped_matmul_grad_weight_block8_device(const void* d_grad, uint64_t rows, uint64_t n, uint64_t grad_stride,
                                                 const void* d_codes, const void* d_scales, uint64_t k,
                                                 const int64_t* d_offsets, uint64_t groups, int out_type, void* d_dw,
                                                 uint64_t dw_stride, uint64_t dw_group_stride, void* d_workspace,
                                                 uint64_t workspace_bytes, void* stream) {
  return guard([&] {
    check_out_type(PXG_BF16, out_type);
    check_size("k", k);
    check_size("n", n);
    if (!d_offsets) config_error("offsets", 0, "must not be null");
    check_groups(groups, d_offsets);
    check_rows(PXG_BF16, "grad", d_grad, rows, n, grad_stride);
    check_packed_rows("codes", d_codes, "scales", d_scales, rows);
    check_rows(out_type, "dw", d_dw, n, k, dw_stride);
    check_matrices_apart("dw_group_stride", groups, n, k, dw_stride, dw_group_stride);
    check_aligned("workspace", d_workspace, 16);
    grad_stride = check_stride(rows, n, grad_stride);
    check_stride(2, k, block8_code_stride(k));
    Product p{d_grad, d_codes, d_dw, d_offsets, grad_stride, block8_code_stride(k), dw_stride, 0, dw_group_stride,
              nullptr, (const uint8_t*)d_scales, block8_scale_stride(k), (int)rows, (int)groups, (int)n, (int)k, 0, false};
    p.workspace = (float*)d_workspace;
    run_product<GRAD_WEIGHT>(PXG_BF16, out_type, p, (hipStream_t)stream, d_workspace ? workspace_bytes : 0);
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
    const uint64_t wide = check_stride(2, k, block8_code_stride(k));
    Product p{d_codes, d_w_codes, d_y, d_offsets, wide, wide, y_stride, n * wide, 0, (const uint8_t*)d_scales,
              (const uint8_t*)d_w_scales, block8_scale_stride(k), (int)rows, (int)groups, (int)rows, (int)n,
              (int)wide, false};
    const hipStream_t s = (hipStream_t)stream;
    if (out_type == PXG_F32) launch_product<FORWARD, __bf16, float, true>(p, 0, s);
    else if (out_type == PXG_F16) launch_product<FORWARD, __bf16, _Float16, true>(p, 0, s);
    else launch_product<FORWARD, __bf16, __bf16, true>(p, 0, s);
  });
}

}  // extern "C"
