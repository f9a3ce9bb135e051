// Layers of ragged groups: the product with a bias, an activation and a
// residual in its epilogue, in 16 bits or over packed rows,
//
//   h[t, :] = x[t, :] w_g^T + b_g,   y[t, :] = f(h[t, :]) + r[t, :]      t in group g
//
// The product's kernels are product_kernels.hpp's; the epilogue takes h from
// the accumulators in f32, so that y is rounded once.
#include "product_kernels.hpp"

namespace pxg {
namespace {

// The epilogue's part of a product of operands of `type`.
void set_epilogue(LinearProduct& p, const pxg_linear& a, int type, void* h) {
  check_bias("bias", type, a.bias_type, a.bias, a.groups, a.n, a.bias_stride);
  check_optional_activation(a.activation);
  if (a.residual) check_rows(a.out_type, "residual", a.residual, a.rows, a.n, a.residual_stride);
  if (h) check_rows(a.out_type, "h", h, a.rows, a.n, a.h_stride);
  p.bias = a.bias;
  p.bias_stride = a.bias_stride;
  p.bias_f32 = a.bias_type == PXG_F32;
  p.activation = (int)a.activation;
  p.residual = a.residual;
  p.rs = a.residual_stride;
  p.kept = h;
  p.hs = a.h_stride;
}

}  // namespace
}  // namespace pxg

using namespace pxg;

extern "C" {

int pxg_grouped_linear_device(const pxg_linear* layer, void* stream) {
  return guard([&] {
    const pxg_linear& a = check_arguments(layer);
    check_type(a.type, false);
    check_out_type(a.type, a.out_type);
    check_size("k", a.k);
    check_size("n", a.n);
    check_groups(a.groups, a.offsets);
    check_rows(a.type, "x", a.x, a.rows, a.k, a.x_stride);
    check_rows(a.type, "w", a.w, a.n, a.k, a.w_stride);
    check_rows(a.out_type, "y", a.y, a.rows, a.n, a.y_stride);
    LinearProduct p{{a.x, a.w, a.y, a.offsets, check_stride(a.rows, a.k, a.x_stride), check_stride(a.n, a.k, a.w_stride),
                     a.y_stride, a.w_group_stride, 0, nullptr, nullptr, 0, (int)a.rows, (int)a.groups, (int)a.rows,
                     (int)a.n, (int)a.k, false}};
    set_epilogue(p, a, a.type, a.h);
    check_rows_apart("y", a.y, a.n * type_bytes((int)a.out_type), a.y_stride * type_bytes((int)a.out_type), a.x, a.k * 2,
                     a.x_stride * 2, a.rows);
    if (a.h)
      check_rows_apart("h", a.h, a.n * type_bytes((int)a.out_type), a.h_stride * type_bytes((int)a.out_type), a.x,
                       a.k * 2, a.x_stride * 2, a.rows);
    if (a.rows == 0) return;
    run_product<FORWARD>(a.type, a.out_type, p, (hipStream_t)stream);
  });
}

int pxg_block8_linear_device(const pxg_linear* layer, void* stream) {
  return guard([&] {
    const pxg_linear& a = check_arguments(layer);
    check_type(a.out_type, true);
    check_size("k", a.k);
    check_size("n", a.n);
    check_groups(a.groups, a.offsets);
    check_packed_rows("x", a.x, "x_scales", a.x_scales, a.rows);
    check_packed_rows("w", a.w, "w_scales", a.w_scales, a.n);
    check_rows(a.out_type, "y", a.y, a.rows, a.n, a.y_stride);
    const uint64_t wide = check_stride(2, a.k, block8_code_stride(a.k));
    LinearProduct p{{a.x, a.w, a.y, a.offsets, wide, wide, a.y_stride, a.n * wide, 0, (const uint8_t*)a.x_scales,
                     (const uint8_t*)a.w_scales, block8_scale_stride(a.k), (int)a.rows, (int)a.groups, (int)a.rows,
                     (int)a.n, (int)wide, false}};
    set_epilogue(p, a, PXG_BF16, nullptr);
    if (a.rows == 0) return;
    const hipStream_t s = (hipStream_t)stream;
    if (a.out_type == PXG_F32) launch_product<FORWARD, __bf16, float, true>(p, 0, s);
    else if (a.out_type == PXG_F16) launch_product<FORWARD, __bf16, _Float16, true>(p, 0, s);
    else launch_product<FORWARD, __bf16, __bf16, true>(p, 0, s);
  });
}

}  // extern "C"
