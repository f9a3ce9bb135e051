// The backward pass of layers of ragged groups (linear.hip) up to the products,
// which are the products' gradients with dh in the place of dy:
//
//   dh = dy f'(h),   db_g = sum over t in g of dh[t, :],   dr = dy
#include <algorithm>

#include "activation.hpp"
#include "common.hpp"
#include "device.hpp"
#include "groups.hpp"
#include "products.hpp"
#include "rows.hpp"

namespace pxg {
namespace {

// The backward pass reads dy and h and writes dh once, and memory bounds it: 16384
// x 4096 in bf16, GELU 77 us, 5.2 TB/s, and 5 us for the bias (88 with dy and h
// in the caches).
// Rows go in tiles of one group; a workgroup takes a tile by 8 p.x columns, a
// thread every 256 / p.x-th row of 8 columns, whose sums it keeps.
// The workgroup's sums are joined in LDS and go to the tile's row of the
// workspace; grad_bias_join adds a group's tiles in order. Without a workspace
// a workgroup takes a whole group by its columns (tile 0: none).
constexpr int GRAD_THREADS = 256, GRAD_BATCH = 4;  // rows that a thread has in flight

struct LinearGrad {
  const void *grad, *h;
  void *dh, *dbias;
  const int64_t* offsets;
  uint64_t gs, hs, ds, bs;  // row strides
  float* workspace;
  int rows, n, groups, tile, x;
};

template <class T, class B, bool VEC, int ACT>
__global__ void __launch_bounds__(GRAD_THREADS) linear_grad_rows(LinearGrad p) {
  __shared__ float sums[GRAD_THREADS * 8];
  const int across = p.x, x = threadIdx.x & (across - 1), y = threadIdx.x / across, high = GRAD_THREADS / across;
  RowTile t;
  if (p.tile) {
    if (!find_row_tile<ALL_TILES>(p.offsets, p.groups, p.rows, p.tile, (int)blockIdx.x, t)) return;
    t.end = t.end - t.row > p.tile ? t.row + p.tile : t.end;
  } else if (!p.offsets) {
    t = {0, 0, p.rows};
  } else {  // groups in order, then the rows of none before and after them
    const int g = (int)blockIdx.x;
    int lo, hi;
    group_range(p.offsets, g < p.groups ? g : g == p.groups ? 0 : p.groups - 1, p.rows, lo, hi);
    t = g < p.groups ? RowTile{g, lo, hi} : g == p.groups ? RowTile{-1, 0, lo} : RowTile{-1, hi, p.rows};
  }
  if constexpr (ACT == NO_ACTIVATION) {
    if (t.group < 0) return;
  }
  const T* grad = (const T*)p.grad;
  const T* h = (const T*)p.h;
  T* dh = (T*)p.dh;
  const uint32_t n = p.n, wide = across * 8;
  for (uint32_t c0 = blockIdx.y * wide; c0 < n; c0 += gridDim.y * wide) {
    const uint32_t c = c0 + x * 8;
    float sum[8] = {};
    if (c < n) {
      for (int r0 = t.row + y; r0 < t.end; r0 += high * GRAD_BATCH) {
        Eight<T> d[GRAD_BATCH], v[GRAD_BATCH];
#pragma unroll
        for (int i = 0; i < GRAD_BATCH; ++i) {
          const int64_t r = r0 + (int64_t)i * high;
          d[i] = v[i] = Eight<T>{};
          if (r >= t.end || t.group < 0) continue;
          d[i] = raw8<T, VEC>(grad + r * p.gs, c, n);
          if constexpr (ACT != NO_ACTIVATION) v[i] = raw8<T, VEC>(h + r * p.hs, c, n);
        }
        __builtin_amdgcn_sched_barrier(0);  // all in flight, and still in T: fewer registers, more wavefronts
#pragma unroll
        for (int i = 0; i < GRAD_BATCH; ++i) {
          const int64_t r = r0 + (int64_t)i * high;
          if (r >= t.end) break;
          float g[8];
          d[i].unpack(g);
          if constexpr (ACT != NO_ACTIVATION) {
            float x[8];
            v[i].unpack(x);
#pragma unroll
            for (int e = 0; e < 8; ++e) g[e] *= act_slope<T, ACT>(x[e]);
            store8<T, VEC>(dh + r * p.ds, c, n, g);
            __builtin_amdgcn_sched_barrier(0);  // a row after another
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) sum[e] += g[e];
        }
      }
    }
    if (!p.dbias || t.group < 0) continue;
    __syncthreads();  // the strip before has been read
#pragma unroll
    for (int e = 0; e < 8; ++e) sums[(y * 8 + e) * across + x] = sum[e];
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < wide; i += GRAD_THREADS) {
      const uint32_t e = i / across, of = i & (across - 1), at = c0 + of * 8 + e;
      float s = 0.0f;
      for (int j = 0; j < high; ++j) s += sums[(j * 8 + e) * across + of];
      if (at >= n) continue;
      if (p.tile) p.workspace[(uint64_t)blockIdx.x * n + at] = s;
      else ((B*)p.dbias)[t.group * p.bs + at] = rounded<B>(s);
    }
  }
}

// A workgroup adds the tiles of one group in 64 columns, a wavefront every
// fourth of them.
template <class B>
__global__ void __launch_bounds__(GRAD_THREADS) grad_bias_join(LinearGrad p) {
  __shared__ float sums[GRAD_THREADS];
  int first, tiles;
  find_group_tiles(p.offsets, p.groups, p.rows, p.tile, (int)blockIdx.x, first, tiles);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t n = p.n;
  for (uint32_t c0 = blockIdx.y * 64; c0 < n; c0 += gridDim.y * 64) {
    const uint32_t c = c0 + lane;
    float s = 0.0f;
    if (c < n) {
      const float* from = p.workspace + (uint64_t)first * n + c;
#pragma unroll 8
      for (int i = wave; i < tiles; i += 4) s += from[(uint64_t)i * n];
    }
    __syncthreads();
    sums[threadIdx.x] = s;
    __syncthreads();
    if (wave == 0 && c < n)
      ((B*)p.dbias)[blockIdx.x * p.bs + c] =
          rounded<B>((sums[lane] + sums[64 + lane]) + (sums[128 + lane] + sums[192 + lane]));
  }
}

// The tile's rows, 0 where each group has a workgroup of its own. About 2048
// workgroups fill the chip; each then joins few sums for the rows it reads. The
// choice goes by the average group, and a group of many that is much longer, or
// rows of none, are then one workgroup's by its columns: 16384 x 4096 in bf16, GELU,
// 71 to 83 us in 64 to 256 equal groups; with half the rows in one group 100 of 64,
// 710 of 128 or 256; with half of them behind the last group 69, and 530 to 540.
struct GradPlan {
  unsigned x;  // threads to a row
  unsigned strips;
  int tile;
  uint64_t tiles, bytes;
};
GradPlan grad_plan(uint64_t rows, uint64_t n, uint64_t groups, bool ragged) {
  GradPlan g{16, 1, 0, 0, 0};
  while (g.x < 32 && g.x * 8 < n) g.x *= 2;
  const uint64_t strips = (n + g.x * 8 - 1) / (g.x * 8), high = GRAD_THREADS / g.x;
  g.strips = (unsigned)std::min<uint64_t>(strips, 1024);
  // one round of a group's rows costs less than a second kernel (35 rows x 3375, GELU, bf16: 11.4 us, 14.8;
  // of four, 120 rows x 1710 in f32 would take 38)
  if (rows <= high * GRAD_BATCH) return g;
  const uint64_t least = high * 2;
  uint64_t tile = std::max((rows * g.strips + 2047) / 2048, (rows >> 21) + 1);
  tile = (tile + least - 1) / least * least;
  if (rows / groups <= tile) return g;
  g.tile = (int)tile;
  g.tiles = row_tiles_max(rows, groups, tile, ragged);
  g.bytes = g.tiles * n * 4;
  return g;
}

template <class T, class B, bool VEC>
void launch_grad(int activation, const LinearGrad& p, const GradPlan& g, hipStream_t s) {
  const dim3 block(GRAD_THREADS);
  const dim3 grid((unsigned)(p.tile ? g.tiles : p.offsets ? p.groups + 2 : 1), g.strips);
  if (activation == PXG_SILU) hipLaunchKernelGGL((linear_grad_rows<T, B, VEC, PXG_SILU>), grid, block, 0, s, p);
  else if (activation == PXG_GELU) hipLaunchKernelGGL((linear_grad_rows<T, B, VEC, PXG_GELU>), grid, block, 0, s, p);
  else hipLaunchKernelGGL((linear_grad_rows<T, B, VEC, NO_ACTIVATION>), grid, block, 0, s, p);
  PXG_HIP(hipGetLastError());
  if (p.dbias && p.tile) {
    const uint64_t strips = ((uint64_t)p.n + 63) / 64;
    hipLaunchKernelGGL(grad_bias_join<B>, dim3((unsigned)p.groups, (unsigned)std::min<uint64_t>(strips, 1024)),
                       dim3(GRAD_THREADS), 0, s, p);
    PXG_HIP(hipGetLastError());
  }
}

}  // namespace
}  // namespace pxg

using namespace pxg;

extern "C" {

uint64_t pxg_grouped_linear_grad_workspace(uint64_t rows, uint64_t n, uint64_t groups) {
  if (rows == 0 || rows > PRODUCT_SIZE_MAX || n == 0 || n > PRODUCT_SIZE_MAX || groups == 0 || groups > (1u << 20))
    return 0;
  return grad_plan(rows, n, groups, true).bytes;
}

int pxg_grouped_linear_grad_device(const pxg_linear_grad* layer, void* stream) {
  return guard([&] {
    const pxg_linear_grad& a = check_arguments(layer);
    check_type(a.type, true);
    check_optional_activation(a.activation);
    check_size("n", a.n);
    check_groups(a.groups, a.offsets);
    check_rows(a.type, "grad", a.grad, a.rows, a.n, a.grad_stride);
    const bool slope = a.activation != NO_ACTIVATION;
    if (slope) {
      check_rows(a.type, "h", a.h, a.rows, a.n, a.h_stride);
      check_rows(a.type, "dh", a.dh, a.rows, a.n, a.dh_stride);
    }
    check_bias("dbias", a.type, a.bias_type, a.dbias, a.groups, a.n, a.dbias_stride);
    check_aligned("workspace", a.workspace, 16);
    if (!slope && !a.dbias) return;
    LinearGrad p{a.grad, a.h, a.dh, a.dbias, a.offsets, a.grad_stride, a.h_stride, a.dh_stride, a.dbias_stride,
                 (float*)a.workspace, (int)a.rows, (int)a.n, (int)a.groups, 0, 0};
    const GradPlan g = grad_plan(a.rows, a.n, a.groups, a.offsets != nullptr);
    if (!a.dbias || (a.workspace && a.workspace_bytes >= g.bytes)) p.tile = g.tile;
    p.x = (int)g.x;
    const bool vec = rows_aligned(a.type, a.grad, a.grad_stride) &&
                     (!slope || (rows_aligned(a.type, a.h, a.h_stride) && rows_aligned(a.type, a.dh, a.dh_stride)));
    by_type(a.type, vec, [&](auto t, auto v) {
      using T = decltype(t);
      constexpr bool V = decltype(v)::value;
      if (a.bias_type == PXG_F32) launch_grad<T, float, V>(a.activation, p, g, (hipStream_t)stream);
      else launch_grad<T, T, V>(a.activation, p, g, (hipStream_t)stream);
    });
  });
}

}  // extern "C"
