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

typedef int i8v __attribute__((ext_vector_type(8)));
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
  bool c_vec;           // four adjacent elements of C, from a multiple of four on, can be stored at once
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
// The tiled product: operands go to LDS by direct copies, 128 bytes of each
// row (or 64 rows, where the summed index runs across them) at a time, into
// one of two stages while the other is multiplied.
// ---------------------------------------------------------------------------
// How an operand lies in memory:
//   ROWS    the summed index along its rows
//   COLS    the summed index across its rows; fragments come out of LDS by
//           transposing reads
//   PACKED  COLS of packed rows; codes are decoded on their way to LDS
enum Layout { ROWS, COLS, PACKED };

struct Fp8 {};  // packed operands multiplied as they are

#if defined(__HIP_DEVICE_COMPILE__)
// A raw buffer resource over [p, p + bytes), from wave-uniform scalars;
// accesses at offsets outside it read zeros.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t tile_rsrc(const void* p, uint64_t bytes) {
  const uint64_t a = (uint64_t)(uintptr_t)p;
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)a);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(a >> 32));
  const int n = __builtin_amdgcn_readfirstlane((int)(uint32_t)(bytes < 0x7FFFFFFF ? bytes : 0x7FFFFFFF));
  return __builtin_amdgcn_make_buffer_rsrc((void*)(uintptr_t)(((uint64_t)hi << 32) | lo), 0, n, 0x00020000);
}

// Copies of 16 (and 4) bytes a lane straight into LDS: lane i's land at
// lds + 16 i (4 i), zeros for offsets outside the resource. Inline asm, so
// that the compiler does not wait for them before every LDS read; nothing
// else in these kernels uses m0. wait_copies() waits for all of them.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void copy16(__amdgpu_buffer_rsrc_t rs, uint32_t offset, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(offset), "s"(rs)
               : "memory", "m0");
}
__device__ __forceinline__ void copy4(__amdgpu_buffer_rsrc_t rs, uint32_t offset, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\tbuffer_load_dword %1, %2, 0 offen lds" ::"s"(lds), "v"(offset), "s"(rs)
               : "memory", "m0");
}
#pragma clang diagnostic pop
__device__ __forceinline__ void wait_copies() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

constexpr uint32_t NOWHERE = 0xFFFFFF00u;  // an offset outside every resource

__device__ __forceinline__ uint32_t lds_address(const void* p) {
  return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) char*)p;
}

// 8 codes times their scale, in bf16.
__device__ __forceinline__ uint4 decode_bf16(uint32_t x, uint32_t y, float s) {
  typedef __bf16 bf2v __attribute__((ext_vector_type(2)));
  const bf2v a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, s, false);
  const bf2v b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, s, true);
  const bf2v c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(y, s, false);
  const bf2v d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(y, s, true);
  return make_uint4(__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b), __builtin_bit_cast(uint32_t, c),
                    __builtin_bit_cast(uint32_t, d));
}

// By how many 16-byte pieces row k of a stage is moved: a transposing read
// takes 32 bytes of rows 8 q + {0..3} (or {4..7}) for each 16 lanes q.
__device__ __forceinline__ int cols_swizzle(int k) { return ((k & 3) | ((k >> 1) & 4)) << 1; }

// Tile `i` of n for this workgroup: workgroups go to the 8 dies in turn, so
// each die takes an eighth of the tiles, in order, and tiles that share
// operands meet in one L2.
__device__ __forceinline__ int die_order(int block, int n) {
  const int die = block & 7, at = block >> 3, each = n >> 3, more = n & 7;
  if (at >= each + (die < more ? 1 : 0)) return -1;
  return die * each + (die < more ? die : more) + at;
}
#endif

// WM x WN wavefronts, each with MT x NT tiles of 16 x 16. T is the type
// multiplied (bf16, f16 or Fp8), O the result's.
template <class T, class O, int FORM, int LA, int LB, int WM, int WN, int MT, int NT>
struct Tiled {
  static constexpr int THREADS = 64 * WM * WN, WAVES = WM * WN;
  static constexpr int TM = 16 * WM * MT, TN = 16 * WN * NT;
  static constexpr bool FP8 = std::is_same_v<T, Fp8>;
  static constexpr int BYTES = FP8 ? 1 : 2;       // of an element
  static constexpr int STEP = 128 / BYTES;        // summed elements a stage holds
  static constexpr int A_BYTES = TM * 128, B_BYTES = TN * 128, STAGE = A_BYTES + B_BYTES;
  static constexpr int SCALES = FP8 ? (TM + TN) * 4 : 0;  // four blocks' scale bytes of each row
  static constexpr int LDS = 2 * (STAGE + SCALES);
};

template <class T, class O, int FORM, int LA, int LB, int WM, int WN, int MT, int NT>
__global__ void __launch_bounds__(64 * WM * WN) product_tiled(Product p) {
#if defined(__HIP_DEVICE_COMPILE__)
  using K = Tiled<T, O, FORM, LA, LB, WM, WN, MT, NT>;
  constexpr int TM = K::TM, TN = K::TN, WAVES = K::WAVES;
  __shared__ __align__(1024) char lds[K::LDS];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WN, wn = wave % WN;

  // this workgroup's tile
  const int tiles_n = (p.n + TN - 1) / TN;
  int m0, n0, rows, cols, steps, group, tail;
  uint64_t a0, b0;  // first bytes of the operands' tiles
  uint64_t first = 0;
  if constexpr (FORM == GRAD_WEIGHT) {
    const int tiles_m = (p.m + TM - 1) / TM, each = tiles_m * tiles_n;
    // a die takes an eighth of every group's tiles: groups differ in length
    const int per = (each + 7) / 8;
    group = (int)(blockIdx.x / (8 * per));
    const int in = (int)(blockIdx.x % (8 * per)), t = (in & 7) * per + (in >> 3);
    if (t >= each) return;
    m0 = t / tiles_n * TM;
    n0 = t % tiles_n * TN;
    int lo, hi;
    group_range(p.offsets, group, p.rows, lo, hi);
    rows = p.m - m0;
    tail = hi - lo;
    steps = (tail + K::STEP - 1) / K::STEP;
    first = lo;
    a0 = ((uint64_t)lo * p.as + m0) * 2;
    b0 = LB == PACKED ? 0 : ((uint64_t)lo * p.bs + n0) * 2;
  } else {
    const int total = count_row_tiles(p.offsets, p.groups, p.rows, TM);
    const int index = die_order(blockIdx.x, total * tiles_n);
    if (index < 0) return;
    // the 32 workgroups that run together on a die share operands best as a
    // block of 4 row tiles by 8
    const int band = index / (4 * tiles_n), in = index - band * 4 * tiles_n;
    const int high = total - band * 4 < 4 ? total - band * 4 : 4;
    RowTile t;
    if (!find_row_tile(p.offsets, p.groups, p.rows, TM, band * 4 + in % high, t)) return;
    m0 = t.row;
    n0 = in / high * TN;
    group = t.group < 0 ? 0 : t.group;
    rows = t.end - m0;
    tail = t.group < 0 ? 0 : p.k;
    steps = (tail + K::STEP - 1) / K::STEP;
    a0 = (uint64_t)m0 * p.as * K::BYTES;
    b0 = (group * p.bg + (LB == ROWS ? (uint64_t)n0 * p.bs : (uint64_t)n0)) * K::BYTES;
  }
  rows = rows < TM ? rows : TM;
  cols = p.n - n0 < TN ? p.n - n0 : TN;

  // Copies. ROWS: a copy of one wavefront fills 8 rows of 128 bytes, 16-byte
  // piece c of row r at place c ^ (r & 7), so that 8 lanes reading piece c of
  // 8 rows meet every bank. COLS: it fills 1024 bytes of rows of 2 TM (2 TN)
  // bytes, piece c of row k at c ^ cols_swizzle(k): of the two quarters of a
  // transposing read that go together, the eight rows lie in different banks.
  const char* pa = (const char*)p.a + a0;
  const char* pb = (const char*)p.b + b0;
  const uint32_t row_a = (lane >> 3) * (uint32_t)(p.as * K::BYTES) + (((lane & 7) ^ (lane >> 3)) << 4);
  const uint32_t row_b = (lane >> 3) * (uint32_t)(p.bs * K::BYTES) + (((lane & 7) ^ (lane >> 3)) << 4);
  constexpr int CA = TM / 8 / WAVES, CB = TN / 8 / WAVES;  // copies a wavefront makes of a stage
  const uint64_t as = p.as * K::BYTES, bs = p.bs * K::BYTES;
  // A lane's offset in copy i of n; NOWHERE where the piece is past the matrix.
  // `me` is its offset in copy 0 (ROWS) and hidden from the compiler inside
  // the loop, which would otherwise keep every copy's in a register.
  auto copy_offset = [&](auto layout, int width, int limit, uint64_t stride, int n, int i, uint32_t me) -> uint32_t {
    constexpr int L = decltype(layout)::value;
    if constexpr (L == ROWS) {
      return (uint32_t)((wave * n + i) * 8 * stride) + me;
    } else {
      const int per = width / 8;  // pieces in a row
      const int k = (wave * n + i) * (64 / per) + lane / per, c = (lane % per) ^ cols_swizzle(k);
      return c * 8 < limit ? (uint32_t)(k * stride) + c * 16 : NOWHERE;
    }
  };

  const uint32_t lds0 = lds_address(lds);
  // Steps past the last one copy zeros.
  auto stage_copies = [&](auto layout, const char* base, int width, int limit, uint64_t stride, auto n, uint32_t me,
                          uint32_t to, int step) {
    constexpr int L = decltype(layout)::value;
    constexpr int N = decltype(n)::value;
    const int left = tail - step * K::STEP;  // summed elements from here on
    const auto rs = L == ROWS ? tile_rsrc(base + (uint64_t)step * 128,
                                          left > 0 ? (limit - 1) * stride + (uint64_t)(left * K::BYTES) : 0)
                              : tile_rsrc(base + (uint64_t)step * K::STEP * stride,
                                          left > 0 ? (left - 1) * stride + limit * 2 : 0);
    if constexpr (L == ROWS) asm volatile("" : "+v"(me));
    // pieces past the rows' end are zeros (packed rows are whole blocks)
    const bool in = L != ROWS || K::FP8 || (((lane & 7) ^ (lane >> 3)) << 4) < left * K::BYTES;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const uint32_t o = copy_offset(layout, width, limit, stride, N, i, me);
      copy16(rs, in ? o : NOWHERE, to + (wave * N + i) * 1024);
    }
  };
  // PACKED: thread t decodes 8 columns of rows t / (TN / 8) + i * THREADS / (TN / 8)
  constexpr int PR = K::THREADS / (TN / 8), PN = K::STEP / PR;
  [[maybe_unused]] uint2 codes[PN];
  [[maybe_unused]] uint32_t bytes[PN];
  auto load_packed = [&](int step) {
    const int c = (threadIdx.x % (TN / 8)) * 8, left = tail - step * K::STEP;
    const uint64_t row = first + (uint64_t)step * K::STEP;
    const auto rc = tile_rsrc((const char*)p.b + row * p.bs + n0, left > 0 ? left * p.bs - n0 : 0);
    const auto rb = tile_rsrc(p.b_scales + row * p.ss + n0 / 128, left > 0 ? left * p.ss - n0 / 128 : 0);
#pragma unroll
    for (int i = 0; i < PN; ++i) {
      const int k = threadIdx.x / (TN / 8) + i * PR;
      typedef int i2v __attribute__((ext_vector_type(2)));
      const i2v w = __builtin_amdgcn_raw_buffer_load_b64(rc, c < cols ? k * (int)p.bs + c : (int)NOWHERE, 0, 0);
      codes[i] = __builtin_bit_cast(uint2, w);
      bytes[i] = __builtin_amdgcn_raw_buffer_load_b8(rb, c < cols ? k * (int)p.ss + c / 128 : (int)NOWHERE, 0, 0);
    }
  };
  auto store_packed = [&](uint32_t to) {
    const int c = threadIdx.x % (TN / 8);
#pragma unroll
    for (int i = 0; i < PN; ++i) {
      const int k = threadIdx.x / (TN / 8) + i * PR;
      *reinterpret_cast<uint4*>(lds + to + k * (TN * 2) + ((c ^ cols_swizzle(k)) << 4)) =
          decode_bf16(codes[i].x, codes[i].y, block8_scale(bytes[i]));
    }
  };
  // Fp8: four blocks' scale bytes of every row of the tiles, one word a lane
  auto scale_copies = [&](int step, int at) {  // part `at` of (TM + TN) / 64, the first TM / 64 A's
    const uint32_t to = lds0 + 2 * K::STAGE + ((step >> 2) & 1) * K::SCALES;
    const bool of_a = at < TM / 64;
    const uint64_t row = of_a ? (uint64_t)m0 : (uint64_t)group * p.n + n0;
    const int r = (of_a ? at : at - TM / 64) * 64 + lane, limit = of_a ? rows : cols;
    const auto rs = tile_rsrc((of_a ? p.a_scales : p.b_scales) + row * p.ss + step,
                              step < p.ss ? limit * p.ss - step : 0);
    copy4(rs, r < limit ? (uint32_t)(r * p.ss) : NOWHERE, to + at * 256);
  };
  auto fetch = [&](int step) {
    const uint32_t to = (step & 1) * K::STAGE;
    stage_copies(std::integral_constant<int, LA>{}, pa, TM, rows, as, std::integral_constant<int, CA>{}, row_a,
                 lds0 + to, step);
    if constexpr (LB != PACKED)
      stage_copies(std::integral_constant<int, LB>{}, pb, TN, cols, bs, std::integral_constant<int, CB>{}, row_b,
                   lds0 + to + K::A_BYTES, step);
    if constexpr (K::FP8)
      if ((step & 3) == 0 && step < steps) scale_copies(step, wave);
  };

  // Fragments. A lane holds row (lane & 15) of a 16-row tile and 8 summed
  // elements from 8 (lane >> 4) on, of every 32 (Fp8: 16 from 16 (lane >> 4)
  // on and 16 from 64 past those, of 128: any order does that A and B share,
  // a block having one scale).
  const int r16 = lane & 15, q = lane >> 4;
  auto rows_at = [&](int wtile, int half) {  // of tile 0 of this wavefront
    return (uint32_t)((wtile * 16 + r16) * 128 + (((half * 4 + q) ^ (r16 & 7)) << 4));
  };
  auto cols_at = [&](int wtile, int width) {
    const int k = 8 * q + (r16 >> 2);
    return (uint32_t)(k * (width * 2) + (((wtile << 1) ^ cols_swizzle(k)) << 4) + (r16 & 3) * 8);
  };
  [[maybe_unused]] const uint32_t rows_half0 = rows_at(0, 0), rows_half1 = rows_at(0, 1);
  [[maybe_unused]] const uint32_t fa0 = LA == ROWS ? rows_at(wm * MT, 0) : cols_at(wm * MT, TM);
  [[maybe_unused]] const uint32_t fb0 = LB == ROWS ? rows_at(wn * NT, 0) : cols_at(wn * NT, TN);
  // tile j of the wavefront, summed elements 32 h to 32 h + 31 (16-bit types)
  auto fragment = [&](auto layout, const char* base, uint32_t at, int j, int h, int width) -> uint4 {
    constexpr int L = decltype(layout)::value;
    if constexpr (L == ROWS) {
      return *reinterpret_cast<const uint4*>(base + (at ^ (h << 6)) + j * 2048);
    } else {
      typedef short s4v __attribute__((ext_vector_type(4)));
      typedef __attribute__((address_space(3))) s4v* lds_s4;
      const char* b = base + (at ^ (j << 5)) + h * 64 * width;
      const s4v x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)b);
      const s4v y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(b + 8 * width));
      const uint2 lo = __builtin_bit_cast(uint2, x), hi = __builtin_bit_cast(uint2, y);
      return make_uint4(lo.x, lo.y, hi.x, hi.y);
    }
  };

  f4v acc[MT][NT] = {};
  if constexpr (!K::FP8) {
    // A step's fragments are two halves of 32 summed elements, each read while
    // the other is multiplied; between a step's halves its stage has been read
    // and the next one has landed, so the barrier there frees the one for the
    // step after next and opens the other.
    struct Half {
      uint4 a[MT], b[NT];
    };
    auto read = [&](Half& f, int step, int h) {
      const char* base = lds + (step & 1) * K::STAGE;
#pragma unroll
      for (int j = 0; j < NT; ++j)
        f.b[j] = fragment(std::integral_constant<int, LB>{}, base + K::A_BYTES, fb0, j, h, TN);
#pragma unroll
      for (int i = 0; i < MT; ++i) f.a[i] = fragment(std::integral_constant<int, LA>{}, base, fa0, i, h, TM);
    };
    auto multiply = [&](const Half& f) {
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = mfma16<T>(f.b[j], f.a[i], acc[i][j]);
    };
    // one LDS read to every few matrix instructions
    auto interleave = [&] {
      constexpr int READS = (LA == ROWS ? 1 : 2) * MT + (LB == ROWS ? 1 : 2) * NT, PER = MT * NT / READS;
#pragma unroll
      for (int i = 0; i < READS; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x008, PER, 0);
      }
      __builtin_amdgcn_sched_group_barrier(0x008, MT * NT - READS * PER, 0);
    };
    auto next = [&](int step) {  // the copies of a step, and of PACKED its codes into registers
      fetch(step);
      if constexpr (LB == PACKED) load_packed(step);
    };
    auto decode = [&](int step) {
      if constexpr (LB == PACKED) store_packed((step & 1) * K::STAGE + K::A_BYTES);
    };
    auto landed = [&] {
      wait_copies();
      __syncthreads();
    };
    if (steps > 0) {
      Half even, odd;
      next(0);
      decode(0);
      landed();
      next(1);
      read(even, 0, 0);
      for (int step = 0; step < steps - 1; ++step) {
        read(odd, step, 1);
        multiply(even);
        interleave();
        decode(step + 1);
        landed();
        next(step + 2);
        read(even, step + 1, 0);
        multiply(odd);
        interleave();
      }
      read(odd, steps - 1, 1);
      multiply(even);
      interleave();
      multiply(odd);
      wait_copies();  // those of the step past the last
    }
  } else {
    // Wavefronts 0 to 3 and 4 to 7, one of each on every SIMD, take turns: one
    // half reads a step's fragments while the other multiplies, with a barrier
    // between the turns. The first half reads step s in turn 2 s and
    // multiplies it in turn 2 s + 1, the second half is a turn behind. Step
    // s's stage has then been read by the end of turn 2 s + 1, is filled for
    // step s + 2 by copies issued in turn 2 s + 2, and has landed by the end of
    // turn 2 s + 3.
    static_assert(K::WAVES == 8, "two wavefronts on a SIMD");
    struct Fragment {
      i8v v;
      int scale;
    };
    auto read = [&](const char* at, int step, int row) {
      Fragment f;
      const uint4 x = *reinterpret_cast<const uint4*>(at + rows_half0);
      const uint4 y = *reinterpret_cast<const uint4*>(at + rows_half1);
      f.v = i8v{(int)x.x, (int)x.y, (int)x.z, (int)x.w, (int)y.x, (int)y.y, (int)y.z, (int)y.w};
      f.scale = (uint8_t)lds[2 * K::STAGE + ((step >> 2) & 1) * K::SCALES + (row + r16) * 4 + (step & 3)];
      return f;
    };
    const bool second = wave >= 4;
    Fragment fa[MT], fb[NT];
    auto read_step = [&](int step) {
      const char* base = lds + (step & 1) * K::STAGE;
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const int row = (wn * NT + j) * 16;
        fb[j] = read(base + K::A_BYTES + row * 128, step, TM + row);
      }
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const int row = (wm * MT + i) * 16;
        fa[i] = read(base + row * 128, step, row);
      }
    };
    auto multiply_row = [&](int i) {
#pragma unroll
      for (int j = 0; j < NT; ++j)
        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fb[j].v, fa[i].v, acc[i][j], 0, 0, 0,
                                                                     fb[j].scale, 0, fa[i].scale);
    };
    auto turn = [&] {  // LDS reads have returned
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_barrier();
      __builtin_amdgcn_sched_barrier(0);
    };
    // the second half's share of a step's copies: all of them, MT parts
    const uint32_t row_off = (lane >> 3) * (uint32_t)p.as + (((lane & 7) ^ (lane >> 3)) << 4);
    auto copy_part = [&](__amdgpu_buffer_rsrc_t ra, __amdgpu_buffer_rsrc_t rb, int step, int i) {
      uint32_t me = row_off;
      asm volatile("" : "+v"(me));
      const int at = (wave & 3) * MT + i;
      const uint32_t to = lds0 + (step & 1) * K::STAGE + at * 1024;
      static_assert(TM == 32 * MT && TN == TM);
      copy16(ra, (uint32_t)(at * 8 * as) + me, to);
      copy16(rb, (uint32_t)(at * 8 * as) + me, to + K::A_BYTES);
    };
    if (steps > 0) {
      fetch(0);
      wait_copies();
      turn();
      if (second) {
        auto copies_of = [&](const char* base, int limit, int step) {
          return tile_rsrc(base + (uint64_t)step * 128, step < steps ? (limit - 1) * as + (tail - step * 128) : 0);
        };
        {
          const auto ra = copies_of(pa, rows, 1), rb = copies_of(pb, cols, 1);
#pragma unroll
          for (int i = 0; i < MT; ++i) copy_part(ra, rb, 1, i);
        }
        turn();
        for (int step = 0; step < steps; ++step) {
          read_step(step);
          wait_copies();
          turn();
          const auto ra = copies_of(pa, rows, step + 2), rb = copies_of(pb, cols, step + 2);
          if (((step + 2) & 3) == 0 && step + 2 < steps) {
            scale_copies(step + 2, (wave & 3) * 2);
            scale_copies(step + 2, (wave & 3) * 2 + 1);
          }
          __builtin_amdgcn_s_setprio(1);
#pragma unroll
          for (int i = 0; i < MT; ++i) {
            multiply_row(i);
            __builtin_amdgcn_sched_barrier(0);
            copy_part(ra, rb, step + 2, i);
            __builtin_amdgcn_sched_barrier(0);
          }
          __builtin_amdgcn_s_setprio(0);
          turn();
        }
        wait_copies();  // those of the steps past the last
      } else {
        for (int step = 0; step < steps; ++step) {
          read_step(step);
          turn();
          __builtin_amdgcn_s_setprio(1);
#pragma unroll
          for (int i = 0; i < MT; ++i) multiply_row(i);
          __builtin_amdgcn_s_setprio(0);
          turn();
        }
        turn();
      }
    }
  }

  // a lane holds columns 4 q to 4 q + 3 of row r16 of each tile
  O* c = (O*)p.c + group * p.cg + (uint64_t)m0 * p.cs + n0;
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int r = (wm * MT + i) * 16 + r16;
    if (r >= rows) continue;
    O* row = c + (uint64_t)r * p.cs;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const int at = (wn * NT + j) * 16 + 4 * q;
      if (p.c_vec && at + 4 <= cols) {
        typedef O o4v __attribute__((ext_vector_type(4)));
        o4v v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (O)acc[i][j][e];
        *reinterpret_cast<o4v*>(row + at) = v;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (at + e < cols) row[at + e] = (O)acc[i][j][e];
      }
    }
  }
#endif
}

// ---------------------------------------------------------------------------
// Few rows in a group: the time is that of reading the matrices. A workgroup
// takes 16 MT rows and 16 rows of a matrix (COLS: 128 of its columns); its
// eight wavefronts read 128 bytes of each row (COLS: 32 rows) in turn, straight
// into the registers that the matrix cores take, and their partial sums are
// added in LDS, in order.
// ---------------------------------------------------------------------------
template <class T, class O, int LB, bool IS_PACKED, int MT>
__global__ void __launch_bounds__(512) product_few(Product p) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr int WAVES = 8, N16 = LB == ROWS ? 1 : 8;     // tiles of 16 columns of C
  constexpr int TN = 16 * N16, PIECES = LB == ROWS ? 2 : 1;  // loads of a row (ROWS) in a round
  constexpr int ROUND = LB == ROWS ? (IS_PACKED ? 128 : 64) : 32;  // summed elements of a wavefront's round
  constexpr int AHEAD = LB == ROWS ? (IS_PACKED || MT > 1 ? (MT > 2 ? 2 : 4) : 8) : 1;  // rounds loaded before they are multiplied
  __shared__ f4v part[WAVES][N16 * MT][64];
  const int lane = threadIdx.x & 63, r16 = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tiles_n = (p.n + TN - 1) / TN;
  RowTile t;
  if (!find_row_tile(p.offsets, p.groups, p.rows, 16 * MT, (int)(blockIdx.x / tiles_n), t)) return;
  const int n0 = (int)(blockIdx.x % tiles_n) * TN;
  const int rows = t.end - t.row < 16 * MT ? t.end - t.row : 16 * MT, cols = p.n - n0 < TN ? p.n - n0 : TN;
  const int k_end = t.group < 0 ? 0 : p.k, group = t.group < 0 ? 0 : t.group;
  constexpr int BYTES = IS_PACKED ? 1 : 2;
  const auto ra = tile_rsrc((const char*)p.a + (uint64_t)t.row * p.as * BYTES,
                            ((uint64_t)(rows - 1) * p.as + p.k) * BYTES);
  uint32_t oa[MT];  // this lane's rows of A
#pragma unroll
  for (int i = 0; i < MT; ++i)
    oa[i] = 16 * i + r16 < rows ? (uint32_t)((16 * i + r16) * p.as * BYTES) + q * 16 : NOWHERE;
  f4v acc[N16][MT] = {};
  typedef uint32_t u4v __attribute__((ext_vector_type(4)));
  auto load = [&](__amdgpu_buffer_rsrc_t rs, uint32_t offset) {
    return __builtin_bit_cast(uint4, (u4v)__builtin_amdgcn_raw_buffer_load_b128(rs, (int)offset, 0, 0));
  };
  if constexpr (LB == ROWS) {
    const uint64_t row = (uint64_t)group * p.n + n0;  // packed: of the codes
    const auto rb = tile_rsrc(IS_PACKED ? (const char*)p.b + row * p.bs : (const char*)p.b + (group * p.bg + n0 * p.bs) * 2,
                              ((uint64_t)(cols - 1) * p.bs + p.k) * BYTES);
    const uint32_t ob = r16 < cols ? (uint32_t)(r16 * p.bs * BYTES) + q * 16 : NOWHERE;
    [[maybe_unused]] __amdgpu_buffer_rsrc_t rsa, rsb;
    if constexpr (IS_PACKED) {
      rsa = tile_rsrc(p.a_scales + (uint64_t)t.row * p.ss, (uint64_t)rows * p.ss);
      rsb = tile_rsrc(p.b_scales + row * p.ss, (uint64_t)cols * p.ss);
    }
    for (int k0 = wave * ROUND; k0 < k_end; k0 += WAVES * ROUND * AHEAD) {
      uint4 b[AHEAD][PIECES], a[AHEAD][PIECES][MT];
      [[maybe_unused]] uint32_t xb[AHEAD], xa[AHEAD][MT];
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        const int k = k0 + u * WAVES * ROUND;
#pragma unroll
        for (int h = 0; h < PIECES; ++h) {
          // past the rows' end: zeros
          const bool in = (k * BYTES + h * 64 + q * 16) < k_end * BYTES;
          b[u][h] = load(rb, in && ob != NOWHERE ? ob + k * BYTES + h * 64 : NOWHERE);
#pragma unroll
          for (int i = 0; i < MT; ++i)
            a[u][h][i] = load(ra, in && oa[i] != NOWHERE ? oa[i] + k * BYTES + h * 64 : NOWHERE);
        }
        if constexpr (IS_PACKED) {
          const bool in = k < k_end;
          xb[u] = __builtin_amdgcn_raw_buffer_load_b8(rsb, in && r16 < cols ? r16 * (int)p.ss + k / 128 : (int)NOWHERE, 0, 0);
#pragma unroll
          for (int i = 0; i < MT; ++i)
            xa[u][i] = __builtin_amdgcn_raw_buffer_load_b8(
                rsa, in && 16 * i + r16 < rows ? (16 * i + r16) * (int)p.ss + k / 128 : (int)NOWHERE, 0, 0);
        }
      }
      __builtin_amdgcn_sched_barrier(0);  // all of them in flight before the first is waited for
#pragma unroll
      for (int u = 0; u < AHEAD; ++u)
#pragma unroll
        for (int h = 0; h < PIECES; ++h) {
          if constexpr (IS_PACKED) {
            // 16 codes a lane: 8 for each of two instructions, of A as of B
            const float sb = block8_scale(xb[u]);
            const uint4 b0 = decode_bf16(b[u][h].x, b[u][h].y, sb), b1 = decode_bf16(b[u][h].z, b[u][h].w, sb);
#pragma unroll
            for (int i = 0; i < MT; ++i) {
              const float sa = block8_scale(xa[u][i]);
              acc[0][i] = mfma16<T>(b0, decode_bf16(a[u][h][i].x, a[u][h][i].y, sa), acc[0][i]);
              acc[0][i] = mfma16<T>(b1, decode_bf16(a[u][h][i].z, a[u][h][i].w, sa), acc[0][i]);
            }
          } else {
#pragma unroll
            for (int i = 0; i < MT; ++i) acc[0][i] = mfma16<T>(b[u][h], a[u][h][i], acc[0][i]);
          }
        }
    }
  } else {
    const auto rb = tile_rsrc((const char*)p.b + (group * p.bg + n0) * 2, ((uint64_t)(p.k - 1) * p.bs + cols) * 2);
    // 8 columns from 8 r16 on of rows 8 q to 8 q + 7
    const uint32_t ob = 8 * r16 < cols ? (uint32_t)(8 * q * p.bs * 2) + r16 * 16 : NOWHERE;
    for (int k0 = wave * ROUND; k0 < k_end; k0 += WAVES * ROUND) {
      uint4 b[8], a[MT];
#pragma unroll
      for (int j = 0; j < 8; ++j)
        b[j] = load(rb, ob != NOWHERE && k0 + 8 * q + j < k_end ? ob + (uint32_t)((k0 + j) * p.bs * 2) : NOWHERE);
#pragma unroll
      for (int i = 0; i < MT; ++i)
        a[i] = load(ra, oa[i] != NOWHERE && k0 + 8 * q < k_end ? oa[i] + k0 * 2 : NOWHERE);
      __builtin_amdgcn_sched_barrier(0);
      // column c of the eight rows, c even and odd: the low and the high halves of word c / 2
      const uint32_t* w = reinterpret_cast<const uint32_t*>(b);
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        uint32_t v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          v[j] = __builtin_amdgcn_perm(w[(2 * j + 1) * 4 + c / 2], w[2 * j * 4 + c / 2], c & 1 ? 0x07060302 : 0x05040100);
        const uint4 f = make_uint4(v[0], v[1], v[2], v[3]);
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[c][i] = mfma16<T>(f, a[i], acc[c][i]);
      }
    }
  }
#pragma unroll
  for (int c = 0; c < N16; ++c)
#pragma unroll
    for (int i = 0; i < MT; ++i) part[wave][c * MT + i][lane] = acc[c][i];
  __syncthreads();
  O* out = (O*)p.c + (uint64_t)t.row * p.cs + n0;
  for (int j = wave; j < N16 * MT; j += WAVES) {
    const int c = j / MT, i = j % MT;
    f4v s = part[0][j][lane];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) s += part[w][j][lane];
    const int r = 16 * i + r16;
    if (r >= rows) continue;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      // tile c holds columns 4 q to 4 q + 3 (COLS: every eighth column from c on)
      const int at = LB == ROWS ? 4 * q + e : 8 * (4 * q + e) + c;
      if (at < cols) out[(uint64_t)r * p.cs + at] = (O)s[e];
    }
  }
#endif
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
void launch_any(const Product& p, hipStream_t s) {
  const uint64_t tm = FORM == GRAD_WEIGHT ? (uint64_t)p.groups * ((p.m + ANY_TILE - 1) / ANY_TILE)
                                          : row_tiles_max(p.rows, p.groups, ANY_TILE, p.offsets != nullptr);
  const uint64_t tn = (p.n + ANY_TILE - 1) / ANY_TILE;
  hipLaunchKernelGGL((product_any<T, O, FORM, PACKED>), dim3(grid_size(tm * tn)), dim3(256), 0, s, p);
  PXG_HIP(hipGetLastError());
}

template <class T, class O, int FORM, int LA, int LB, int WM, int WN, int MT, int NT>
void launch_tiled(const Product& p, hipStream_t s) {
  using K = Tiled<T, O, FORM, LA, LB, WM, WN, MT, NT>;
  const uint64_t tn = (p.n + K::TN - 1) / K::TN;
  uint64_t tiles;
  if (FORM == GRAD_WEIGHT) tiles = (((p.m + K::TM - 1) / K::TM * tn + 7) / 8) * 8 * p.groups;
  else tiles = (row_tiles_max(p.rows, p.groups, K::TM, p.offsets != nullptr) * tn + 7) / 8 * 8;
  hipLaunchKernelGGL((product_tiled<T, O, FORM, LA, LB, WM, WN, MT, NT>), dim3(grid_size(tiles)), dim3(K::THREADS), 0, s,
                     p);
  PXG_HIP(hipGetLastError());
}

// Whether the tiled product can copy an operand: 16-byte pieces that all
// belong to one row, and a tile's offsets in 31 bits.
bool copies(int bytes, const void* d, uint64_t cols, uint64_t stride, uint64_t group_stride) {
  return ((uint64_t)(uintptr_t)d | cols * bytes | stride * bytes | group_stride * bytes) % 16 == 0 &&
         stride * bytes <= (1u << 22);
}

template <class T, class O, int LB, bool IS_PACKED, int MT>
void launch_few(const Product& p, hipStream_t s) {
  constexpr uint64_t TN = LB == ROWS ? 16 : 128;
  const uint64_t tiles = row_tiles_max(p.rows, p.groups, 16 * MT, p.offsets != nullptr) * ((p.n + TN - 1) / TN);
  hipLaunchKernelGGL((product_few<T, O, LB, IS_PACKED, MT>), dim3(grid_size(tiles)), dim3(512), 0, s, p);
  PXG_HIP(hipGetLastError());
}

template <int FORM, class T, class O, bool IS_PACKED>
void launch_product(Product p, hipStream_t s) {
  p.c_vec = ((uint64_t)(uintptr_t)p.c | p.cs * sizeof(O) | p.cg * sizeof(O)) % (4 * sizeof(O)) == 0;
  constexpr int LA = FORM == GRAD_WEIGHT ? COLS : ROWS;
  constexpr int LB = FORM == FORWARD ? ROWS : FORM == GRAD_INPUT ? COLS : IS_PACKED ? PACKED : COLS;
  constexpr int bytes = FORM == FORWARD && IS_PACKED ? 1 : 2;
  const uint64_t acols = FORM == GRAD_WEIGHT ? p.m : p.k, bcols = FORM == FORWARD ? p.k : p.n;
  if (!copies(bytes, p.a, acols, p.as, 0) || (LB != PACKED && !copies(bytes, p.b, bcols, p.bs, p.bg)))
    return launch_any<FORM, T, O, IS_PACKED>(p, s);
  const uint64_t each = ((uint64_t)p.rows + p.groups - 1) / p.groups;  // rows of a group, on average
  if constexpr (FORM != GRAD_WEIGHT) {
    // COLS spans a matrix' rows with one resource
    if (LB == ROWS || p.k * p.bs * 2 <= 0x7FFFFFFF) {
      if (each <= 16) return launch_few<T, O, LB, IS_PACKED, 1>(p, s);
      if (each <= 32) return launch_few<T, O, LB, IS_PACKED, 2>(p, s);
      if constexpr (LB == ROWS)
        if (each <= 64) return launch_few<T, O, LB, IS_PACKED, 4>(p, s);
    }
  }
  if constexpr (FORM == FORWARD && IS_PACKED) {
    if constexpr (!std::is_same_v<O, float>)
      if (each >= 256) return launch_tiled<Fp8, O, FORM, ROWS, ROWS, 2, 4, 8, 4>(p, s);
    return launch_any<FORM, T, O, IS_PACKED>(p, s);
  } else {
    launch_tiled<T, O, FORM, LA, LB, 2, 4, 8, 4>(p, s);
  }
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
    if (rows == 0) return;
    Product p{d_grad, d_w, d_dx, d_offsets, grad_stride, w_stride, dx_stride, w_group_stride, 0, nullptr, nullptr, 0, (int)rows,
              (int)groups, (int)rows, (int)k, (int)n, false};
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
              (int)groups, (int)n, (int)k, 0, false};
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
              nullptr, (const uint8_t*)d_scales, block8_scale_stride(k), (int)rows, (int)groups, (int)n, (int)k, 0, false};
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
    Product p{d_codes, d_w_codes, d_y, d_offsets, wide, wide, y_stride, n * wide, 0, (const uint8_t*)d_scales,
              (const uint8_t*)d_w_scales, block8_scale_stride(k), (int)rows, (int)groups, (int)rows, (int)n,
              (int)wide, false};
    const hipStream_t s = (hipStream_t)stream;
    if (out_type == PXG_F32) launch_product<FORWARD, __bf16, float, true>(p, s);
    else if (out_type == PXG_F16) launch_product<FORWARD, __bf16, _Float16, true>(p, s);
    else launch_product<FORWARD, __bf16, __bf16, true>(p, s);
  });
}

}  // extern "C"
