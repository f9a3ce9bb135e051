// Matrix products of rows in ragged groups, each group with a matrix of its
// own (expert layers), their gradients, and the same product over packed
// 8-bit rows (block8.hpp).
//
//   forward      y[t, :]  = x[t, :] w_g^T        t in group g, w_g n x k
//   grad input   dx[t, :] = dy[t, :] w_g
//   grad weight  dw_g     = sum over t in g of dy[t, :]^T x[t, :]
//
// Sums of 16-bit products are held in f32 on the matrix cores and rounded
// once, to the output's type; so are those of packed rows into f32. Packed rows
// into 16 bits may be multiplied on the 8-bit cores, which cut products before
// they sum them (run8 below says by how much).
//
// Two kernels. Many rows: the matrix cores bound it, and product_tiled keeps
// them fed. Few: the matrices' bytes do, and product_few streams them. Measured
// in bf16, TFLOP/s (a library product of 8192 x 4096 x 4096 reaches 1385, in 8
// bits without scales 2830; a copy 5.2 TB/s):
//   8192 rows, 4096 -> 4096                    forward 1227, input gradient 1260, weight gradient 1378, packed 2430
//   16384 rows, 2048 -> 2048                           1220,                1150,                 1105,        2080
//   the same in 16 uneven groups                        915,                 880,                  840,        1560
//   8 groups of one row, 2048 -> 2048: 67 MB of matrices in 16 us, input gradient 14, packed 10
#include <algorithm>
#include <cmath>
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
  bool c_vec;           // C's rows are 16-byte aligned
  int limit = 0;        // grad weight: longer groups are summed in parts (groups.hpp),
  float* workspace = nullptr;  // in slots of m x n
  unsigned first = 0;   // workgroups of the launches before this one
};

template <class T>
__device__ __forceinline__ f4v mfma16(uint4 a, uint4 b, f4v c) {
  if constexpr (std::is_same_v<T, __bf16>)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8v, a), __builtin_bit_cast(bf8v, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(hf8v, a), __builtin_bit_cast(hf8v, b), c, 0, 0, 0);
}

// ---------------------------------------------------------------------------
// The tiled product: operands go to LDS by direct copies, 128 bytes of each
// row (or 64 rows, where the summed index runs across them) at a time, into
// one of two stages while the other is multiplied. A 256 x 256 tile takes 128
// FLOP from each byte that it copies, 43 from each that it reads out of LDS;
// its two stages fill 128 KB of the 160. What bounds it at many rows is the
// matrix cores' clock under that load; in uneven groups, the partial tiles and
// the last round of tiles.
// ---------------------------------------------------------------------------
// How an operand lies in memory:
//   ROWS    the summed index along its rows
//   COLS    the summed index across its rows; fragments come out of LDS by
//           transposing reads
//   PACKED_ROWS, PACKED_COLS  the same of packed rows; codes are decoded on
//           their way to LDS
//   ANY_ROWS, ANY_COLS  the same of rows that are not whole 16-byte pieces;
//           they are shifted into place on their way to LDS
enum Layout { ROWS, COLS, PACKED_ROWS, PACKED_COLS, ANY_ROWS, ANY_COLS };
constexpr bool is_packed(int l) { return l == PACKED_ROWS || l == PACKED_COLS; }
constexpr bool is_any(int l) { return l == ANY_ROWS || l == ANY_COLS; }
constexpr bool is_rows(int l) { return l == ROWS || l == PACKED_ROWS || l == ANY_ROWS; }
constexpr bool is_copied(int l) { return l == ROWS || l == COLS; }

struct Fp8 {};  // packed operands multiplied as they are

#if defined(__HIP_DEVICE_COMPILE__)
// A workgroup's place among all of a product's launches.
__device__ __forceinline__ unsigned workgroup(const Product& p) { return p.first + blockIdx.x; }

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
// else in these kernels uses m0. Inside asm the compiler adds no wait
// states: a copy needs one after m0's write, and five after a vector
// instruction (a readfirstlane) wrote part of its resource. The resources are
// made further ahead than that, which a test of the built library checks; all
// five inside the asm cost 2% (16384 rows in 32 groups, 2048 -> 2048: input
// gradient 170, 174 us; 8 bits 92, 94). wait_copies() waits for all of them,
// wait_copies_but<N>() for all but the last N.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void copy16(__amdgpu_buffer_rsrc_t rs, uint32_t offset, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(offset), "s"(rs)
               : "memory", "m0");
}
__device__ __forceinline__ void copy4(__amdgpu_buffer_rsrc_t rs, uint32_t offset, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds" ::"s"(lds), "v"(offset), "s"(rs)
               : "memory", "m0");
}
#pragma clang diagnostic pop
template <int N>
__device__ __forceinline__ void wait_copies_but() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ void wait_copies() { wait_copies_but<0>(); }

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

// A barrier after the wavefront's LDS accesses; copies stay in flight.
__device__ __forceinline__ void lds_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// By how many 16-byte pieces row k of a stage is moved: a transposing read
// takes 32 bytes of rows 8 q + {0..3} (or {4..7}) for each 16 lanes q. Rows of
// 64 elements have four such pieces only.
template <int WIDTH>
__device__ __forceinline__ int cols_swizzle(int k) {
  return (WIDTH == 64 ? k & 3 : (k & 3) | ((k >> 1) & 4)) << 1;
}

// Part `die` of n cut into eight, the larger parts first: its first and size.
__device__ __forceinline__ void eighth(int n, int die, int& first, int& size) {
  const int each = n >> 3, more = n & 7;
  first = die * each + (die < more ? die : more);
  size = each + (die < more ? 1 : 0);
}
#endif

// WM x WN wavefronts, each with MT x NT tiles of 16 x 16. T is the type
// multiplied: bf16, f16 or Fp8.
template <class T, int WM, int WN, int MT, int NT>
struct Tiled {
  static constexpr int THREADS = 64 * WM * WN, WAVES = WM * WN;
  static constexpr int TM = 16 * WM * MT, TN = 16 * WN * NT;
  static constexpr bool FP8 = std::is_same_v<T, Fp8>;
  static constexpr int BYTES = FP8 ? 1 : 2;       // of an element
  static constexpr int STEP = 128 / BYTES;        // summed elements a stage holds
  static constexpr int A_BYTES = TM * 128, B_BYTES = TN * 128, STAGE = A_BYTES + B_BYTES;
  static constexpr int SCALES = FP8 ? (TM + TN) * 4 : 0;  // four blocks' scale bytes of each row
  // a large tile's stages, or three of half its rows
  static constexpr int LDS = std::max(2 * (STAGE + SCALES), THREADS == 512 && !FP8 ? 3 * (STAGE - A_BYTES / 2) : 0);
};

template <class T, class O, int FORM, int LA, int LB, int WM, int WN, int MT, int NT>
__global__ void __launch_bounds__(64 * WM * WN) product_tiled(Product p) {
#if defined(__HIP_DEVICE_COMPILE__)
  using K = Tiled<T, WM, WN, MT, NT>;
  constexpr int TM = K::TM, TN = K::TN, WAVES = K::WAVES;
  __shared__ __align__(1024) char lds[K::LDS];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WN, wn = wave % WN;

  // This workgroup's tile. Workgroups go to the eight dies in turn. Each die
  // takes an eighth of the tiles, in order, so that tiles that share operands
  // meet in one L2; the longest come first, as what begins last ends last.
  const int tiles_n = (p.n + TN - 1) / TN;
  // weight gradients fit one launch (their first place added costs 1 to 4%)
  const unsigned place = FORM == GRAD_WEIGHT ? blockIdx.x : workgroup(p);
  const int die = place & 7, at = place >> 3;
  int m0, n0, rows, cols, steps, group, tail;
  uint64_t a0, b0;  // first elements of the operands' tiles
  [[maybe_unused]] uint64_t sa0 = 0, sb0 = 0;  // and their rows, packed
  [[maybe_unused]] int slot = -1;              // of the workspace, for a group summed in parts
  if constexpr (FORM == GRAD_WEIGHT) {
    // an eighth of every part's tiles, the longest part first
    const int tiles_m = (p.m + TM - 1) / TM, each = tiles_m * tiles_n, per = (each + 7) / 8;
    const int t = die * per + at % per;
    GroupPart part;
    if (t >= each || !find_group_part(p.offsets, p.groups, p.rows, p.limit, at / per, part)) return;
    group = part.group;
    slot = part.parts > 1 ? part.slot : -1;
    const int lo = part.lo, hi = part.hi;
    m0 = t / tiles_n * TM;
    n0 = t % tiles_n * TN;
    rows = p.m - m0;
    tail = hi - lo;
    a0 = (uint64_t)lo * p.as + m0;
    b0 = (uint64_t)lo * p.bs + n0;
    sb0 = (uint64_t)lo * p.ss + n0 / 128;
  } else {
    // an eighth of the whole row tiles, then of the partial ones. The 32
    // workgroups that run together on a die share operands best as a block of
    // 4 row tiles by 8 (8192 rows, 4096 -> 4096: 224 us; in rows of tiles 229).
    int whole, partial, first, size;
    // one load of the offsets (8 groups of 8192 rows, 1024 -> 4096: 2 us less than rounds of them)
    const bool few = p.offsets && p.groups <= SEGMENT_GROUPS;
    Segments segments{};
    if (few) {
      segments = load_segments(p.offsets, p.groups, p.rows);
      count_segments(segments, TM, whole, partial);
    } else {
      count_row_tiles(p.offsets, p.groups, p.rows, TM, whole, partial);
    }
    eighth(whole * tiles_n, die, first, size);
    const bool is_whole = at < size;
    int index = first + at, count = whole;
    if (!is_whole) {
      index = at - size;
      eighth(partial * tiles_n, 7 - die, first, size);
      if (index >= size) return;
      index += first;
      count = partial;
    }
    const int band = index / (4 * tiles_n), in = index - band * 4 * tiles_n;
    const int high = count - band * 4 < 4 ? count - band * 4 : 4;
    RowTile t;
    const int nth = band * 4 + in % high;
    if (few) {
      if (is_whole) pick_row_tile<WHOLE_TILES>(segments, p.groups, TM, nth, t);
      else pick_row_tile<PARTIAL_TILES>(segments, p.groups, TM, nth, t);
    } else {
      if (is_whole) find_row_tile<WHOLE_TILES>(p.offsets, p.groups, p.rows, TM, nth, t);
      else find_row_tile<PARTIAL_TILES>(p.offsets, p.groups, p.rows, TM, nth, t);
    }
    m0 = t.row;
    n0 = in / high * TN;
    group = t.group < 0 ? 0 : t.group;
    rows = t.end - m0;
    tail = t.group < 0 ? 0 : p.k;
    a0 = (uint64_t)m0 * p.as;
    b0 = group * p.bg + (is_rows(LB) ? (uint64_t)n0 * p.bs : (uint64_t)n0);
    sa0 = (uint64_t)m0 * p.ss;
    sb0 = ((uint64_t)group * p.n + n0) * p.ss;
  }
  steps = (tail + K::STEP - 1) / K::STEP;
  rows = rows < TM ? rows : TM;
  cols = p.n - n0 < TN ? p.n - n0 : TN;

  // Dies begin at different places of the sum: rows a power of two apart
  // otherwise have all of them read the same memory channels (32 groups of 128
  // rows, 2048 -> 2048: forward 52 us, 59 without). Four steps share a word of
  // scale bytes.
  const int spin = !K::FP8 ? steps / 8 * die : steps % 4 == 0 ? steps / 32 * 4 * die : 0;
  int source = spin;  // of the step copied last: its place in the sum
  auto advance = [&] { source = source + 1 < steps ? source + 1 : 0; };

  // Copies. ROWS: a copy of one wavefront fills 8 rows of 128 bytes, 16-byte
  // piece c of row r at place c ^ (r & 7), so that 8 lanes reading piece c of
  // 8 rows meet every bank. COLS: it fills 1024 bytes of rows of 2 TM (2 TN)
  // bytes, piece c of row k at c ^ cols_swizzle(k): of the two quarters of a
  // transposing read that go together, the eight rows lie in different banks.
  struct Operand {
    const char* base;  // the tile's first element
    const uint8_t* scales;
    uint64_t stride;  // bytes from row to row
    int limit;        // rows (COLS: columns) of the tile inside the matrix
    uint32_t row;     // ROWS: this lane's offset in copy 0
  };
  auto operand = [&](const void* base, uint64_t first, const uint8_t* scales, uint64_t row, uint64_t stride, int limit,
                     int bytes) {
    return Operand{(const char*)base + first * bytes, scales + row, stride * bytes, limit,
                   (lane >> 3) * (uint32_t)(stride * bytes) + (((lane & 7) ^ (lane >> 3)) << 4)};
  };
  const Operand A = operand(p.a, a0, p.a_scales, sa0, p.as, rows, is_packed(LA) ? 1 : K::BYTES);
  const Operand B = operand(p.b, b0, p.b_scales, sb0, p.bs, cols, is_packed(LB) ? 1 : K::BYTES);
  const uint32_t lds0 = lds_address(lds);
  // A step's elements of an operand from the tile's first on; none past the
  // last step, whose copies then write zeros without reading.
  auto stage_resource = [&](auto layout, const Operand& o, int step) {
    const int left = tail - source * K::STEP;  // summed elements from here on
    return decltype(layout)::value == ROWS
               ? tile_rsrc(o.base + (uint64_t)source * 128,
                           step < steps ? (o.limit - 1) * o.stride + (uint64_t)(left * K::BYTES) : 0)
               : tile_rsrc(o.base + (uint64_t)source * K::STEP * o.stride,
                           step < steps ? (left - 1) * o.stride + o.limit * 2 : 0);
  };
  // one wavefront's part of its copies, to an operand's place in a stage
  auto stage_copy = [&](auto layout, auto width, const Operand& o, __amdgpu_buffer_rsrc_t rs, int place, int part) {
    const uint32_t to = lds0 + place + part * 1024;
    if constexpr (decltype(layout)::value == ROWS) {
      uint32_t at = o.row;
      asm volatile("" : "+v"(at));  // keeps one register for all parts, not one for each
      // pieces past the rows' end are zeros (packed rows are whole blocks)
      const bool in = K::FP8 || (((lane & 7) ^ (lane >> 3)) << 4) < (tail - source * K::STEP) * K::BYTES;
      copy16(rs, in ? (uint32_t)(part * 8 * o.stride) + at : NOWHERE, to);
    } else {
      constexpr int PER = decltype(width)::value / 8;  // pieces in a row
      int me = lane;
      if constexpr (is_packed(LB)) asm volatile("" : "+v"(me));  // registers are short there
      const int k = part * (64 / PER) + me / PER, c = (me % PER) ^ cols_swizzle<decltype(width)::value>(k);
      copy16(rs, c * 8 < o.limit ? (uint32_t)(k * (int)o.stride) + c * 16 : NOWHERE, to);
    }
  };
  using LayoutA = std::integral_constant<int, LA>;
  using LayoutB = std::integral_constant<int, LB>;
  using WidthA = std::integral_constant<int, TM>;
  using WidthB = std::integral_constant<int, TN>;
  auto stage_copies = [&](auto layout, auto width, const Operand& o, int step, int place) {
    if constexpr (is_copied(decltype(layout)::value)) {
      constexpr int N = decltype(width)::value / 8 / WAVES;
      const auto rs = stage_resource(layout, o, step);
#pragma unroll
      for (int i = 0; i < N; ++i) stage_copy(layout, width, o, rs, place, wave * N + i);
    }
  };
  // Packed: a thread takes 8 codes at a time, of row (COLS: summed element)
  // `line`, piece `c` of 8, reads them a step ahead and decodes them.
  // ANY: the same with 16 elements. Rows begin at any multiple of two bytes,
  // so the nine words that the elements touch are read and shifted. A word
  // that the row shares with a neighbour is read whole; elements of other rows
  // are set to zero.
  struct Staged {
    uint4 lo[4], hi[2];
    uint32_t last[4];  // ANY: the ninth word; packed: the scale byte
  };
  auto pieces = [&](auto layout, auto width, auto f) {
    constexpr int L = decltype(layout)::value, W = decltype(width)::value, SIZE = is_any(L) ? 16 : 8;
    constexpr int PER = (is_rows(L) ? K::STEP : W) / SIZE;  // pieces in a line
    constexpr int N = W * K::STEP / SIZE / K::THREADS;
    static_assert(N <= (is_any(L) ? 2 : 4));
#pragma unroll
    for (int i = 0; i < N; ++i) f(i, (int)threadIdx.x / PER + i * (K::THREADS / PER), (int)threadIdx.x % PER);
  };
  auto load_staged = [&](auto layout, auto width, const Operand& o, int step, Staged& x) {
    constexpr int L = decltype(layout)::value;
    const int left = step < steps ? tail - source * K::STEP : 0;
    [[maybe_unused]] auto load = [](__amdgpu_buffer_rsrc_t rs, uint32_t at) {
      typedef uint32_t u4v __attribute__((ext_vector_type(4)));
      return __builtin_bit_cast(uint4, (u4v)__builtin_amdgcn_raw_buffer_load_b128(rs, (int)at, 0, 0));
    };
    if constexpr (is_packed(L)) {
      typedef int i2v __attribute__((ext_vector_type(2)));
      const uint64_t lines = L == PACKED_ROWS ? (left > 0 ? o.limit : 0) : left > 0 ? left : 0;
      // resources end with the last line that counts; a line's own end is a multiple of 128 columns
      const uint64_t codes0 = L == PACKED_ROWS ? (uint64_t)source * 64 : (uint64_t)source * K::STEP * o.stride;
      const uint64_t scales0 = L == PACKED_ROWS ? (uint64_t)source / 2 : (uint64_t)source * K::STEP * p.ss;
      const uint64_t skip = L == PACKED_ROWS ? codes0 : n0, skip_s = L == PACKED_ROWS ? scales0 : n0 / 128;
      const auto rc = tile_rsrc(o.base + codes0, lines ? lines * o.stride - skip : 0);
      const auto rb = tile_rsrc(o.scales + scales0, lines ? lines * p.ss - skip_s : 0);
      // of a block, the columns before the tile's first
      const int before = L == PACKED_ROWS ? 0 : n0 % 128;
      pieces(layout, width, [&](int i, int line, int c) {
        const bool in = L == PACKED_ROWS ? line < o.limit : c * 8 < o.limit;
        const i2v w = __builtin_amdgcn_raw_buffer_load_b64(rc, in ? line * (int)o.stride + c * 8 : (int)NOWHERE, 0, 0);
        x.lo[i].x = w[0];
        x.lo[i].y = w[1];
        x.last[i] = __builtin_amdgcn_raw_buffer_load_b8(
            rb, in ? line * (int)p.ss + (L == PACKED_ROWS ? 0 : (before + c * 8) / 128) : (int)NOWHERE, 0, 0);
      });
    } else if constexpr (is_any(L)) {
      const int odd = (int)((uintptr_t)o.base & 2);
      const uint64_t end = L == ANY_ROWS ? (o.limit - 1) * o.stride + (uint64_t)left * 2
                                         : (uint64_t)(left - 1) * o.stride + o.limit * 2;
      const auto rs = tile_rsrc(o.base - odd + (L == ANY_ROWS ? (uint64_t)source * 128 : (uint64_t)source * K::STEP * o.stride),
                                left > 0 ? (end + odd + 3) & ~3ull : 0);
      pieces(layout, width, [&](int i, int line, int c) {
        const bool in = L == ANY_ROWS ? line < o.limit && c * 16 < left : line < left && c * 16 < o.limit;
        const uint32_t at = in ? (odd + line * (uint32_t)o.stride + c * 32) & ~3u : NOWHERE;
        x.lo[i] = load(rs, at);
        x.hi[i] = load(rs, in ? at + 16 : NOWHERE);
        x.last[i] = __builtin_amdgcn_raw_buffer_load_b32(rs, in ? (int)at + 32 : (int)NOWHERE, 0, 0);
      });
    }
  };
  auto store_staged = [&](auto layout, auto width, const Operand& o, int at, const Staged& x) {
    constexpr int L = decltype(layout)::value, W = decltype(width)::value;
    char* to = lds + at;
    auto place = [&](int line, int c) {
      return reinterpret_cast<uint4*>(
          to + (is_rows(L) ? line * 128 + ((c ^ (line & 7)) << 4) : line * (W * 2) + ((c ^ cols_swizzle<W>(line)) << 4)));
    };
    if constexpr (is_packed(L)) {
      pieces(layout, width, [&](int i, int line, int c) {
        *place(line, c) = decode_bf16(x.lo[i].x, x.lo[i].y, block8_scale(x.last[i]));
      });
    } else if constexpr (is_any(L)) {
      const int left = tail - source * K::STEP;
      pieces(layout, width, [&](int i, int line, int c) {
        const uint32_t shift = (((uint32_t)(uintptr_t)o.base + line * (uint32_t)o.stride) & 2) * 8;
        const int valid = (L == ANY_ROWS ? left : o.limit) - c * 16;
        const uint32_t w[9] = {x.lo[i].x, x.lo[i].y, x.lo[i].z, x.lo[i].w, x.hi[i].x,
                               x.hi[i].y, x.hi[i].z, x.hi[i].w, x.last[i]};
        uint32_t v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t both = __builtin_amdgcn_alignbit(w[e + 1], w[e], shift);
          v[e] = valid > 2 * e + 1 ? both : valid > 2 * e ? both & 0xFFFF : 0;
        }
        *place(line, 2 * c) = make_uint4(v[0], v[1], v[2], v[3]);
        *place(line, 2 * c + 1) = make_uint4(v[4], v[5], v[6], v[7]);
      });
    }
  };

  // Fragments. A lane holds row (lane & 15) of a 16-row tile and 8 summed
  // elements from 8 (lane >> 4) on, of every 32 (Fp8: 16 from 16 (lane >> 4)
  // on and 16 from 64 past those, of 128: any order does that A and B share,
  // a block having one scale). Tile i of wavefront row wm is tile i WM + wm of
  // A's, so that a partial tile's rows are spread over all wavefronts; B's
  // tiles of a wavefront are adjacent.
  const int r16 = lane & 15, q = lane >> 4;
  auto rows_at = [&](int tile, int half) {
    return (uint32_t)((tile * 16 + r16) * 128 + (((half * 4 + q) ^ (r16 & 7)) << 4));
  };
  auto cols_at = [&](int tile, auto width) {
    constexpr int W = decltype(width)::value;
    const int k = 8 * q + (r16 >> 2);
    return (uint32_t)(k * (W * 2) + (((tile << 1) ^ cols_swizzle<W>(k)) << 4) + (r16 & 3) * 8);
  };

  f4v acc[MT][NT] = {};
  // LIVE of a wavefront's MT row tiles are inside the matrix.
  [[maybe_unused]] auto run16 = [&](auto live) {
    // A step's fragments are two halves of 32 summed elements, each read while
    // the other is multiplied; between a step's halves its stage has been read
    // and the next one has landed, so the barrier there frees the one for the
    // step after next and opens the other.
    constexpr int LIVE = decltype(live)::value;
    // A partial row tile of at most half the rows has room for a third stage,
    // which its little work needs to hide the copies' latency (32 groups of 128
    // rows, 2048 -> 2048: forward 51 us, 59 with two; without a loop for half the
    // rows 62. Uneven groups gain nothing: 16384 rows in 16, 160 us of either).
    constexpr bool DEEP = FORM != GRAD_WEIGHT && is_copied(LB) && K::THREADS == 512 && 2 * LIVE <= MT;
    constexpr int STAGES = DEEP ? 3 : 2, AW = DEEP ? TM / 2 : TM, STAGE = AW * 128 + K::B_BYTES;
    constexpr int COPIES = (AW + TN) / 8 / WAVES;  // of a wavefront in a step
    static_assert(STAGES * STAGE <= K::LDS);
    using WideA = std::integral_constant<int, AW>;
    const uint32_t fa0 = is_rows(LA) ? rows_at(wm, 0) : cols_at(wm, WidthA{});
    const uint32_t fb0 = is_rows(LB) ? rows_at(wn * NT, 0) : cols_at(wn * NT, WidthB{});
    // the tile j tiles on, summed elements 32 h to 32 h + 31
    auto fragment = [&](auto layout, auto width, const char* base, uint32_t at, int j, int h) -> uint4 {
      if constexpr (is_rows(decltype(layout)::value)) {
        return *reinterpret_cast<const uint4*>(base + (at ^ (h << 6)) + j * 2048);
      } else {
        constexpr int W = decltype(width)::value;
        typedef short s4v __attribute__((ext_vector_type(4)));
        typedef __attribute__((address_space(3))) s4v* lds_s4;
        const char* b = base + (at ^ (j << 5)) + h * 64 * W;
        const s4v x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)b);
        const s4v y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(b + 8 * W));
        const uint2 lo = __builtin_bit_cast(uint2, x), hi = __builtin_bit_cast(uint2, y);
        return make_uint4(lo.x, lo.y, hi.x, hi.y);
      }
    };
    struct Half {
      uint4 a[LIVE], b[NT];
    };
    int slot = 0;  // the stage of the step being multiplied
    auto later = [&](int by) { return slot + by < STAGES ? slot + by : slot + by - STAGES; };
    auto read = [&](Half& f, int at, int h) {
      const char* base = lds + at * STAGE;
#pragma unroll
      for (int j = 0; j < NT; ++j) f.b[j] = fragment(LayoutB{}, WidthB{}, base + AW * 128, fb0, j, h);
#pragma unroll
      for (int i = 0; i < LIVE; ++i) f.a[i] = fragment(LayoutA{}, WidthA{}, base, fa0, i * WM, h);
    };
    auto multiply = [&](const Half& f) {
#pragma unroll
      for (int i = 0; i < LIVE; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = mfma16<T>(f.b[j], f.a[i], acc[i][j]);
    };
    // one LDS read to every few matrix instructions
    auto interleave = [&] {
      constexpr int READS = (is_rows(LA) ? 1 : 2) * LIVE + (is_rows(LB) ? 1 : 2) * NT, PER = LIVE * NT / READS;
      if constexpr (PER > 0) {
#pragma unroll
        for (int i = 0; i < READS; ++i) {
          __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x008, PER, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, LIVE * NT - READS * PER, 0);
      }
    };
    Staged xa, xb;
    auto next = [&](int step, int at) {  // a step's copies, and what goes through registers
      if (step > 0) advance();
      stage_copies(LayoutA{}, WideA{}, A, step, at * STAGE);
      stage_copies(LayoutB{}, WidthB{}, B, step, at * STAGE + AW * 128);
      load_staged(LayoutA{}, WidthA{}, A, step, xa);
      load_staged(LayoutB{}, WidthB{}, B, step, xb);
    };
    auto stage = [&](int at) {
      store_staged(LayoutA{}, WidthA{}, A, at * STAGE, xa);
      store_staged(LayoutB{}, WidthB{}, B, at * STAGE + AW * 128, xb);
    };
    Half even, odd;
    if constexpr (is_copied(LA) && is_copied(LB)) {  // all stages' copies fly together
#pragma unroll
      for (int step = 0; step < STAGES; ++step) next(step, step);
      wait_copies_but<(STAGES - 1) * COPIES>();
      lds_barrier();
    } else {
      next(0, 0);
      stage(0);
      wait_copies();
      lds_barrier();
      next(1, 1);
    }
    read(even, 0, 0);
    for (int step = 0; step < steps - 1; ++step) {
      read(odd, slot, 1);
      multiply(even);
      interleave();
      stage(later(1));
      if constexpr (is_copied(LA) && is_copied(LB)) wait_copies_but<(STAGES - 2) * COPIES>();
      else wait_copies();
      lds_barrier();
      next(step + STAGES, slot);
      slot = later(1);
      read(even, slot, 0);
      multiply(odd);
      interleave();
    }
    read(odd, slot, 1);
    multiply(even);
    interleave();
    multiply(odd);
    wait_copies();  // those of the steps past the last
  };
  [[maybe_unused]] auto run8 = [&](auto live) {
    // Wavefronts 0 to 3 and 4 to 7, one of each on every SIMD, take turns: one
    // half reads a step's fragments while the other multiplies, with a barrier
    // between the turns. The first half reads step s in turn 2 s and
    // multiplies it in turn 2 s + 1, the second half is a turn behind and makes
    // the copies, between its matrix instructions. Step s's stage has been
    // read by the end of turn 2 s + 1, is filled for step s + 2 by copies
    // issued in turn 2 s + 2, and has landed by the end of turn 2 s + 3.
    //
    // What the instruction sums (probed over all pairs of codes): of each eight
    // neighbouring products it cuts every one toward zero to a multiple of
    // 2^(E - 13), E the largest sum of two codes' exponents among the eight (-6
    // for a subnormal code; zeros do not count), and adds the eights' sums and
    // the accumulator in f32. A product of normal codes whose exponents' sum is
    // within 7 of E loses nothing. As a whole the result is off by 1.5e-5 of itself for normal
    // data, 2.7e-5 with columns' magnitudes spread as exp(0.7 normal), 7.6e-5
    // with exp(2 normal) (8192 x 4096 x 4096). Rounding to f16 costs 2.08e-4,
    // to bf16 1.66e-3, so that an f16 result's error grows by 0.3, 0.8 and 6%
    // and a bf16 one's by 0.1% at most; packing has cost 2.6e-2 before. Of
    // single elements 7, 10 and 21% (f16; bf16 1, 2 and 4%) are not the exact
    // sum's nearest value.
    constexpr int LIVE = decltype(live)::value;
    static_assert(WAVES == 8 && TM == 32 * MT && TN == TM);
    struct Fragment {
      i8v v;
      int scale;
    };
    Fragment fa[LIVE], fb[NT];
    const uint32_t half0 = rows_at(0, 0), half1 = rows_at(0, 1);
    auto read = [&](const char* at, int step, int row) {
      Fragment f;
      const uint4 x = *reinterpret_cast<const uint4*>(at + half0);
      const uint4 y = *reinterpret_cast<const uint4*>(at + half1);
      f.v = i8v{(int)x.x, (int)x.y, (int)x.z, (int)x.w, (int)y.x, (int)y.y, (int)y.z, (int)y.w};
      f.scale = (uint8_t)lds[2 * K::STAGE + ((step >> 2) & 1) * K::SCALES + (row + r16) * 4 + (step & 3)];
      return f;
    };
    auto read_step = [&](int step) {
      const char* base = lds + (step & 1) * K::STAGE;
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const int row = (wn * NT + j) * 16;
        fb[j] = read(base + K::A_BYTES + row * 128, step, TM + row);
      }
#pragma unroll
      for (int i = 0; i < LIVE; ++i) {
        const int row = (i * WM + wm) * 16;
        fa[i] = read(base + row * 128, step, row);
      }
    };
    auto multiply_row = [&](int i) {
      if (i < LIVE)
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
    // four blocks' scale bytes of every row of the tiles, one word a lane:
    // part `at` of (TM + TN) / 64, the first TM / 64 A's
    auto scale_copies = [&](int step, int at) {
      const uint32_t to = lds0 + 2 * K::STAGE + ((step >> 2) & 1) * K::SCALES;
      const bool of_a = at < TM / 64;
      const int r = (of_a ? at : at - TM / 64) * 64 + lane, limit = of_a ? rows : cols;
      const auto rs = tile_rsrc((of_a ? A.scales : B.scales) + source, step < steps ? limit * p.ss - source : 0);
      copy4(rs, r < limit ? (uint32_t)(r * p.ss) : NOWHERE, to + at * 256);
    };
    stage_copies(LayoutA{}, WidthA{}, A, 0, 0);
    stage_copies(LayoutB{}, WidthB{}, B, 0, K::A_BYTES);
    scale_copies(0, wave);
    if (wave >= 4) {
      auto part = [&](__amdgpu_buffer_rsrc_t ra, __amdgpu_buffer_rsrc_t rb, int step, int i) {
        stage_copy(LayoutA{}, WidthA{}, A, ra, (step & 1) * K::STAGE, (wave & 3) * MT + i);
        stage_copy(LayoutB{}, WidthB{}, B, rb, (step & 1) * K::STAGE + K::A_BYTES, (wave & 3) * MT + i);
      };
      {
        advance();
        const auto ra = stage_resource(LayoutA{}, A, 1), rb = stage_resource(LayoutB{}, B, 1);
#pragma unroll
        for (int i = 0; i < MT; ++i) part(ra, rb, 1, i);
      }
      wait_copies_but<2 * MT>();
      turn();
      turn();
      for (int step = 0; step < steps; ++step) {
        read_step(step);
        wait_copies();
        turn();
        advance();
        const auto ra = stage_resource(LayoutA{}, A, step + 2), rb = stage_resource(LayoutB{}, B, step + 2);
        if (((step + 2) & 3) == 0) {
          scale_copies(step + 2, (wave & 3) * 2);
          scale_copies(step + 2, (wave & 3) * 2 + 1);
        }
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          multiply_row(i);
          __builtin_amdgcn_sched_barrier(0);
          part(ra, rb, step + 2, i);
          __builtin_amdgcn_sched_barrier(0);
        }
        __builtin_amdgcn_s_setprio(0);
        turn();
      }
      wait_copies();  // those of the steps past the last
    } else {
      wait_copies();
      turn();
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
  };
  auto run = [&](auto live) {
    if constexpr (K::FP8) run8(live);
    else run16(live);
  };
  if (steps > 0) {
    // weight gradients have a partial tile only at the matrix' edge (the other
    // loop's registers cost 16 uneven groups, 2048 x 2048, 177 us for 164)
    if (FORM != GRAD_WEIGHT && rows <= TM / 2) run(std::integral_constant<int, MT / 2>{});
    else run(std::integral_constant<int, MT>{});
  }

  // A lane holds columns 4 q to 4 q + 3 of row r16 of each tile. Through LDS,
  // 16 rows of the wavefront's columns at a time, so that what is stored
  // together is whole rows of them and not 8 bytes of each of 16.
  auto store = [&](auto type, void* result, uint64_t stride, bool whole) {
    using R = decltype(type);
    constexpr int EACH = 16 / sizeof(R), PER = NT * 16 / EACH;  // a lane's elements, lanes to a row
    constexpr int PITCH = NT * 16 * sizeof(R) + 16;             // 16 bytes more spread the rows over the banks
    static_assert(WAVES * 16 * PITCH <= K::LDS);
    char* mine = lds + wave * (16 * PITCH);
    R* c = (R*)result + (uint64_t)m0 * stride + n0;
    const int col = wn * NT * 16 + lane % PER * EACH;
#pragma unroll
    for (int i = 0; i < MT; ++i) {
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        typedef R r4v __attribute__((ext_vector_type(4)));
        r4v v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (R)acc[i][j][e];
        *reinterpret_cast<r4v*>(mine + r16 * PITCH + (j * 16 + 4 * q) * sizeof(R)) = v;
      }
      if (whole) {
#pragma unroll
        for (int h = 0; h < 16 * PER / 64; ++h) {
          const int r = lane / PER + h * (64 / PER), row = (i * WM + wm) * 16 + r;
          const uint4 v = *reinterpret_cast<const uint4*>(mine + r * PITCH + lane % PER * 16);
          if (row >= rows) continue;
          R* to = c + (uint64_t)row * stride + col;
          if (col + EACH <= cols) {
            *reinterpret_cast<uint4*>(to) = v;
          } else {
            R x[EACH];
            *reinterpret_cast<uint4*>(x) = v;
#pragma unroll
            for (int e = 0; e < EACH; ++e)
              if (col + e < cols) to[e] = x[e];
          }
        }
      } else {
        // rows that are not 16-byte aligned: an element a lane, of one row or two
        // (8192 rows packed, 2049 -> 1027: 39 us; the pieces' elements in turn 46)
        constexpr int W = NT * 16;
#pragma unroll
        for (int h = 0; h < 16 * W / 64; ++h) {
          const int r = lane / W + h * (64 / W), row = (i * WM + wm) * 16 + r, at = lane % W;
          const R v = *reinterpret_cast<const R*>(mine + r * PITCH + at * sizeof(R));
          if (row < rows && wn * W + at < cols) c[(uint64_t)row * stride + wn * W + at] = v;
        }
      }
    }
  };
  lds_barrier();
  O* result = (O*)p.c + group * p.cg;
  if constexpr (FORM == GRAD_WEIGHT) {
    float* part = p.workspace + (uint64_t)(slot < 0 ? 0 : slot) * p.m * p.n;
    const bool apart = slot >= 0;
    if constexpr (std::is_same_v<O, float>) {  // one piece of code for both
      store(O{}, apart ? part : result, apart ? p.n : p.cs, apart ? p.n % 4 == 0 : p.c_vec);
    } else if (apart) {
      store(float{}, part, p.n, p.n % 4 == 0);
    } else {
      store(O{}, result, p.cs, p.c_vec);
    }
  } else {
    store(O{}, result, p.cs, p.c_vec);
  }
#endif
}

// ---------------------------------------------------------------------------
// Few rows: the time is that of reading the matrices. A workgroup takes 16 rows
// and 16 rows of a matrix (COLS: 128 of its columns); its eight wavefronts read
// 128 bytes of each row (COLS: 32 rows) in turn, straight into the registers
// that the matrix cores take, and their partial sums are added in LDS, in
// order. Through LDS, a step would wait for its barrier with little to
// multiply. Two workgroups on a CU read while one another's sums are joined:
// two rounds of loads in registers are faster than eight with one workgroup
// (16 groups of one row, 2048 -> 2048: 29 us, 41; one row, 4096 -> 4096: 8.8, 8.9).
// ---------------------------------------------------------------------------
template <class T, class O, int LB, bool IS_PACKED>
__global__ void __launch_bounds__(512, 4) product_few(Product p) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr int WAVES = 8, N16 = LB == ROWS ? 1 : 8;     // tiles of 16 columns of C
  constexpr int TN = 16 * N16, PIECES = LB == ROWS ? 2 : 1;  // loads of a row (ROWS) in a round
  constexpr int ROUND = LB == ROWS ? (IS_PACKED ? 128 : 64) : 32;  // summed elements of a wavefront's round
  constexpr int AHEAD = IS_PACKED ? 1 : 2;  // ROWS: rounds loaded before they are multiplied
  __shared__ f4v part[WAVES][N16][64];
  const int lane = threadIdx.x & 63, r16 = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tiles_n = (p.n + TN - 1) / TN;
  RowTile t;
  if (!find_row_tile<ALL_TILES>(p.offsets, p.groups, p.rows, 16, (int)(workgroup(p) / tiles_n), t)) return;
  const int n0 = (int)(workgroup(p) % tiles_n) * TN;
  const int rows = t.end - t.row < 16 ? t.end - t.row : 16, cols = p.n - n0 < TN ? p.n - n0 : TN;
  const int k_end = t.group < 0 ? 0 : p.k, group = t.group < 0 ? 0 : t.group;
  constexpr int BYTES = IS_PACKED ? 1 : 2;
  const auto ra = tile_rsrc((const char*)p.a + (uint64_t)t.row * p.as * BYTES,
                            ((uint64_t)(rows - 1) * p.as + p.k) * BYTES);
  const uint32_t oa = r16 < rows ? (uint32_t)(r16 * p.as * BYTES) + q * 16 : NOWHERE;  // this lane's row of A
  f4v acc[N16] = {};
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
      uint4 b[AHEAD][PIECES], a[AHEAD][PIECES];
      [[maybe_unused]] uint32_t xb[AHEAD], xa[AHEAD];
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        const int k = k0 + u * WAVES * ROUND;
#pragma unroll
        for (int h = 0; h < PIECES; ++h) {
          // past the rows' end: zeros
          const bool in = (k * BYTES + h * 64 + q * 16) < k_end * BYTES;
          b[u][h] = load(rb, in && ob != NOWHERE ? ob + k * BYTES + h * 64 : NOWHERE);
          a[u][h] = load(ra, in && oa != NOWHERE ? oa + k * BYTES + h * 64 : NOWHERE);
        }
        if constexpr (IS_PACKED) {
          const bool in = k < k_end;
          xb[u] = __builtin_amdgcn_raw_buffer_load_b8(rsb, in && r16 < cols ? r16 * (int)p.ss + k / 128 : (int)NOWHERE, 0, 0);
          xa[u] = __builtin_amdgcn_raw_buffer_load_b8(rsa, in && r16 < rows ? r16 * (int)p.ss + k / 128 : (int)NOWHERE, 0, 0);
        }
      }
      __builtin_amdgcn_sched_barrier(0);  // all of them in flight before the first is waited for
#pragma unroll
      for (int u = 0; u < AHEAD; ++u)
#pragma unroll
        for (int h = 0; h < PIECES; ++h) {
          if constexpr (IS_PACKED) {
            // 16 codes a lane: 8 for each of two instructions, of A as of B
            const uint4 x = a[u][h], y = b[u][h];
            const float sa = block8_scale(xa[u]), sb = block8_scale(xb[u]);
            acc[0] = mfma16<T>(decode_bf16(y.x, y.y, sb), decode_bf16(x.x, x.y, sa), acc[0]);
            acc[0] = mfma16<T>(decode_bf16(y.z, y.w, sb), decode_bf16(x.z, x.w, sa), acc[0]);
          } else {
            acc[0] = mfma16<T>(b[u][h], a[u][h], acc[0]);
          }
        }
    }
  } else {
    const auto rb = tile_rsrc((const char*)p.b + (group * p.bg + n0) * 2, ((uint64_t)(p.k - 1) * p.bs + cols) * 2);
    // 8 columns from 8 r16 on of rows 8 q to 8 q + 7
    const uint32_t ob = 8 * r16 < cols ? (uint32_t)(8 * q * p.bs * 2) + r16 * 16 : NOWHERE;
    for (int k0 = wave * ROUND; k0 < k_end; k0 += WAVES * ROUND) {
      uint4 b[8];
#pragma unroll
      for (int j = 0; j < 8; ++j)
        b[j] = load(rb, ob != NOWHERE && k0 + 8 * q + j < k_end ? ob + (uint32_t)((k0 + j) * p.bs * 2) : NOWHERE);
      const uint4 a = load(ra, oa != NOWHERE && k0 + 8 * q < k_end ? oa + k0 * 2 : NOWHERE);
      __builtin_amdgcn_sched_barrier(0);
      // column c of the eight rows, c even and odd: the low and the high halves of word c / 2
      const uint32_t* w = reinterpret_cast<const uint32_t*>(b);
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        uint32_t v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          v[j] = __builtin_amdgcn_perm(w[(2 * j + 1) * 4 + c / 2], w[2 * j * 4 + c / 2], c & 1 ? 0x07060302 : 0x05040100);
        acc[c] = mfma16<T>(make_uint4(v[0], v[1], v[2], v[3]), a, acc[c]);
      }
    }
  }
#pragma unroll
  for (int c = 0; c < N16; ++c) part[wave][c][lane] = acc[c];
  __syncthreads();
  O* out = (O*)p.c + (uint64_t)t.row * p.cs + n0;
  for (int c = wave; c < N16; c += WAVES) {
    f4v s = part[0][c][lane];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) s += part[w][c][lane];
    if (r16 >= rows) continue;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      // tile c holds columns 4 q to 4 q + 3 (COLS: every eighth column from c on)
      const int at = LB == ROWS ? 4 * q + e : 8 * (4 * q + e) + c;
      if (at < cols) out[(uint64_t)r16 * p.cs + at] = (O)s[e];
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

// Calls launch(workgroups) for a product's tiles, p.first being those before: a
// launch has less than 2^32 work-items along x. Each launch begins with a
// multiple of eight, so that the dies take tiles in turn.
template <class F>
void by_tiles(uint64_t tiles, Product& p, F launch) {
  if (tiles > PRODUCT_SIZE_MAX) config_error("rows", tiles, "gives more tiles than there are places for");
  by_launches(tiles, [&](uint64_t a, uint64_t m) {
    p.first = (unsigned)a;
    launch(dim3((unsigned)m));
    PXG_HIP(hipGetLastError());
  });
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

// The sums of divided groups: a grid of (such group, some rows of dw) by 1024
// columns adds the parts of each element in order.
constexpr int JOIN_ROWS = 512;  // workgroups to a group
template <class O>
__global__ void __launch_bounds__(256) join_parts(Product p) {
  const int each = p.m < JOIN_ROWS ? p.m : JOIN_ROWS;
  GroupPart g;
  if (!find_divided_group(p.offsets, p.groups, p.rows, p.limit, (int)blockIdx.x / each, g)) return;
  const int c = (blockIdx.y * 256 + threadIdx.x) * 4;
  if (c >= p.n) return;
  const uint64_t part = (uint64_t)p.m * p.n;
  for (int row = (int)blockIdx.x % each; row < p.m; row += each) {
    const float* from = p.workspace + g.slot * part + (uint64_t)row * p.n + c;
    O* to = (O*)p.c + g.group * p.cg + row * p.cs + c;
    if (p.n % 4 == 0) {
      f4v x = *reinterpret_cast<const f4v*>(from);
      for (int s = 1; s < g.parts; ++s) x += *reinterpret_cast<const f4v*>(from + s * part);
#pragma unroll
      for (int e = 0; e < 4; ++e) to[e] = (O)x[e];
    } else {
      for (int e = 0; e < 4 && c + e < p.n; ++e) {
        float x = from[e];
        for (int s = 1; s < g.parts; ++s) x += from[s * part + e];
        to[e] = (O)x;
      }
    }
  }
}

// The kernel asked for on this thread (0: the cheapest), and the last one launched.
thread_local int g_kernel = 0;
thread_local uint32_t g_last_kernel = 0;

template <class T, class O, int FORM, int LA, int LB, int WM, int WN, int MT, int NT>
void launch_tiled(Product p, hipStream_t s) {
  using K = Tiled<T, WM, WN, MT, NT>;
  const uint64_t tn = (p.n + K::TN - 1) / K::TN;
  uint64_t tiles;
  if (FORM == GRAD_WEIGHT)
    tiles = (((p.m + K::TM - 1) / K::TM * tn + 7) / 8) * 8 * group_parts_max(p.rows, p.groups, p.limit);
  else tiles = (row_tiles_max(p.rows, p.groups, K::TM, p.offsets != nullptr) * tn / 8 + 2) * 8;  // both kinds' eighths
  auto launch = [&](dim3 grid) {
    hipLaunchKernelGGL((product_tiled<T, O, FORM, LA, LB, WM, WN, MT, NT>), grid, dim3(K::THREADS), 0, s, p);
  };
  if (FORM == GRAD_WEIGHT) {
    if (tiles > PRODUCT_SIZE_MAX) config_error("n", tiles, "gives more tiles than a launch has workgroups");
    launch(dim3((unsigned)tiles));
    PXG_HIP(hipGetLastError());
  } else {
    by_tiles(tiles, p, launch);
  }
  g_last_kernel = K::TM | (K::FP8 ? PXG_KERNEL_8_BIT : 0) | (is_any(LA) ? PXG_KERNEL_UNALIGNED : 0) |
                  (p.limit ? PXG_KERNEL_PARTS : 0);
}

// Whether an operand can be copied: 16-byte pieces that all belong to one row.
bool copies(int bytes, const void* d, uint64_t cols, uint64_t stride, uint64_t group_stride) {
  return ((uint64_t)(uintptr_t)d | cols * bytes | stride * bytes | group_stride * bytes) % 16 == 0;
}

template <class T, class O, int LB, bool IS_PACKED>
void launch_few(Product p, hipStream_t s) {
  constexpr uint64_t TN = LB == ROWS ? 16 : 128;
  const uint64_t tiles = row_tiles_max(p.rows, p.groups, 16, p.offsets != nullptr) * ((p.n + TN - 1) / TN);
  by_tiles(tiles, p, [&](dim3 grid) {
    hipLaunchKernelGGL((product_few<T, O, LB, IS_PACKED>), grid, dim3(512), 0, s, p);
  });
  g_last_kernel = 16;
}

// Which tiles a product takes: the cheapest by what was measured, in us. A
// tile takes `fixed` and then `step` for 64 summed elements, `least` of it
// alone on its CU and `more` where the chip is full (256 x 256 tiles one on a
// CU, 128 x 128 two, 64 x 64 four). Groups end inside a tile. Measured with
// 256, 128 and 64:
//   16384 rows, 2048 -> 2048   forward 115, 150, 211; weight gradient 300, 188, 265
//   4096 rows, 768 -> 768               23,  14,  12;                  79,  50,  36
//   8192 rows in 8 uneven groups, 1024 -> 4096   weight gradient        63,  86, 123
// Packed rows: 256 are the 8-bit cores' tiles, for results of 16 bits only: what
// these cores cut off products (run8 above) is under a 16-bit result's rounding
// and far over an f32 one's. Decoded to bf16, which is exact, products are
// summed in f32.
// Measured on the 8-bit cores and decoded:
//   8 groups of 1024 rows, 2048 -> 2048    35, 107
//   32 groups of 128 rows, 2048 -> 2048    30,  57
//   8 groups of 24 rows, 2048 -> 2048      23,  26
//   333 rows, 1000 -> 1500                 26,  15
struct Tile {
  int size, slots;
  double fixed, least, more;
};
constexpr Tile TILES[3] = {{256, 256, 6, 1.15, 0.45}, {128, 512, 4, 0.7, 0.35}, {64, 1024, 3, 0.42, 0.3}};
constexpr Tile PACKED_TILES[3] = {{256, 256, 6, 0.6, 0.25}, {128, 512, 4, 0.95, 0.45}, {64, 1024, 3, 0.6, 0.4}};
// Joining the parts of divided groups: a launch, and their bytes twice.
constexpr double JOIN_US = 4, JOIN_BYTES_PER_US = 4e6;

struct Cost {
  double best = 1e30, fp8 = 1e30;
  int tile = 64, limit = 0;
};
// packed: the first of PACKED_TILES is the fp8 product's, not among the choice.
// Weight gradients: routers' groups are uneven, so the longest of g is taken as
// sqrt(g) averages; its tiles, or its parts', are the last to end. Between one part a
// group and many, in us at each one's best tile (a part's greatest length):
//   1 group of 16384 rows, 2048 x 2048            188 -> 122 (4096)
//   1 of 4096, 768 x 768                           36 ->  21 (1536)
//   8 uneven ones, 16384 rows in all, 512 x 512    39 ->  30 (1024)
//   8 uneven, 8192 rows, 4096 x 1024               63 ->  87 (2048): the parts' traffic
Cost product_cost(int form, const Product& p, bool packed, uint64_t room = 0, int tile_asked = 0) {
  Cost best;
  const double average = form == GRAD_WEIGHT ? (double)p.rows / p.groups : p.k;
  const double longest = form == GRAD_WEIGHT ? average * std::sqrt((double)p.groups) : p.k;
  for (int i = 0; i < 3; ++i) {
    const Tile& t = packed ? PACKED_TILES[i] : TILES[i];
    if (tile_asked && tile_asked != t.size) continue;
    const uint64_t tn = ((uint64_t)p.n + t.size - 1) / t.size;
    const uint64_t tiles = form == GRAD_WEIGHT ? (((uint64_t)p.m + t.size - 1) / t.size) * tn
                                               : (p.rows + (uint64_t)p.groups * t.size / 2 + t.size - 1) / t.size * tn;
    for (int parts = 1; parts <= 32; parts *= 2) {
      const uint64_t limit = parts == 1 ? 0 : ((uint64_t)(longest / parts) + 63) / 64 * 64;
      uint64_t all = tiles, bytes = 0;
      if (form == GRAD_WEIGHT) {
        const uint64_t slots = group_slots_max(p.rows, p.groups, limit);
        bytes = 4 * slots * p.m * p.n;
        if (parts > 1 && (limit < 128 || p.groups > SEGMENT_GROUPS || bytes > room)) break;
        all *= group_parts_max(p.rows, p.groups, limit);
      } else if (parts > 1) {
        break;
      }
      const double step = t.least + t.more * std::min(1.0, (double)all / t.slots);
      const double summed = form == GRAD_WEIGHT ? (double)tiles * p.rows / all : p.k;
      // one group's half tile of padding does not begin a round, up to 7680
      // columns; of more it does, and 128 x 128 tiles are taken where 256 x 256
      // would be faster (2048 rows, 4096 -> 8192: 150 us, 108)
      const double rounds = std::ceil((double)all / t.slots - (p.groups == 1 ? 0.12 : 0.0));
      double us = std::max(1.0, rounds) * (t.fixed + std::ceil(summed / 64) * step);
      us = std::max(us, t.fixed + (limit ? (double)limit : longest) / 64 * step);
      if (limit) us += JOIN_US + 2.0 * bytes / JOIN_BYTES_PER_US;
      if (packed && i == 0) {
        best.fp8 = us;
      } else if (us < best.best) {
        best.best = us;
        best.tile = t.size;
        best.limit = (int)limit;
      }
    }
  }
  // A much longer group than assumed: where it alone would take half as long
  // again as all tiles together, and dividing it saves more than its parts'
  // traffic costs. Packed, into f32, whole and divided, with the longest of 8
  // groups of 8192 rows, 1024 -> 4096: 5500 rows 155, 99; 4200 rows 127, 103;
  // none divided 92, 94. Of 16 of 16384, 2048 -> 2048: 7799 rows 269, 206 us.
  if (form == GRAD_WEIGHT && !best.limit && p.groups > 1 && p.groups <= SEGMENT_GROUPS) {
    const Tile& t = TILES[best.tile == 256 ? 0 : best.tile == 128 ? 1 : 2];
    const uint64_t tiles = (((uint64_t)p.m + t.size - 1) / t.size) * (((uint64_t)p.n + t.size - 1) / t.size);
    const uint64_t limit = (p.rows * tiles * 3 / 2 / t.slots + 63) / 64 * 64, slot = 4ull * p.m * p.n;
    const double saved = limit / 128.0 * (t.least + t.more), join = JOIN_US + 4.0 * slot / JOIN_BYTES_PER_US;
    if (limit < (uint64_t)p.rows && saved > join && group_slots_max(p.rows, p.groups, limit) * slot <= room)
      best.limit = (int)limit;
  }
  return best;
}

// What product_few takes, in us: a start, and its row tiles' matrices at the
// rate that it reads them, which falls with the rows beside them. COLS reads
// them again out of the caches, and k rows one after another. Tiles are bound
// by their own cost or by the matrices' bytes. Few and tiled, measured:
//   16 rows, 4096 -> 4096              forward 11, 35; input gradient 18, 36; packed 9, 41
//   64 rows, the same                          33, 35;                18, 36;        25, 43
//   16 groups of 1 row, 2048 -> 2048           29, 23;                22, 23;        17, 32
//   8 groups of 64 rows, 1024 -> 1024          19,  9;                10,  9;        14, 14
double few_cost(int b, bool packed, const Product& p) {
  const double used = std::min(p.rows, p.groups);
  const double tiles = p.groups == 1 ? (p.rows + 15) / 16 : std::max(used, p.rows / 16.0 + p.groups / 2.0);
  const double matrix = (double)p.n * p.k * (packed ? 1 : 2), full = p.rows / (16 * tiles);
  if (b == COLS) return 2 + std::max(matrix * (used * (1 + full / 7) / 6e6 + (tiles - used) / 12e6), p.k * 0.0033);
  return 2 + matrix * tiles * (packed ? (1 + full / 2) / 4.5e6 : (1 + full / 3) / 5e6);
}
double tiled_cost(double cost, bool packed, const Product& p) {
  return std::max(cost, (double)std::min(p.rows, p.groups) * p.n * p.k * (packed ? 1 : 2) / 5.9e6);
}

// The tile asked for on this thread, 0 if any; packed rows into f32 have no 256.
int asked_tile(bool packed_into_f32) {
  return g_kernel == 16 || (packed_into_f32 && g_kernel == 256) ? 0 : g_kernel;
}

// `room`: bytes of p.workspace.
template <int FORM, class T, class O, bool IS_PACKED>
void launch_product(Product p, uint64_t room, hipStream_t s) {
  p.c_vec = ((uint64_t)(uintptr_t)p.c | p.cs * sizeof(O) | p.cg * sizeof(O)) % 16 == 0;
  constexpr int LA = FORM == GRAD_WEIGHT ? COLS : FORM == FORWARD && IS_PACKED ? PACKED_ROWS : ROWS;
  constexpr int LB = FORM == GRAD_INPUT ? COLS : FORM == GRAD_WEIGHT ? (IS_PACKED ? PACKED_COLS : COLS) : LA;
  const uint64_t acols = FORM == GRAD_WEIGHT ? p.m : p.k, bcols = FORM == FORWARD ? p.k : p.n;
  const bool copied = (is_packed(LA) || copies(2, p.a, acols, p.as, 0)) &&
                      (is_packed(LB) || copies(2, p.b, bcols, p.bs, p.bg));
  constexpr bool PACKED_FORWARD = FORM == FORWARD && IS_PACKED;
  const Cost cost = product_cost(FORM, p, PACKED_FORWARD, room, asked_tile(PACKED_FORWARD && std::is_same_v<O, float>));
  if constexpr (FORM != GRAD_WEIGHT) {
    constexpr int B = FORM == GRAD_INPUT ? COLS : ROWS;
    // COLS spans a matrix' rows with one resource
    const bool reaches = B == ROWS || p.k * p.bs * 2 <= 0x7FFFFFFF;
    const double tiled = std::is_same_v<O, float> ? cost.best : std::min(cost.best, cost.fp8);
    const bool few = g_kernel ? g_kernel == 16 : few_cost(B, IS_PACKED, p) <= tiled_cost(tiled, IS_PACKED, p);
    if (copied && reaches && few) return launch_few<T, O, B, IS_PACKED>(p, s);
  }
  if constexpr (FORM == GRAD_WEIGHT) p.limit = cost.limit;
  if constexpr (FORM == FORWARD && IS_PACKED && !std::is_same_v<O, float>)
    if (cost.fp8 <= cost.best) return launch_tiled<Fp8, O, FORM, ROWS, ROWS, 2, 4, 8, 4>(p, s);
  if (copied) {
    if (LA != PACKED_ROWS && cost.tile == 256) {
      if constexpr (LA != PACKED_ROWS) launch_tiled<T, O, FORM, LA, LB, 2, 4, 8, 4>(p, s);
    } else if (cost.tile >= 128) {
      launch_tiled<T, O, FORM, LA, LB, 2, 2, 4, 4>(p, s);
    } else {
      launch_tiled<T, O, FORM, LA, LB, 2, 2, 2, 2>(p, s);
    }
  } else if constexpr (!is_packed(LA)) {
    constexpr int AA = FORM == GRAD_WEIGHT ? ANY_COLS : ANY_ROWS;
    constexpr int AB = is_packed(LB) ? LB : FORM == FORWARD ? ANY_ROWS : ANY_COLS;
    if (cost.tile >= 128) launch_tiled<T, O, FORM, AA, AB, 2, 2, 4, 4>(p, s);
    else launch_tiled<T, O, FORM, AA, AB, 2, 2, 2, 2>(p, s);
  }
  if (FORM == GRAD_WEIGHT && p.limit) {
    const uint64_t divided = std::min<uint64_t>(p.groups, p.rows / p.limit);
    if (divided) {
      const dim3 grid((unsigned)(divided * std::min(p.m, JOIN_ROWS)), (unsigned)(((uint64_t)p.n + 1023) / 1024));
      hipLaunchKernelGGL(join_parts<O>, grid, dim3(256), 0, s, p);
      PXG_HIP(hipGetLastError());
    }
  }
}

template <int FORM>
void run_product(int type, int out_type, const Product& p, hipStream_t s, uint64_t room = 0) {
  by_types(type, out_type, [&](auto t, auto o) {
    using T = decltype(t);
    using O = decltype(o);
    if constexpr (FORM == GRAD_WEIGHT && std::is_same_v<T, __bf16>) {
      if (p.b_scales) return launch_product<FORM, T, O, true>(p, room, s);
    }
    launch_product<FORM, T, O, false>(p, room, s);
  });
}

}  // namespace
}  // namespace pxg

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
