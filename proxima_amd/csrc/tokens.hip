// A whole expert layer for a few tokens:
//
//   y_t = r_t + sum over picks j of g_tj (W2_e f(W1_e x_t + b1_e) [* W3_e x_t] + b2_e),   e = experts_tj
//
// For a few tokens the time is that of reading the matrices of the experts in
// use, once, so nothing else may wait for memory. Two kernels, or three:
//
//   tokens_hidden  a workgroup takes an expert in use and 16 rows of its W1 (and
//                  W3), finds the expert's tokens from the ids, and leaves
//                  a = g f(h) [* up] of them in the workspace;
//   tokens_out     a workgroup takes 16 rows of every W2. A token's row of the
//                  matrix instruction is the same for all experts (zeros where it
//                  did not pick one), so that the sum over experts and hidden
//                  columns is one sum in registers, the wavefronts' shares joined
//                  at the end. Where such workgroups do not fill the chip it takes
//                  8 rows (up to 8 tokens; the instruction's other half is another
//                  piece of the sum), or a slice of the sum;
//   tokens_join    adds the slices, where there are any. tokens_plan chooses.
//
// Tokens go in blocks of 64 (a bit mask of them is one scalar register pair).
// Sums are held in f32. a is kept as planes of bf16 whose sum it is: three (all
// of f32's 24 bits) for f32 results, two for 16-bit ones. There the second keeps 8
// bits of what is below the first's last, so that up to 2^-16 of a is lost, beside a
// rounding of the result of 2^-8 (bf16) or 2^-11 (f16); a third would cost 4 to 14%
// (us with two, and of the same into f32: 8 x 2 of 16 gated experts, 2048 -> 4096 ->
// 2048 89, 94; 32 x 4 of 64 packed ones, 2048 -> 1024 -> 2048 56, 64; 64 x 8 of 64,
// 1024 -> 512 -> 1024 56, 61). Matrices in f16 are taken apart into two bf16 for the
// second product, which is exact but for 2^-40 (rest() says why), so that a's range
// is f32's.
#include "activation.hpp"
#include "block8.hpp"
#include "common.hpp"
#include "device.hpp"
#include "groups.hpp"
#include "matrix_cores.hpp"
#include "products.hpp"
#include "rows.hpp"

namespace pxg {
namespace {

constexpr int BLOCK_TOKENS = 64, PICKS_MAX = 16;
[[maybe_unused]] constexpr int ENTRIES_MAX = BLOCK_TOKENS * PICKS_MAX;  // experts in use of a block
constexpr uint64_t EXPERTS_MAX = 1u << 16, TOKENS_MAX = 1u << 16;
constexpr uint64_t SLICE_BYTES = 32 << 10;
constexpr int TOKENS_WAVES = 8, TOKENS_THREADS = 64 * TOKENS_WAVES;

struct ExpertMatrix {  // of every expert; strides in elements (packed: bytes of codes)
  const void* p;
  uint64_t stride, group;
  const uint8_t* scales;  // packed: rows `scale_stride` apart
  uint64_t scale_stride;
};

// An expert in use: its tokens of a block, and how many pairs of the block have a lower id.
struct Entry {
  int expert, offset;
  uint64_t tokens;
};

struct TokenLayer {
  const void* x;
  uint64_t xs;
  const int64_t* ids;
  const float* gates;
  uint64_t is, gs;
  ExpertMatrix w1, up, w2;
  const void *bias1, *bias2;
  uint64_t b1s, b2s;
  const void* residual;
  void* y;
  uint64_t rs, ys;
  char* planes;      // row (pair of a block) by plane by column
  Entry* entries;    // entries_max + 1 of a block, the first's expert their number
  float* partial;    // tokens_out's sums by slice, row and column
  int rows, k, hidden, wide, n, picks, experts, entries_max, slices;
  unsigned first = 0;  // tokens_out's workgroups (along x) of the launches before this one
  int activation;
  bool bias_f32;
};

#if defined(__HIP_DEVICE_COMPILE__)
// 16 rows of a matrix, 64 bytes of summed elements (ROUND of them a wavefront)
// at a time: what a lane reads, and the fragments it makes of it.
template <class T, bool PACKED, bool ANY>
struct MatrixTile {
  static constexpr int ROUND = PACKED ? 128 : 64;
  struct Round {
    Piece<ANY && !PACKED> w[2];
    uint32_t scale;
  };
  __amdgpu_buffer_rsrc_t rs, scales;
  uint32_t at, scale_at;  // this lane's row
  bool in;

  // TILE rows from row0 on; with fewer than 16 of them lanes share rows, and take other columns by load's k
  template <int TILE>
  __device__ __forceinline__ void set(const ExpertMatrix& m, int expert, int height, int row0, int rows, int cols,
                                      int lane) {
    const int row = (lane & 15) % TILE, q = lane >> 4;
    uint32_t odd = 0;
    constexpr int BYTES = PACKED ? 1 : 2;
    const char* p = (const char*)m.p + (expert * m.group + row0 * m.stride) * BYTES;
    rs = rows_rsrc<ANY && !PACKED>(p, ((uint64_t)(rows - 1) * m.stride + cols) * BYTES, odd);
    in = row < rows;
    at = odd + (uint32_t)(row * m.stride * BYTES) + q * 16;
    if constexpr (PACKED) {
      scales = tile_rsrc(m.scales + ((uint64_t)expert * height + row0) * m.scale_stride, rows * m.scale_stride);
      scale_at = row * (uint32_t)m.scale_stride;
    }
  }
  // `cols` is the matrix' width: packed, a multiple of 128
  __device__ __forceinline__ Round load(int k, int cols, int q) const {
    Round r;
    constexpr int BYTES = PACKED ? 1 : 2, EACH = PACKED ? 16 : 8;
#pragma unroll
    for (int h = 0; h < 2; ++h)
      r.w[h] = load_piece<ANY && !PACKED>(rs, at + k * BYTES + h * 64, in && k + h * 4 * EACH + q * EACH < cols);
    if constexpr (PACKED)
      r.scale = __builtin_amdgcn_raw_buffer_load_b8(scales, (int)(in && k < cols ? scale_at + k / 128 : NOWHERE), 0, 0);
    return r;
  }
  // fragment f (of 2, packed 4): 8 summed elements of this lane's row, from element column(f, q) of the round on
  static constexpr int FRAGMENTS = PACKED ? 4 : 2;
  __device__ static __forceinline__ int column(int f, int q) { return PACKED ? (f >> 1) * 64 + q * 16 + (f & 1) * 8 : f * 32 + q * 8; }
  __device__ __forceinline__ uint4 fragment(const Round& r, int f, int k, int cols, int q) const {
    if constexpr (PACKED) {
      const uint4 c = r.w[f >> 1].v;
      return f & 1 ? decode_bf16(c.z, c.w, block8_scale(r.scale)) : decode_bf16(c.x, c.y, block8_scale(r.scale));
    } else {
      return elements(r.w[f], at, cols - k - column(f, q));
    }
  }
};

// v cut after bf16's bits, toward zero, so that v - cut(v) is exact.
__device__ __forceinline__ float cut(float v) { return __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, v) & 0xFFFF0000u); }
__device__ __forceinline__ uint32_t high_half(float v) { return __builtin_bit_cast(uint32_t, v) >> 16; }
// What is left of v; of what 16 bits hold exactly 2^-40 of it rather than nothing, as zero times an infinity of the other
// factor is not a number. (From |v| = 2^-86 on, where there are three planes 2^-46: below, that is less than bf16's
// smallest normal value. f16 matrices, 8 x 2 of 16 gated experts: 84.9 us, 84.3 without.)
__device__ __forceinline__ float rest(float v, float c) {
  return fabsf(v) < __builtin_inff() ? __builtin_fmaf(c, 0x1p-40f, v - c) : v;
}
#endif

// D: one matrix, or two (gated). RT: row tiles of 16 tokens that a block may need.
template <class T, bool PACKED, bool ANY, int D, int RT, int PLANES>
__global__ void __launch_bounds__(TOKENS_THREADS, 4) tokens_hidden(TokenLayer p) {
#if defined(__HIP_DEVICE_COMPILE__)
  using M = MatrixTile<T, PACKED, ANY>;
  constexpr int AHEAD = RT == 1 ? 2 : 1;  // rounds loaded before they are multiplied
  constexpr bool EARLY = !PACKED || RT < 4;  // so are x's, where they fit the registers
  __shared__ uint32_t used[EXPERTS_MAX / 32];
  __shared__ int ids[ENTRIES_MAX];
  __shared__ f4v part[TOKENS_WAVES][D * RT][64];
  const int lane = threadIdx.x & 63, r16 = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // along x the tiles of a matrix, then the experts in use, then the blocks of tokens
  const int n0 = (int)blockIdx.x * 16, nth = (int)blockIdx.y;
  const int t0 = blockIdx.z * BLOCK_TOKENS, tokens = p.rows - t0 < BLOCK_TOKENS ? p.rows - t0 : BLOCK_TOKENS;
  Entry* entries = p.entries + (uint64_t)blockIdx.z * (p.entries_max + 1);

  // the nth expert in use
  const int words = (p.experts + 31) / 32;
  for (int i = threadIdx.x; i < words; i += TOKENS_THREADS) used[i] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < tokens * p.picks; i += TOKENS_THREADS) {
    const int64_t id = p.ids[(uint64_t)(t0 + i / p.picks) * p.is + i % p.picks];
    const bool is = (uint64_t)id < (uint64_t)p.experts;
    if (is) atomicOr(&used[id >> 5], 1u << (id & 31));
    ids[i] = is ? (int)id : 1 << 30;
  }
  __syncthreads();
  const int per = (words + 63) / 64;
  int have = 0;
  for (int i = 0; i < per; ++i) have += lane * per + i < words ? __popc(used[lane * per + i]) : 0;
  const int upto = wave_sum_scan(have, lane);
  const int all = __builtin_amdgcn_readlane(upto, 63);
  if (nth == 0 && n0 == 0 && threadIdx.x == 0) entries[0].expert = all;
  if (nth >= all) return;
  const int owner = __builtin_ctzll(__ballot(upto > nth));
  int left = nth - (__builtin_amdgcn_readlane(upto, owner) - __builtin_amdgcn_readlane(have, owner)), word = owner * per;
  uint32_t bits = __builtin_amdgcn_readfirstlane(used[word]);
  while (left >= __popc(bits)) {
    left -= __popc(bits);
    bits = __builtin_amdgcn_readfirstlane(used[++word]);
  }
  for (; left; --left) bits &= bits - 1;
  const int expert = word * 32 + __builtin_ctz(bits);

  const int cols = p.hidden - n0 < 16 ? p.hidden - n0 : 16;
  const int k_wide = PACKED ? (int)p.w1.stride : p.k;
  M w[D];
  w[0].template set<16>(p.w1, expert, p.hidden, n0, cols, k_wide, lane);
  if constexpr (D == 2) w[1].template set<16>(p.up, expert, p.hidden, n0, cols, k_wide, lane);
  // its tokens, a lane each, and their gates; then lane r has the r-th of them
  bool mine = false;
  float gate = 0.0f;
  int lower = 0;
  if (lane < tokens)
    for (int j = 0; j < p.picks; ++j) {
      const int id = ids[lane * p.picks + j];
      lower += id < expert;
      if (id == expert) {
        mine = true;
        gate += p.gates[(uint64_t)(t0 + lane) * p.gs + j];
      }
    }
  const uint64_t mask = __ballot(mine);
  const int count = __popcll(mask);
  const int offset = __builtin_amdgcn_readlane(wave_sum_scan(lower, lane), 63);
  const int rank = __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
  // the others push to lanes past the last token's (there are as many of both)
  const int to = mine ? rank : count + lane - rank;
  const int token = __builtin_amdgcn_ds_permute(to * 4, lane);
  gate = __builtin_bit_cast(float, __builtin_amdgcn_ds_permute(to * 4, __builtin_bit_cast(int, gate)));
  if (n0 == 0 && threadIdx.x == 0) entries[nth + 1] = {expert, offset, mask};

  uint32_t odd;
  const auto rx = rows_rsrc<ANY>((const char*)p.x + (uint64_t)t0 * p.xs * 2,
                                 ((uint64_t)(tokens - 1) * p.xs + p.k) * 2, odd);
  uint32_t xat[RT];
  bool xin[RT];
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    xin[i] = i * 16 + r16 < count;
    xat[i] = odd + (uint32_t)(__shfl(token, i * 16 + r16) * p.xs * 2);
  }
  f4v acc[D][RT] = {};
  for (int k0 = wave * M::ROUND; k0 < k_wide; k0 += TOKENS_WAVES * M::ROUND * AHEAD) {
    typename M::Round b[AHEAD][D];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u)
#pragma unroll
      for (int d = 0; d < D; ++d) b[u][d] = w[d].load(k0 + u * TOKENS_WAVES * M::ROUND, k_wide, q);
    Piece<ANY> a[AHEAD][RT][M::FRAGMENTS];
    auto load_x = [&](int u, int i, int f) {
      const int at = k0 + u * TOKENS_WAVES * M::ROUND + M::column(f, q);
      a[u][i][f] = load_piece<ANY>(rx, xat[i] + at * 2, xin[i] && at < p.k);
    };
    if constexpr (EARLY) {
#pragma unroll
      for (int u = 0; u < AHEAD; ++u)
#pragma unroll
        for (int i = 0; i < RT; ++i)
          if (i == 0 || i * 16 < count)
#pragma unroll
            for (int f = 0; f < M::FRAGMENTS; ++f) load_x(u, i, f);
      __builtin_amdgcn_sched_barrier(0);  // all of them in flight before the first is waited for
    }
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int k = k0 + u * TOKENS_WAVES * M::ROUND;
#pragma unroll
      for (int f = 0; f < M::FRAGMENTS; ++f) {
        uint4 wf[D];
#pragma unroll
        for (int d = 0; d < D; ++d) wf[d] = w[d].fragment(b[u][d], f, k, k_wide, q);
#pragma unroll
        for (int i = 0; i < RT; ++i)
          if (i == 0 || i * 16 < count) {
            if constexpr (!EARLY) load_x(u, i, f);
            const uint4 xf = elements(a[u][i][f], xat[i], p.k - k - M::column(f, q));
#pragma unroll
            for (int d = 0; d < D; ++d) acc[d][i] = mfma16<T>(wf[d], xf, acc[d][i]);
          }
      }
    }
  }
#pragma unroll
  for (int d = 0; d < D; ++d)
#pragma unroll
    for (int i = 0; i < RT; ++i) part[wave][i * D + d][lane] = acc[d][i];
  __syncthreads();
  const int i = wave;  // a wavefront ends a row tile
  if (i >= RT || i * 16 >= count) return;
  f4v h[D];
#pragma unroll
  for (int d = 0; d < D; ++d) {
    h[d] = part[0][i * D + d][lane];
#pragma unroll
    for (int o = 1; o < TOKENS_WAVES; ++o) h[d] += part[o][i * D + d][lane];
  }
  // a lane has columns 4 q to 4 q + 3 of the (16 i + r16)-th token
  const float g = __shfl(gate, i * 16 + r16);
  if (i * 16 + r16 >= count) return;
  float v[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int at = n0 + 4 * q + e;
    v[e] = h[0][e];
    if (p.bias1 && at < p.hidden)
      v[e] += p.bias_f32 ? ((const float*)p.bias1)[expert * p.b1s + at] : (float)((const T*)p.bias1)[expert * p.b1s + at];
  }
  activate<std::conditional_t<PLANES == 3, float, T>>(v, p.activation);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if constexpr (D == 2) v[e] *= h[1][e];
    v[e] = 4 * q + e < cols ? v[e] * g : 0.0f;
  }
  const uint64_t row = (uint64_t)t0 * p.picks + offset + i * 16 + r16;
  char* to_row = p.planes + row * PLANES * p.wide * 2;
#pragma unroll
  for (int plane = 0; plane < PLANES; ++plane) {
    uint32_t bits16[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (plane == PLANES - 1) {
        bits16[e] = __builtin_bit_cast(uint16_t, (__bf16)v[e]);
      } else {
        const float c = cut(v[e]);
        bits16[e] = high_half(c);
        v[e] = rest(v[e], c);
      }
    }
    char* to_plane = to_row + (uint64_t)plane * p.wide * 2;
    *reinterpret_cast<uint2*>(to_plane + (n0 + 4 * q) * 2) =
        make_uint2(bits16[0] | bits16[1] << 16, bits16[2] | bits16[3] << 16);
    if (n0 + 16 >= p.hidden)  // the columns past the last are multiplied by zeros
      for (int at = n0 + 16 + 4 * q; at < p.wide; at += 16) *reinterpret_cast<uint2*>(to_plane + at * 2) = make_uint2(0, 0);
  }
#endif
}

// y from the sum over experts: b2 by the token's picks, and the residual.
template <class T, class O>
__device__ __forceinline__ void finish(const TokenLayer& p, int token, int col, float v) {
  if (p.bias2)
    for (int j = 0; j < p.picks; ++j) {
      const int64_t id = p.ids[(uint64_t)token * p.is + j];
      if ((uint64_t)id < (uint64_t)p.experts) {
        const uint64_t at = id * p.b2s + col;
        v += p.gates[(uint64_t)token * p.gs + j] * (p.bias_f32 ? ((const float*)p.bias2)[at] : (float)((const T*)p.bias2)[at]);
      }
    }
  if (p.residual) v += (float)((const O*)p.residual)[(uint64_t)token * p.rs + col];
  ((O*)p.y)[(uint64_t)token * p.ys + col] = rounded<O>(v);
}

// PARTS (1 or 2): the matrix instruction's 16 rows are 16 / PARTS of a matrix by PARTS neighbouring pieces of the sum,
// its 16 columns as many tokens by the same pieces; of the products, those of a piece with itself count. RT: row tiles
// of 16 / PARTS tokens.
template <class T, bool PACKED, bool ANY, int RT, class O, int PARTS, int WAVES>
__global__ void __launch_bounds__(64 * WAVES, 4) tokens_out(TokenLayer p) {
#if defined(__HIP_DEVICE_COMPILE__)
  using M = MatrixTile<T, PACKED, ANY>;
  constexpr int PLANES = std::is_same_v<O, float> ? 3 : 2;
  constexpr int AHEAD = RT > 1 || ANY ? 2 : PACKED ? 4 - PLANES : PLANES == 3 ? 2 : std::is_same_v<T, __bf16> ? 4 : 3;  // chunks loaded before they are multiplied
  constexpr int TILE = 16 / PARTS, THREADS = 64 * WAVES;
  __shared__ Entry entries[ENTRIES_MAX];
  __shared__ f4v part[WAVES][RT][64];
  const int lane = threadIdx.x & 63, r16 = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tiles = (p.n + TILE - 1) / TILE, place = (int)(p.first + blockIdx.x);
  const int n0 = place % tiles * TILE, slice = place / tiles;
  const int t0 = blockIdx.y * BLOCK_TOKENS, tokens = p.rows - t0 < BLOCK_TOKENS ? p.rows - t0 : BLOCK_TOKENS;
  const Entry* from = p.entries + (uint64_t)blockIdx.y * (p.entries_max + 1);
  const int all = __builtin_amdgcn_readfirstlane(from[0].expert);
  for (int i = threadIdx.x; i < all; i += THREADS) entries[i] = from[i + 1];
  __syncthreads();

  const int cols = p.n - n0 < TILE ? p.n - n0 : TILE, wide = PACKED ? p.wide : p.hidden;
  const int chunks = (wide + PARTS * M::ROUND - 1) / (PARTS * M::ROUND);  // of an expert's hidden columns
  const int mine_of = r16 % TILE, piece = r16 / TILE * M::ROUND;  // this lane's token of a row tile, and its columns
  const int64_t total = (int64_t)all * chunks;
  const int begin = (int)(total * slice / p.slices), end = (int)(total * (slice + 1) / p.slices);
  uint64_t below[RT];  // tokens before this lane's of row tile i
#pragma unroll
  for (int i = 0; i < RT; ++i) below[i] = (1ull << (i * TILE + mine_of)) - 1;
  f4v acc[RT] = {};
  // a row tile's fragments of a: zeros in the rows of tokens that did not pick the expert
  auto load_a = [&](const Entry& e, int i, int k, uint4 (&a)[PLANES][M::FRAGMENTS]) {
    const uint64_t row_bytes = (uint64_t)PLANES * p.wide * 2;
    const auto ra = tile_rsrc(p.planes + ((uint64_t)t0 * p.picks + e.offset) * row_bytes, __popcll(e.tokens) * row_bytes);
    const bool in = e.tokens >> (i * TILE + mine_of) & 1;
    const uint32_t at = __popcll(e.tokens & below[i]) * (uint32_t)row_bytes;
#pragma unroll
    for (int plane = 0; plane < PLANES; ++plane)
#pragma unroll
      for (int f = 0; f < M::FRAGMENTS; ++f) {
        const int c = k + M::column(f, q);
        a[plane][f] = load_piece<false>(ra, at + (uint32_t)plane * p.wide * 2 + c * 2, in && c < p.wide).v;
      }
  };
  auto multiply = [&](uint4 w, const uint4 (&a)[PLANES][M::FRAGMENTS], int f, f4v& c) {
    if constexpr (std::is_same_v<T, _Float16>) {
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        typedef _Float16 h2v __attribute__((ext_vector_type(2)));
        const h2v h = __builtin_bit_cast(h2v, e == 0 ? w.x : e == 1 ? w.y : e == 2 ? w.z : w.w);
        const float x = (float)h[0], y = (float)h[1], cx = cut(x), cy = cut(y);
        hi[e] = high_half(cx) | (__builtin_bit_cast(uint32_t, cy) & 0xFFFF0000u);
        lo[e] = high_half(rest(x, cx)) | (__builtin_bit_cast(uint32_t, rest(y, cy)) & 0xFFFF0000u);
      }
      const uint4 wh = make_uint4(hi[0], hi[1], hi[2], hi[3]), wl = make_uint4(lo[0], lo[1], lo[2], lo[3]);
#pragma unroll
      for (int plane = PLANES - 1; plane >= 0; --plane) {
        c = mfma16<__bf16>(wl, a[plane][f], c);
        c = mfma16<__bf16>(wh, a[plane][f], c);
      }
    } else {
#pragma unroll
      for (int plane = PLANES - 1; plane >= 0; --plane) c = mfma16<__bf16>(w, a[plane][f], c);
    }
  };
  auto entry_at = [&](int i) {
    Entry e = entries[i];
    e.expert = __builtin_amdgcn_readfirstlane(e.expert);
    e.offset = __builtin_amdgcn_readfirstlane(e.offset);
    e.tokens = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)e.tokens) |
               (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(e.tokens >> 32)) << 32;
    return e;
  };
  // chunk `c`: of the nth expert, from column `chunk` rounds on
  int c = begin + wave, nth = c / chunks, chunk = c % chunks;
  auto next = [&] {
    c += WAVES;
    chunk += WAVES;
    while (chunk >= chunks) {
      chunk -= chunks;
      ++nth;
    }
  };
  while (c < end) {
    M w[AHEAD];
    typename M::Round b[AHEAD];
    uint4 a[AHEAD][PLANES][M::FRAGMENTS];
    Entry e[AHEAD];
    int k[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      e[u] = entry_at(c < end ? nth : 0);
      if (c >= end) e[u].tokens = 0;
      k[u] = (c < end ? chunk * (PARTS * M::ROUND) : wide) + piece;  // past the end: zeros
      w[u].template set<TILE>(p.w2, e[u].expert, p.n, n0, cols, wide, lane);
      b[u] = w[u].load(k[u], wide, q);
      if constexpr (RT == 1) load_a(e[u], 0, k[u], a[u]);
      next();
    }
    if constexpr (RT == 1) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      uint4 wf[M::FRAGMENTS];
#pragma unroll
      for (int f = 0; f < M::FRAGMENTS; ++f) wf[f] = w[u].fragment(b[u], f, k[u], wide, q);
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        if (RT > 1 && !(e[u].tokens >> (i * TILE) & ((1 << TILE) - 1))) continue;
        if constexpr (RT > 1) load_a(e[u], i, k[u], a[u]);
        f4v sum = {};
#pragma unroll
        for (int f = 0; f < M::FRAGMENTS; ++f) multiply(wf[f], a[u], f, sum);
        // zeros times an infinity of another token's expert stay out
        if (e[u].tokens >> (i * TILE + mine_of) & 1) acc[i] += sum;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < RT; ++i) part[wave][i][lane] = acc[i];
  __syncthreads();
  const int i = wave, t = i * TILE + r16;  // a wavefront ends a row tile
  if (i >= RT || r16 >= TILE || q >= 4 / PARTS || t >= tokens) return;
  f4v s = {};
#pragma unroll 4
  for (int o = 0; o < WAVES; ++o)
#pragma unroll
    for (int h = 0; h < PARTS; ++h) s += part[o][i][lane + h * (64 / PARTS + TILE)];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (4 * q + e >= cols) break;
    if (p.slices == 1) finish<T, O>(p, t0 + t, n0 + 4 * q + e, s[e]);
    else p.partial[((uint64_t)slice * p.rows + t0 + t) * p.n + n0 + 4 * q + e] = s[e];
  }
#endif
}

// The slices' sums, in order. (The last of them to end could add them up instead
// of a kernel, but its fences empty the L2s: 8 tokens x 2 of 16 experts 209 us, 84 with this.)
template <class T, class O>
__global__ void __launch_bounds__(256) tokens_join(TokenLayer p) {
  const uint64_t all = (uint64_t)p.rows * p.n;
  for (uint64_t i = blockIdx.x * 256ull + threadIdx.x; i < all; i += gridDim.x * 256ull) {
    float v = 0.0f;
#pragma unroll 4
    for (int s = 0; s < p.slices; ++s) v += p.partial[s * all + i];
    finish<T, O>(p, (int)(i / p.n), (int)(i % p.n), v);
  }
}

// --- host ------------------------------------------------------------------------------
struct TokensPlan {
  uint64_t blocks, entries_max, wide, planes_bytes, entries_bytes, partial_bytes;
  int slices, parts, waves;
};
uint64_t pieces_of(uint64_t bytes) { return (bytes + 255) / 256 * 256; }

TokensPlan tokens_plan(uint64_t rows, uint64_t picks, uint64_t experts, uint64_t hidden, uint64_t n, bool f32_out,
                       bool packed) {
  TokensPlan t;
  t.blocks = (rows + BLOCK_TOKENS - 1) / BLOCK_TOKENS;
  const uint64_t pairs = std::min<uint64_t>(rows, BLOCK_TOKENS) * picks;
  t.entries_max = std::min(experts, pairs);
  t.wide = (hidden + 127) / 128 * 128;
  t.planes_bytes = pieces_of(rows * picks * (f32_out ? 3 : 2) * t.wide * 2);
  t.entries_bytes = pieces_of(t.blocks * (t.entries_max + 1) * sizeof(Entry));
  // The second kernel wants 256 workgroups, one with 16 wavefronts on each CU. Where 16
  // rows of a matrix each make fewer, 8 do it for up to 8 tokens (8 x 2 of 16 gated
  // experts, 2048 -> 4096 -> 2048: 38 us, 34 and 5 with slices and two kernels; 32 x 4 of
  // 64 packed ones, 2048 -> 1024 -> 2048: 38, for 26 and 5). Else the sum is cut into
  // slices that a third kernel joins: as many as fill the chip, of at least 32 KB
  // each, two chunks for each wavefront of a workgroup (of at least 96 KB: 18 tokens,
  // 512 -> 3904 -> 387, 3 gated experts 33 us for 25; 53 tokens, 2672 -> 1193 -> 1344, 2
  // experts 40 for 33).
  const uint64_t tiles = (n + 15) / 16 * t.blocks, bytes = t.entries_max * 16 * hidden * (packed ? 1 : 2);
  t.parts = tiles < 256 && tiles >= 128 && rows <= 8 ? 2 : 1;
  t.waves = tiles * t.parts >= 256 ? 16 : TOKENS_WAVES;
  t.slices = t.waves == 16 ? 1 : (int)std::max<uint64_t>(1, std::min({(uint64_t)512 / tiles, bytes / SLICE_BYTES, (uint64_t)32}));
  t.partial_bytes = t.slices > 1 ? pieces_of(4 * t.slices * rows * n) : 0;
  return t;
}

template <class T, bool PACKED, class O>
void run_tokens(TokenLayer p, const TokensPlan& t, hipStream_t s) {
  constexpr int PLANES = std::is_same_v<O, float> ? 3 : 2;
  auto hidden = [&](auto any, auto gated, auto rt) {
    const dim3 grid((unsigned)((p.hidden + 15) / 16), (unsigned)t.entries_max, (unsigned)t.blocks);
    hipLaunchKernelGGL((tokens_hidden<T, PACKED, decltype(any)::value, decltype(gated)::value, decltype(rt)::value, PLANES>),
                       grid, dim3(TOKENS_THREADS), 0, s, p);
    PXG_HIP(hipGetLastError());
  };
  auto out_of = [&](auto any, auto rt, auto parts, auto waves) {
    constexpr int PARTS = decltype(parts)::value, WAVES = decltype(waves)::value;
    constexpr uint64_t MOST = LAUNCH_ROWS / 2;  // of 1024 threads
    const uint64_t all = (uint64_t)p.slices * (((uint64_t)p.n + 16 / PARTS - 1) / (16 / PARTS));
    for (uint64_t a = 0; a < all; a += MOST) {
      p.first = (unsigned)a;
      hipLaunchKernelGGL((tokens_out<T, PACKED, decltype(any)::value, decltype(rt)::value, O, PARTS, WAVES>),
                         dim3((unsigned)std::min(MOST, all - a), (unsigned)t.blocks), dim3(64 * WAVES), 0, s, p);
      PXG_HIP(hipGetLastError());
    }
  };
  auto aligned = [](const void* d, uint64_t cols, uint64_t stride, uint64_t group) {
    return ((uint64_t)(uintptr_t)d | cols * 2 | stride * 2 | group * 2) % 16 == 0;
  };
  const bool any1 = !aligned(p.x, p.k, p.xs, 0) || (!PACKED && (!aligned(p.w1.p, p.k, p.w1.stride, p.w1.group) ||
                                                               (p.up.p && !aligned(p.up.p, p.k, p.up.stride, p.up.group))));
  const bool any2 = !PACKED && !aligned(p.w2.p, p.hidden, p.w2.stride, p.w2.group);
  using Yes = std::true_type;
  using No = std::false_type;
  using One = std::integral_constant<int, 1>;
  using Two = std::integral_constant<int, 2>;
  using Four = std::integral_constant<int, 4>;
  auto out = [&](auto any, auto rt) {
    using Few = std::integral_constant<int, TOKENS_WAVES>;
    using Many = std::integral_constant<int, 16>;
    if (t.parts == 2) {
      out_of(any, One{}, Two{}, Many{});
    } else if (t.waves == 16) {
      out_of(any, rt, One{}, Many{});
    } else {
      out_of(any, rt, One{}, Few{});
    }
  };
  auto by_rows = [&](auto f) {
    if (p.rows <= 16) f(One{});
    else if (p.rows <= 32) f(Two{});
    else f(Four{});
  };
  by_rows([&](auto rt) {
    auto by_matrices = [&](auto any) {
      if (p.up.p) hidden(any, Two{}, rt);
      else hidden(any, One{}, rt);
    };
    if (any1) by_matrices(Yes{});
    else by_matrices(No{});
    if constexpr (!PACKED) {
      if (any2) return out(Yes{}, rt);
    }
    out(No{}, rt);
  });
  if (p.slices > 1) {
    const uint64_t all = (uint64_t)p.rows * p.n;
    hipLaunchKernelGGL((tokens_join<T, O>), dim3((unsigned)std::min<uint64_t>((all + 255) / 256, 4096)), dim3(256), 0, s, p);
    PXG_HIP(hipGetLastError());
  }
}

uint64_t workspace_bytes_of(const TokensPlan& t) { return t.planes_bytes + t.entries_bytes + t.partial_bytes; }

void check_tokens(uint64_t rows, uint64_t picks, uint64_t experts) {
  if (rows > TOKENS_MAX) config_error("rows", rows, "must be at most 65536");
  if (picks == 0 || picks > PICKS_MAX) config_error("picks", picks, "must be between 1 and 16");
  if (experts == 0 || experts > EXPERTS_MAX) config_error("experts", experts, "must be between 1 and 65536");
}
// Sizes whose rows' bytes tiles count in 31 bits.
void check_width(const char* name, uint64_t size) {
  if (size == 0 || size > (1u << 22)) config_error(name, size, "must be between 1 and 4194304");
}

}  // namespace
}  // namespace pxg

using namespace pxg;

extern "C" {

uint64_t pxg_expert_layer_workspace(uint64_t rows, uint64_t picks, uint64_t experts, uint64_t hidden, uint64_t n,
                                    int out_type) {
  if (rows == 0 || rows > TOKENS_MAX || picks == 0 || picks > PICKS_MAX || experts == 0 || experts > EXPERTS_MAX ||
      hidden == 0 || hidden > (1u << 22) || n == 0 || n > PRODUCT_SIZE_MAX)
    return 0;
  // enough for packed matrices as for others, whose slices are more
  return workspace_bytes_of(tokens_plan(rows, picks, experts, hidden, n, out_type == PXG_F32, false));
}

int pxg_expert_layer_device(const pxg_expert_layer* layer, void* stream) {
  return guard([&] {
    const pxg_expert_layer& a = check_arguments(layer);
    const bool packed = a.packed != 0;
    check_type(a.type, false);
    if (packed && a.type != PXG_BF16) config_error("type", (uint64_t)a.type, "must be bf16 with packed matrices");
    check_out_type(a.type, a.out_type);
    check_tokens(a.rows, a.picks, a.experts);
    check_width("k", a.k);
    check_width("hidden", a.hidden);
    check_size("n", a.n);
    check_optional_activation(a.activation);
    check_rows(a.type, "x", a.x, a.rows, a.k, a.x_stride);
    check_rows(PXG_F32, "gates", a.gates, a.rows, a.picks, a.gates_stride);
    check_rows(PXG_F32, "ids", a.ids, a.rows, a.picks, a.ids_stride);
    check_aligned("ids", a.ids, 8);
    auto matrix = [&](const char* name, const pxg_expert_matrix& m, uint64_t height, uint64_t width) {
      if (!m.data) config_error(name, 0, "must not be null");
      if (packed) {
        check_packed_rows(name, m.data, name, m.scales, height);
        const uint64_t wide = check_stride(2, width, block8_code_stride(width));
        return ExpertMatrix{m.data, wide, height * wide, (const uint8_t*)m.scales, block8_scale_stride(width)};
      }
      check_rows(a.type, name, m.data, height, width, m.stride);
      return ExpertMatrix{m.data, check_stride(height, width, m.stride), m.group_stride, nullptr, 0};
    };
    TokenLayer p{};
    p.w1 = matrix("w1", a.w1, a.hidden, a.k);
    if (a.up.data) p.up = matrix("up", a.up, a.hidden, a.k);
    p.w2 = matrix("w2", a.w2, a.n, a.hidden);
    check_bias("bias1", a.type, a.bias_type, a.bias1, a.experts, a.hidden, a.bias1_stride);
    check_bias("bias2", a.type, a.bias_type, a.bias2, a.experts, a.n, a.bias2_stride);
    if (a.residual) check_rows(a.out_type, "residual", a.residual, a.rows, a.n, a.residual_stride);
    check_rows(a.out_type, "y", a.y, a.rows, a.n, a.y_stride);
    p.xs = check_stride(a.rows, a.k, a.x_stride);
    if (a.rows == 0) return;
    const TokensPlan t = tokens_plan(a.rows, a.picks, a.experts, a.hidden, a.n, a.out_type == PXG_F32, packed);
    check_aligned("workspace", a.workspace, 16);
    if (!a.workspace || a.workspace_bytes < workspace_bytes_of(t))
      config_error("workspace_bytes", a.workspace_bytes, "must be what pxg_expert_layer_workspace says");
    p.x = a.x;
    p.ids = a.ids;
    p.gates = a.gates;
    p.is = a.ids_stride;
    p.gs = a.gates_stride;
    p.bias1 = a.bias1;
    p.bias2 = a.bias2;
    p.b1s = a.bias1_stride;
    p.b2s = a.bias2_stride;
    p.residual = a.residual;
    p.rs = a.residual_stride;
    p.y = a.y;
    p.ys = a.y_stride;
    p.planes = (char*)a.workspace;
    p.entries = (Entry*)(p.planes + t.planes_bytes);
    p.partial = (float*)(p.planes + t.planes_bytes + t.entries_bytes);
    p.rows = (int)a.rows;
    p.k = (int)a.k;
    p.hidden = (int)a.hidden;
    p.wide = (int)t.wide;
    p.n = (int)a.n;
    p.picks = (int)a.picks;
    p.experts = (int)a.experts;
    p.entries_max = (int)t.entries_max;
    p.slices = t.slices;
    p.activation = (int)a.activation;
    p.bias_f32 = a.bias_type == PXG_F32;
    const hipStream_t s = (hipStream_t)stream;
    const bool f32_out = a.out_type == PXG_F32;
    if (packed) {
      if (f32_out) run_tokens<__bf16, true, float>(p, t, s);
      else run_tokens<__bf16, true, __bf16>(p, t, s);
    } else if (a.type == PXG_F16) {
      if (f32_out) run_tokens<_Float16, false, float>(p, t, s);
      else run_tokens<_Float16, false, _Float16>(p, t, s);
    } else {
      if (f32_out) run_tokens<__bf16, false, float>(p, t, s);
      else run_tokens<__bf16, false, __bf16>(p, t, s);
    }
  });
}

}  // extern "C"
