// Ragged groups of rows, from offsets that stay on the device.
//
// Group g is the rows from offsets[g] to offsets[g + 1]. The offsets are
// clamped: each to [0, rows], then to no less than those before it, so that
// any values give disjoint ranges inside the matrix. Rows before the first
// group and after the last belong to none.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "device.hpp"

namespace pxg {

__device__ __forceinline__ int clamp_offset(int64_t o, int rows) {
  return o < 0 ? 0 : o > rows ? rows : (int)o;
}

__device__ __forceinline__ int wave_max_scan(int v, int lane) {
#pragma unroll
  for (int o = 1; o < WAVE; o <<= 1) {
    const int u = __shfl_up(v, o, WAVE);
    v = lane >= o && u > v ? u : v;
  }
  return v;
}
__device__ __forceinline__ int wave_sum_scan(int v, int lane) {
#pragma unroll
  for (int o = 1; o < WAVE; o <<= 1) {
    const int u = __shfl_up(v, o, WAVE);
    v += lane >= o ? u : 0;
  }
  return v;
}

// The rows of group g, by a wavefront whose lanes all call it.
__device__ __forceinline__ void group_range(const int64_t* __restrict__ offsets, int g, int rows, int& lo, int& hi) {
  const int lane = threadIdx.x & (WAVE - 1);
  int m = 0;
  for (int i = lane; i <= g; i += WAVE) {
    const int o = clamp_offset(offsets[i], rows);
    m = o > m ? o : m;
  }
#pragma unroll
  for (int o = WAVE / 2; o > 0; o >>= 1) {
    const int u = __shfl_xor(m, o, WAVE);
    m = u > m ? u : m;
  }
  lo = __builtin_amdgcn_readfirstlane(m);
  const int h = __builtin_amdgcn_readfirstlane(clamp_offset(offsets[g + 1], rows));
  hi = h > lo ? h : lo;
}

// One tile of at most `size` rows: its group (-1: rows of no group, whose
// results are zero), its first row and the end of its segment.
struct RowTile {
  int group, row, end;
};

// The tiles of `size` rows that the groups, and the rows of none at either
// end, are cut into: all of them in order, only the whole ones, or only the
// last, partial ones of each.
enum RowTileKind { ALL_TILES, WHOLE_TILES, PARTIAL_TILES };

template <int KIND>
__device__ __forceinline__ int row_tiles_of(int rows, int size) {
  return KIND == ALL_TILES ? (rows + size - 1) / size : KIND == WHOLE_TILES ? rows / size : rows % size ? 1 : 0;
}

// Tile `index` of its kind; false past the last. `offsets` NULL is one group
// of all rows. A wavefront's lanes all call it and get the same.
template <int KIND>
__device__ __forceinline__ bool find_row_tile(const int64_t* __restrict__ offsets, int groups, int rows, int size,
                                              int index, RowTile& t) {
  if (!offsets) {
    t = {0, (KIND == PARTIAL_TILES ? rows / size + index : index) * size, rows};
    return index < row_tiles_of<KIND>(rows, size);
  }
  const int lane = threadIdx.x & (WAVE - 1);
  int begin = 0, before = 0;  // rows and tiles before the segments of this round
  // segment s ends at offsets[s]; segment 0 and segment groups + 1 are the rows of no group
  for (int s0 = 0; s0 < groups + 2; s0 += WAVE) {
    const int s = s0 + lane;
    int end = s <= groups ? clamp_offset(offsets[s], rows) : rows;
    end = wave_max_scan(end > begin ? end : begin, lane);
    int first = __shfl_up(end, 1, WAVE);
    if (lane == 0) first = begin;
    const int tiles = row_tiles_of<KIND>(end - first, size);
    const int last = before + wave_sum_scan(tiles, lane);
    const uint64_t hit = __ballot(index < last);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      const int f = __builtin_amdgcn_readlane(first, l), n = __builtin_amdgcn_readlane(tiles, l);
      const int k = index - (__builtin_amdgcn_readlane(last, l) - n);
      t.group = s0 + l == 0 || s0 + l > groups ? -1 : s0 + l - 1;
      t.end = __builtin_amdgcn_readlane(end, l);
      t.row = KIND == PARTIAL_TILES ? f + (t.end - f) / size * size : f + k * size;
      return true;
    }
    begin = __builtin_amdgcn_readlane(end, WAVE - 1);
    before = __builtin_amdgcn_readlane(last, WAVE - 1);
  }
  return false;
}

// How many whole and partial tiles there are.
__device__ __forceinline__ void count_row_tiles(const int64_t* __restrict__ offsets, int groups, int rows, int size,
                                                int& whole, int& partial) {
  if (!offsets) {
    whole = row_tiles_of<WHOLE_TILES>(rows, size);
    partial = row_tiles_of<PARTIAL_TILES>(rows, size);
    return;
  }
  const int lane = threadIdx.x & (WAVE - 1);
  int begin = 0;
  whole = partial = 0;
  for (int s0 = 0; s0 < groups + 2; s0 += WAVE) {
    const int s = s0 + lane;
    int end = s <= groups ? clamp_offset(offsets[s], rows) : rows;
    end = wave_max_scan(end > begin ? end : begin, lane);
    int first = __shfl_up(end, 1, WAVE);
    if (lane == 0) first = begin;
    partial += __popcll(__ballot(row_tiles_of<PARTIAL_TILES>(end - first, size)));
    whole += __builtin_amdgcn_readlane(wave_sum_scan(row_tiles_of<WHOLE_TILES>(end - first, size), lane), WAVE - 1);
    begin = __builtin_amdgcn_readlane(end, WAVE - 1);
  }
}

// The segments of up to 62 groups, one a lane: segment s is rows first to end,
// segments 0 and groups + 1 (and the empty ones past it) those of no group.
struct Segments {
  int first, end;
};
constexpr int SEGMENT_GROUPS = WAVE - 2;
__device__ __forceinline__ Segments load_segments(const int64_t* __restrict__ offsets, int groups, int rows) {
  const int lane = threadIdx.x & (WAVE - 1);
  Segments s;
  s.end = wave_max_scan(lane <= groups ? clamp_offset(offsets[lane], rows) : rows, lane);
  s.first = __shfl_up(s.end, 1, WAVE);
  if (lane == 0) s.first = 0;
  return s;
}

// Tile `index` of its kind, as find_row_tile.
template <int KIND>
__device__ __forceinline__ bool pick_row_tile(const Segments& s, int groups, int size, int index, RowTile& t) {
  const int lane = threadIdx.x & (WAVE - 1);
  const int tiles = row_tiles_of<KIND>(s.end - s.first, size);
  const int last = wave_sum_scan(tiles, lane);
  const uint64_t hit = __ballot(index < last);
  if (!hit) return false;
  const int l = __builtin_ctzll(hit);
  const int f = __builtin_amdgcn_readlane(s.first, l), n = __builtin_amdgcn_readlane(tiles, l);
  const int k = index - (__builtin_amdgcn_readlane(last, l) - n);
  t.group = l == 0 || l > groups ? -1 : l - 1;
  t.end = __builtin_amdgcn_readlane(s.end, l);
  t.row = KIND == PARTIAL_TILES ? f + (t.end - f) / size * size : f + k * size;
  return true;
}
__device__ __forceinline__ void count_segments(const Segments& s, int size, int& whole, int& partial) {
  const int lane = threadIdx.x & (WAVE - 1);
  partial = __popcll(__ballot(row_tiles_of<PARTIAL_TILES>(s.end - s.first, size)));
  whole = __builtin_amdgcn_readlane(wave_sum_scan(row_tiles_of<WHOLE_TILES>(s.end - s.first, size), lane), WAVE - 1);
}

// The group, and its rows, at a place in the order of falling sizes (ties by
// index), by a wavefront whose lanes all call it; above 62 groups the order is
// the groups' own.
__device__ __forceinline__ int group_by_size(const int64_t* __restrict__ offsets, int groups, int rows, int place,
                                             int& lo, int& hi) {
  if (groups > SEGMENT_GROUPS) {
    group_range(offsets, place, rows, lo, hi);
    return place;
  }
  const int lane = threadIdx.x & (WAVE - 1);
  const Segments s = load_segments(offsets, groups, rows);
  const int size = lane >= 1 && lane <= groups ? s.end - s.first : -1;
  int rank = 0;
  for (int g = 1; g <= groups; ++g) {
    const int o = __builtin_amdgcn_readlane(size, g);
    rank += o > size || (o == size && g < lane) ? 1 : 0;
  }
  const int l = __builtin_ctzll(__ballot(size >= 0 && rank == place));
  lo = __builtin_amdgcn_readlane(s.first, l);
  hi = __builtin_amdgcn_readlane(s.end, l);
  return l - 1;
}

// No more tiles than this come out of `rows` rows in `groups` groups, the
// rows of no group at either end counted as two more.
inline uint64_t row_tiles_max(uint64_t rows, uint64_t groups, uint64_t size, bool ragged) {
  const uint64_t full = (rows + size - 1) / size;
  if (!ragged) return full;
  const uint64_t parts = groups + 2 < rows ? groups + 2 : rows;
  return rows / size + parts < full ? full : rows / size + parts;
}

}  // namespace pxg
