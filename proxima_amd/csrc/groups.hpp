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
  int begin = 0, before = 0;  // rows and tiles before the segments of this pass
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

// A group's rows are summed in one part, or, longer than `limit` rows
// (limit > 0), in as few parts as keep each within it, whole steps of 64 rows.
// Parts of divided groups have slots of a workspace, in the groups' order.
// Above 62 groups none is divided.
struct GroupPart {
  int group, lo, hi;
  int parts, slot;  // of the group; this part's slot where there are several
};
__host__ __device__ __forceinline__ int group_parts(int size, int limit) {
  return limit > 0 && size > limit ? (size - 1) / limit + 1 : 1;  // size + limit may pass 2^31
}
// The rows of each of several parts but the last, which may have fewer.
__host__ __device__ __forceinline__ int group_part_length(int size, int parts) {
  return ((size - 1) / parts / 64 + 1) * 64;
}

// The part at a place in the order of falling lengths (ties by index; above 62
// groups the groups' own order), by a wavefront whose lanes all call it; false
// past the last.
__device__ __forceinline__ bool find_group_part(const int64_t* __restrict__ offsets, int groups, int rows, int limit,
                                                int place, GroupPart& g) {
  if (groups > SEGMENT_GROUPS) {
    if (place >= groups) return false;
    group_range(offsets, place, rows, g.lo, g.hi);
    g.group = place;
    g.parts = 1;
    g.slot = 0;
    return true;
  }
  const int lane = threadIdx.x & (WAVE - 1);
  const Segments s = load_segments(offsets, groups, rows);
  const bool real = lane >= 1 && lane <= groups;
  const int size = s.end - s.first, parts = real ? group_parts(size, limit) : 0;
  const int length = parts > 1 ? group_part_length(size, parts) : size;
  int before = 0;
  for (int o = 1; o <= groups; ++o) {
    const int l = __builtin_amdgcn_readlane(length, o), n = __builtin_amdgcn_readlane(parts, o);
    before += l > length || (l == length && o < lane) ? n : 0;
  }
  const int slots = parts > 1 ? parts : 0, slot = wave_sum_scan(slots, lane) - slots;
  const uint64_t hit = __ballot(real && place >= before && place < before + parts);
  if (!hit) return false;
  const int l = __builtin_ctzll(hit), k = place - __builtin_amdgcn_readlane(before, l);
  const int first = __builtin_amdgcn_readlane(s.first, l), end = __builtin_amdgcn_readlane(s.end, l);
  const int64_t from = first + (int64_t)k * __builtin_amdgcn_readlane(length, l);
  const int64_t to = from + __builtin_amdgcn_readlane(length, l);
  g.group = l - 1;
  g.lo = from < end ? (int)from : end;
  g.hi = to < end ? (int)to : end;
  g.parts = __builtin_amdgcn_readlane(parts, l);
  g.slot = __builtin_amdgcn_readlane(slot, l) + k;
  return true;
}

// Divided group `index` in the groups' order: itself, its parts and its first
// slot; false past the last.
__device__ __forceinline__ bool find_divided_group(const int64_t* __restrict__ offsets, int groups, int rows, int limit,
                                                   int index, GroupPart& g) {
  const int lane = threadIdx.x & (WAVE - 1);
  const Segments s = load_segments(offsets, groups, rows);
  const int parts = lane >= 1 && lane <= groups ? group_parts(s.end - s.first, limit) : 0;
  const int slots = parts > 1 ? parts : 0, slot = wave_sum_scan(slots, lane) - slots;
  const int nth = wave_sum_scan(parts > 1 ? 1 : 0, lane);
  const uint64_t hit = __ballot(parts > 1 && nth == index + 1);
  if (!hit) return false;
  const int l = __builtin_ctzll(hit);
  g = {l - 1, __builtin_amdgcn_readlane(s.first, l), __builtin_amdgcn_readlane(s.end, l),
       __builtin_amdgcn_readlane(parts, l), __builtin_amdgcn_readlane(slot, l)};
  return true;
}

// No more parts, and no more slots, than this.
inline uint64_t group_parts_max(uint64_t rows, uint64_t groups, uint64_t limit) {
  if (groups == 1 && limit) return (rows + limit - 1) / limit;
  return limit ? groups + rows / limit : groups;
}
inline uint64_t group_slots_max(uint64_t rows, uint64_t groups, uint64_t limit) {
  if (groups == 1 && limit) return (rows + limit - 1) / limit;
  const uint64_t divided = limit ? rows / limit : 0;
  return divided + (divided < groups ? divided : groups);
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
