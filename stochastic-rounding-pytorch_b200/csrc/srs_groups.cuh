// Rows in groups: group g has rows ends[g-1] .. ends[g] - 1 of a matrix (from 0 for the
// first), rows from the last end on belong to none.  `ends` is in device memory and the
// host never reads it: grids are sized by a bound and every CTA finds its own part.
//
// Ends are read as their running maximum, cut to 0 .. rows: whatever the array holds, the
// groups lie inside the matrix, do not overlap, and their tiles stay within the bound
//   rows / edge + groups
// that buffers and grids are sized by.
#pragma once

#include <cstdint>
#include <cuda_runtime.h>

namespace srs {

constexpr int kMaxGroups = 1024;

__device__ __forceinline__ int64_t token_at(const int32_t* order, int place, int tokens) {
  const int t = __ldg(order + place);
  return t >= 0 && t < tokens ? t : 0;  // an entry that names no token reads the first
}

__device__ __forceinline__ int warp_scan_sum(int v, int lane) {
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int u = __shfl_up_sync(0xFFFFFFFFu, v, d);
    if (lane >= d) v += u;
  }
  return v;
}

__device__ __forceinline__ int warp_scan_max(int v, int lane) {
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int u = __shfl_up_sync(0xFFFFFFFFu, v, d);
    if (lane >= d) v = max(v, u);
  }
  return v;
}

// The ends of up to 128 groups from the first on, one a lane, asked for together.
struct EndsAhead {
  int e[4];
  __device__ __forceinline__ EndsAhead(const int32_t* __restrict__ ends, int groups, int lane) {
#pragma unroll
    for (int i = 0; i < 4; ++i) e[i] = 32 * i + lane < groups ? __ldg(ends + 32 * i + lane) : 0;
  }
  __device__ __forceinline__ int at(const int32_t* __restrict__ ends, int groups, int base,
                                    int lane) const {
    if (base >= 128) return base + lane < groups ? __ldg(ends + base + lane) : 0;
    return base < 64 ? (base < 32 ? e[0] : e[1]) : (base < 96 ? e[2] : e[3]);
  }
};

// Groups base .. base + 31 for a warp, one a lane; `carry`: end of the group before.
// Groups from `groups` on are empty.
__device__ __forceinline__ void group_span(const int32_t* __restrict__ ends, const EndsAhead& ahead,
                                           int groups, int rows, int base, int lane, int* carry,
                                           int* start, int* end) {
  int e = min(max(ahead.at(ends, groups, base, lane), 0), rows);
  e = max(warp_scan_max(base + lane < groups ? e : 0, lane), *carry);
  const int before = __shfl_up_sync(0xFFFFFFFFu, e, 1);
  *start = lane == 0 ? *carry : before;
  *end = e;
  *carry = __shfl_sync(0xFFFFFFFFu, e, 31);
}

// One tile of `edge` rows at most, counted from its group's first row.
struct GroupTile {
  int group;      // -1: there is no such tile
  int row0, end;  // first row of the tile, end of its group
  int start;      // first row of its group
  int rank;       // groups with rows before it
  int quads;      // 4 * (words of 4 tiles that groups before it take) + tiles before it in its own
};

// Tile `index` of all groups' tiles in order, found by a warp (the same in all lanes).
__device__ __forceinline__ GroupTile find_group_tile(const int32_t* __restrict__ ends, int groups,
                                                     int rows, int edge, int index, int lane) {
  GroupTile r{-1, 0, 0, 0, 0, 0};
  int carry = 0, tiles_before = 0, quads_before = 0, rank = 0;
  const EndsAhead ahead(ends, groups, lane);
  for (int base = 0; base < groups; base += 32) {
    int start, end;
    group_span(ends, ahead, groups, rows, base, lane, &carry, &start, &end);
    const int tiles = (end - start + edge - 1) / edge, quads = (tiles + 3) & ~3;
    const int upto = tiles_before + warp_scan_sum(tiles, lane);
    const int quads_upto = quads_before + warp_scan_sum(quads, lane);
    const unsigned found = __ballot_sync(0xFFFFFFFFu, upto > index);
    const unsigned some = __ballot_sync(0xFFFFFFFFu, tiles > 0);
    if (found != 0u) {
      const int at = __ffs(found) - 1, inside = index - (upto - tiles);
      r.group = base + at;
      r.row0 = __shfl_sync(0xFFFFFFFFu, start + inside * edge, at);
      r.end = __shfl_sync(0xFFFFFFFFu, end, at);
      r.start = __shfl_sync(0xFFFFFFFFu, start, at);
      r.rank = rank + __popc(some & ((1u << at) - 1u));
      r.quads = __shfl_sync(0xFFFFFFFFu, quads_upto - quads + inside, at);
      return r;
    }
    tiles_before = __shfl_sync(0xFFFFFFFFu, upto, 31);
    quads_before = __shfl_sync(0xFFFFFFFFu, quads_upto, 31);
    rank += __popc(some);
  }
  return r;
}

// Most tiles of `edge` rows that `groups` groups of `rows` rows in all can have.
inline int64_t most_group_tiles(int64_t rows, int64_t groups, int64_t edge) {
  // every group with rows has at most one tile that is not full
  return rows / edge + (groups < rows ? groups : rows);
}

}  // namespace srs
