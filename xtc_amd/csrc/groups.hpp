// SPDX-License-Identifier: BSD-3-Clause
// Rows sorted by group: which rows a group has, and which tile of which group
// a workgroup computes.
//
// sizes[e] says how many rows group e has; the groups follow one another from
// row 0.  A negative size counts as none and rows past T belong to nobody:
//   begin(e) = min(T, sum_{i<e} max(sizes[i], 0)),  end(e) = begin(e + 1)
// Sums saturate at T, which needs 2 T < 2^32 and keeps any sizes harmless.
//
// The host does not know the sizes, so every wave of a workgroup finds its own
// group: 64 sizes a step, two prefix sums over the lanes.  For E <= 64 that is
// one load and twelve lane shuffles, below a microsecond.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace xtc_hip {

struct RowGroup {
  int e;      // group; E for the rows past the last group, -1 for no tile
  int begin;  // first row of the tile
  int end;    // one past the last row of the group
};

namespace groups {

__device__ __forceinline__ unsigned sat_add(unsigned a, unsigned b, unsigned top) { return min(a + b, top); }

// inclusive prefix sums over the 64 lanes, saturating at `top`
__device__ __forceinline__ unsigned scan(unsigned v, unsigned top, int lane) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const unsigned u = __shfl_up(v, d);
    v = lane >= d ? sat_add(u, v, top) : v;
  }
  return v;
}

}  // namespace groups

// Tile `mt` of the tiles of BM rows, group after group, the rows past the last
// group (if any) as group E.  Wave-uniform.
template <int BM>
__device__ __forceinline__ RowGroup find_tile(const int* sizes, int E, int T, int mt) {
  const int lane = threadIdx.x & 63;
  unsigned rows = 0, tiles = 0;  // before this step's groups
  for (int e0 = 0; e0 <= E; e0 += 64) {
    const int e = e0 + lane;
    const unsigned n = e < E ? min((unsigned)max(sizes[e], 0), (unsigned)T) : 0u;
    unsigned end = groups::sat_add(rows, groups::scan(n, T, lane), T);
    if (e >= E) end = T;  // the pseudo-group of the rows past the last group
    unsigned begin = __shfl_up(end, 1);
    if (lane == 0) begin = rows;
    const unsigned mine = e <= E ? (end - begin + BM - 1) / BM : 0u;
    const unsigned upto = tiles + groups::scan(mine, 0x7fffffffu, lane);
    const uint64_t hit = __ballot((int)(upto - mine) <= mt && mt < (int)upto);
    if (hit) {
      const int at = __builtin_ctzll(hit);
      RowGroup r;
      r.e = e0 + at;
      const int first = __builtin_amdgcn_readlane((int)begin, at);
      const int skip = mt - __builtin_amdgcn_readlane((int)(upto - mine), at);
      r.begin = first + skip * BM;
      r.end = __builtin_amdgcn_readlane((int)end, at);
      return r;
    }
    rows = __builtin_amdgcn_readlane((int)end, 63);
    tiles = __builtin_amdgcn_readlane((int)upto, 63);
  }
  return RowGroup{-1, 0, 0};
}

// All rows of group e.  Wave-uniform.
__device__ __forceinline__ RowGroup find_group(const int* sizes, int E, int T, int e) {
  const int lane = threadIdx.x & 63;
  unsigned rows = 0;
  for (int e0 = 0;; e0 += 64) {
    const int i = e0 + lane;
    const unsigned n = i < E ? min((unsigned)max(sizes[i], 0), (unsigned)T) : 0u;
    const unsigned end = groups::sat_add(rows, groups::scan(n, T, lane), T);
    if (e < e0 + 64) {
      RowGroup r;
      r.e = e;
      r.end = __builtin_amdgcn_readlane((int)end, e - e0);
      r.begin = e == e0 ? (int)rows : __builtin_amdgcn_readlane((int)end, e - e0 - 1);
      return r;
    }
    rows = __builtin_amdgcn_readlane((int)end, 63);
  }
}

// Tiles of BM rows that E groups and the rows past them can have, T rows in
// all: each of n parts that are not empty ends in one partial tile at most.
inline int64_t most_tiles(int64_t T, int64_t E, int BM) {
  const int64_t n = T < E + 1 ? T : E + 1;
  return (T + n * (BM - 1)) / BM;
}

}  // namespace xtc_hip
