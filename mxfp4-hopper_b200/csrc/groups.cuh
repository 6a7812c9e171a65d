// Ragged groups: rows sorted by expert, expert e owning rows [off[e], off[e + 1])
// with off the running sum of m_splits, which lives in device memory so that no
// host synchronisation is needed.  A negative split counts as zero and rows are
// never taken beyond M, whatever the splits say.
#pragma once
#include <cstdint>

#include "common.cuh"
#include "mxfp4_b200.h"

namespace mxb {

constexpr int kGroupTableInts = 2 * (MXB_MAX_EXPERTS + 1);

struct GroupTable {
  int32_t* off;   // [E + 1] first row of each expert
  int32_t* tile;  // [E + 1] first tile of each expert
};

// Built by one warp.  Expert e has tiles_of(rows) tiles; m_splits may be NULL
// for a single group of all M rows.
template <typename F>
__device__ __forceinline__ void build_groups(const GroupTable& g, const int32_t* m_splits, int E,
                                             int64_t M, F tiles_of) {
  const int lane = threadIdx.x & 31;
  int64_t rows_before = 0;
  int tiles_before = 0;
  for (int e0 = 0; e0 < E; e0 += 32) {
    const int e = e0 + lane;
    int64_t m = 0;
    if (e < E) m = m_splits ? max(m_splits[e], 0) : M;
    int64_t end = m;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t v = __shfl_up_sync(0xffffffffu, end, d);
      if (lane >= d) end += v;
    }
    end += rows_before;
    rows_before = __shfl_sync(0xffffffffu, end, 31);
    const int32_t a = (int32_t)min(end - m, M), b = (int32_t)min(end, M);
    const int tiles = e < E ? tiles_of(b - a) : 0;
    int tend = tiles;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, tend, d);
      if (lane >= d) tend += v;
    }
    tend += tiles_before;
    tiles_before = __shfl_sync(0xffffffffu, tend, 31);
    if (e < E) {
      g.off[e + 1] = b;
      g.tile[e + 1] = tend;
    }
  }
  if (lane == 0) g.off[0] = g.tile[0] = 0;
}

// The expert that tile t (< tile[E]) belongs to.
__device__ __forceinline__ int find_group(const int32_t* tile, int E, int t) {
  int lo = 0, hi = E - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (tile[mid + 1] > t) hi = mid; else lo = mid + 1;
  }
  return lo;
}

}  // namespace mxb
