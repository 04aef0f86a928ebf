// fp8_groups.cuh -- the groups of a grouped 8-bit product and their tiles.
#pragma once
#include "fp8.h"

namespace vx {

// A group's rows and queries from its (untrusted) offsets, clamped to the operands.
struct Fp8Group {
  int64_t row0, nrows, query0, nqueries;
  int64_t query_tiles, tiles;
  int width;  // queries of a tile
};

__device__ __forceinline__ int64_t clamp_to(int64_t v, int64_t hi) { return v < 0 ? 0 : v > hi ? hi : v; }

__device__ __forceinline__ Fp8Group fp8_group(const Fp8Groups& a, int64_t g) {
  Fp8Group r;
  r.row0 = clamp_to(a.row_off[g], a.nrows);
  r.nrows = clamp_to(clamp_to(a.row_off[g + 1], a.nrows) - r.row0, a.max_cols);
  r.query0 = clamp_to(a.query_off[g], a.nq);
  r.nqueries = clamp_to(clamp_to(a.query_off[g + 1], a.nq) - r.query0, a.nq);
  // rows and queries are below 2^31: 32-bit division
  r.query_tiles = (uint32_t)(r.nqueries + kFp8MaxWidth - 1) / (uint32_t)kFp8MaxWidth;
  r.width = r.query_tiles == 0 ? 32
                               : (int)(((uint32_t)(r.nqueries + r.query_tiles - 1) / (uint32_t)r.query_tiles + 31) / 32 * 32);
  r.tiles = (int64_t)((uint32_t)(r.nrows + a.tile_rows - 1) / (uint32_t)a.tile_rows) * r.query_tiles;
  return r;
}

// Tiles before each group (a.tile_off [groups + 1]), by one block of kThreads threads, each with a run
// of consecutive groups.
template <int kThreads>
__device__ __forceinline__ void fp8_count_tiles(const Fp8Groups& a) {
  __shared__ int64_t warp_sum[kThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t per = (a.groups + kThreads - 1) / kThreads;
  const int64_t g0 = tid * per, g1 = g0 + per < a.groups ? g0 + per : a.groups;
  int64_t mine = 0;
#pragma unroll 4
  for (int64_t g = g0; g < g1; g++) mine += fp8_group(a, g).tiles;
  int64_t incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t v = __shfl_up_sync(0xFFFFFFFFu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) warp_sum[warp] = incl;
  __syncthreads();
  int64_t before = incl - mine;
  for (int i = 0; i < warp; i++) before += warp_sum[i];
#pragma unroll 4
  for (int64_t g = g0; g < g1; g++) {
    a.tile_off[g] = before;
    before += fp8_group(a, g).tiles;
  }
  if (g0 < a.groups && g1 == a.groups) a.tile_off[a.groups] = before;
}

}  // namespace vx
