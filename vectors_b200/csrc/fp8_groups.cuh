// fp8_groups.cuh -- the groups of a grouped 8-bit product and their tiles.
#pragma once
#include "fp8.h"

namespace vx {

// A group's rows and queries, within the operands, and its tiles.
struct Fp8Group {
  int row0, nrows, query0, nqueries;
  uint32_t query_tiles, row_tiles;
  int width;      // queries of a tile, a multiple of 32
  int tile_rows;  // rows of a tile, a multiple of 32
  __device__ __forceinline__ int64_t tiles() const { return (int64_t)row_tiles * query_tiles; }
};

__device__ __forceinline__ int64_t clamp_to(int64_t v, int64_t hi) { return v < 0 ? 0 : v > hi ? hi : v; }

// (first row, rows, first query, queries) of group g from its untrusted offsets.
__device__ __forceinline__ int4 fp8_group_bounds(const Fp8Groups& a, int64_t g) {
  const int64_t row0 = clamp_to(a.row_off[g], a.nrows), query0 = clamp_to(a.query_off[g], a.nq);
  return make_int4((int)row0, (int)clamp_to(clamp_to(a.row_off[g + 1], a.nrows) - row0, a.max_cols), (int)query0,
                   (int)clamp_to(clamp_to(a.query_off[g + 1], a.nq) - query0, a.nq));
}

__device__ __forceinline__ Fp8Group fp8_group(const int4& b) {
  Fp8Group r;
  r.row0 = b.x, r.nrows = b.y, r.query0 = b.z, r.nqueries = b.w;
  r.query_tiles = (uint32_t)(r.nqueries + (kFp8MaxWidth - 1)) / kFp8MaxWidth;
  r.row_tiles = (uint32_t)(r.nrows + (kFp8TileRows - 1)) / kFp8TileRows;
  // equal tiles, up to a multiple of 32
  r.width = r.query_tiles == 0 ? 32 : (int)(((uint32_t)r.nqueries + r.query_tiles - 1) / r.query_tiles + 31) / 32 * 32;
  r.tile_rows = r.row_tiles == 0 ? 32 : (int)(((uint32_t)r.nrows + r.row_tiles - 1) / r.row_tiles + 31) / 32 * 32;
  return r;
}

// Tile t of a group (t % query_tiles its query tile), and a tile in 16 bytes.
__device__ __forceinline__ Fp8Tile fp8_group_tile(const Fp8Group& g, int64_t t) {
  const int64_t rt = (uint64_t)t >> 32 ? t / g.query_tiles : (int64_t)((uint32_t)t / g.query_tiles);
  const int64_t qt = t - rt * g.query_tiles;
  Fp8Tile x;
  x.col = (uint32_t)(rt * g.tile_rows);
  x.row = (uint32_t)g.row0 + x.col;
  x.query = (uint32_t)(g.query0 + qt * g.width);
  const int rows = g.nrows - (int)x.col, queries = g.nqueries - (int)(qt * g.width);
  x.rows = rows < g.tile_rows ? rows : g.tile_rows;
  x.queries = queries < g.width ? queries : g.width;
  x.width = (x.queries + 31) / 32 * 32;
  x.half = g.tile_rows >> 1;
  return x;
}
__device__ __forceinline__ ulonglong2 pack_tile(const Fp8Tile& t) {
  return make_ulonglong2((uint64_t)t.row << 32 | t.query,
                         (uint64_t)t.col << 32 | (uint32_t)t.rows << 23 | (uint32_t)t.queries << 15 |
                             (uint32_t)t.width / 32 << 8 | (uint32_t)t.half);
}
__device__ __forceinline__ Fp8Tile unpack_tile(uint64_t x, uint64_t y) {
  const uint32_t v = (uint32_t)y;
  return Fp8Tile{(uint32_t)(x >> 32),  (uint32_t)x,              (uint32_t)(y >> 32), (int)(v >> 23),
                 (int)(v >> 15 & 255), (int)(v >> 8 & 127) * 32, (int)(v & 255)};
}

// Each group's bounds (a.bounds [groups]) and the tiles before it (a.tile_off [groups + 1]), and the
// first tiles (a.first), by one block of kThreads threads, each with a run of consecutive groups.
template <int kThreads>
__device__ __forceinline__ void fp8_count_tiles(const Fp8Groups& a) {
  __shared__ int64_t warp_sum[kThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t per = (a.groups + kThreads - 1) / kThreads;
  const int64_t g0 = tid * per, g1 = g0 + per < a.groups ? g0 + per : a.groups;
  int64_t mine = 0;
#pragma unroll 4
  for (int64_t g = g0; g < g1; g++) {
    const int4 b = fp8_group_bounds(a, g);
    a.bounds[g] = b;
    mine += fp8_group(b).tiles();
  }
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
    before += fp8_group(a.bounds[g]).tiles();
  }
  if (g0 < a.groups && g1 == a.groups) a.tile_off[a.groups] = before;
  __syncthreads();
  // thread p: the group with tile_off[lo] <= p < tile_off[hi]
  for (int p = tid; p < a.firsts; p += kThreads) {
    int64_t lo = 0, hi = a.groups;
    if (p >= a.tile_off[hi]) {
      a.first[p] = make_ulonglong2(0, 0);
      continue;
    }
    // the first groups hold the first tiles: doubling steps, then bisection
    for (int64_t by = 1; lo + by < hi; by *= 2) {
      if (a.tile_off[lo + by] > p) {
        hi = lo + by;
        break;
      }
      lo += by;
    }
    while (hi - lo > 1) {
      const int64_t mid = (lo + hi) >> 1;
      if (a.tile_off[mid] <= p) lo = mid;
      else hi = mid;
    }
    a.first[p] = pack_tile(fp8_group_tile(fp8_group(a.bounds[lo]), p - a.tile_off[lo]));
  }
}

}  // namespace vx
