// fp8.h -- rows kept as e4m3 codes with one power-of-two scale per block of 128 dimensions:
// quantising rows into a store, reading them back, and the score products on them (fp8.cu,
// fp8_scores.cu).
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace vx {

constexpr int kFp8Block = 128;        // dimensions that share a scale
constexpr int kFp8MaxDim = 1 << 16;
constexpr int kFp8MaxWidth = 224;     // most queries of one product tile (TMEM columns per accumulator)
constexpr int kFp8TileRows = 256;     // most stored rows of one
// Batches of at most this many rows find repeated slots by comparing slots directly (fp8.cu): one launch and
// no scratch.  Rows x 768 fp32, direct / by a cluster: 7.5 / 10.7 us a call up to 512 rows and 10.3 / 10.7 at
// 1,000 (launches bound them); on the device, as in a captured graph, 3.0 / 3.4 us at 128 rows, 5.3 / 3.8 at
// 512, 7.7 / 4.7 at 1,000.
constexpr int64_t kFp8DirectSlots = 512;

inline int fp8_blocks(int dim) { return (dim + kFp8Block - 1) / kFp8Block; }
inline int fp8_code_pitch(int dim) { return fp8_blocks(dim) * kFp8Block; }  // bytes of codes per row
inline int fp8_scale_pitch(int dim) { return (fp8_blocks(dim) + 3) / 4 * 4; }  // bytes of scales per row

// A grouped product's offsets, the sizes they are clamped to, and where each group's bounds and the
// tiles before it go.
struct Fp8Groups {
  const int64_t* row_off;    // [groups + 1]; null: one group of every row and query
  const int64_t* query_off;  // [groups + 1]
  int64_t groups;
  int64_t nrows, nq;
  int64_t max_cols;   // results kept per query (groups with more rows are cut there)
  int4* bounds;       // [groups]
  int64_t* tile_off;  // [groups + 1]
  ulonglong2* first;  // [firsts] the first tiles, packed (width 0: there are fewer)
  int firsts;
};

// One tile of a product: rows [row, row + rows) against queries [query, query + queries), results from
// column `col`.
struct Fp8Tile {
  uint32_t row, query, col;  // below 2^31
  int rows, queries;
  int width;  // MMA N: queries rounded up to 32; 0: no more tiles
  int half;   // rows of each CTA: the leader's are the first `half`
};

struct Fp8WriteArgs {
  const void* rows;  // [n] rows, `stride` elements apart
  int type;          // vx_dtype of the rows
  int64_t n;
  int dim;
  int64_t stride;
  const void* slots;  // destination of each row, or null: first, first + 1, ...
  int slot_bytes;     // 4 or 8
  int64_t first;
  uint8_t* codes;
  uint8_t* scales;
  int64_t capacity;
  int32_t* owner;  // [capacity] scratch; needed for more than kFp8DirectSlots rows with slots
  int num_sms;
};

struct Fp8ReadArgs {
  const uint8_t* codes;
  const uint8_t* scales;
  int64_t capacity;
  int dim;
  const void* slots;
  int slot_bytes;
  int64_t first, n;
  void* out;
  int type;
  int64_t stride;
};

cudaError_t launch_fp8_write(const Fp8WriteArgs& a, int* launches, cudaStream_t st);
// Before a product: quantises its queries (a.rows null: they are stored rows already) and counts the
// groups' tiles (g.row_off null: no groups), in one launch that lets a dependent one begin early; clears
// *counter, unless null.
cudaError_t launch_fp8_prepare(const Fp8WriteArgs& a, const Fp8Groups& g, unsigned long long* counter, cudaStream_t st);
cudaError_t launch_fp8_read(const Fp8ReadArgs& a, cudaStream_t st);

struct Fp8ScoreArgs {
  const uint8_t* row_scales;
  int64_t nrows;
  const uint8_t* query_scales;
  int64_t nq;
  int scale_words;  // 32-bit scale words per row
  int kchunks;      // 128-byte chunks of a row
  void* out;
  int64_t ldo;  // elements between two queries' results
  Fp8Groups groups;
  uint64_t timeout_ns;
  int32_t* err;
  unsigned long long* next_tile;  // zero at the launch: tiles are taken from here; null: in fixed turns
  int64_t tiles;      // without groups
  int query_tiles;    // without groups
  int width;          // queries of the widest tile, a multiple of 32
  int tile_rows;      // stored rows of a tile
  // A few float queries that every cluster quantises for itself (resident queries): type a vx_dtype
  const void* queries;  // null: query_scales and the tensor maps tell of stored rows
  int query_type;
  int dim;
  int64_t query_stride;
  // filled in by launch_fp8_scores
  int stages;
  int stage_bytes;
  int tile_slots;
  int wait_first;
};

// The operands' tensor maps: rows[0] with boxes of half a tile's rows and queries[0] with boxes of half a
// tile's queries; with groups, whose tiles differ, rows[i] and queries[i] with boxes of 128 >> i rows.
struct Fp8Maps {
  CUtensorMap rows[4];
  CUtensorMap queries[4];
};

// The tiling of a product: tile sizes and, without groups, the number of tiles.
struct Fp8Tiling {
  int width, tile_rows, query_tiles;
  int64_t tiles;
};
// Whether a product's float queries are quantised inside it: few of them, and blocks for one round of
// its epilogue warps.
bool fp8_resident(int64_t nq, int dim, const Fp8Tiling& t);
Fp8Tiling fp8_tiling(int64_t nrows, int64_t nq, int64_t groups, int num_sms);
// after_prep: the launch before this one on `st` is launch_fp8_prepare's; this one may begin before it
// ends.
cudaError_t launch_fp8_scores(const Fp8Maps& maps, const Fp8ScoreArgs& a, int out_type, int num_sms, bool after_prep,
                              cudaStream_t st);

}  // namespace vx
