// fp8_scores.cu -- score products on 8-bit rows: S[i][j] = sum over 128-dim blocks b of
// 2^(eq[i][b] + er[j][b]) * sum_k q[i][k] r[j][k], for one group of all rows and queries or for
// many groups of different sizes (each group's queries against its own rows).
//
// Tensor cores.  tcgen05 block scaling (kind::mxf8f6f4) multiplies e4m3 operands and applies the
// two power-of-two scales inside the instruction, for every 32 elements of K; a block of 128 is four
// instructions with the same scales.  The whole sum over K stays in the fp32 accumulator in TMEM,
// and no scale passes through the epilogue.  (With arbitrary fp32 scales each 128-element partial
// sum would have to be read from TMEM and multiplied in the FP32 pipe, which takes as long as the
// MMAs themselves.)
//
// Tiling.  2-CTA clusters (cta_group::2), up to 256 stored rows x up to 224 queries.  The stored rows
// are the MMA's M operand, so a TMEM lane holds one stored row and an epilogue warp has 32 consecutive
// results of each query, which it stores as they are: 32 lanes, 4 (or 2) bytes each.  (16 bytes a
// lane, brought together by shuffles or through shared memory, or TMA stores from there, were
// slower: 400 MB of fp32 results 115, 90 and 89 us against 85; 200 MB of bf16 84, 68 and 91 against
// 50.)  The queries are its N operand, any multiple of 32, so few queries cost few MMA cycles and the
// kernel then streams the stored rows at HBM speed (one query x 2M x 768: 7.0 TB/s); each CTA stages
// its half of the rows and of the queries of a 128-byte K chunk by TMA (128-byte swizzle).  224 and
// not 256 queries: two accumulators take 448 of the 512 TMEM columns and leave 60 for a ring of five
// scale slots.  At 8192 x 65536 x 1024 with bf16 results the tensor pipe is busy 81 % of a lone call
// (434 us, 2.5 PFLOP/s); back to back the card's power limit holds it to 2.0.
//
// Scales.  A slot holds the scale words of four K chunks (512 dimensions): 128 words for the CTA's
// rows and up to 256 for the queries.  A stored row's scale bytes are consecutive, so a 32-bit load
// gives four chunks' exponents, which go to TMEM as they are (the descriptor's scale id picks the
// byte).  Three warps copy them to shared memory (cp.async), a fourth hands a slot that has landed
// to the MMA thread, which copies it to TMEM (tcgen05.cp) in the tensor core's own order ahead of
// its MMAs.  (Stored from registers with tcgen05.st, or handed over with a plain release at cluster
// scope, a slot took 1,400-2,000 cycles, more than its MMAs: 2M x 768, one query, 256 -> 349 us.  The
// second CTA's slots are released by the completion of an asynchronous store instead, which costs
// nothing that could be measured.)
//
// Tiles.  Clusters take tiles from a counter where there are many: with large results the SMs' shares of
// the write bandwidth differ (the slowest unit of 1000 x 100k x 128 in fixed turns took 87 us with the
// median at 67).  One warp of the leader finds the next tile, with groups by looking at 128 groups'
// offsets at once, and sends its description to every role of both CTAs; a cluster's first tile waits
// for nobody.
//
// Few float queries.  Up to 64 queries of 128 blocks in all are quantised by each cluster for itself, into
// shared memory in the MMA's layout, where they stay for all its tiles: one launch and no scratch
// (when it came, one query x 10k x 768: 10.8 -> 8.2 us a call; x 100k: 20.7 -> 18.5; 37 x 5,003 x 300:
// 10.8 -> 10.2; x 100k is 19.2 since the CTAs meet before they allocate).
//
// Warps: 0 rows by TMA, 1 TMEM and (leader CTA) MMA, 2 row scales, 3-4 query scales, 5 hand-over of
// scales, 6 queries by TMA, 7 (leader CTA) tiles, 8-15 epilogue (two per TMEM lane quarter, taking
// 32-query groups in turn).  Every wait is bounded; on expiry the error word is set, the roles unwind
// and TMEM is released.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>

#include "../../include/vx.h"
#include "fp8.h"
#include "fp8_encode.cuh"
#include "fp8_groups.cuh"
#include "sm100.cuh"

namespace vx {
namespace {

using namespace sm100;

constexpr int kThreads = 512;
constexpr int kTmemCols = 512;
constexpr int kRowBytes = 128 * 128;  // a CTA's stored-row operand per stage
constexpr int kScaleSlots = 5;
constexpr int kSlotCols = 12;
constexpr int kSlotBytes = 1536;  // 128 row words, then up to 256 query words
constexpr uint32_t kScaleBase = 2 * kFp8MaxWidth;
constexpr size_t kMaxSmem = 232448;
constexpr int kMaxResident = 64 << 10;  // bytes of a CTA's resident queries
constexpr size_t kTailBytes = kScaleSlots * kSlotBytes + 1024;  // scale slots, barriers, tiles
constexpr int kMaxStages = 12;
constexpr int kTileSlots = 8;  // most tiles on their way

static_assert(2 * kMaxStages + 3 * kScaleSlots + 4 + 2 * kTileSlots + 2 <= 64, "barriers");
static_assert(kScaleBase + kScaleSlots * kSlotCols <= kTmemCols, "TMEM columns");

__host__ __device__ constexpr size_t stage_bytes(int width) { return kRowBytes + (size_t)width / 2 * 128; }

using Tile = Fp8Tile;

// Tile (rt, qt) of an ungrouped product; all load queries by boxes of half the width.
__device__ __forceinline__ Tile tile_at(const Fp8ScoreArgs& a, uint32_t rt, uint32_t qt) {
  Tile x;
  x.row = x.col = rt * (uint32_t)a.tile_rows;
  x.query = qt * (uint32_t)a.width;
  const int64_t rows = a.nrows - x.row, queries = a.nq - x.query;
  x.rows = rows < a.tile_rows ? (int)rows : a.tile_rows;
  x.queries = queries < a.width ? (int)queries : a.width;
  x.width = a.width;
  x.half = a.tile_rows >> 1;
  return x;
}

// Finds tiles by number, in ascending order, with a whole warp.  One group: tile p is (row tile
// p / query_tiles, query tile p % query_tiles).
struct Finder {
  const Fp8ScoreArgs& a;
  Fp8Group g;
  int64_t group, first, tiles;  // current group, the tiles before it, all tiles
  __device__ __forceinline__ explicit Finder(const Fp8ScoreArgs& args) : a(args), group(-1), first(0) {
    tiles = a.groups.row_off ? a.groups.tile_off[a.groups.groups] : a.tiles;
  }
  static __device__ __forceinline__ int64_t divide(int64_t x, int64_t by) {
    return ((uint64_t)x | (uint64_t)by) >> 32 ? x / by : (int64_t)((uint32_t)x / (uint32_t)by);
  }
  __device__ __forceinline__ Tile find(int64_t p) {
    const int lane = threadIdx.x & 31;
    Tile x{0, 0, 0, 0, 0, 0, 0};
    if (!a.groups.row_off) {
      if (p >= tiles) return x;
      const int64_t rt = divide(p, a.query_tiles);
      return tile_at(a, (uint32_t)rt, (uint32_t)(p - rt * a.query_tiles));
    }
    const int64_t* off = a.groups.tile_off;
    int64_t lo = group < 0 ? 0 : group, hi = a.groups.groups;  // off[lo] <= p < off[hi]
    // usually within the next 128 groups, whose offsets are looked at together; else 32 places of the
    // rest at a time
    int k = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int64_t at = lo + 1 + i * 32 + lane;
      k += __popc(__ballot_sync(0xFFFFFFFFu, at < hi && off[at] <= p));
    }
    lo += k;
    if (k < 128) hi = lo + 1;
    while (hi - lo > 1) {
      const int64_t by = (hi - lo + 31) >> 5;
      const int64_t at = lo + by * (lane + 1);
      k = __popc(__ballot_sync(0xFFFFFFFFu, at < hi && off[at] <= p));
      lo += by * k;
      if (lo + by < hi) hi = lo + by;
    }
    if (p >= tiles) return x;
    if (lo != group) {
      group = lo;
      first = off[lo];
      g = fp8_group(a.groups.bounds[lo]);
    }
    return fp8_group_tile(g, p - first);
  }
};

template <int kType>
struct Out;
template <>
struct Out<VX_F32> {
  using T = float;
  static __device__ __forceinline__ T of(uint32_t v) { return __uint_as_float(v); }
};
template <>
struct Out<VX_F16> {
  using T = __half;
  static __device__ __forceinline__ T of(uint32_t v) { return __float2half_rn(__uint_as_float(v)); }
};
template <>
struct Out<VX_BF16> {
  using T = __nv_bfloat16;
  static __device__ __forceinline__ T of(uint32_t v) { return __float2bfloat16_rn(__uint_as_float(v)); }
};

// Shared memory of resident queries: this CTA's half of the codes, chunk by chunk with 128-byte swizzle,
// and every query's scale words as scale slots have them.
__host__ __device__ __forceinline__ uint32_t resident_codes(const Fp8ScoreArgs& a) {
  return (uint32_t)(a.width / 2 * 128 * a.kchunks);
}
__host__ __device__ __forceinline__ uint32_t resident_words(const Fp8ScoreArgs& a) {
  return (uint32_t)((a.kchunks + 3) / 4 * 512);
}

// Quantises the queries, by the eight epilogue warps: every query's scales and this CTA's half of the
// codes.  Places past the last query keep what they hold: they reach only columns that are not stored.
template <class T>
__device__ __forceinline__ void encode_resident(const Fp8ScoreArgs& a, uint8_t* codes, uint8_t* words, uint32_t rank) {
  constexpr int kWords = (int)sizeof(T);  // of a piece of 4
  const int part = threadIdx.x & 7, group = ((int)threadIdx.x - 256) >> 3;
  const int blocks = (int)a.nq * a.kchunks, half = a.width >> 1;
  const bool vec = ((uintptr_t)a.queries | (uintptr_t)(a.query_stride * (int64_t)sizeof(T))) % (4 * sizeof(T)) == 0;
  uint32_t r[4][4 * kWords];
#pragma unroll
  for (int j = 0; j < 4; j++) {  // at most 128 blocks: all on their way at once
    const int block = j * 32 + group;
    if (block >= blocks) continue;
    const int q = block / a.kchunks, k = block % a.kchunks * kFp8Block;
    const T* x = (const T*)a.queries + q * a.query_stride;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int at = k + (i * 8 + part) * 4;
      if (vec) load_piece<T, 4, true>(x, at, a.dim, r[j] + i * kWords);
      else load_piece<T, 4, false>(x, at, a.dim, r[j] + i * kWords);
    }
  }
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const int block = j * 32 + group;
    uint32_t m = block < blocks ? largest<T>(r[j]) : 0u;
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
    if (block >= blocks) continue;
    const int q = block / a.kchunks, kc = block % a.kchunks;
    const int b = scale_byte(m);
    if (part == 0) words[kc / 4 * 512 + (q & 31) * 16 + (q >> 5) * 4 + (kc & 3)] = (uint8_t)b;
    const int row = q - (int)rank * half;
    if (row < 0 || row >= half) continue;
    uint8_t* to = codes + (kc * half + row) * 128;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int at = (i * 8 + part) * 4;
      *(uint32_t*)(to + (((at >> 4) ^ (row & 7)) << 4 | (at & 15))) = four_codes<T>(r[j] + i * kWords, 0, b);
    }
  }
}

template <int kType, bool kResident>
__global__ void __launch_bounds__(kThreads, 1)
    fp8_scores_kernel(const __grid_constant__ Fp8Maps maps, const __grid_constant__ Fp8ScoreArgs a) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* stages = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  const int n_stages = a.stages;
  const uint32_t stage_size = (uint32_t)a.stage_bytes;
  uint8_t* resident = stages + n_stages * stage_size;  // queries quantised here: codes, then scale words
  uint8_t* resident_scales = resident + (kResident ? resident_codes(a) : 0);
  uint8_t* slots = resident_scales + (kResident ? resident_words(a) : 0);
  uint64_t* full = (uint64_t*)(slots + kScaleSlots * kSlotBytes);
  uint64_t* empty = full + kMaxStages;
  uint64_t* landed = empty + kMaxStages;
  uint64_t* sfull = landed + kScaleSlots;
  uint64_t* sempty = sfull + kScaleSlots;
  uint64_t* tfull = sempty + kScaleSlots;
  uint64_t* tempty = tfull + 2;
  uint64_t* nfull = tempty + 2;
  uint64_t* nempty = nfull + kTileSlots;
  uint64_t* drained = nempty + kTileSlots;
  uint64_t* encoded = drained + 1;
  uint64_t* tile_slots = full + 64;  // 16-byte aligned
  uint32_t* tmem_slot = (uint32_t*)(tile_slots + 2 * kTileSlots);
  volatile int* abort_flag = (volatile int*)(tmem_slot + 1);

  const int warp = __shfl_sync(0xFFFFFFFFu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  cluster_arrive();
  const int64_t unit = blockIdx.x >> 1, units = gridDim.x >> 1;
  if (warp == 0 && lane < 2 && (lane == 0 || !kResident)) prefetch_tmap(lane == 0 ? &maps.rows[0] : &maps.queries[0]);

  if (threadIdx.x == 0) {
    for (int s = 0; s < n_stages; s++) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < kScaleSlots; s++) {
      mbar_init(&landed[s], kResident ? 32 : 96);  // the lanes of the loading warps
      mbar_init(&sfull[s], 2);    // each CTA's hand-over
      mbar_init(&sempty[s], 1);
    }
    for (int b = 0; b < 2; b++) {
      mbar_init(&tfull[b], 1);
      mbar_init(&tempty[b], 16);  // eight epilogue warps of each CTA
    }
    for (int s = 0; s < kTileSlots; s++) {
      mbar_init(&nfull[s], 1);    // the leader's tile warp
      mbar_init(&nempty[s], 16);  // the epilogue warps: a tile that is stored has gone through every role
    }
    mbar_init(drained, 1);
    mbar_init(encoded, 16);  // the epilogue warps of both CTAs
    *abort_flag = 0;
    fence_mbar_init();
  }
  // A pair's tensor memory is allocated by both CTAs together, so not before both have started: an
  // allocation that one began alone, on a busy device, could wait for good.
  __syncwarp();
  cluster_wait();
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, kTmemCols);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncwarp();
  cluster_sync();  // both CTAs' barriers are initialised before any remote arrive
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  // The launch before this one wrote the encoded queries, the groups' tile counts and the counter of
  // tiles: every role waits for it before it needs them, and before a bounded wait that would take it
  // in.  Without groups, stored rows and their scales are loaded without it, as far as there is room; that
  // helps after a small preparation only, since a cluster starts when one that fills the device has left
  // two SMs free.
  const bool grouped = a.groups.row_off != nullptr;
  bool waited = !a.wait_first;
  auto wait_for_prep = [&]() {
    if (!waited) asm volatile("griddepcontrol.wait;" ::: "memory");
    waited = true;
  };

  auto give_up = [&]() {
    *abort_flag = 1;
    record_error(a.err, kDevWaitTimeout);
  };
  // Shared memory of this CTA that the pair's tensor cores may read, announced to the leader's MMA thread:
  // released and acquired at cluster scope.
  const uint32_t leader_bars = mapa_shared(smem_addr(full), 0), nothing = mapa_shared(smem_addr(tmem_slot + 2), 0);
  auto announce = [&](uint64_t* bar) {
    if (leader) mbar_arrive(bar);
    else mbar_arrive_cluster_async(leader_bars + (uint32_t)((uint8_t*)bar - (uint8_t*)full), nothing);
  };
  // Each role takes the tiles in order; false: no more, or given up.  A cluster's first tile is the one of
  // its number: without groups known at once, with groups one of those that the launch before this one
  // left.
  int nslot = 0;
  uint32_t nphase = 0;
  bool first_tile = true;
  const bool only_tile = !grouped && a.tiles <= units;
  bool ended = false;
  auto next_tile = [&](Tile& t) {
    if (first_tile) {
      first_tile = false;
      if (grouped) {
        wait_for_prep();
        const ulonglong2 v = a.groups.first[unit];
        t = unpack_tile(v.x, v.y);
        if (t.width == 0) ended = true;
        return t.width != 0;
      }
      const uint32_t rt = (uint32_t)unit / (uint32_t)a.query_tiles, qt = (uint32_t)unit - rt * (uint32_t)a.query_tiles;
      t = tile_at(a, rt, qt);
      return true;
    }
    if (only_tile || ended) return false;
    wait_for_prep();
    if (*abort_flag || !mbar_wait<true>(&nfull[nslot], nphase, a.timeout_ns, abort_flag)) {
      give_up();
      return false;
    }
    const volatile uint64_t* v = tile_slots + 2 * nslot;
    t = unpack_tile(v[0], v[1]);
    if (++nslot == a.tile_slots) {
      nslot = 0;
      nphase ^= 1u;
    }
    return t.width != 0;
  };

  if (warp == 0 || warp == 6) {
    // ---------------- TMA: warp 0 the stored rows, warp 6 the queries
    if ((warp == 0 || !kResident) && elect_one()) {
      const bool rows = warp == 0;
      const CUtensorMap* map = rows ? maps.rows : maps.queries;
      // query tiles are read again for every row tile
      const uint64_t policy = rows ? policy_evict_normal() : policy_evict_last();
      const uint32_t full0 = mapa_shared(smem_addr(&full[0]), 0);
      int stage = 0;
      uint32_t phase = 0;
      if (!rows) wait_for_prep();
      int room = n_stages;
      Tile t;
      while (next_tile(t)) {
        const int count = rows ? t.half : t.width >> 1;  // operand rows of this CTA
        const int32_t y0 = (int32_t)(rows ? t.row : t.query) + (int)rank * count;
        for (int kc = 0; kc < a.kchunks; kc++) {
          if (room-- == 0) wait_for_prep();
          if (!mbar_wait(&empty[stage], phase ^ 1u, a.timeout_ns, abort_flag)) {
            give_up();
            break;
          }
          uint8_t* s = stages + stage * stage_size + (rows ? 0 : kRowBytes);
          const uint32_t bar = full0 + (uint32_t)(stage * 8);
          if (rows && leader)
            mbar_arrive_expect_tx(&full[stage], 2u * 128u * (uint32_t)(count + (kResident ? 0 : t.width >> 1)));
          if (!grouped) {
            tma_load_2d_pair(s, map, bar, kc * 128, y0, policy);
          } else {
            int32_t y = y0;
#pragma unroll
            for (int i = 0; i < 4; i++) {  // boxes of 128, 64, 32 and 16 rows
              const int box = 128 >> i;
              if (count & box) {
                tma_load_2d_pair(s, map + i, bar, kc * 128, y, policy);
                s += box * 128;
                y += box;
              }
            }
          }
          if (++stage == n_stages) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      if (rows) {
        // tcgen05.commit's arrivals come by themselves, and the cluster's barrier does not wait for them: this
        // CTA stays for the last hand-back of each stage (the epilogue takes longer)
        wait_for_prep();
        for (int i = 0; i < n_stages; i++) {
          mbar_settle(&empty[stage], phase ^ 1u);
          if (++stage == n_stages) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      if (*abort_flag) {
        // Let the loads already issued land before the cluster's shared memory is released.
        const uint64_t until = globaltimer_ns() + 2000000ull;
        while (globaltimer_ns() < until) {
        }
      }
    }
  } else if (warp == 1) {
    if (leader && elect_one()) {
      int stage = 0, slot = 0;
      uint32_t phase = 0, sphase = 0;
      const uint64_t desc0 = sw128_kmajor_desc(smem_addr(stages));
      const uint32_t desc_lo0 = (uint32_t)desc0, desc_hi = (uint32_t)(desc0 >> 32);
      const uint32_t stage_step = stage_size >> 4;
      uint32_t desc_lo = desc_lo0;
      // the queries' operand: behind the rows' in each stage, or resident
      const uint32_t resident_lo = (uint32_t)sw128_kmajor_desc(smem_addr(resident));
      const uint32_t resident_step = (uint32_t)(a.width / 2 * 128) >> 4;
      const uint64_t resident_ds = scale_block_desc(smem_addr(resident_scales));
      wait_for_prep();
      if (kResident && !mbar_wait<true>(encoded, 0, a.timeout_ns, abort_flag)) give_up();
      Tile t;
      for (uint32_t li = 0; next_tile(t); li++) {
        const int acc = (int)(li & 1);
        if (!mbar_wait(&tempty[acc], ((li >> 1) & 1u) ^ 1u, a.timeout_ns, abort_flag)) {
          give_up();
          break;
        }
        tc_fence_after();
        const uint32_t d = tmem_base + (uint32_t)(acc * kFp8MaxWidth);
        const uint32_t idesc0 = idesc_mxf8(256, t.width, 0);
        bool ok = true;
        for (int kc = 0; kc < a.kchunks && ok; kc += 4) {  // a scale slot's chunks
          if (!mbar_wait<true>(&sfull[slot], sphase, a.timeout_ns, abort_flag)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t scales = tmem_base + kScaleBase + (uint32_t)(slot * kSlotCols);
          const uint64_t ds = scale_block_desc(smem_addr(slots) + (uint32_t)(slot * kSlotBytes));
          tmem_cp_scales_pair(scales, ds);
          tmem_cp_scales_pair(scales + 4, kResident ? resident_ds + (uint64_t)(kc * (512 / 4) >> 4) : ds + (512 >> 4));
          if (t.width > 128) tmem_cp_scales_pair(scales + 8, ds + (1024 >> 4));
#pragma unroll
          for (int sub = 0; sub < 4; sub++) {
            if (kc + sub >= a.kchunks) break;
            if (!mbar_wait<true>(&full[stage], phase, a.timeout_ns, abort_flag)) {
              ok = false;
              break;
            }
            tc_fence_after();
            const uint32_t b_lo = kResident ? resident_lo + (uint32_t)(kc + sub) * resident_step : desc_lo + (kRowBytes >> 4);
            mma_mxf8_pair_chunk(d, desc_lo, b_lo, desc_hi, idesc0 | sub << 4 | (uint32_t)sub << 29,
                                scales, scales + 4, (uint32_t)(kc + sub));
            mma_commit_pair_mc(&empty[stage], (uint16_t)0x3);
            desc_lo += stage_step;
            if (++stage == n_stages) {
              stage = 0;
              phase ^= 1u;
              desc_lo = desc_lo0;
            }
          }
          mma_commit_pair_mc(&sempty[slot], (uint16_t)0x3);
          if (++slot == kScaleSlots) {
            slot = 0;
            sphase ^= 1u;
          }
        }
        if (!ok) give_up();
        if (!ok) break;
        mma_commit_pair_mc(&tfull[acc], (uint16_t)0x3);
      }
      // MMAs in flight end before their TMEM and shared memory are released, whoever else has given up
      mma_commit_pair_mc(drained, (uint16_t)0x1);
      mbar_settle(drained, 0);
    }
  } else if (warp >= 8) {
    // ---------------- epilogue: one stored row per lane, one query per TMEM column
    using T = typename Out<kType>::T;
    const int quarter = warp & 3;
    const int first = (warp >> 2 & 1) * 32;  // this warp's 32-query groups: every other one
    const uint32_t tempty0 = mapa_shared(smem_addr(&tempty[0]), 0), nempty0 = mapa_shared(smem_addr(&nempty[0]), 0);
    wait_for_prep();
    if constexpr (kResident) {
      if (a.query_type == VX_F32) encode_resident<float>(a, resident, resident_scales, rank);
      else if (a.query_type == VX_F16) encode_resident<__half>(a, resident, resident_scales, rank);
      else encode_resident<__nv_bfloat16>(a, resident, resident_scales, rank);
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) announce(encoded);
    }
    for (uint32_t li = 0;; li++) {
      Tile t;
      const bool sent = !first_tile;  // by the tile warp, in slot nslot
      const uint32_t nempty_bar = nempty0 + (uint32_t)(nslot * 8);
      if (!__all_sync(0xFFFFFFFFu, next_tile(t))) break;
      const int acc = (int)(li & 1);
      // this warp's rows of the tile
      int rows = t.rows - (int)rank * t.half;
      rows = (rows < t.half ? rows : t.half) - quarter * 32;
      T* o = (T*)a.out + (int64_t)(t.query + first) * a.ldo + t.col + (int)rank * t.half + quarter * 32;
      const bool ok = !*abort_flag && mbar_wait(&tfull[acc], (li >> 1) & 1u, a.timeout_ns, abort_flag);
      if (!__all_sync(0xFFFFFFFFu, ok)) {
        if (lane == 0) give_up();
        break;
      }
      tc_fence_after();
      const uint32_t taddr = tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(acc * kFp8MaxWidth);
      for (int c0 = first; c0 < t.queries; c0 += 64) {
        uint32_t v[32];
        __syncwarp();
        tmem_ld_32x32b_x32(taddr + (uint32_t)c0, v);
        tmem_ld_wait_v(v);
        const int lim = t.queries - c0;
        if (lane < rows) {
          T* at = o + lane;
          if (lim >= 32) {
#pragma unroll
            for (int j = 0; j < 32; j++) {
              *at = Out<kType>::of(v[j]);
              at += a.ldo;
            }
          } else {
#pragma unroll
            for (int j = 0; j < 32; j++) {
              if (j < lim) *at = Out<kType>::of(v[j]);
              at += a.ldo;
            }
          }
        }
        o += 64 * a.ldo;
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive_cluster_relaxed(tempty0 + (uint32_t)(acc * 8));  // the leader issues the next MMA
        if (sent) mbar_arrive_cluster_relaxed(nempty_bar);
      }
    }
  } else if (warp < 5) {
    // ---------------- scales: warp 2 the CTA's 128 rows, warps 3 and 4 the tile's queries 0-127 and
    // 128-223, lane l the words of rows l, 32 + l, 64 + l and 96 + l (the order TMEM has them in)
    const int part = warp - 2;
    const uint8_t* src = part == 0 ? a.row_scales : a.query_scales;
    const int64_t limit = part == 0 ? a.nrows : a.nq;
    const int slots_per_tile = (a.kchunks + 3) >> 2;
    int slot = 0;
    uint32_t sphase = 0;
    if (part > 0) wait_for_prep();
    int room = kScaleSlots;
    Tile t;
    while ((part == 0 || !kResident) && __all_sync(0xFFFFFFFFu, next_tile(t))) {
      const int64_t first = (part == 0 ? t.row + rank * (uint32_t)t.half : t.query + (uint32_t)(part - 1) * 128u) + lane;
      const int count = part == 0 ? t.half : t.width - (part - 1) * 128;
      const uint8_t* at[4];
      bool in[4];
#pragma unroll
      for (int c = 0; c < 4; c++) {
        const int64_t row = first + c * 32;
        in[c] = c * 32 + lane < count && row < limit;
        at[c] = in[c] ? src + row * (4 * (int64_t)a.scale_words) : src;
      }
      bool ok = true;
      for (int w = 0; w < slots_per_tile; w++) {
        if (room-- == 0) wait_for_prep();
        ok = !*abort_flag && mbar_wait(&sempty[slot], sphase ^ 1u, a.timeout_ns, abort_flag);
        ok = __all_sync(0xFFFFFFFFu, ok);
        if (!ok) {
          if (lane == 0) give_up();
          break;
        }
        const uint32_t dst = smem_addr(slots + slot * kSlotBytes + part * 512 + lane * 16);
#pragma unroll
        for (int c = 0; c < 4; c++) cp_async_4(dst + 4 * c, at[c] + 4 * w, in[c]);
        cp_async_arrive(&landed[slot]);
        if (++slot == kScaleSlots) {
          slot = 0;
          sphase ^= 1u;
        }
      }
      if (!ok) break;
    }
    if (part == 0) {  // the last hand-back of each slot, as of the stages
      wait_for_prep();
      for (int i = 0; i < kScaleSlots; i++) {
        mbar_settle(&sempty[slot], sphase ^ 1u);
        if (++slot == kScaleSlots) {
          slot = 0;
          sphase ^= 1u;
        }
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  } else if (warp == 5) {
    // ---------------- slots that have landed go to the leader's MMA thread
    if (elect_one()) {
      wait_for_prep();
      int slot = 0;
      uint32_t sphase = 0;
      Tile t;
      while (next_tile(t)) {
        for (int w = (a.kchunks + 3) >> 2; w > 0; w--) {
          if (!mbar_wait(&landed[slot], sphase, a.timeout_ns, abort_flag)) {
            give_up();
            break;
          }
          fence_proxy_async();
          announce(&sfull[slot]);
          if (++slot == kScaleSlots) {
            slot = 0;
            sphase ^= 1u;
          }
        }
      }
    }
  } else if (leader && !only_tile) {
    // ---------------- warp 7: tiles, to the same place in both CTAs
    if (grouped || a.next_tile) wait_for_prep();
    const uint32_t at[2] = {mapa_shared(smem_addr(tile_slots), 0), mapa_shared(smem_addr(tile_slots), 1)};
    const uint32_t bar[2] = {mapa_shared(smem_addr(nfull), 0), mapa_shared(smem_addr(nfull), 1)};
    Tile own;
    if (next_tile(own)) {  // a cluster without a first tile has no role that would wait for a second
      Finder finder(a);
      // The cluster's first tile is known to every role.  With groups the number after the one in hand is on
      // its way while the group is looked up.
      unsigned long long taken = 0;
      auto take = [&]() {
        if (a.next_tile && lane == 0) taken = atomicAdd(a.next_tile, 1ull);
      };
      int64_t p = unit;
      auto advance = [&]() {
        if (!grouped) take();
        p = a.next_tile ? units + (int64_t)__shfl_sync(0xFFFFFFFFu, taken, 0) : p + units;
        if (grouped) take();
      };
      if (grouped) take();
      advance();
      for (int width = 1; width != 0; advance()) {
        const Tile t = finder.find(p);
        width = t.width;
        const bool ok = mbar_wait(&nempty[nslot], nphase ^ 1u, a.timeout_ns, abort_flag);
        if (!__all_sync(0xFFFFFFFFu, ok)) {
          if (lane == 0) give_up();
          break;
        }
        const ulonglong2 v = pack_tile(t);
        if (lane < 2) store_cluster_16(at[lane] + (uint32_t)nslot * 16u, bar[lane] + (uint32_t)nslot * 8u, v.x, v.y);
        if (++nslot == a.tile_slots) {
          nslot = 0;
          nphase ^= 1u;
        }
      }
    }
  }

  wait_for_prep();
  tc_fence_before();
  cluster_sync();  // the pair's MMAs, loads and epilogues are done with TMEM and shared memory
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, kTmemCols);
    __syncwarp();
  }
  // Nor does the cluster's barrier wait for asynchronous stores (tiles).  A role that ends in order has seen
  // them all; a CTA that gave up stays for what the other may have sent it until then.
  if (warp == 7 && *abort_flag) {
    const uint64_t until = globaltimer_ns() + 2000000ull;
    while (globaltimer_ns() < until) {
    }
    __syncwarp();
  }
  cluster_meet();  // a pair frees its tensor memory together: neither CTA ends before both have
}

template <int kType, bool kResident>
cudaError_t launch_typed(const Fp8Maps& maps, const Fp8ScoreArgs& a, int units, size_t smem, bool after_prep,
                         cudaStream_t st) {
  auto kern = fp8_scores_kernel<kType, kResident>;
  static std::atomic<uint64_t> sized{0};  // bit d: done for device d
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return e;
  if (device >= 64 || !((sized.load() >> device) & 1)) {
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMaxSmem);
    if (e != cudaSuccess) return e;
    if (device < 64) sized.fetch_or(1ull << device);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(2 * units));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = after_prep ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kern, maps, a);
}

template <int kType>
cudaError_t launch_out(const Fp8Maps& maps, const Fp8ScoreArgs& a, int units, size_t smem, bool after_prep,
                       cudaStream_t st) {
  return a.queries ? launch_typed<kType, true>(maps, a, units, smem, after_prep, st)
                   : launch_typed<kType, false>(maps, a, units, smem, after_prep, st);
}

}  // namespace

Fp8Tiling fp8_tiling(int64_t nrows, int64_t nq, int64_t groups, int num_sms) {
  Fp8Tiling t{};
  t.tile_rows = kFp8TileRows;
  t.query_tiles = (int)((nq + kFp8MaxWidth - 1) / kFp8MaxWidth);
  if (groups > 0) {  // the widest tile any group can have; its rows go by the group
    t.width = (int)(nq < kFp8MaxWidth ? (nq + 31) / 32 * 32 : kFp8MaxWidth);
    return t;
  }
  // equal tiles of at most kFp8MaxWidth queries
  t.width = (int)(((nq + t.query_tiles - 1) / t.query_tiles + 31) / 32 * 32);
  t.tiles = (nrows + t.tile_rows - 1) / t.tile_rows * t.query_tiles;
  // Few queries and few tiles per cluster: the stored rows are what takes the time, so each cluster's
  // turns get equal shares of them.
  const int64_t units = num_sms / 2, turns = (t.tiles + units - 1) / units;
  if (t.width <= 64 && turns > 1 && turns <= 8) {
    const int64_t share = (nrows + turns * units - 1) / (turns * units);
    t.tile_rows = (int)((share + 7) / 8 * 8);
    t.tiles = (nrows + t.tile_rows - 1) / t.tile_rows;
  }
  return t;
}

bool fp8_resident(int64_t nq, int dim, const Fp8Tiling& t) {
  return t.query_tiles == 1 && t.width <= 64 && nq * fp8_blocks(dim) <= 128 &&
         t.width / 2 * fp8_code_pitch(dim) <= kMaxResident;
}

cudaError_t launch_fp8_scores(const Fp8Maps& maps, const Fp8ScoreArgs& args, int out_type, int num_sms, bool after_prep,
                              cudaStream_t st) {
  Fp8ScoreArgs a = args;
  int64_t units = num_sms / 2;
  if (!a.groups.row_off && units > a.tiles) units = a.tiles;
  if (units < 1) units = 1;
  const size_t tail = kTailBytes + (a.queries ? resident_codes(a) + resident_words(a) : 0);
  a.stage_bytes = (int)(a.queries ? kRowBytes : stage_bytes(a.width));
  a.stages = (int)((kMaxSmem - 1024 - tail) / a.stage_bytes);
  if (a.stages > kMaxStages) a.stages = kMaxStages;
  if (tail + 1024 + 4 * (size_t)a.stage_bytes > kMaxSmem) return cudaErrorInvalidValue;
  // Tiles on their way in a cluster: one multiplied, one stored, and those that the stages can hold
  // beyond (fewer leave the end of the work better shared out).
  a.tile_slots = 2 + (a.stages + a.kchunks - 1) / a.kchunks;
  if (a.tile_slots > kTileSlots) a.tile_slots = kTileSlots;
  a.wait_first = after_prep;
  const size_t smem = 1024 + (size_t)a.stages * a.stage_bytes + tail;
  switch (out_type) {
    case VX_F32: return launch_out<VX_F32>(maps, a, (int)units, smem, after_prep, st);
    case VX_F16: return launch_out<VX_F16>(maps, a, (int)units, smem, after_prep, st);
    case VX_BF16: return launch_out<VX_BF16>(maps, a, (int)units, smem, after_prep, st);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace vx
