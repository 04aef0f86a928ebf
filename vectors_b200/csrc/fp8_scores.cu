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
// Tiling.  2-CTA clusters (cta_group::2), 256 stored rows x up to 224 queries.  The stored rows are
// the MMA's M operand, so a TMEM lane holds one stored row and an epilogue warp writes 32
// consecutive results of one query at a time: coalesced, with no transposition.  The queries are
// its N operand, any multiple of 32, so few queries cost few MMA cycles and the kernel then streams
// the stored rows at HBM speed; each CTA stages its 128 rows and half the queries of a 128-byte K
// chunk by TMA (128-byte swizzle).  224 and not 256 queries: two accumulators take 448 of the 512
// TMEM columns and leave 60 for a ring of five scale slots.
//
// Scales.  A slot holds the scale words of four K chunks (512 dimensions): 128 words for the CTA's
// rows and up to 256 for the queries.  A stored row's scale bytes are consecutive, so a 32-bit load
// gives four chunks' exponents, which go to TMEM as they are (the descriptor's scale id picks the
// byte).  Three warps copy them to shared memory (cp.async), a fourth hands a slot that has landed
// to the MMA thread, which copies it to TMEM (tcgen05.cp) in the tensor core's own order ahead of
// its MMAs.  (Stored from registers with tcgen05.st, or handed over with a release at cluster scope,
// a slot took 1,400-2,000 cycles, more than its MMAs.)
//
// Warps: 0 rows by TMA, 1 TMEM and (leader CTA) MMA, 2 row scales, 3-4 query scales, 5 hand-over of
// scales, 6 queries by TMA, 8-15 epilogue (two per TMEM lane quarter, taking 32-query groups in
// turn).  Every wait is bounded; on expiry the error word is set, the roles unwind and
// TMEM is released.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>

#include "../../include/vx.h"
#include "fp8.h"
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
constexpr size_t kTailBytes = kScaleSlots * kSlotBytes + 512;  // scale slots and barriers
constexpr int kMaxStages = 12;

static_assert(kScaleBase + kScaleSlots * kSlotCols <= kTmemCols, "TMEM columns");

__host__ __device__ constexpr size_t stage_bytes(int width) { return kRowBytes + (size_t)width / 2 * 128; }

// One tile: rows [row, row + rows) against queries [query, query + queries).
struct Tile {
  int64_t row, query;
  int64_t col;  // column of the first row's results
  int rows, queries;
  int width;    // MMA N: queries rounded up to 32
};

// The tiles of a work unit, in order, from number `p` of its range to before `end`.  One group: tile p
// is (row tile p / query_tiles, query tile p % query_tiles), and the clusters take tiles in turn, so
// that they work side by side (results of one query in neighbouring DRAM pages).  Several groups:
// each cluster takes a run of consecutive tiles, so that stepping from group to group stays cheap.
struct Walk {
  const Fp8ScoreArgs& a;
  Fp8Group g;
  int64_t p, end, step;
  int64_t group;   // current group (groups only)
  int64_t rt, qt;  // row and query tile within it
  int64_t step_rt, step_qt;
  __device__ __forceinline__ Walk(const Fp8ScoreArgs& args, int64_t unit, int64_t units) : a(args), group(0) {
    if (!a.groups.row_off) {
      g.row0 = g.query0 = 0;
      g.nrows = a.nrows;
      g.nqueries = a.nq;
      g.query_tiles = a.query_tiles;
      g.width = a.width;
      p = unit;
      end = a.tiles;
      step = units;
      rt = p / a.query_tiles;
      qt = p % a.query_tiles;
      step_rt = units / a.query_tiles;
      step_qt = units % a.query_tiles;
      return;
    }
    const int64_t total = a.groups.tile_off[a.groups.groups];
    p = total * unit / units;
    end = total * (unit + 1) / units;
    step = step_qt = 1;
    step_rt = rt = qt = 0;
    if (p >= end) return;
    int64_t lo = 0, hi = a.groups.groups;  // tile_off[lo] <= p < tile_off[hi]; 32 places tried at once
    while (hi - lo > 1) {
      const int64_t by = (hi - lo + 31) >> 5;
      const int64_t at = lo + by * ((threadIdx.x & 31) + 1);
      const int k = __popc(__ballot_sync(0xFFFFFFFFu, at < hi && a.groups.tile_off[at] <= p));
      lo += by * k;
      if (lo + by < hi) hi = lo + by;
    }
    group = lo;
    g = fp8_group(a.groups, lo);
    const int64_t t = p - a.groups.tile_off[lo];
    rt = t / (g.query_tiles > 0 ? g.query_tiles : 1);
    qt = t - rt * g.query_tiles;
  }
  __device__ __forceinline__ bool more() const { return p < end; }
  __device__ __forceinline__ int64_t count() const { return p < end ? (end - p + step - 1) / step : 0; }
  __device__ __forceinline__ void next() {
    p += step;
    qt += step_qt;
    rt += step_rt;
    if (qt >= g.query_tiles) {
      qt -= g.query_tiles;
      rt++;
    }
    if (a.groups.row_off && rt * 256 >= g.nrows && p < end) {  // on to the next group that has tiles
      do {
        if (group + 1 >= a.groups.groups) {  // only if the offsets changed during the call
          end = p;
          return;
        }
        group++;
        g = fp8_group(a.groups, group);
      } while (g.tiles == 0);
      rt = qt = 0;
    }
  }
  __device__ __forceinline__ Tile tile() const {
    Tile x;
    x.row = g.row0 + rt * 256;
    x.col = a.groups.row_off ? rt * 256 : x.row;
    const int64_t rl = g.nrows - rt * 256;
    x.rows = rl < 256 ? (int)rl : 256;
    x.query = g.query0 + qt * g.width;
    const int64_t ql = g.nqueries - qt * g.width;
    x.queries = ql < g.width ? (int)(ql < 0 ? 0 : ql) : g.width;
    // ungrouped tiles all load queries by boxes of half the width
    x.width = !a.groups.row_off ? a.width : x.queries > 0 ? (x.queries + 31) / 32 * 32 : 32;
    return x;
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

template <int kType>
__global__ void __launch_bounds__(kThreads, 1)
    fp8_scores_kernel(const __grid_constant__ Fp8Maps maps, const __grid_constant__ Fp8ScoreArgs a) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* stages = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  const int n_stages = a.stages;
  const size_t stage_size = stage_bytes(a.width);
  uint8_t* slots = stages + n_stages * stage_size;
  uint64_t* full = (uint64_t*)(slots + kScaleSlots * kSlotBytes);
  uint64_t* empty = full + kMaxStages;
  uint64_t* landed = empty + kMaxStages;
  uint64_t* sfull = landed + kScaleSlots;
  uint64_t* sempty = sfull + kScaleSlots;
  uint64_t* tfull = sempty + kScaleSlots;
  uint64_t* tempty = tfull + 2;
  uint64_t* drained = tempty + 2;
  uint32_t* tmem_slot = (uint32_t*)(drained + 1);
  volatile int* abort_flag = (volatile int*)(tmem_slot + 1);

  const int warp = __shfl_sync(0xFFFFFFFFu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const int64_t unit = blockIdx.x >> 1, units = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < n_stages; s++) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < kScaleSlots; s++) {
      mbar_init(&landed[s], 96);  // the lanes of the three loading warps
      mbar_init(&sfull[s], 2);    // each CTA's hand-over
      mbar_init(&sempty[s], 1);
    }
    for (int b = 0; b < 2; b++) {
      mbar_init(&tfull[b], 1);
      mbar_init(&tempty[b], 16);  // eight epilogue warps of each CTA
    }
    mbar_init(drained, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, kTmemCols);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  cluster_sync();  // both CTAs' barriers are initialised before any remote arrive
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  // The launch before this one wrote the encoded queries, the groups' tile counts or both.
  if (a.wait_first) asm volatile("griddepcontrol.wait;" ::: "memory");

  Walk walk(a, unit, units);
  const bool any = walk.more();

  auto give_up = [&]() {
    *abort_flag = 1;
    record_error(a.err, kDevWaitTimeout);
  };

  if (warp == 0 || warp == 6) {
    // ---------------- TMA: warp 0 the stored rows, warp 6 the queries
    if (any && elect_one()) {
      const bool rows = warp == 0;
      if (rows) prefetch_tmap(&maps.rows);
      else prefetch_tmap(&maps.queries[0]);
      // query tiles are read again for every row tile
      const uint64_t policy = rows ? policy_evict_normal() : policy_evict_last();
      const uint32_t full0 = mapa_shared(smem_addr(&full[0]), 0);
      int stage = 0;
      uint32_t phase = 0;
      for (; walk.more() && !*abort_flag; walk.next()) {
        const Tile t = walk.tile();
        const int half = t.width >> 1;  // query rows of this CTA
        const int32_t y0 = rows ? (int32_t)t.row + (int)rank * 128 : (int32_t)t.query + (int)rank * half;
        for (int kc = 0; kc < a.kchunks; kc++) {
          if (!mbar_wait(&empty[stage], phase ^ 1u, a.timeout_ns, abort_flag)) {
            give_up();
            break;
          }
          uint8_t* s = stages + stage * stage_size;
          const uint32_t bar = full0 + (uint32_t)(stage * 8);
          if (rows) {
            if (leader) mbar_arrive_expect_tx(&full[stage], 2u * (uint32_t)stage_bytes(t.width));
            tma_load_2d_pair(s, &maps.rows, bar, kc * 128, y0, policy);
          } else if (!a.groups.row_off) {
            tma_load_2d_pair(s + kRowBytes, &maps.queries[0], bar, kc * 128, y0, policy);
          } else {
            int32_t y = y0;
            s += kRowBytes;
#pragma unroll
            for (int i = 0; i < 3; i++) {  // the half's rows as boxes of 64, 32 and 16
              const int box = 64 >> i;
              if (half & box) {
                tma_load_2d_pair(s, &maps.queries[i], bar, kc * 128, y, policy);
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
      if (*abort_flag) {
        // Let the loads already issued land before the cluster's shared memory is released.
        const uint64_t until = globaltimer_ns() + 2000000ull;
        while (globaltimer_ns() < until) {
        }
      }
    }
  } else if (warp == 1) {
    if (leader && any && elect_one()) {
      int stage = 0, slot = 0;
      uint32_t phase = 0, sphase = 0;
      uint32_t li = 0;
      for (; walk.more() && !*abort_flag; walk.next(), li++) {
        const Tile t = walk.tile();
        const int acc = (int)(li & 1);
        if (!mbar_wait(&tempty[acc], ((li >> 1) & 1u) ^ 1u, a.timeout_ns, abort_flag)) {
          give_up();
          break;
        }
        tc_fence_after();
        const uint32_t d = tmem_base + (uint32_t)(acc * kFp8MaxWidth);
        const uint32_t idesc0 = idesc_mxf8(256, t.width, 0);
        bool ok = true;
        for (int kc = 0; kc < a.kchunks; kc++) {
          const int sub = kc & 3;
          const uint32_t scales = tmem_base + kScaleBase + (uint32_t)(slot * kSlotCols);
          if (sub == 0) {
            if (!mbar_wait(&sfull[slot], sphase, a.timeout_ns, abort_flag)) {
              ok = false;
              give_up();
              break;
            }
            tc_fence_after();
            const uint64_t ds = scale_block_desc(smem_addr(slots + slot * kSlotBytes));
            tmem_cp_scales_pair(scales, ds);
            tmem_cp_scales_pair(scales + 4, ds + (512 >> 4));
            if (t.width > 128) tmem_cp_scales_pair(scales + 8, ds + (1024 >> 4));
          }
          if (!mbar_wait(&full[stage], phase, a.timeout_ns, abort_flag)) {
            ok = false;
            give_up();
            break;
          }
          tc_fence_after();
          const uint32_t sa = smem_addr(stages + stage * stage_size);
          const uint64_t da = sw128_kmajor_desc(sa), db = sw128_kmajor_desc(sa + kRowBytes);
          const uint32_t idesc = idesc0 | ((uint32_t)sub << 4) | ((uint32_t)sub << 29);
#pragma unroll
          for (int kk = 0; kk < 4; kk++)
            mma_mxf8_pair(d, da + 2ull * kk, db + 2ull * kk, idesc, scales, scales + 4, (kc | kk) != 0 ? 1u : 0u);
          mma_commit_pair_mc(&empty[stage], (uint16_t)0x3);
          if (++stage == n_stages) {
            stage = 0;
            phase ^= 1u;
          }
          if (sub == 3 || kc + 1 == a.kchunks) {
            mma_commit_pair_mc(&sempty[slot], (uint16_t)0x3);
            if (++slot == kScaleSlots) {
              slot = 0;
              sphase ^= 1u;
            }
          }
        }
        if (!ok) break;
        mma_commit_pair_mc(&tfull[acc], (uint16_t)0x3);
      }
      if (*abort_flag) {  // MMAs in flight end before their TMEM and shared memory are released
        mma_commit_pair_mc(drained, (uint16_t)0x1);
        const uint64_t until = globaltimer_ns() + 2000000ull;
        while (!mbar_try_wait(drained, 0) && globaltimer_ns() < until) {
        }
      }
    }
  } else if (warp >= 8) {
    // ---------------- epilogue: one stored row per lane, one query per TMEM column
    using T = typename Out<kType>::T;
    const int quarter = warp & 3;
    const int first = (warp >> 2 & 1) * 32;  // this warp's 32-query groups: every other one
    const int my_row = (int)rank * 128 + quarter * 32 + lane;
    const uint32_t tempty0 = mapa_shared(smem_addr(&tempty[0]), 0);
    uint32_t li = 0;
    for (; walk.more(); walk.next(), li++) {
      const Tile t = walk.tile();
      const int acc = (int)(li & 1);
      const bool row_in = my_row < t.rows;
      T* o = (T*)a.out + (t.query + first) * a.ldo + t.col + my_row;
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
        if (row_in) {
          if (lim >= 32) {
#pragma unroll
            for (int j = 0; j < 32; j++) {
              *o = Out<kType>::of(v[j]);
              o += a.ldo;
            }
          } else {
#pragma unroll
            for (int j = 0; j < 32; j++) {
              if (j < lim) *o = Out<kType>::of(v[j]);
              o += a.ldo;
            }
          }
          o += 32 * a.ldo;
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster_relaxed(tempty0 + (uint32_t)(acc * 8));  // the leader issues the next MMA
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
    for (; walk.more(); walk.next()) {
      const Tile t = walk.tile();
      const int64_t first = (part == 0 ? t.row + (int)rank * 128 : t.query + (part - 1) * 128) + lane;
      const int count = part == 0 ? 128 : t.width - (part - 1) * 128;
      const uint8_t* at[4];
      bool in[4];
#pragma unroll
      for (int c = 0; c < 4; c++) {
        const int64_t row = first + c * 32;
        in[c] = c * 32 < count && row < limit;
        at[c] = in[c] ? src + row * (4 * (int64_t)a.scale_words) : src;
      }
      bool ok = true;
      for (int w = 0; w < slots_per_tile; w++) {
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
    asm volatile("cp.async.wait_all;" ::: "memory");
  } else if (warp == 5 && any && elect_one()) {
    // ---------------- slots that have landed go to the leader's MMA thread
    const uint32_t sfull0 = mapa_shared(smem_addr(&sfull[0]), 0);
    int slot = 0;
    uint32_t sphase = 0;
    for (int64_t left = walk.count() * ((a.kchunks + 3) >> 2); left > 0; left--) {
      if (*abort_flag || !mbar_wait(&landed[slot], sphase, a.timeout_ns, abort_flag)) {
        give_up();
        break;
      }
      fence_proxy_async();
      mbar_arrive_pair(sfull0 + (uint32_t)(slot * 8));
      if (++slot == kScaleSlots) {
        slot = 0;
        sphase ^= 1u;
      }
    }
  }

  tc_fence_before();
  cluster_sync();  // the pair's MMAs, loads and epilogues are done with TMEM and shared memory
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, kTmemCols);
  }
}

template <int kType>
cudaError_t launch_typed(const Fp8Maps& maps, const Fp8ScoreArgs& a, int units, size_t smem, bool after_prep,
                         cudaStream_t st) {
  auto kern = fp8_scores_kernel<kType>;
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

}  // namespace

cudaError_t launch_fp8_scores(const Fp8Maps& maps, const Fp8ScoreArgs& args, int out_type, int num_sms, bool after_prep,
                              cudaStream_t st) {
  Fp8ScoreArgs a = args;
  const int64_t qt = (a.nq + kFp8MaxWidth - 1) / kFp8MaxWidth;
  int64_t units = num_sms / 2;
  if (a.groups.row_off) {
    a.width = (int)(a.nq < kFp8MaxWidth ? (a.nq + 31) / 32 * 32 : kFp8MaxWidth);  // widest possible tile
  } else {
    a.query_tiles = (int)qt;
    a.width = fp8_query_width(a.nq);
    a.tiles = (a.nrows + 255) / 256 * qt;
    if (units > a.tiles) units = a.tiles;
  }
  if (units < 1) units = 1;
  a.stages = (int)((kMaxSmem - 1024 - kTailBytes) / stage_bytes(a.width));
  if (a.stages > kMaxStages) a.stages = kMaxStages;
  a.wait_first = after_prep;
  const size_t smem = 1024 + a.stages * stage_bytes(a.width) + kTailBytes;
  switch (out_type) {
    case VX_F32: return launch_typed<VX_F32>(maps, a, (int)units, smem, after_prep, st);
    case VX_F16: return launch_typed<VX_F16>(maps, a, (int)units, smem, after_prep, st);
    case VX_BF16: return launch_typed<VX_BF16>(maps, a, (int)units, smem, after_prep, st);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace vx
