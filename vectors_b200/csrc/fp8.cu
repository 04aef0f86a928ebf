// fp8.cu -- quantising rows into an 8-bit store as they are written, and reading them back.
//
// Stored form of a row x: blocks of 128 dimensions, each with one scale 2^e, e the smallest
// integer >= -127 with max |x| <= 448 * 2^e (448 is e4m3's largest value), kept as the byte
// e + 127; each element as the nearest e4m3 value of x / 2^e, ties to even: |error| <= 2^-4 |x|, or
// 2^-10 * 2^e for elements below 2^-6 * 2^e.  For the larger elements a power of two is as good as
// an arbitrary scale (e4m3 has its own exponent); it may be up to twice that scale, so the small
// elements' absolute error may be up to twice what it would be.  In return the scaling itself is exact, a
// scale takes one byte, and the tensor cores apply it inside the product (fp8_scores.cu).  A block that
// holds a NaN or an infinity is NaN throughout: scale byte 255, codes 0x7f (past dim too).
//
// Both kernels stream: per row they move dim elements and pitch(dim) codes + scales.
//   write  8 lanes take a block, 16 elements each in pieces of 16 (or 8) bytes, so that both sides are
//          consecutive, the block's maximum is three shuffles away, and rows of any number of blocks
//          fill the warps.  (A prefetched next block costs more in resident warps than it hides.)
//          400k x 1024 fp32: 299-316 us, 6.5-6.9 TB/s; 100k x 768 bf16: 43 us, 5.4 TB/s.
//   read   one warp takes up to 8 blocks of a row, 4 elements a lane and block, so that the wider
//          side, its stores, is consecutive.  300k scattered rows x 1000 to fp16: 147-160 us, 5.7-6.2 TB/s.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <atomic>
#include <type_traits>

#include "../../include/vx.h"
#include "common.cuh"
#include "fp8.h"
#include "fp8_encode.cuh"
#include "fp8_groups.cuh"
#include "sm100.cuh"

namespace vx {
namespace {

constexpr int kThreads = 256;


__device__ __forceinline__ int64_t slot_at(const void* slots, int slot_bytes, int64_t i) {
  return slot_bytes == 4 ? (int64_t)((const int32_t*)slots)[i] : ((const int64_t*)slots)[i];
}

// ---------------------------------------------------------------- element types
template <class T>
__device__ __forceinline__ T from_f32(float v) {
  if constexpr (sizeof(T) == 4) return v;
  else if constexpr (std::is_same<T, __half>::value) return __float2half_rn(v);
  else return __float2bfloat16_rn(v);
}
template <class T>
struct alignas(4 * sizeof(T)) Four {
  T v[4];
};
// ---------------------------------------------------------------- repeated slots
// Where several rows of a batch name one slot, the last of them is kept.  Up to kFp8DirectSlots
// rows: the lanes of a block look for its slot among the later rows.  Above: owner[slot] becomes the
// largest row index that names the slot, without clearing `owner` first: every row stores its index
// (some row's index is left), then every row raises the entry to its own.  Up to kClusterRows rows one
// cluster does both (4,000 rows: 10.5 us a call, 12.4 with two launches; 30,000: 24.6 and 20.5).  The
// launches overlap: each begins before the one before it ends and waits for it where it needs its
// results.
__device__ __forceinline__ void launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_launch_before() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

template <bool kMax>
__global__ void owner_kernel(const void* slots, int slot_bytes, int64_t n, int64_t capacity, int32_t* owner) {
  launch_dependents();
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const int64_t s = i < n ? slot_at(slots, slot_bytes, i) : -1;
  if (kMax) wait_for_launch_before();
  if (s < 0 || s >= capacity) return;
  if (kMax) atomicMax(&owner[s], (int32_t)i);
  else owner[s] = (int32_t)i;
}

// Both steps by one cluster, a row a thread, for up to kClusterRows rows.
constexpr int kOwnerCtas = 8, kOwnerThreads = 1024;
constexpr int64_t kClusterRows = kOwnerCtas * kOwnerThreads;
__global__ void __cluster_dims__(kOwnerCtas, 1, 1) __launch_bounds__(kOwnerThreads)
    owner_cluster_kernel(const void* slots, int slot_bytes, int64_t n, int64_t capacity, int32_t* owner) {
  launch_dependents();
  const int i = blockIdx.x * kOwnerThreads + threadIdx.x;
  int64_t s = i < n ? slot_at(slots, slot_bytes, i) : -1;
  if (s >= capacity) s = -1;
  if (s >= 0) owner[s] = i;
  sm100::cluster_sync();
  if (s >= 0) atomicMax(&owner[s], i);
}

// ---------------------------------------------------------------- write
// Work is counted in blocks of 128 dimensions, row after row; a CTA takes kRun of them at a time and
// goes on gridDim.x runs further.  kGroups: CTA 0 counts a grouped product's tiles instead.
constexpr int kRun = kThreads / 8;

template <class T, int kE, bool kVec, bool kGroups>
__global__ void __launch_bounds__(kThreads, 6) fp8_write_kernel(const Fp8WriteArgs a, const Fp8Groups groups,
                                                             unsigned long long* counter) {
  launch_dependents();
  if (counter && blockIdx.x == 0 && threadIdx.x == 0) *counter = 0;
  const uint32_t ctas = gridDim.x - (kGroups ? 1 : 0);
  if constexpr (kGroups) {
    if (blockIdx.x == 0) {
      fp8_count_tiles<kThreads>(groups);
      return;
    }
  }
  constexpr int kPieces = 16 / kE, kWords = kE * (int)sizeof(T) / 4;
  const int part = threadIdx.x & 7;
  const uint32_t nb = (uint32_t)(a.dim + kFp8Block - 1) / kFp8Block;
  const uint32_t scale_pitch = (nb + 3) / 4 * 4;
  const uint64_t begin = (uint64_t)(blockIdx.x - (kGroups ? 1 : 0)) * kRun + (threadIdx.x >> 3), step = (uint64_t)ctas * kRun;
  const auto divide = [nb](uint64_t x) { return x >> 32 ? x / nb : (uint64_t)((uint32_t)x / nb); };
  int64_t row = (int64_t)divide(begin);
  uint32_t at = (uint32_t)(begin - (uint64_t)row * nb);  // block within the row
  const int64_t step_row = (int64_t)divide(step);
  const uint32_t step_at = (uint32_t)(step - (uint64_t)step_row * nb);

  bool first = true;
  for (; __any_sync(0xFFFFFFFFu, row < a.n); first = false) {
    uint32_t r[kPieces * kWords];
    int64_t slot = -1;
    if (row < a.n) {
      const T* x = (const T*)a.rows + row * a.stride;
#pragma unroll
      for (int i = 0; i < kPieces; i++)
        load_piece<T, kE, kVec>(x, (int)at * kFp8Block + (i * 8 + part) * kE, a.dim, r + i * kWords);
      slot = a.slots ? slot_at(a.slots, a.slot_bytes, row) : a.first + row;
      if (slot >= a.capacity) slot = -1;
    }
    if (a.owner && first) wait_for_launch_before();
    bool keep = slot >= 0;
    if (a.owner) {
      if (keep) keep = __ldcg(a.owner + slot) == (int32_t)row;
    } else if (a.slots) {
      if (keep)
        for (int j = (int)row + 1 + part; j < (int)a.n; j += 8) keep &= slot_at(a.slots, a.slot_bytes, j) != slot;
      keep = (__ballot_sync(0xFFFFFFFFu, !keep) >> (threadIdx.x & 24) & 0xFFu) == 0;
    }
    uint32_t m = keep ? largest<T>(r) : 0u;
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
    if (keep) {
      const int b = scale_byte(m);
      uint8_t* codes = a.codes + slot * ((int64_t)nb * kFp8Block) + at * kFp8Block + part * kE;
#pragma unroll
      for (int i = 0; i < kPieces; i++) {
        uint32_t c[kE / 4];
#pragma unroll
        for (int q = 0; q < kE / 4; q++) c[q] = four_codes<T>(r + i * kWords, 4 * q, b);
        if constexpr (kE == 8) *(uint2*)(codes + i * 64) = make_uint2(c[0], c[1]);
        else *(uint32_t*)(codes + i * 32) = c[0];
      }
      // the scale's byte, and after the last block's the zeros up to a word
      uint8_t* scale = a.scales + slot * (int64_t)scale_pitch + at;
      if (part == 0) *scale = (uint8_t)b;
      else if (at + 1 == nb && at + part < scale_pitch) scale[part] = 0;
    }
    row += step_row;
    at += step_at;
    if (at >= nb) {
      at -= nb;
      row++;
    }
  }
  if (a.owner && first) wait_for_launch_before();  // no CTA ends before the launches before it
}

__global__ void __launch_bounds__(1024) fp8_count_tiles_kernel(const Fp8Groups groups, unsigned long long* counter) {
  launch_dependents();
  if (counter && threadIdx.x == 0) *counter = 0;
  if (!groups.row_off) return;
  fp8_count_tiles<1024>(groups);
}

// ---------------------------------------------------------------- read
template <class T, bool kVec, int kWords>
__global__ void __launch_bounds__(kThreads) fp8_read_kernel(const Fp8ReadArgs a, uint32_t parts) {
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)(blockIdx.x / parts) * (kThreads / 32) + (threadIdx.x >> 5);
  const int first = (int)(blockIdx.x % parts) * kWords * 4;
  if (row >= a.n) return;
  const int64_t slot = a.slots ? slot_at(a.slots, a.slot_bytes, row) : a.first + row;
  const bool in = slot >= 0 && slot < a.capacity;
  const int nb = (a.dim + kFp8Block - 1) / kFp8Block;
  const uint8_t* codes = a.codes + (in ? slot : 0) * ((int64_t)nb * kFp8Block);
  const uint8_t* scales = a.scales + (in ? slot : 0) * (int64_t)((nb + 3) / 4 * 4);
  uint32_t c[kWords * 4], word[kWords];
#pragma unroll
  for (int w = 0; w < kWords; w++)
    word[w] = in && first + 4 * w < nb ? __ldg((const uint32_t*)(scales + first + 4 * w)) : 0u;
#pragma unroll
  for (int j = 0; j < kWords * 4; j++)
    c[j] = in && first + j < nb ? __ldcs((const uint32_t*)(codes + (first + j) * kFp8Block + lane * 4)) : 0u;
  T* y = (T*)a.out + row * a.stride;
#pragma unroll
  for (int j = 0; j < kWords * 4; j++) {
    const int k = (first + j) * kFp8Block + lane * 4;
    if (k >= a.dim) break;
    const uint32_t b = (word[j >> 2] >> (8 * (j & 3))) & 0xFFu;
    // 2^(b - 127); b = 0 is the subnormal 2^-127, 255 is NaN
    const float s = __uint_as_float(b == 255u ? 0x7FC00000u : b == 0u ? 0x00400000u : b << 23);
    const __half2 lo = __half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(c[j] & 0xFFFFu), __NV_E4M3));
    const __half2 hi = __half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(c[j] >> 16), __NV_E4M3));
    const float2 f = __half22float2(lo), g = __half22float2(hi);
    Four<T> o;
    o.v[0] = from_f32<T>(f.x * s);
    o.v[1] = from_f32<T>(f.y * s);
    o.v[2] = from_f32<T>(g.x * s);
    o.v[3] = from_f32<T>(g.y * s);
    if (kVec && k + 4 <= a.dim) {
      *reinterpret_cast<Four<T>*>(y + k) = o;
    } else {
#pragma unroll
      for (int i = 0; i < 4; i++)
        if (k + i < a.dim) y[k + i] = o.v[i];
    }
  }
}

template <class T>
bool four_aligned(const void* p, int64_t stride) {
  return (uintptr_t)p % (4 * sizeof(T)) == 0 && stride % 4 == 0;
}

// Parts of a row of `words` scale words that a warp each takes.
int parts_of(int words, int per) { return (words + per - 1) / per; }

// Launches `kern`, allowed to begin before the launch before it ends if `dependent`.
template <class... P, class... A>
cudaError_t launch(void (*kern)(P...), unsigned grid, int threads, bool dependent, cudaStream_t st, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = dependent ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kern, args...);
}

// As many CTAs as stay on the device at once, or as there are runs of work; where that leaves each
// more than 8 runs, CTAs of 4 that the device shares out as they end (400k x 1024 fp32: 304 us, 348 in
// one wave; 16k x 1024 bf16: 10.8 us in one wave, 13.2 in CTAs of 4).
template <class T, int kE, bool kVec, bool kGroups>
cudaError_t write_variant(const Fp8WriteArgs& a, const Fp8Groups& g, unsigned long long* counter, cudaStream_t st) {
  static std::atomic<int> per_sm{0};
  auto kern = fp8_write_kernel<T, kE, kVec, kGroups>;
  int n = per_sm.load();
  if (n == 0) {
    cudaError_t e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kern, kThreads, 0);
    if (e != cudaSuccess) return e;
    per_sm.store(n);
  }
  const int64_t runs = (a.n * fp8_blocks(a.dim) + kRun - 1) / kRun;
  const int64_t most = (int64_t)n * a.num_sms - (kGroups ? 1 : 0);
  int64_t grid = runs < most ? runs : most;
  if (runs > 8 * most) grid = (runs + 3) / 4;
  grid += kGroups ? 1 : 0;
  if (grid > 0x7FFFFFFF) return cudaErrorInvalidValue;
  return launch(kern, (unsigned)grid, kThreads, a.owner != nullptr, st, a, g, counter);
}

template <class T, bool kGroups>
cudaError_t write_typed(const Fp8WriteArgs& a, const Fp8Groups& g, unsigned long long* counter, cudaStream_t st) {
  // the widest loads that every row's first element is aligned for
  const uintptr_t bits = (uintptr_t)a.rows | (uintptr_t)(a.stride * (int64_t)sizeof(T));
  if (bits % 16 == 0) return write_variant<T, 16 / sizeof(T), true, kGroups>(a, g, counter, st);
  if (sizeof(T) == 2 && bits % 8 == 0) return write_variant<T, 4, true, kGroups>(a, g, counter, st);
  return write_variant<T, 4, false, kGroups>(a, g, counter, st);
}

template <bool kGroups>
cudaError_t write_any(const Fp8WriteArgs& a, const Fp8Groups& g, unsigned long long* counter, cudaStream_t st) {
  switch (a.type) {
    case VX_F32: return write_typed<float, kGroups>(a, g, counter, st);
    case VX_F16: return write_typed<__half, kGroups>(a, g, counter, st);
    case VX_BF16: return write_typed<__nv_bfloat16, kGroups>(a, g, counter, st);
    default: return cudaErrorInvalidValue;
  }
}

template <class T, int kWords>
cudaError_t read_words(const Fp8ReadArgs& a, int words, cudaStream_t st) {
  const int parts = parts_of(words, kWords);
  const int64_t grid = (a.n + kThreads / 32 - 1) / (kThreads / 32) * parts;
  if (grid > 0x7FFFFFFF) return cudaErrorInvalidValue;
  if (four_aligned<T>(a.out, a.stride))
    return launch(fp8_read_kernel<T, true, kWords>, (unsigned)grid, kThreads, false, st, a, (uint32_t)parts);
  return launch(fp8_read_kernel<T, false, kWords>, (unsigned)grid, kThreads, false, st, a, (uint32_t)parts);
}

template <class T>
cudaError_t read_typed(const Fp8ReadArgs& a, cudaStream_t st) {
  const int words = fp8_scale_pitch(a.dim) / 4;
  return words > 1 ? read_words<T, 2>(a, words, st) : read_words<T, 1>(a, words, st);
}

}  // namespace

cudaError_t launch_fp8_write(const Fp8WriteArgs& a, int* launches, cudaStream_t st) {
  *launches = 1;
  if (a.owner && a.n <= kClusterRows) {
    const cudaError_t e =
        launch(owner_cluster_kernel, kOwnerCtas, kOwnerThreads, false, st, a.slots, a.slot_bytes, a.n, a.capacity, a.owner);
    if (e != cudaSuccess) return e;
    *launches = 2;
  } else if (a.owner) {
    const unsigned g = (unsigned)((a.n + kThreads - 1) / kThreads);
    cudaError_t e = launch(owner_kernel<false>, g, kThreads, false, st, a.slots, a.slot_bytes, a.n, a.capacity, a.owner);
    if (e == cudaSuccess)
      e = launch(owner_kernel<true>, g, kThreads, true, st, a.slots, a.slot_bytes, a.n, a.capacity, a.owner);
    if (e != cudaSuccess) return e;
    *launches = 3;
  }
  return write_any<false>(a, Fp8Groups{}, nullptr, st);
}

cudaError_t launch_fp8_prepare(const Fp8WriteArgs& a, const Fp8Groups& g, unsigned long long* counter, cudaStream_t st) {
  if (!a.rows) return launch(fp8_count_tiles_kernel, 1u, 1024, false, st, g, counter);
  return g.row_off ? write_any<true>(a, g, counter, st) : write_any<false>(a, g, counter, st);
}

cudaError_t launch_fp8_read(const Fp8ReadArgs& a, cudaStream_t st) {
  switch (a.type) {
    case VX_F32: return read_typed<float>(a, st);
    case VX_F16: return read_typed<__half>(a, st);
    case VX_BF16: return read_typed<__nv_bfloat16>(a, st);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace vx
