// fp8.cu -- quantising rows into an 8-bit store as they are written, and reading them back.
//
// Stored form of a row x: blocks of 128 dimensions, each with one scale 2^e, e the smallest
// integer >= -127 with max |x| <= 448 * 2^e (448 is e4m3's largest value), kept as the byte
// e + 127; each element as the nearest e4m3 value of x / 2^e, ties to even.  A power of two costs
// no accuracy against an arbitrary scale (e4m3 has its own exponent: |error| <= 2^-4 |x|, or
// 2^-10 * 2^e for elements below 2^-6 * 2^e), the scaling itself is exact, a scale takes one
// byte, and the tensor cores apply it inside the product (fp8_scores.cu).  A block that holds a
// NaN or an infinity is NaN throughout: scale byte 255, codes 0x7f.
//
// Both kernels stream: per row they move dim elements and pitch(dim) codes + scales.  One warp takes
// up to kWords x 4 blocks of one row, 4 elements a lane and block: their loads are in flight
// together, every access of the warp is consecutive, and four blocks' scales make one 32-bit word.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <cstring>
#include <type_traits>

#include "../../include/vx.h"
#include "common.cuh"
#include "fp8.h"
#include "fp8_groups.cuh"

namespace vx {
namespace {

constexpr int kThreads = 256;
constexpr uint32_t kInf = 0x7F800000u;

__device__ __forceinline__ int64_t slot_at(const void* slots, int slot_bytes, int64_t i) {
  return slot_bytes == 4 ? (int64_t)((const int32_t*)slots)[i] : ((const int64_t*)slots)[i];
}

// ---------------------------------------------------------------- element types
template <class T>
__device__ __forceinline__ float to_f32(T v) {
  if constexpr (sizeof(T) == 4) return v;
  else if constexpr (std::is_same<T, __half>::value) return __half2float(v);
  else return __bfloat162float(v);
}
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
// Four elements that this kernel reads once.
template <class T>
__device__ __forceinline__ Four<T> load_four(const T* p) {
  if constexpr (sizeof(T) == 4) {
    const float4 f = __ldcs(reinterpret_cast<const float4*>(p));
    return Four<T>{{f.x, f.y, f.z, f.w}};
  } else {
    const uint2 u = __ldcs(reinterpret_cast<const uint2*>(p));
    Four<T> f;
    memcpy(&f, &u, 8);
    return f;
  }
}

// Elements k .. k + 3 of a row; zero from dim on.
template <class T, bool kVec>
__device__ __forceinline__ void load4(const T* row, int k, int dim, float (&x)[4]) {
  if (kVec && k + 4 <= dim) {
    const Four<T> f = load_four<T>(row + k);
#pragma unroll
    for (int i = 0; i < 4; i++) x[i] = to_f32<T>(f.v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++) x[i] = k + i < dim ? to_f32<T>(row[k + i]) : 0.0f;
  }
}

// Scale byte of a block from the bits of its largest magnitude: with amax = 1.m 2^(p - 127) and
// 448 = 1.75 * 2^8, the smallest e with amax <= 448 * 2^e is p - 127 - 8, plus one where 1.m > 1.75.
__device__ __forceinline__ int scale_byte(uint32_t amax_bits) {
  if (amax_bits >= kInf) return 255;
  const int b = (int)(amax_bits >> 23) - 8 + ((amax_bits & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  return b > 0 ? b : 0;
}

// ---------------------------------------------------------------- repeated slots
// Where several rows of a batch name one slot, the last of them is kept.  Up to kFp8DirectSlots
// rows: each row looks for its slot among the later rows.  Above: owner[slot] becomes the largest
// row index that names the slot, without clearing `owner` first: every row stores its index (some
// row's index is left), then every row raises the entry to its own.  The three launches overlap:
// each begins before the one before it ends and waits for it where it needs its results.
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

// ---------------------------------------------------------------- write
// Blocks of 8 warps; block b takes rows 8 (b / parts) + warp, part b % parts of their words.
// kGroups: block 0 counts a grouped product's tiles instead.
template <class T, bool kVec, int kWords, bool kGroups>
__global__ void __launch_bounds__(kThreads) fp8_write_kernel(const Fp8WriteArgs a, const Fp8Groups groups,
                                                             unsigned long long* counter, uint32_t parts) {
  launch_dependents();
  if (counter && blockIdx.x == 0 && threadIdx.x == 0) *counter = 0;
  uint32_t block = blockIdx.x;
  if constexpr (kGroups) {
    if (block == 0) {
      fp8_count_tiles<kThreads>(groups);
      return;
    }
    block--;
  }
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)(block / parts) * (kThreads / 32) + (threadIdx.x >> 5);
  const int first = (int)(block % parts) * kWords * 4;  // first block of the row's
  const int nb = (a.dim + kFp8Block - 1) / kFp8Block;
  const T* x = (const T*)a.rows + row * a.stride;
  float v[kWords * 4][4];
  int64_t slot = -1;
  if (row < a.n) {
#pragma unroll
    for (int j = 0; j < kWords * 4; j++) load4<T, kVec>(x, (first + j) * kFp8Block + lane * 4, a.dim, v[j]);
    slot = a.slots ? slot_at(a.slots, a.slot_bytes, row) : a.first + row;
  }
  if (a.owner) wait_for_launch_before();  // every thread: no block ends before the launches before it
  if (slot < 0 || slot >= a.capacity) return;
  if (a.slots) {
    if (a.owner) {
      if (__ldcg(a.owner + slot) != (int32_t)row) return;
    } else {
      bool later = false;
      for (int64_t j = row + 1 + lane; j < a.n; j += 32) later |= slot_at(a.slots, a.slot_bytes, j) == slot;
      if (__any_sync(0xFFFFFFFFu, later)) return;
    }
  }
  uint8_t* codes = a.codes + slot * ((int64_t)nb * kFp8Block);
  uint8_t* scales = a.scales + slot * (int64_t)((nb + 3) / 4 * 4);
#pragma unroll
  for (int w = 0; w < kWords; w++) {
    if (first + 4 * w >= nb) break;
    uint32_t word = 0;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const float(&y)[4] = v[4 * w + j];
      const int k = first + 4 * w + j;
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < 4; i++) m = max(m, __float_as_uint(y[i]) & 0x7FFFFFFFu);
      m = __reduce_max_sync(0xFFFFFFFFu, m);
      if (k >= nb) break;
      const int b = scale_byte(m);
      word |= (uint32_t)b << (8 * j);
      uint32_t c = 0x7F7F7F7Fu;
      if (b != 255) {
        const float inv = __uint_as_float((uint32_t)(254 - b) << 23);  // 2^(127 - b), b <= 247
        const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(y[0] * inv, y[1] * inv), __NV_SATFINITE, __NV_E4M3);
        const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(y[2] * inv, y[3] * inv), __NV_SATFINITE, __NV_E4M3);
        c = lo | (hi << 16);
      }
      *(uint32_t*)(codes + k * kFp8Block + lane * 4) = c;
    }
    if (lane == 0) *(uint32_t*)(scales + first + 4 * w) = word;
  }
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

// Parts of a row of `words` scale words that a warp each takes, and the blocks for n rows.
int parts_of(int words, int per) { return (words + per - 1) / per; }
bool grid_for(int64_t n, int parts, int extra, unsigned* grid) {
  const int64_t g = (n + kThreads / 32 - 1) / (kThreads / 32) * parts + extra;
  *grid = (unsigned)g;
  return g <= 0x7FFFFFFF;
}

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

template <class T, int kWords, bool kGroups>
cudaError_t write_words(const Fp8WriteArgs& a, const Fp8Groups& g, unsigned long long* counter, int words, cudaStream_t st) {
  const int parts = parts_of(words, kWords);
  unsigned grid;
  if (!grid_for(a.n, parts, kGroups ? 1 : 0, &grid)) return cudaErrorInvalidValue;
  const bool dependent = a.owner != nullptr;
  if (four_aligned<T>(a.rows, a.stride))
    return launch(fp8_write_kernel<T, true, kWords, kGroups>, grid, kThreads, dependent, st, a, g, counter, (uint32_t)parts);
  return launch(fp8_write_kernel<T, false, kWords, kGroups>, grid, kThreads, dependent, st, a, g, counter, (uint32_t)parts);
}

// Rows of more than 512 dimensions: a warp takes 8 blocks (kWords 2), else 4.
template <class T, bool kGroups>
cudaError_t write_typed(const Fp8WriteArgs& a, const Fp8Groups& g, unsigned long long* counter, cudaStream_t st) {
  const int words = fp8_scale_pitch(a.dim) / 4;
  return words > 1 ? write_words<T, 2, kGroups>(a, g, counter, words, st)
                   : write_words<T, 1, kGroups>(a, g, counter, words, st);
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
  unsigned grid;
  if (!grid_for(a.n, parts, 0, &grid)) return cudaErrorInvalidValue;
  if (four_aligned<T>(a.out, a.stride))
    return launch(fp8_read_kernel<T, true, kWords>, grid, kThreads, false, st, a, (uint32_t)parts);
  return launch(fp8_read_kernel<T, false, kWords>, grid, kThreads, false, st, a, (uint32_t)parts);
}

template <class T>
cudaError_t read_typed(const Fp8ReadArgs& a, cudaStream_t st) {
  const int words = fp8_scale_pitch(a.dim) / 4;
  return words > 1 ? read_words<T, 2>(a, words, st) : read_words<T, 1>(a, words, st);
}

}  // namespace

cudaError_t launch_fp8_write(const Fp8WriteArgs& a, int* launches, cudaStream_t st) {
  *launches = 1;
  if (a.owner) {
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
