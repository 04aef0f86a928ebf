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
// Both kernels stream: per row they move dim elements and pitch(dim) codes + scales, and one warp
// takes four blocks (512 dimensions) of one row, 4 elements a lane and block, so that the four
// blocks' loads are in flight together and their scales make one 32-bit word.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <cstring>
#include <type_traits>

#include "../../include/vx.h"
#include "common.cuh"
#include "fp8.h"

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
// row's index is left), then every row raises the entry to its own.
__global__ void owner_store_kernel(const void* slots, int slot_bytes, int64_t n, int64_t capacity, int32_t* owner) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= n) return;
  const int64_t s = slot_at(slots, slot_bytes, i);
  if (s >= 0 && s < capacity) owner[s] = (int32_t)i;
}
__global__ void owner_max_kernel(const void* slots, int slot_bytes, int64_t n, int64_t capacity, int32_t* owner) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= n) return;
  const int64_t s = slot_at(slots, slot_bytes, i);
  if (s >= 0 && s < capacity) atomicMax(&owner[s], (int32_t)i);
}

// ---------------------------------------------------------------- write
template <class T, bool kVec>
__global__ void __launch_bounds__(kThreads) fp8_write_kernel(const Fp8WriteArgs a, int words, bool early) {
  if (early) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int lane = threadIdx.x & 31;
  const int64_t unit = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  const int64_t row = unit / words;
  const int w = (int)(unit % words);  // blocks 4w .. 4w + 3
  if (row >= a.n) return;
  int64_t slot = a.first + row;
  if (a.slots) {
    slot = slot_at(a.slots, a.slot_bytes, row);
    if (slot < 0 || slot >= a.capacity) return;
    if (a.owner) {
      if (a.owner[slot] != (int32_t)row) return;
    } else {
      bool later = false;
      for (int64_t j = row + 1 + lane; j < a.n; j += 32) later |= slot_at(a.slots, a.slot_bytes, j) == slot;
      if (__any_sync(0xFFFFFFFFu, later)) return;
    }
  }
  const int nb = (a.dim + kFp8Block - 1) / kFp8Block;
  const T* x = (const T*)a.rows + row * a.stride;
  float v[4][4];
#pragma unroll
  for (int j = 0; j < 4; j++) load4<T, kVec>(x, (4 * w + j) * kFp8Block + lane * 4, a.dim, v[j]);
  uint32_t word = 0;
  uint8_t* codes = a.codes + slot * ((int64_t)nb * kFp8Block);
#pragma unroll
  for (int j = 0; j < 4; j++) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) m = max(m, __float_as_uint(v[j][i]) & 0x7FFFFFFFu);
    m = __reduce_max_sync(0xFFFFFFFFu, m);
    if (4 * w + j >= nb) break;
    const int b = scale_byte(m);
    word |= (uint32_t)b << (8 * j);
    uint32_t c = 0x7F7F7F7Fu;
    if (b != 255) {
      const float inv = __uint_as_float((uint32_t)(254 - b) << 23);  // 2^(127 - b), b <= 247
      const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(v[j][0] * inv, v[j][1] * inv), __NV_SATFINITE, __NV_E4M3);
      const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(v[j][2] * inv, v[j][3] * inv), __NV_SATFINITE, __NV_E4M3);
      c = lo | (hi << 16);
    }
    *(uint32_t*)(codes + (4 * w + j) * kFp8Block + lane * 4) = c;
  }
  if (lane == 0) *(uint32_t*)(a.scales + slot * (4 * (int64_t)words) + 4 * w) = word;
}

// ---------------------------------------------------------------- read
template <class T, bool kVec>
__global__ void __launch_bounds__(kThreads) fp8_read_kernel(const Fp8ReadArgs a, int words) {
  const int lane = threadIdx.x & 31;
  const int64_t unit = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  const int64_t row = unit / words;
  const int w = (int)(unit % words);
  if (row >= a.n) return;
  const int64_t slot = a.slots ? slot_at(a.slots, a.slot_bytes, row) : a.first + row;
  const bool in = slot >= 0 && slot < a.capacity;
  const int nb = (a.dim + kFp8Block - 1) / kFp8Block;
  const uint8_t* codes = a.codes + (in ? slot : 0) * ((int64_t)nb * kFp8Block);
  uint32_t c[4], word = 0;
  if (in) word = __ldg((const uint32_t*)(a.scales + slot * (4 * (int64_t)words) + 4 * w));
#pragma unroll
  for (int j = 0; j < 4; j++)
    c[j] = in && 4 * w + j < nb ? __ldcs((const uint32_t*)(codes + (4 * w + j) * kFp8Block + lane * 4)) : 0u;
  T* y = (T*)a.out + row * a.stride;
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const int k = (4 * w + j) * kFp8Block + lane * 4;
    if (k >= a.dim) break;
    const uint32_t b = (word >> (8 * j)) & 0xFFu;
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

template <class T>
cudaError_t write_typed(const Fp8WriteArgs& a, bool early, int words, unsigned grid, cudaStream_t st) {
  if (four_aligned<T>(a.rows, a.stride))
    fp8_write_kernel<T, true><<<grid, kThreads, 0, st>>>(a, words, early);
  else
    fp8_write_kernel<T, false><<<grid, kThreads, 0, st>>>(a, words, early);
  return cudaGetLastError();
}

template <class T>
cudaError_t read_typed(const Fp8ReadArgs& a, int words, unsigned grid, cudaStream_t st) {
  if (four_aligned<T>(a.out, a.stride))
    fp8_read_kernel<T, true><<<grid, kThreads, 0, st>>>(a, words);
  else
    fp8_read_kernel<T, false><<<grid, kThreads, 0, st>>>(a, words);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_fp8_write(const Fp8WriteArgs& a, bool early, int* launches, cudaStream_t st) {
  const int words = fp8_scale_pitch(a.dim) / 4;
  *launches = 1;
  if (a.owner) {
    const unsigned g = (unsigned)((a.n + kThreads - 1) / kThreads);
    owner_store_kernel<<<g, kThreads, 0, st>>>(a.slots, a.slot_bytes, a.n, a.capacity, a.owner);
    owner_max_kernel<<<g, kThreads, 0, st>>>(a.slots, a.slot_bytes, a.n, a.capacity, a.owner);
    *launches = 3;
  }
  const int64_t grid = (a.n * words + kThreads / 32 - 1) / (kThreads / 32);
  if (grid > 0x7FFFFFFF) return cudaErrorInvalidValue;
  switch (a.type) {
    case VX_F32: return write_typed<float>(a, early, words, (unsigned)grid, st);
    case VX_F16: return write_typed<__half>(a, early, words, (unsigned)grid, st);
    case VX_BF16: return write_typed<__nv_bfloat16>(a, early, words, (unsigned)grid, st);
    default: return cudaErrorInvalidValue;
  }
}

cudaError_t launch_fp8_read(const Fp8ReadArgs& a, cudaStream_t st) {
  const int words = fp8_scale_pitch(a.dim) / 4;
  const int64_t grid = (a.n * words + kThreads / 32 - 1) / (kThreads / 32);
  if (grid > 0x7FFFFFFF) return cudaErrorInvalidValue;
  switch (a.type) {
    case VX_F32: return read_typed<float>(a, words, (unsigned)grid, st);
    case VX_F16: return read_typed<__half>(a, words, (unsigned)grid, st);
    case VX_BF16: return read_typed<__nv_bfloat16>(a, words, (unsigned)grid, st);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace vx
