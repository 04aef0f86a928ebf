// fp8_encode.cuh -- quantising a block of 128 elements by 8 lanes, 16 elements each (fp8.cu, and the
// queries of small products in fp8_scores.cu).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <type_traits>

#include "fp8.h"

namespace vx {

// Elements k .. k + kE - 1 of a row as they are, zero from dim on; kVec: by one load where all exist.
template <class T, int kE, bool kVec>
__device__ __forceinline__ void load_piece(const T* row, int k, int dim, uint32_t* r) {
  constexpr int kWords = kE * (int)sizeof(T) / 4;
  if (kVec && k + kE <= dim) {
    if constexpr (kWords == 4) {
      const uint4 u = __ldcs((const uint4*)(row + k));
      r[0] = u.x, r[1] = u.y, r[2] = u.z, r[3] = u.w;
    } else {
      const uint2 u = __ldcs((const uint2*)(row + k));
      r[0] = u.x, r[1] = u.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < kWords; i++) {
      if constexpr (sizeof(T) == 4) {
        r[i] = k + i < dim ? __float_as_uint(row[k + i]) : 0u;
      } else {
        const uint16_t* x = (const uint16_t*)row + k + 2 * i;
        r[i] = k + 2 * i < dim ? x[0] : 0u;
        if (k + 2 * i + 1 < dim) r[i] |= (uint32_t)x[1] << 16;
      }
    }
  }
}
// Element i of a piece.
template <class T>
__device__ __forceinline__ float element(const uint32_t* r, int i) {
  if constexpr (sizeof(T) == 4) return __uint_as_float(r[i]);
  else if constexpr (std::is_same<T, __nv_bfloat16>::value)
    return __uint_as_float(i & 1 ? r[i / 2] & 0xFFFF0000u : r[i / 2] << 16);
  else return __half2float(__ushort_as_half((unsigned short)(i & 1 ? r[i / 2] >> 16 : r[i / 2] & 0xFFFFu)));
}

// Bits of the largest magnitude of 16 elements, as float32's.
template <class T>
__device__ __forceinline__ uint32_t largest(const uint32_t (&r)[4 * sizeof(T)]) {
  uint32_t m = 0;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 16; i++) m = max(m, r[i] & 0x7FFFFFFFu);
    return m;
  } else {  // magnitudes of 16 bits order as integers
#pragma unroll
    for (int i = 0; i < 8; i++) m = __vmaxu2(m, r[i] & 0x7FFF7FFFu);
    m = max(m >> 16, m & 0xFFFFu);
    return __float_as_uint(element<T>(&m, 0));
  }
}

// Scale byte of a block from the bits of its largest magnitude: with amax = 1.m 2^(p - 127) and
// 448 = 1.75 * 2^8, the smallest e with amax <= 448 * 2^e is p - 127 - 8, plus one where 1.m > 1.75.
__device__ __forceinline__ int scale_byte(uint32_t amax_bits) {
  if (amax_bits >= 0x7F800000u) return 255;
  const int b = (int)(amax_bits >> 23) - 8 + ((amax_bits & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  return b > 0 ? b : 0;
}

// Codes of elements i .. i + 3 of a piece under scale byte b.
template <class T>
__device__ __forceinline__ uint32_t four_codes(const uint32_t* r, int i, int b) {
  if (b == 255) return 0x7F7F7F7Fu;
  const float inv = __uint_as_float((uint32_t)(254 - b) << 23);  // 2^(127 - b), b <= 247
  const float2 lo = make_float2(element<T>(r, i) * inv, element<T>(r, i + 1) * inv);
  const float2 hi = make_float2(element<T>(r, i + 2) * inv, element<T>(r, i + 3) * inv);
  return (uint32_t)__nv_cvt_float2_to_fp8x2(lo, __NV_SATFINITE, __NV_E4M3) |
         (uint32_t)__nv_cvt_float2_to_fp8x2(hi, __NV_SATFINITE, __NV_E4M3) << 16;
}

}  // namespace vx
