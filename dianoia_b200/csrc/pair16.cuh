// Pairs of 16-bit elements (f16, bf16) as the tensor cores' fragments hold them.
#pragma once

#include "elem.cuh"

namespace dn {

template <typename T>
struct Pair;
// A softmax's base stands kLift (log2) below the largest score of the time it
// was set, and stays until a score passes that by kSlack: weights reach
// 2^(kLift + kSlack). bf16 has f32's exponents. f16's least number is 2^-24,
// and a weight below half of that would count in the sum and not among the
// values (128k keys of weight e^-18 beside one of 1 are 0.2% of the whole):
// raised by 2^7, weights are kept down to 2^-32 of the largest. 2^12 leaves
// room below f16's 2^16 for scores so large that they are rounded to units.
template <>
struct Pair<__half> {
  static constexpr float kLift = 7.0f, kSlack = 5.0f;
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    uint32_t u;
    memcpy(&u, &h, 4);
    return u;
  }
  // Whether either half is an infinity or a NaN.
  static __device__ __forceinline__ bool unbounded(uint32_t u) {
    return (u & 0x7c00u) == 0x7c00u || (u & 0x7c000000u) == 0x7c000000u;
  }
};
template <>
struct Pair<__nv_bfloat16> {
  static constexpr float kLift = 0.0f, kSlack = 8.0f;
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    uint32_t u;
    memcpy(&u, &h, 4);
    return u;
  }
  static __device__ __forceinline__ bool unbounded(uint32_t u) {
    return (u & 0x7f80u) == 0x7f80u || (u & 0x7f800000u) == 0x7f800000u;
  }
};

template <typename T>
__device__ __forceinline__ bool unbounded16(const void* p) {
  const uint4 v = *static_cast<const uint4*>(p);
  return Pair<T>::unbounded(v.x) || Pair<T>::unbounded(v.y) || Pair<T>::unbounded(v.z) || Pair<T>::unbounded(v.w);
}

// Two elements of a row; `pairs`: every row is 4-byte aligned.
template <typename T>
__device__ __forceinline__ uint32_t load_pair(const T* p, bool pairs) {
  if (pairs) return *reinterpret_cast<const uint32_t*>(p);
  const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
  return h[0] | (uint32_t)h[1] << 16;
}
template <typename T>
__device__ __forceinline__ void store_pair(T* p, uint32_t v, bool pairs) {
  if (pairs) {
    *reinterpret_cast<uint32_t*>(p) = v;
  } else {
    uint16_t* h = reinterpret_cast<uint16_t*>(p);
    h[0] = (uint16_t)v;
    h[1] = (uint16_t)(v >> 16);
  }
}

}  // namespace dn
