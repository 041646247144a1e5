// Elements of the paged cache and of logits: f32, f16 and bf16 in memory, f32
// in registers. Conversions to f32 are exact; each from f32 rounds to nearest
// even, once.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include <type_traits>

namespace dn {

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// V consecutive elements as f32; 16- or 8-byte accesses where the run has that
// size and alignment (the caller's promise for V > 1), else one at a time.
template <typename T, int V>
__device__ __forceinline__ void load_run(const T* p, float (&x)[V]) {
  if constexpr (V * sizeof(T) % 16 == 0) {
#pragma unroll
    for (int u = 0; u < (int)(V * sizeof(T) / 16); u++) {
      const uint4 w = reinterpret_cast<const uint4*>(p)[u];
      T e[16 / sizeof(T)];
      memcpy(e, &w, 16);
#pragma unroll
      for (int i = 0; i < (int)(16 / sizeof(T)); i++) x[u * (16 / sizeof(T)) + i] = to_f32<T>(e[i]);
    }
  } else if constexpr (V * sizeof(T) == 8) {
    const uint2 w = *reinterpret_cast<const uint2*>(p);
    T e[V];
    memcpy(e, &w, 8);
#pragma unroll
    for (int i = 0; i < V; i++) x[i] = to_f32<T>(e[i]);
  } else {
#pragma unroll
    for (int i = 0; i < V; i++) x[i] = to_f32<T>(p[i]);
  }
}

template <typename T, int V>
__device__ __forceinline__ void store_run(T* p, const float (&x)[V]) {
  if constexpr (V * sizeof(T) % 16 == 0) {
#pragma unroll
    for (int u = 0; u < (int)(V * sizeof(T) / 16); u++) {
      T e[16 / sizeof(T)];
#pragma unroll
      for (int i = 0; i < (int)(16 / sizeof(T)); i++) e[i] = from_f32<T>(x[u * (16 / sizeof(T)) + i]);
      uint4 w;
      memcpy(&w, e, 16);
      reinterpret_cast<uint4*>(p)[u] = w;
    }
  } else if constexpr (V * sizeof(T) == 8) {
    T e[V];
#pragma unroll
    for (int i = 0; i < V; i++) e[i] = from_f32<T>(x[i]);
    uint2 w;
    memcpy(&w, e, 8);
    *reinterpret_cast<uint2*>(p) = w;
  } else {
#pragma unroll
    for (int i = 0; i < V; i++) p[i] = from_f32<T>(x[i]);
  }
}

// A run of V elements as it lies in memory, read once (16 bytes at a time
// where it has that size: the caller's promise of alignment).
template <typename T, int V>
struct Raw {
  static constexpr int kBytes = V * (int)sizeof(T);
  T e[V];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < V; i++) e[i] = from_f32<T>(0.0f);
  }
  // The run as elements of TC (the same bits where that is T).
  template <typename TC>
  __device__ __forceinline__ void store(TC* p) const {
    if constexpr (sizeof(T) == sizeof(TC) && kBytes % 16 == 0 && std::is_same<T, TC>::value) {
#pragma unroll
      for (int u = 0; u < kBytes / 16; u++) {
        uint4 w;
        memcpy(&w, reinterpret_cast<const char*>(e) + 16 * u, 16);
        reinterpret_cast<uint4*>(p)[u] = w;
      }
    } else {
      float x[V];
#pragma unroll
      for (int i = 0; i < V; i++) x[i] = to_f32<T>(e[i]);
      store_run<TC, V>(p, x);
    }
  }
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (kBytes % 16 == 0) {
#pragma unroll
      for (int u = 0; u < kBytes / 16; u++) {
        const uint4 w = __ldcs(reinterpret_cast<const uint4*>(p) + u);
        memcpy(reinterpret_cast<char*>(e) + 16 * u, &w, 16);
      }
    } else {
#pragma unroll
      for (int i = 0; i < V; i++) e[i] = p[i];
    }
  }
};

}  // namespace dn
