// Appends a step's keys and values to a paged cache and rotates its queries
// and keys on the way (dn_paged_append).
//
// Per head of a token: x' = w x / sqrt(mean(x^2) + eps) (optional), then for
// j < rot / 2  y[j] = x'[j] c[j] - x'[j + rot/2] s[j],
//              y[j + rot/2] = x'[j + rot/2] c[j] + x'[j] s[j],
// y[j] = x'[j] from rot on; values are only moved. All in f32, rounded once to
// the cache's type.
//
// Bytes-bound: every value is read and written once. A head belongs to a
// group of G lanes; a lane holds two runs of V values, the two halves of a
// rotation pair (runs past rot are held two by two), so that the rotation
// needs no exchange, the norm one shuffle reduction of G lanes, and memory
// moves in 16-byte accesses. G is the smallest power of two that holds the
// head: 8 lanes for 128 values, four heads to a warp.
#include "dn_common.cuh"
#include "dn_launch.h"
#include "elem.cuh"

namespace dn {
namespace {

constexpr int kThreads = 256;

template <typename TI, typename TC, int V, int G, int ITER>
__global__ void __launch_bounds__(kThreads) paged_append_kernel(const __grid_constant__ PagedAppendArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  const int hd = (int)a.cache.hd, heads = (int)a.heads, kvh = (int)a.cache.kv_heads;
  const uint32_t per_token = (uint32_t)(heads + 2 * kvh);
  const int64_t unit = (int64_t)blockIdx.x * (kThreads / G) + threadIdx.x / G;
  if (unit >= a.n * per_token) return;  // whole groups leave together
  const uint32_t t = (uint32_t)unit / per_token, h = (uint32_t)unit % per_token;
  const int lane = threadIdx.x % G;
  const unsigned group = G == 32 ? 0xffffffffu : ((1u << G) - 1) << (threadIdx.x % 32 / G * G);
  const bool is_q = (int)h < heads, is_k = !is_q && (int)h < heads + kvh;
  const int head = is_q ? (int)h : is_k ? (int)h - heads : (int)h - heads - kvh;
  const TI* src = is_q   ? static_cast<const TI*>(a.q) + (int64_t)t * a.q_stride
                  : is_k ? static_cast<const TI*>(a.k) + (int64_t)t * a.k_stride
                         : static_cast<const TI*>(a.v) + (int64_t)t * a.v_stride;
  src += (int64_t)head * hd;
  const int rot = is_q || is_k ? (int)a.rot : 0;

  // A slot's two runs: (s, s + rot / 2) for the rotated pairs, then the rest.
  const int pairs = rot / 2 / V, slots = (hd / V + 1) / 2;
  int first[ITER], second[ITER];
  float x[ITER][V], y[ITER][V];
#pragma unroll
  for (int i = 0; i < ITER; i++) {
    const int s = lane + i * G;
    first[i] = s < pairs ? s * V : rot + 2 * (s - pairs) * V;
    second[i] = s < pairs ? first[i] + rot / 2 : first[i] + V;
#pragma unroll
    for (int e = 0; e < V; e++) x[i][e] = y[i][e] = 0.0f;
    if (s < slots) {
      load_run<TI, V>(src + first[i], x[i]);
      if (second[i] < hd) load_run<TI, V>(src + second[i], y[i]);
    }
  }

  // Where the token goes; -1: nowhere.
  const int seq = a.seq[t], pos = a.pos[t];
  int64_t page = -1;
  const int entry = pos / (int)a.cache.page_size;
  if (seq >= 0 && seq < a.cache.sequences && pos >= 0 && entry < a.cache.table_stride &&
      (a.rot == 0 || pos < a.rope_rows))
    page = a.cache.table[seq * a.cache.table_stride + entry];
  const bool held = page >= 0 && page < a.cache.pages;
  if (!held) {
    if (is_q) {
      const float zero[V] = {};
      TC* dst = static_cast<TC*>(a.q_out) + (int64_t)t * a.q_out_stride + (int64_t)head * hd;
#pragma unroll
      for (int i = 0; i < ITER; i++) {
        if (lane + i * G >= slots) break;
        store_run<TC, V>(dst + first[i], zero);
        if (second[i] < hd) store_run<TC, V>(dst + second[i], zero);
      }
    }
    return;  // the whole group
  }

  const float* w = is_q ? a.q_norm : is_k ? a.k_norm : nullptr;
  if (w != nullptr) {
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < ITER; i++)
#pragma unroll
      for (int e = 0; e < V; e++) sum += x[i][e] * x[i][e] + y[i][e] * y[i][e];
#pragma unroll
    for (int off = G / 2; off >= 1; off >>= 1) sum += __shfl_xor_sync(group, sum, off);
    const float r = 1.0f / sqrtf(sum / (float)hd + a.eps);
#pragma unroll
    for (int i = 0; i < ITER; i++) {
      if (lane + i * G >= slots) break;
      float wx[V], wy[V] = {};
      load_run<float, V>(w + first[i], wx);
      if (second[i] < hd) load_run<float, V>(w + second[i], wy);
#pragma unroll
      for (int e = 0; e < V; e++) {
        x[i][e] *= r * wx[e];
        y[i][e] *= r * wy[e];
      }
    }
  }
  const float* tab = a.rope + (int64_t)pos * a.rot;
  const int slot = pos - entry * (int)a.cache.page_size;
  TC* dst;
  if (is_q) {
    dst = static_cast<TC*>(a.q_out) + (int64_t)t * a.q_out_stride + (int64_t)head * hd;
  } else {
    dst = static_cast<TC*>(is_k ? a.cache.keys : a.cache.values) + page * a.cache.page_stride +
          (head * a.cache.page_size + slot) * hd;
  }
#pragma unroll
  for (int i = 0; i < ITER; i++) {
    const int s = lane + i * G;
    if (s >= slots) break;
    if (s < pairs) {
      float c[V], n[V];
      load_run<float, V>(tab + first[i], c);
      load_run<float, V>(tab + rot / 2 + first[i], n);
#pragma unroll
      for (int e = 0; e < V; e++) {
        const float p = x[i][e], q = y[i][e];
        x[i][e] = p * c[e] - q * n[e];
        y[i][e] = q * c[e] + p * n[e];
      }
    }
    store_run<TC, V>(dst + first[i], x[i]);
    if (second[i] < hd) store_run<TC, V>(dst + second[i], y[i]);
  }
}

template <typename TI, typename TC, int V, int G, int ITER>
cudaError_t launch_group(const PagedAppendArgs& a, cudaStream_t stream, bool pdl) {
  const int64_t units = a.n * (a.heads + 2 * a.cache.kv_heads);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((units * G + kThreads - 1) / kThreads));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl ? 1 : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, paged_append_kernel<TI, TC, V, G, ITER>, a);
}

template <typename TI, typename TC>
cudaError_t launch_types(const PagedAppendArgs& a, cudaStream_t stream, bool pdl) {
  // Runs of 16 bytes of the narrower type, where sizes, strides and addresses
  // allow 16-byte accesses; else one value at a time.
  constexpr int V = sizeof(TI) == 4 && sizeof(TC) == 4 ? 4 : 8;
  const uintptr_t addr = (uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.q_out |
                         (uintptr_t)a.cache.keys | (uintptr_t)a.cache.values | (uintptr_t)a.rope |
                         (uintptr_t)a.q_norm | (uintptr_t)a.k_norm;
  const int64_t step = a.q_stride | a.k_stride | a.v_stride | a.q_out_stride | a.cache.page_stride | a.cache.hd |
                       a.rot / 2;
  if ((addr & 15) != 0 || step % V != 0) return launch_group<TI, TC, 1, 32, 4>(a, stream, pdl);
  const int64_t slots = (a.cache.hd / V + 1) / 2;
  if (slots <= 4) return launch_group<TI, TC, V, 4, 1>(a, stream, pdl);
  if (slots <= 8) return launch_group<TI, TC, V, 8, 1>(a, stream, pdl);
  if (slots <= 16) return launch_group<TI, TC, V, 16, 1>(a, stream, pdl);
  if constexpr (V == 4) return launch_group<TI, TC, V, 32, 1>(a, stream, pdl);
  return cudaErrorInvalidValue;  // hd over kMaxPagedHd, which the entry refuses
}

template <typename TI>
cudaError_t launch_in(const PagedAppendArgs& a, cudaStream_t stream, bool pdl) {
  switch (a.cache.type) {
    case kF32: return launch_types<TI, float>(a, stream, pdl);
    case kF16: return launch_types<TI, __half>(a, stream, pdl);
    default: return launch_types<TI, __nv_bfloat16>(a, stream, pdl);
  }
}

}  // namespace

cudaError_t launch_paged_append(const PagedAppendArgs& a, cudaStream_t stream, bool pdl) {
  if (a.n <= 0) return cudaSuccess;
  switch (a.type) {
    case kF32: return launch_in<float>(a, stream, pdl);
    case kF16: return launch_in<__half>(a, stream, pdl);
    default: return launch_in<__nv_bfloat16>(a, stream, pdl);
  }
}

}  // namespace dn
