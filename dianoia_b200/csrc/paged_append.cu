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
// moves in 16-byte accesses. For long prompts a group takes six heads of a
// token, whose loads are then in flight together before the chain sequence,
// position, page is followed, and which share the turns. G is the smallest
// power of two that holds the head: 8 lanes for 128 values, four heads to a
// warp.
// Measured: 16384 tokens of 32 + 8 + 8 heads of 128 bf16 values in 87 us (4.7
// TB/s in and out, where a plain copy does 6.5; one head a group 114 us, two
// 104, eight 125): the six heads' registers (127) leave two blocks to an SM,
// whose loads wait while their stores leave. Reads that stay out of the way of
// the cache lines just written (evict-first) are a fifth of that. 8000 tokens
// from f32 into an f32 cache take 80 us (4.9 TB/s), into a bf16 one 82 (3.6). 16
// tokens of a decode step take 3 us, the latency of the chain.
#include "dn_common.cuh"
#include "dn_launch.h"
#include "elem.cuh"

namespace dn {
namespace {

constexpr int kThreads = 256;

template <typename TI, typename TC, int V, int G, int ITER, int U>
__global__ void __launch_bounds__(kThreads) paged_append_kernel(const __grid_constant__ PagedAppendArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  const int hd = (int)a.cache.hd, heads = (int)a.heads, kvh = (int)a.cache.kv_heads;
  const uint32_t slots_all = (uint32_t)(heads + 2 * kvh), per_token = (slots_all + U - 1) / U;
  const int64_t unit = (int64_t)blockIdx.x * (kThreads / G) + threadIdx.x / G;
  if (unit >= a.n * per_token) return;  // whole groups leave together
  const uint32_t t = (uint32_t)unit / per_token, h0 = (uint32_t)unit % per_token * U;
  const int lane = threadIdx.x % G;
  const unsigned group = G == 32 ? 0xffffffffu : ((1u << G) - 1) << (threadIdx.x % 32 / G * G);

  // A slot's two runs: (s, s + rot / 2) for the rotated pairs, then the rest;
  // of a value, which does not turn, runs 2 s and 2 s + 1. Runs that are not
  // there stay zeros.
  const int rot = (int)a.rot, pairs = rot / 2 / V, slots = (hd / V + 1) / 2;
  int first[2][ITER], second[2][ITER];  // [of a value, of a query or a key]
#pragma unroll
  for (int i = 0; i < ITER; i++) {
    const int s = lane + i * G;
    first[0][i] = 2 * s * V;
    second[0][i] = first[0][i] + V;
    first[1][i] = s < pairs ? s * V : rot + 2 * (s - pairs) * V;
    second[1][i] = s < pairs ? first[1][i] + rot / 2 : first[1][i] + V;
  }
  const TI* tq = static_cast<const TI*>(a.q) + (int64_t)t * a.q_stride;
  const TI* tk = static_cast<const TI*>(a.k) + (int64_t)t * a.k_stride;
  const TI* tv = static_cast<const TI*>(a.v) + (int64_t)t * a.v_stride;
  Raw<TI, V> x[U][ITER], y[U][ITER];
#pragma unroll
  for (int u = 0; u < U; u++) {
    const int h = (int)h0 + u;
    const bool turns = h < heads + kvh;
    const TI* src = h < heads ? tq + h * hd : turns ? tk + (h - heads) * hd : tv + (h - heads - kvh) * hd;
#pragma unroll
    for (int i = 0; i < ITER; i++) {
      x[u][i].clear();
      y[u][i].clear();
      if (h >= (int)slots_all || lane + i * G >= slots) continue;
      x[u][i].load(src + (turns ? first[1][i] : first[0][i]));
      const int two = turns ? second[1][i] : second[0][i];
      if (two < hd) y[u][i].load(src + two);
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
  TC* out = static_cast<TC*>(a.q_out) + (int64_t)t * a.q_out_stride;
  if (!held) {  // the whole group
    const float zero[V] = {};
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
      for (int i = 0; i < ITER; i++) {
        const int h = (int)h0 + u;
        if (h >= heads || lane + i * G >= slots) continue;
        store_run<TC, V>(out + h * hd + first[1][i], zero);
        if (second[1][i] < hd) store_run<TC, V>(out + h * hd + second[1][i], zero);
      }
    return;
  }
  const int slot = pos - entry * (int)a.cache.page_size, head_step = (int)a.cache.page_size * hd;
  TC* keys = static_cast<TC*>(a.cache.keys) + page * a.cache.page_stride + slot * hd;
  TC* vals = static_cast<TC*>(a.cache.values) + page * a.cache.page_stride + slot * hd;
  // The token's turns, for every head that this lane holds a part of.
  float c[ITER][V], n[ITER][V];
  const float* tab = a.rope + (int64_t)pos * rot;
#pragma unroll
  for (int i = 0; i < ITER; i++) {
    if (lane + i * G >= pairs) continue;
    load_run<float, V>(tab + first[1][i], c[i]);
    load_run<float, V>(tab + rot / 2 + first[1][i], n[i]);
  }
#pragma unroll
  for (int u = 0; u < U; u++) {
    const int h = (int)h0 + u;
    if (h >= (int)slots_all) break;  // whole groups alike
    if (h >= heads + kvh) {          // a value: moved
      TC* dst = vals + (int64_t)(h - heads - kvh) * head_step;
#pragma unroll
      for (int i = 0; i < ITER; i++) {
        if (lane + i * G >= slots) continue;
        x[u][i].template store<TC>(dst + first[0][i]);
        if (second[0][i] < hd) y[u][i].template store<TC>(dst + second[0][i]);
      }
      continue;
    }
    float p[ITER][V], q[ITER][V];
#pragma unroll
    for (int i = 0; i < ITER; i++)
#pragma unroll
      for (int e = 0; e < V; e++) {
        p[i][e] = to_f32<TI>(x[u][i].e[e]);
        q[i][e] = to_f32<TI>(y[u][i].e[e]);
      }
    const float* w = h < heads ? a.q_norm : a.k_norm;
    if (w != nullptr) {
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < ITER; i++)
#pragma unroll
        for (int e = 0; e < V; e++) sum += p[i][e] * p[i][e] + q[i][e] * q[i][e];
#pragma unroll
      for (int off = G / 2; off >= 1; off >>= 1) sum += __shfl_xor_sync(group, sum, off);
      const float r = 1.0f / sqrtf(sum / (float)hd + a.eps);
#pragma unroll
      for (int i = 0; i < ITER; i++) {
        if (lane + i * G >= slots) continue;
        float wx[V], wy[V] = {};
        load_run<float, V>(w + first[1][i], wx);
        if (second[1][i] < hd) load_run<float, V>(w + second[1][i], wy);
#pragma unroll
        for (int e = 0; e < V; e++) {
          p[i][e] *= r * wx[e];
          q[i][e] *= r * wy[e];
        }
      }
    }
    TC* dst = h < heads ? out + h * hd : keys + (int64_t)(h - heads) * head_step;
#pragma unroll
    for (int i = 0; i < ITER; i++) {
      if (lane + i * G >= slots) continue;
      if (lane + i * G < pairs) {
#pragma unroll
        for (int e = 0; e < V; e++) {
          const float f = p[i][e], g = q[i][e];
          p[i][e] = f * c[i][e] - g * n[i][e];
          q[i][e] = g * c[i][e] + f * n[i][e];
        }
      }
      store_run<TC, V>(dst + first[1][i], p[i]);
      if (second[1][i] < hd) store_run<TC, V>(dst + second[1][i], q[i]);
    }
  }
}

template <typename TI, typename TC, int V, int G, int ITER, int U>
cudaError_t launch_units(const PagedAppendArgs& a, cudaStream_t stream, bool pdl) {
  const int64_t units = a.n * ((a.heads + 2 * a.cache.kv_heads + U - 1) / U);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((units * G + kThreads - 1) / kThreads));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl ? 1 : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, paged_append_kernel<TI, TC, V, G, ITER, U>, a);
}

template <typename TI, typename TC, int V, int G>
cudaError_t launch_group(const PagedAppendArgs& a, cudaStream_t stream, bool pdl) {
  // Six heads a group, once that leaves every SM its 2048 threads twice.
  const int64_t threads = a.n * (a.heads + 2 * a.cache.kv_heads) * G;
  return threads >= (int64_t)8 * 148 * 2048 ? launch_units<TI, TC, V, G, 1, 6>(a, stream, pdl)
                                            : launch_units<TI, TC, V, G, 1, 1>(a, stream, pdl);
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
  if ((addr & 15) != 0 || step % V != 0) return launch_units<TI, TC, 1, 32, 4, 1>(a, stream, pdl);
  const int64_t slots = (a.cache.hd / V + 1) / 2;
  if (slots <= 4) return launch_group<TI, TC, V, 4>(a, stream, pdl);
  if (slots <= 8) return launch_group<TI, TC, V, 8>(a, stream, pdl);
  if (slots <= 16) return launch_group<TI, TC, V, 16>(a, stream, pdl);
  if constexpr (V == 4) return launch_group<TI, TC, V, 32>(a, stream, pdl);
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
