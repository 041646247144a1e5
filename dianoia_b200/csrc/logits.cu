// The rules on a batch's logits: penalties for repeated tokens, biases and
// grammar masks (dn_logits_apply).
//
// Per row and token v, with c = how often v was generated and s = whether it
// is in the history at all:
//   x1 = s ? (x > 0 ? x / r : x r) : x,  x2 = x1 - (c f + [c > 0] p),
//   x3 = x2 + the row's biases of v in list order,  y = allowed(v) ? x3 : -inf.
//
// Bytes-bound: logits in and out, once. A CTA owns kChunk tokens of one row.
// Its logits are loaded into registers first; while they are on their way it
// counts the history's tokens that fall into its range in shared memory
// (integer atomics: their order changes nothing), adds up the biases there
// (one warp, in list order) and takes its words of the mask. So there is no
// count array in memory, one launch, and the scan of the history, which every
// CTA of the row reads from L2, hides behind the logits.
#include "dn_common.cuh"
#include "dn_launch.h"
#include "elem.cuh"

namespace dn {
namespace {

constexpr int kThreads = 256;
constexpr int kChunk = 4096;
constexpr uint32_t kBiased = 1u << 31;

template <typename T, int V>
__global__ void __launch_bounds__(kThreads) logits_kernel(const __grid_constant__ LogitsArgs a, int chunks) {
  pdl_launch_dependents();
  pdl_wait();
  constexpr int kRuns = kChunk / (kThreads * V);
  // Of each token of the range: bit 0 whether seen, bit 31 whether it has a
  // bias (then biases holds it), between them how often it was generated. A
  // run of tokens without any of it, nearly all of them, costs one load.
  __shared__ __align__(16) uint32_t marks[kChunk];
  __shared__ float biases[kChunk];
  __shared__ uint32_t words[kChunk / 32 + 2];
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.x / (unsigned)chunks;
  const int chunk = (int)(blockIdx.x % (unsigned)chunks);
  const T* in = static_cast<const T*>(a.logits) + row * a.stride;
  T* out = static_cast<T*>(a.out) + row * a.out_stride;
  // V > 1: ranges start where rows have 16-byte aligned runs, up to V - 1
  // tokens before the row's first (which are then left out).
  const int shift = V > 1 ? (int)(((uintptr_t)in & 15) / sizeof(T)) : 0;
  const int base = chunk * kChunk - shift, vocab = (int)a.vocab;
  const LogitRules& r = a.rules;

  Raw<T, V> x[kRuns];
#pragma unroll
  for (int i = 0; i < kRuns; i++) {
    const int v = base + (i * kThreads + tid) * V;
    if (v >= 0 && v + V <= vocab) {
      x[i].load(in + v);
    } else {
#pragma unroll
      for (int e = 0; e < V; e++)
        if (v + e >= 0 && v + e < vocab) x[i].e[e] = in[v + e];
    }
  }
  const int64_t h0 = r.history != nullptr ? r.history[row] : 0;
  const int64_t h1 = r.history != nullptr ? r.history[row + 1] : 0;
  const int64_t b0 = r.bias_start != nullptr ? r.bias_start[row] : 0;
  const int64_t b1 = r.bias_start != nullptr ? r.bias_start[row + 1] : 0;
  const float rep = r.repetition != nullptr ? r.repetition[row] : 1.0f;
  const float freq = r.frequency != nullptr ? r.frequency[row] : 0.0f;
  const float pres = r.presence != nullptr ? r.presence[row] : 0.0f;
  const int64_t mrow = r.mask == nullptr ? -1 : r.mask_row != nullptr ? r.mask_row[row] : row;
  const uint32_t* mask = mrow >= 0 && mrow < r.mask_rows ? r.mask + mrow * r.mask_stride : nullptr;
  const bool counted = h1 > h0, biased = b1 > b0;
  const int word0 = (base < 0 ? 0 : base) / 32;  // of words[0]
  const bool marked = counted || biased;
  if (marked)
    for (int i = tid; i < kChunk / 4; i += kThreads) reinterpret_cast<uint4*>(marks)[i] = make_uint4(0, 0, 0, 0);
  if (mask != nullptr)
    for (int i = tid; i < kChunk / 32 + 2; i += kThreads)
      words[i] = word0 + i < (vocab + 31) / 32 ? mask[word0 + i] : 0;
  __syncthreads();
  if (counted) {
    const int64_t made = r.generated != nullptr ? h1 - r.generated[row] : h0;
    constexpr int kAtOnce = 4;
    for (int64_t i0 = h0 + tid; i0 < h1; i0 += kThreads * kAtOnce) {
      int v[kAtOnce];
#pragma unroll
      for (int k = 0; k < kAtOnce; k++) v[k] = i0 + k * kThreads < h1 ? r.tokens[i0 + k * kThreads] : -1;
#pragma unroll
      for (int k = 0; k < kAtOnce; k++) {
        const uint32_t at = (uint32_t)v[k] - (uint32_t)base;
        if (v[k] >= 0 && v[k] < vocab && at < kChunk) {
          atomicOr(&marks[at], 1u);
          if (i0 + k * kThreads >= made) atomicAdd(&marks[at], 2u);
        }
      }
    }
  }
  if (biased && tid >= kThreads - 32) {
    const int lane = tid % 32;
    constexpr int kAtOnce = 4;
    for (int64_t i0 = b0; i0 < b1; i0 += 32 * kAtOnce) {
      int v[kAtOnce];
      float add[kAtOnce];
#pragma unroll
      for (int k = 0; k < kAtOnce; k++) {
        const int64_t i = i0 + 32 * k + lane;
        v[k] = i < b1 ? r.bias_tokens[i] : -1;
        add[k] = i < b1 ? r.bias[i] : 0.0f;
      }
#pragma unroll
      for (int k = 0; k < kAtOnce; k++) {
        const uint32_t at = (uint32_t)v[k] - (uint32_t)base;
        unsigned left = __ballot_sync(0xffffffffu, v[k] >= 0 && v[k] < vocab && at < kChunk);
        while (left != 0) {  // in list order
          const int src = __ffs(left) - 1;
          left &= left - 1;
          if (lane == src) {
            biases[at] = (atomicOr(&marks[at], kBiased) & kBiased) != 0 ? biases[at] + add[k] : 0.0f + add[k];
          }
          __syncwarp();
        }
      }
    }
  }
  __syncthreads();

#pragma unroll
  for (int i = 0; i < kRuns; i++) {
    const int at = (i * kThreads + tid) * V, v = base + at;
    if (v >= vocab) break;
    uint32_t allowed = 0xffffffffu;  // of tokens v .. v + V - 1
    if (mask != nullptr) {
      const int w = (v < 0 ? 0 : v) / 32 - word0;
      allowed = v >= 0 ? __funnelshift_r(words[w], words[w + 1], v % 32) : words[w] << -v;
    }
    float y[V];
    uint32_t c[V], any = 0;
    if (marked) {
      if constexpr (V % 4 == 0) {
#pragma unroll
        for (int e = 0; e < V; e += 4) {
          const uint4 four = *reinterpret_cast<const uint4*>(&marks[at + e]);
          c[e] = four.x;
          c[e + 1] = four.y;
          c[e + 2] = four.z;
          c[e + 3] = four.w;
        }
      } else {
#pragma unroll
        for (int e = 0; e < V; e++) c[e] = marks[at + e];
      }
#pragma unroll
      for (int e = 0; e < V; e++) any |= c[e];
    }
#pragma unroll
    for (int e = 0; e < V; e++) y[e] = to_f32<T>(x[i].e[e]);
    if (any != 0) {
#pragma unroll
      for (int e = 0; e < V; e++) {
        if ((c[e] & ~kBiased) != 0) {
          y[e] = y[e] > 0.0f ? y[e] / rep : y[e] * rep;
          const float times = (float)((c[e] & ~kBiased) >> 1);
          y[e] -= times * freq + (times > 0.0f ? pres : 0.0f);
        }
        if ((c[e] & kBiased) != 0) y[e] += biases[at + e];
      }
    }
#pragma unroll
    for (int e = 0; e < V; e++) y[e] = (allowed >> e & 1u) != 0 ? y[e] : -INFINITY;
    if (v >= 0 && v + V <= vocab) {
      store_run<T, V>(out + v, y);
    } else {
#pragma unroll
      for (int e = 0; e < V; e++)
        if (v + e >= 0 && v + e < vocab) out[v + e] = from_f32<T>(y[e]);
    }
  }
}

template <typename T, int V>
cudaError_t launch_run(const LogitsArgs& a, cudaStream_t stream, bool pdl) {
  const int64_t chunks = (a.vocab + V - 1 + kChunk - 1) / kChunk;
  if (chunks * a.n > 0x7fffffff) return cudaErrorInvalidValue;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(chunks * a.n));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl ? 1 : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, logits_kernel<T, V>, a, (int)chunks);
}

template <typename T>
cudaError_t launch_type(const LogitsArgs& a, cudaStream_t stream, bool pdl) {
  // 16-byte runs where every row of out starts at the alignment of its row of
  // logits, whatever that is; else one value at a time.
  constexpr int V = 16 / sizeof(T);
  const bool same = (((uintptr_t)a.logits ^ (uintptr_t)a.out) & 15) == 0 &&
                    (a.n <= 1 || (a.stride - a.out_stride) % V == 0);
  return same ? launch_run<T, V>(a, stream, pdl) : launch_run<T, 1>(a, stream, pdl);
}

}  // namespace

cudaError_t launch_logits(const LogitsArgs& a, cudaStream_t stream, bool pdl) {
  if (a.n <= 0 || a.vocab <= 0) return cudaSuccess;
  switch (a.type) {
    case kF32: return launch_type<float>(a, stream, pdl);
    case kF16: return launch_type<__half>(a, stream, pdl);
    default: return launch_type<__nv_bfloat16>(a, stream, pdl);
  }
}

}  // namespace dn
