// The rules on a batch's logits: penalties for repeated tokens, biases and
// grammar masks (dn_logits_apply).
//
// Per row and token v, with c = how often v was generated and s = whether it
// is in the history at all:
//   x1 = s ? (x > 0 ? x / r : x r) : x,  x2 = x1 - (c f + [c > 0] p),
//   x3 = x2 + the row's biases of v in list order,  y = allowed(v) ? x3 : -inf.
//
// Bytes-bound: logits in and out, once. A CTA owns kChunk tokens of one row.
// It counts the history's tokens that fall into its range in shared memory
// (integer atomics: their order changes nothing), adds up the biases there
// (one lane, in list order), and then passes over its logits once, so that
// there is no count array in memory and one launch. The history is read by
// every CTA of the row, from L2.
#include "dn_common.cuh"
#include "dn_launch.h"
#include "elem.cuh"

namespace dn {
namespace {

constexpr int kThreads = 256;
constexpr int kChunk = 4096;

template <typename T, int V>
__global__ void __launch_bounds__(kThreads) logits_kernel(const __grid_constant__ LogitsArgs a, int chunks) {
  pdl_launch_dependents();
  pdl_wait();
  __shared__ uint32_t counts[kChunk];  // 2 * times generated + whether seen
  __shared__ float biases[kChunk];
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

  const int64_t h0 = r.history != nullptr ? r.history[row] : 0;
  const int64_t h1 = r.history != nullptr ? r.history[row + 1] : 0;
  const int64_t b0 = r.bias_start != nullptr ? r.bias_start[row] : 0;
  const int64_t b1 = r.bias_start != nullptr ? r.bias_start[row + 1] : 0;
  const bool counted = h1 > h0, biased = b1 > b0;
  if (counted)
    for (int i = tid; i < kChunk; i += kThreads) counts[i] = 0;
  if (biased)
    for (int i = tid; i < kChunk; i += kThreads) biases[i] = 0.0f;
  __syncthreads();
  if (counted) {
    const int64_t made = r.generated != nullptr ? h1 - r.generated[row] : h0;
    for (int64_t i = h0 + tid; i < h1; i += kThreads) {
      const int v = r.tokens[i];
      const uint32_t at = (uint32_t)v - (uint32_t)base;
      if (v >= 0 && v < vocab && at < kChunk) {
        atomicOr(&counts[at], 1u);
        if (i >= made) atomicAdd(&counts[at], 2u);
      }
    }
  }
  if (biased && tid < 32) {
    for (int64_t i0 = b0; i0 < b1; i0 += 32) {
      const int64_t i = i0 + tid;
      const int v = i < b1 ? r.bias_tokens[i] : -1;
      const uint32_t at = (uint32_t)v - (uint32_t)base;
      const bool mine = v >= 0 && v < vocab && at < kChunk;
      const float add = mine ? r.bias[i] : 0.0f;
      unsigned left = __ballot_sync(0xffffffffu, mine);
      while (left != 0) {  // in list order
        const int src = __ffs(left) - 1;
        left &= left - 1;
        if (tid == src) biases[at] += add;
        __syncwarp();
      }
    }
  }
  const float rep = r.repetition != nullptr ? r.repetition[row] : 1.0f;
  const float freq = r.frequency != nullptr ? r.frequency[row] : 0.0f;
  const float pres = r.presence != nullptr ? r.presence[row] : 0.0f;
  const int64_t mrow = r.mask == nullptr ? -1 : r.mask_row != nullptr ? r.mask_row[row] : row;
  const uint32_t* mask = mrow >= 0 && mrow < r.mask_rows ? r.mask + mrow * r.mask_stride : nullptr;
  const int words = (vocab + 31) / 32;
  __syncthreads();

  auto rule = [&](float x, int at, bool allowed) {
    if (counted) {
      const uint32_t c = counts[at];
      if (c != 0) {
        x = x > 0.0f ? x / rep : x * rep;
        const float times = (float)(c >> 1);
        x -= times * freq + (times > 0.0f ? pres : 0.0f);
      }
    }
    if (biased) x += biases[at];
    return allowed ? x : -INFINITY;
  };
  for (int at = tid * V; at < kChunk; at += kThreads * V) {
    const int v = base + at;
    if (v >= vocab) break;
    uint32_t bits = 0xffffffffu;  // of tokens v .. v + V - 1
    if (mask != nullptr) {
      const int w = v >= 0 ? v / 32 : 0;
      const uint32_t lo = mask[w], hi = w + 1 < words ? mask[w + 1] : 0;
      bits = v >= 0 ? __funnelshift_r(lo, hi, v % 32) : lo << -v;
    }
    if (v >= 0 && v + V <= vocab) {
      float x[V];
      load_run<T, V>(in + v, x);
#pragma unroll
      for (int e = 0; e < V; e++) x[e] = rule(x[e], at + e, (bits >> e & 1u) != 0);
      store_run<T, V>(out + v, x);
    } else {
      for (int e = 0; e < V; e++)
        if (v + e >= 0 && v + e < vocab)
          out[v + e] = from_f32<T>(rule(to_f32<T>(in[v + e]), at + e, (bits >> e & 1u) != 0));
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
