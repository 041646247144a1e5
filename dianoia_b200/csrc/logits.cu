// The rules on a batch's logits: penalties for repeated tokens, biases and
// grammar masks (dn_logits_apply).
//
// Per row and token v, with c = how often v was generated and s = whether it
// is in the history at all:
//   x1 = s ? (x > 0 ? x / r : x r) : x,  x2 = x1 - (c f + [c > 0] p),
//   x3 = x2 + the row's biases of v in list order,  y = allowed(v) ? x3 : -inf.
//
// Bytes-bound: logits in and out, once, and what stands between is latency:
// the row's rules, its history, the marks. So a CTA's kChunk tokens of one row
// come to shared memory by one bulk copy, which costs no registers (six
// CTAs to an SM keep 96 KB on the way), and leave by another. Meanwhile the
// CTA counts the history's tokens that fall into its range (integer atomics:
// their order changes nothing) and lists them with those that have biases;
// then the listed tokens, few of the range, are worked out one a thread, which
// adds the token's biases in list order (one warp does where a range has more
// than kFew of them), and under a mask the range is passed over once. There is
// no count array in memory and one launch; the history is read by every CTA of
// the row, from L2.
// Measured: 256 rows of 151936 f32 logits in 64 us (4.9 TB/s of logits in and
// out; holding them in registers 83 us); 64 rows behind histories of 3000 tokens
// with 150 biases 28 us, of which the histories are 9 and the biases 2 (5 where
// one warp adds them all).
#include "dn_common.cuh"
#include "dn_launch.h"
#include "elem.cuh"
#include "kernel_smem.h"

namespace dn {
namespace {

constexpr int kThreads = 256;
constexpr int kChunk = 4096;
constexpr int kListed = 512;  // tokens the list holds; with more, all of the range are looked at
constexpr int kFew = 32;       // biases of a range that their tokens' threads add themselves
constexpr uint32_t kBiased = 1u << 31;

__device__ __forceinline__ void bulk_s2g(void* dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(smem_u32(src)), "r"(bytes)
               : "memory");
}

// BULK: rows of out start at the alignment of their rows of logits, so that
// 16-byte aligned parts of both can be copied whole.
template <typename T, bool BULK>
__global__ void __launch_bounds__(kThreads) logits_kernel(const __grid_constant__ LogitsArgs a, int chunks) {
  pdl_launch_dependents();
  pdl_wait();
  constexpr int V = 16 / sizeof(T);
  __shared__ __align__(128) T x[kChunk];
  // Of each token of the range: bit 0 whether seen, bit 31 whether it has a
  // bias, between them how often it was generated.
  __shared__ __align__(16) uint32_t marks[kChunk];
  __shared__ uint16_t list[kListed];
  __shared__ uint32_t words[kChunk / 32 + 2];
  __shared__ int listed, few;  // tokens listed; biases of the range
  __shared__ int few_at[kFew], few_order[kFew];
  __shared__ float few_add[kFew];
  __shared__ uint64_t full;
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.x / (unsigned)chunks;
  const int chunk = (int)(blockIdx.x % (unsigned)chunks);
  const T* in = static_cast<const T*>(a.logits) + row * a.stride;
  T* out = static_cast<T*>(a.out) + row * a.out_stride;
  // Ranges start at 16-byte boundaries: up to V - 1 tokens before the row's
  // first, which are then left out.
  const int shift = BULK ? (int)(((uintptr_t)in & 15) / sizeof(T)) : 0;
  const int base = chunk * kChunk - shift, vocab = (int)a.vocab;
  // The chunks are counted for the largest shift: a row of a smaller one may
  // have no token left for its last.
  if (base >= vocab) return;
  // The range's tokens of the row, begin .. end - 1 past base (one at least);
  // whole 16 bytes of them, from .. to - 1.
  const int begin = base < 0 ? -base : 0, end = min(base + kChunk, vocab) - base;
  const int from = BULK ? begin > 0 ? V : 0 : end, to = BULK && end > from ? from + (end - from) / V * V : from;
  const LogitRules& r = a.rules;
  if (tid == 0) {
    mbar_init(&full, 1);
    fence_mbar_init();
    if (to > from) {
      mbar_arrive_expect_tx(&full, (uint32_t)((to - from) * sizeof(T)));
      bulk_g2s(&x[from], in + base + from, (uint32_t)((to - from) * sizeof(T)), &full);
    }
    listed = few = 0;
  }
  // What no bulk copy takes (all of it without BULK).
  for (int at = begin + tid; at < min(from, end); at += kThreads) x[at] = in[base + at];
  for (int at = max(to, begin) + tid; BULK && at < end; at += kThreads) x[at] = in[base + at];

  int seen = 0, made = 0, biased = 0;  // tokens of the history, those before the generated ones, biases
  const int* tokens = nullptr;
  const int* bias_tokens = nullptr;
  const float* bias = nullptr;
  if (r.history != nullptr) {
    const int64_t h0 = r.history[row], h1 = r.history[row + 1];
    tokens = r.tokens + h0;
    seen = (int)min64(h1 - h0, INT32_MAX - 2 * kChunk);
    made = r.generated != nullptr ? seen - r.generated[row] : 0;
  }
  if (r.bias_start != nullptr) {
    const int64_t b0 = r.bias_start[row], b1 = r.bias_start[row + 1];
    bias_tokens = r.bias_tokens + b0;
    bias = r.bias + b0;
    biased = (int)min64(b1 - b0, INT32_MAX - 2 * kChunk);
  }
  const int64_t mrow = r.mask == nullptr ? -1 : r.mask_row != nullptr ? r.mask_row[row] : row;
  const uint32_t* mask = mrow >= 0 && mrow < r.mask_rows ? r.mask + mrow * r.mask_stride : nullptr;
  const bool marked = seen > 0 || biased > 0;
  // The first tokens and biases are on their way while the marks are cleared.
  constexpr int kAtOnce = 8;
  uint32_t at[kAtOnce], first_bias = tid < biased ? (uint32_t)bias_tokens[tid] - (uint32_t)base : 0xffffffffu;
  auto load_tokens = [&](int i0) {
#pragma unroll
    for (int k = 0; k < kAtOnce; k++)
      at[k] = i0 + k * kThreads < seen ? (uint32_t)tokens[i0 + k * kThreads] - (uint32_t)base : 0xffffffffu;
  };
  load_tokens(tid);
  const int word0 = (base + begin) / 32;  // of words[0]
  if (marked) {
#pragma unroll
    for (int i = 0; i < kChunk / 4 / kThreads; i++)
      reinterpret_cast<uint4*>(marks)[i * kThreads + tid] = make_uint4(0, 0, 0, 0);
  }
  if (mask != nullptr && tid < kChunk / 32 + 2) words[tid] = word0 + tid < (vocab + 31) / 32 ? mask[word0 + tid] : 0;
  __syncthreads();
  auto add_to_list = [&](uint32_t at) {
    const int j = atomicAdd(&listed, 1);
    if (j < kListed) list[j] = (uint16_t)at;
  };
  auto mine = [&](uint32_t at) { return at - (uint32_t)begin < (uint32_t)(end - begin); };
  for (int i0 = tid; i0 < seen; i0 += kThreads * kAtOnce) {
    if (i0 != tid) load_tokens(i0);
#pragma unroll
    for (int k = 0; k < kAtOnce; k++)
      if (mine(at[k])) {
        if (atomicOr(&marks[at[k]], 1u) == 0) add_to_list(at[k]);
        if (i0 + k * kThreads >= made) atomicAdd(&marks[at[k]], 2u);
      }
  }
  for (int i = tid; i < biased; i += kThreads) {
    const uint32_t v = i == tid ? first_bias : (uint32_t)bias_tokens[i] - (uint32_t)base;
    if (!mine(v)) continue;
    const int j = atomicAdd(&few, 1);
    if (j < kFew) {
      few_at[j] = (int)v;
      few_order[j] = i;
      few_add[j] = bias[i];
    }
    if (atomicOr(&marks[v], kBiased) == 0) add_to_list(v);
  }
  const bool landed = to <= from || mbar_wait_bounded(&full, 0, a.status, kStatusTmaTimeout);
  if (!landed) mbar_land(&full, 0);
  if (!__syncthreads_and(landed)) return;

  // The marked tokens.
  const int count = marked ? listed : 0;
  const bool fits = count <= kListed;
  auto each_marked = [&](auto&& f) {
    if (fits) {
      for (int j = tid; j < count; j += kThreads) f((int)list[j]);
    } else {
      for (int at = begin + tid; at < end; at += kThreads) f(at);
    }
  };
  if (count > 0) {
    const float rep = r.repetition != nullptr ? r.repetition[row] : 1.0f;
    const float freq = r.frequency != nullptr ? r.frequency[row] : 0.0f;
    const float pres = r.presence != nullptr ? r.presence[row] : 0.0f;
    auto penalized = [&](int at, uint32_t mark) {
      float z = to_f32<T>(x[at]);
      if (mark != 0) {
        z = z > 0.0f ? z / rep : z * rep;
        const float times = (float)(mark >> 1);
        z -= times * freq + (times > 0.0f ? pres : 0.0f);
      }
      return z;
    };
    const int adds = few;
    if (adds <= kFew) {
      each_marked([&](int at) {
        const uint32_t mark = marks[at];
        if (mark == 0) return;
        float z = penalized(at, mark & ~kBiased);
        if ((mark & kBiased) != 0) {
          for (int last = -1;;) {  // its biases in list order
            int next = INT32_MAX, from = 0;
            for (int j = 0; j < adds; j++)
              if (few_at[j] == at && few_order[j] > last && few_order[j] < next) {
                next = few_order[j];
                from = j;
              }
            if (next == INT32_MAX) break;
            z += few_add[from];
            last = next;
          }
        }
        x[at] = from_f32<T>(z);
      });
    } else {
      // f32 results in place of the marks; one warp adds the biases to them.
      each_marked([&](int at) { marks[at] = __float_as_uint(penalized(at, marks[at] & ~kBiased)); });
      __syncthreads();
      if (tid < 32) {
        for (int i0 = tid; i0 - tid < biased; i0 += 32) {
          const uint32_t at = i0 < biased ? (uint32_t)bias_tokens[i0] - (uint32_t)base : 0xffffffffu;
          const bool here = mine(at);
          unsigned left = __ballot_sync(0xffffffffu, here);
          const float add = here ? bias[i0] : 0.0f;
          while (left != 0) {  // in list order
            const int src = __ffs(left) - 1;
            left &= left - 1;
            if (tid == src) marks[at] = __float_as_uint(__uint_as_float(marks[at]) + add);
            __syncwarp();
          }
        }
      }
      __syncthreads();
      each_marked([&](int at) { x[at] = from_f32<T>(__uint_as_float(marks[at])); });
    }
  }
  if (mask != nullptr) {
    if (count > 0) __syncthreads();
    for (int at = begin + tid; at < end; at += kThreads) {
      const int v = base + at;
      if ((words[v / 32 - word0] >> (v % 32) & 1u) == 0) x[at] = from_f32<T>(-INFINITY);
    }
  }
  if (count > 0 || mask != nullptr) fence_proxy_async_smem();  // the threads' writes, before the bulk copy reads them
  __syncthreads();
  if (to > from && tid == 0) {
    bulk_s2g(out + base + from, &x[from], (uint32_t)((to - from) * sizeof(T)));
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
  }
  for (int at = begin + tid; at < min(from, end); at += kThreads) out[base + at] = x[at];
  for (int at = max(to, begin) + tid; BULK && at < end; at += kThreads) out[base + at] = x[at];
  if (to > from && tid == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
}

template <typename T, bool BULK>
cudaError_t launch_copies(const LogitsArgs& a, cudaStream_t stream, bool pdl) {
  const int64_t chunks = (a.vocab + 16 / (int64_t)sizeof(T) - 1 + kChunk - 1) / kChunk;
  if (chunks * a.n > 0x7fffffff) return cudaErrorInvalidValue;
  if (cudaError_t e = allow_smem<logits_kernel<T, BULK>>(0); e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(chunks * a.n));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl ? 1 : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, logits_kernel<T, BULK>, a, (int)chunks);
}

template <typename T>
cudaError_t launch_type(const LogitsArgs& a, cudaStream_t stream, bool pdl) {
  constexpr int V = 16 / sizeof(T);
  const bool same = (((uintptr_t)a.logits ^ (uintptr_t)a.out) & 15) == 0 &&
                    (a.n <= 1 || (a.stride - a.out_stride) % V == 0);
  return same ? launch_copies<T, true>(a, stream, pdl) : launch_copies<T, false>(a, stream, pdl);
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
