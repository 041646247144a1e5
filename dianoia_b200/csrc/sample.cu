// The choice of a token from a row of logits (dn_sample).
//
// w_v = exp((x_v - max) / T) as whole steps of 2^-44 (64 bits hold the sum of
// 2^19 of them), so that sums have no rounding and no order. The kept tokens
// are a prefix of the row ordered by logit, equal ones by index: those above a
// border logit and the first few equal to it. Logits map to ordered 32-bit
// keys, the border is found bit by bit, each bit one pass of the row.
#include "dn_common.cuh"
#include "dn_launch.h"
#include "elem.cuh"

namespace dn {
namespace {

constexpr int kThreads = 1024;
constexpr double kOne = 17592186044416.0;  // 2^44, the largest weight

// Ordered as the floats are, -0 as +0; 0 for what is no token.
__device__ __forceinline__ uint32_t key_of(float x) {
  if (!(x > -INFINITY)) return 0;
  const uint32_t u = __float_as_uint(x + 0.0f);
  return (u >> 31) != 0 ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ uint64_t block_sum(uint64_t s, uint64_t* red) {
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
  __syncthreads();
  if (threadIdx.x % 32 == 0) red[threadIdx.x / 32] = s;
  __syncthreads();
  s = red[threadIdx.x % 32];
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
  return s;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_kernel(const __grid_constant__ SampleArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  __shared__ uint64_t red[32];
  __shared__ uint32_t tops[32];
  const int row = blockIdx.x, tid = threadIdx.x, vocab = (int)a.vocab;
  const T* in = static_cast<const T*>(a.logits) + (int64_t)row * a.stride;
  const Sampling& how = a.how;
  const float temperature = how.temperature != nullptr ? how.temperature[row] : 1.0f;
  const bool greedy = !(temperature > 0.0f);
  const int top_k = how.top_k != nullptr ? how.top_k[row] : 0;
  const float top_p = how.top_p != nullptr ? how.top_p[row] : 1.0f;
  const float min_p = how.min_p != nullptr ? how.min_p[row] : 0.0f;
  const float u = how.uniform[row];
  auto key_at = [&](int v) { return key_of(to_f32<T>(in[v])); };
  // Sums f(v) over the row.
  auto sum_of = [&](auto&& f) {
    uint64_t s = 0;
    for (int v = tid; v < vocab; v += kThreads) s += f(v);
    return block_sum(s, red);
  };
  uint32_t top = 0;
  for (int v = tid; v < vocab; v += kThreads) top = max(top, key_at(v));
  top = __reduce_max_sync(0xffffffffu, top);
  if (tid % 32 == 0) tops[tid / 32] = top;
  __syncthreads();
  top = __reduce_max_sync(0xffffffffu, tops[tid % 32]);
  if (top == 0) {
    if (tid == 0) {
      a.tokens[row] = -1;
      if (a.logprobs != nullptr) a.logprobs[row] = -INFINITY;
      if (a.kept != nullptr) a.kept[row] = 0;
    }
    return;
  }
  const double largest = (double)__uint_as_float((top >> 31) != 0 ? top & 0x7fffffffu : ~top);
  const double inv = greedy ? 0.0 : 1.0 / (double)temperature;
  auto share = [&](int v, uint32_t key) {
    if (key == top) return 1.0;
    if (key == 0 || greedy || isinf(largest)) return 0.0;
    return exp(((double)to_f32<T>(in[v]) - largest) * inv);
  };
  auto weight = [&](int v, uint32_t key) { return (uint64_t)__double2ull_rn(share(v, key) * kOne); };
  // The largest key of which f(key) >= want, f falling; f(1) >= want.
  auto border_of = [&](uint64_t want, auto&& f) {
    uint32_t key = 0;
    for (int bit = 31; bit >= 0; bit--) {
      const uint32_t next = key | 1u << bit;
      if (f(next) >= want) key = next;
    }
    return key;
  };
  uint32_t border = 1;          // tokens below it are out,
  uint64_t ties = vocab;        // of those at it the first so many are in
  auto count_from = [&](uint32_t k) { return sum_of([&](int v) { return (uint64_t)(key_at(v) >= k); }); };
  if (greedy || min_p > 1.0f) {  // the first token alone
    border = top;
    ties = 1;
  } else {
    if (top_k > 0 && count_from(1) > (uint64_t)top_k) {
      border = border_of((uint64_t)top_k, count_from);
      ties = (uint64_t)top_k - (border == ~0u ? 0 : count_from(border + 1));
    }
    if (top_p < 1.0f) {
      auto mass_from = [&](uint32_t k) {
        return sum_of([&](int v) {
          const uint32_t key = key_at(v);
          return key >= k ? weight(v, key) : 0;
        });
      };
      // What top_k leaves: all above the border, `ties` at it.
      auto at_border = [&](uint32_t k) {
        return sum_of([&](int v) {
          const uint32_t key = key_at(v);
          return key == k ? ((uint64_t)1 << 44) + 0 : 0;
        }) >> 44;
      };
      const uint64_t tied = at_border(border);
      const uint64_t in_border = tied == 0 ? 0 : (mass_from(border) - mass_from(border + 1)) / tied * (ties < tied ? ties : tied);
      const uint64_t total = mass_from(border + 1) + in_border;
      const double share_p = top_p > 0.0f ? (double)top_p * (double)total : 0.0;
      uint64_t want = (uint64_t)ceil(share_p);
      if (want < 1) want = 1;
      auto mass_kept = [&](uint32_t k) {  // of the tokens that top_k leaves
        const uint64_t above = mass_from(k > border ? k : border + 1);
        return k > border ? above : above + in_border;
      };
      const uint32_t at = border_of(want, mass_kept);
      if (at >= border) {
        const uint64_t above = mass_from(at + 1);
        const uint64_t many = at_border(at);
        const uint64_t each = (mass_from(at) - above) / many;
        const uint64_t need = (want - above + each - 1) / each;
        if (at > border || need < ties) ties = need;
        border = at;
      }
    }
  }
  auto in_min = [&](int v, uint32_t key) { return key == top || !(min_p > 0.0f) || share(v, key) >= (double)min_p; };
  // The index of the last tie that is in.
  int last_tie = vocab;
  if (ties < (uint64_t)vocab) {
    int lo = -1, hi = vocab - 1;  // the smallest hi with `ties` ties up to it
    while (hi - lo > 1) {
      const int mid = lo + (hi - lo) / 2;
      if (sum_of([&](int v) { return (uint64_t)(v <= mid && key_at(v) == border); }) >= ties) hi = mid; else lo = mid;
    }
    last_tie = hi;
  }
  auto kept = [&](int v) {
    const uint32_t key = key_at(v);
    return key != 0 && (key > border || (key == border && v <= last_tie)) && in_min(v, key);
  };
  const uint64_t count = sum_of([&](int v) { return (uint64_t)kept(v); });
  const uint64_t mass = sum_of([&](int v) { return kept(v) ? weight(v, key_at(v)) : 0; });
  const double share_u = u > 0.0f ? (double)u * (double)mass : 0.0;
  uint64_t target = share_u >= (double)mass ? mass - 1 : (uint64_t)share_u;
  if (target >= mass) target = mass - 1;
  int lo = -1, hi = vocab - 1;  // the smallest hi up to which the kept mass is more than the target
  while (hi - lo > 1) {
    const int mid = lo + (hi - lo) / 2;
    if (sum_of([&](int v) { return v <= mid && kept(v) ? weight(v, key_at(v)) : 0; }) > target) hi = mid; else lo = mid;
  }
  if (tid == 0) {
    a.tokens[row] = hi;
    if (a.logprobs != nullptr) a.logprobs[row] = (float)log((double)weight(hi, key_at(hi)) / (double)mass);
    if (a.kept != nullptr) a.kept[row] = (int)count;
  }
}

template <typename T>
cudaError_t launch_type(const SampleArgs& a, cudaStream_t stream, bool pdl) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)a.n);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl ? 1 : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, sample_kernel<T>, a);
}

}  // namespace

cudaError_t launch_sample(const SampleArgs& a, cudaStream_t stream, bool pdl) {
  if (a.n <= 0) return cudaSuccess;
  switch (a.type) {
    case kF32: return launch_type<float>(a, stream, pdl);
    case kF16: return launch_type<__half>(a, stream, pdl);
    default: return launch_type<__nv_bfloat16>(a, stream, pdl);
  }
}

}  // namespace dn
