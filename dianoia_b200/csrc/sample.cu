// The choice of a token from a row of logits (dn_sample).
//
// w_v = exp((x_v - max) / T) as whole steps of 2^-44 (64 bits hold the sum of
// 2^19 of them), so that sums have no rounding and no order. The kept tokens
// are a prefix of the row ordered by logit, equal ones by index: top_k cuts it
// by count, top_p by the sum of weights, min_p by the weight itself. Logits map
// to ordered 32-bit keys.
//
// Bytes-bound for many rows, latency for few: a row should be read from memory
// once, and few steps follow one another. So a cluster of blocks holds a row in
// its shared memory (38 KB a block of a 151936-token row of f32 over 16 blocks,
// four blocks to an SM), finds the largest logit, and then the few tokens that
// can matter:
//  - top_k: the threads' own largest logits, one for each 37 tokens or so, in a
//    histogram of their distance from the largest one: at least k tokens are as
//    near as the k-th of these;
//  - min_p: the weight says it;
//  - top_p: the weights by their log2, roughly, in a histogram: as many of the
//    largest as hold that share. The rest only adds to the sum (below 2^-20 from
//    f32 exponentials, in the same steps).
// Their weights (f64) and keys go to the first block's shared memory, which sorts
// them and decides alone while the others leave. Where more tokens matter than its
// lists hold (flat distributions, many ties, thousands of top_k) the border is
// found eight bits of the key at a time over all of the row in the cluster's
// shared memory; without a rule but the temperature every token has its f64
// weight and the block that the random number falls to looks for the token.
#include <cooperative_groups.h>

#include "dn_common.cuh"
#include "dn_launch.h"
#include "elem.cuh"
#include "kernel_smem.h"

namespace dn {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxBlocks = 16;  // of a cluster
constexpr int kListed = 512;    // tokens that a block lists
constexpr int kSorted = 2048;   // that the first one sorts, over its part of the row
constexpr int kMostK = 1536;    // top_k up to which the histogram is asked
constexpr int kBins = 256;
constexpr double kOne = 17592186044416.0;  // 2^44, the largest weight
constexpr int kLevels = 24;      // log2 of the weights that top_p may list
constexpr float kExact = -20.0f;  // log2 of the weights that count in f64

// Ordered as the floats are, -0 as +0; 0 for what is no token.
__device__ __forceinline__ uint32_t key_of(float x) {
  if (!(x > -INFINITY)) return 0;
  const uint32_t u = __float_as_uint(x + 0.0f);
  return (u >> 31) != 0 ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float((key >> 31) != 0 ? key & 0x7fffffffu : ~key);
}

// What the blocks of a cluster read of one another.
struct Shared {
  uint64_t hist[kBins];
  uint32_t near[kBins];
  uint64_t list_weight[kListed];
  uint32_t list_key[kListed];
  uint16_t list_at[kListed];
  uint64_t scan[kWarps];  // of this block alone, as the next two
  uint64_t head, tail;    // sums of the listed weights, and of the others
  uint64_t mass;
  uint32_t top;
  int listed, ties, count, first;
  int border_bin;  // of this block alone
  uint64_t border_above;
};

// The sum over the cluster's blocks of f(what a block shares), the same in every
// lane; the blocks before `upto` in `before`. A lane asks a block.
template <typename F>
__device__ __forceinline__ uint64_t over_blocks(cg::cluster_group& cluster, Shared& sh, F&& f, int upto, uint64_t& before) {
  const int lane = threadIdx.x % 32;
  uint64_t v = lane < (int)cluster.num_blocks() ? (uint64_t)f(*cluster.map_shared_rank(&sh, lane)) : 0;
  uint64_t b = lane < upto ? v : 0;
#pragma unroll
  for (int off = 8; off >= 1; off >>= 1) {
    v += __shfl_xor_sync(0xffffffffu, v, off);
    b += __shfl_xor_sync(0xffffffffu, b, off);
  }
  before = __shfl_sync(0xffffffffu, b, 0);
  return __shfl_sync(0xffffffffu, v, 0);
}
template <typename F>
__device__ __forceinline__ uint64_t over_blocks(cg::cluster_group& cluster, Shared& sh, F&& f) {
  uint64_t before;
  return over_blocks(cluster, sh, f, 0, before);
}

template <typename T>
struct Row {
  const T* x;     // this block's part of the row
  int n, first;   // its elements (some before the row's begin or past its end hold -inf), the token of the first
  float largest;
  double inv;     // 1 / temperature
  uint32_t top;

  __device__ __forceinline__ uint32_t key(int at) const { return key_of(to_f32<T>(x[at])); }
  // exp((x - largest) / temperature), 0 for what is no token.
  __device__ __forceinline__ double share(uint32_t key) const {
    if (key == top) return 1.0;
    if (key == 0 || isinf(largest)) return 0.0;
    return exp(((double)value_of(key) - (double)largest) * inv);
  }
  __device__ __forceinline__ uint64_t weight(uint32_t key) const { return (uint64_t)__double2ull_rn(share(key) * kOne); }
};

// The sum of s over the threads before this one, and over all of them in `all`.
__device__ __forceinline__ uint64_t scan_block(uint64_t s, uint64_t* warps, uint64_t& all) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  uint64_t up = s;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const uint64_t y = __shfl_up_sync(0xffffffffu, up, off);
    if (lane >= off) up += y;
  }
  __syncthreads();
  if (lane == 31) warps[warp] = up;
  __syncthreads();
  uint64_t before = 0;
  all = 0;
#pragma unroll
  for (int w = 0; w < kWarps; w++) {
    if (w < warp) before += warps[w];
    all += warps[w];
  }
  return before + up - s;
}

// Sorts n (a power of two) pairs by their first, largest first.
__device__ __forceinline__ void sort_block(uint64_t* by, uint64_t* with, int n) {
  for (int size = 2; size <= n; size <<= 1)
    for (int step = size / 2; step >= 1; step >>= 1) {
      __syncthreads();
      for (int i = threadIdx.x; i < n / 2; i += kThreads) {
        const int lo = (i & -step) * 2 | (i & (step - 1)), hi = lo + step;
        const uint64_t p = by[lo], q = by[hi];
        if ((p < q) == ((lo & size) == 0)) {
          by[lo] = q;
          by[hi] = p;
          const uint64_t w = with[lo];
          with[lo] = with[hi];
          with[hi] = w;
        }
      }
    }
  __syncthreads();
}

__device__ __forceinline__ int power_of_two(int n) { return n <= 2 ? 2 : 1 << (32 - __clz(n - 1)); }

// What top_p asks of a sum, and the place that a random number has in one.
__device__ __forceinline__ uint64_t wanted_of(float top_p, uint64_t total) {
  const double want = top_p > 0.0f ? ceil((double)top_p * (double)total) : 0.0;
  return want >= 1.0 ? (uint64_t)want : 1;
}
__device__ __forceinline__ uint64_t target_of(float u, uint64_t mass) {
  const double at = u > 0.0f ? (double)u * (double)mass : 0.0;
  return at >= (double)mass ? mass - 1 : min((unsigned long long)at, (unsigned long long)(mass - 1));
}

__device__ __forceinline__ void answer(const SampleArgs& a, int64_t row, int token, float logprob, int kept) {
  a.tokens[row] = token;
  if (a.logprobs != nullptr) a.logprobs[row] = logprob;
  if (a.kept != nullptr) a.kept[row] = kept;
}

__device__ __forceinline__ float log_share(uint64_t weight, uint64_t mass) {
  return weight == mass ? 0.0f : (float)log((double)weight / (double)mass);
}

// The largest key from which on f (counts or weights) sum to at least `want`
// over the row, eight bits at a time, and the sum of the keys above it. `f`
// gives a key's part of the sum; `less` of the sum is left out at key `at_key`.
// All blocks of the cluster come to the same.
template <typename T, typename F>
__device__ uint32_t border_of(cg::cluster_group& cluster, Shared& sh, const Row<T>& r, uint64_t want, uint64_t& above, F&& f,
                              uint32_t at_key, uint64_t less) {
  const int tid = threadIdx.x, blocks = (int)cluster.num_blocks();
  uint32_t prefix = 0;
  above = 0;
  for (int shift = 24; shift >= 0; shift -= 8) {
    sh.hist[tid] = 0;
    __syncthreads();
    for (int at = tid; at < r.n; at += kThreads) {
      const uint32_t key = r.key(at);
      if (key != 0 && (shift == 24 || key >> (shift + 8) == prefix))
        if (const uint64_t part = f(key); part != 0)
          atomicAdd(reinterpret_cast<unsigned long long*>(&sh.hist[key >> shift & 255]), (unsigned long long)part);
    }
    cluster.sync();
    // Thread t has bin 255 - t: the sums before it are those above it.
    const int bin = 255 - tid;
    uint64_t own = 0;
#pragma unroll
    for (int b = 0; b < kMaxBlocks; b++) own += b < blocks ? cluster.map_shared_rank(&sh, b)->hist[bin] : 0;
    if (less != 0 && (shift == 24 || at_key >> (shift + 8) == prefix) && (int)(at_key >> shift & 255) == bin) own -= less;
    uint64_t all;
    const uint64_t before = above + scan_block(own, sh.scan, all);
    if (before < want && before + own >= want) {
      sh.border_bin = bin;
      sh.border_above = before;
    }
    cluster.sync();  // and the block's own barrier
    prefix = prefix << 8 | (uint32_t)sh.border_bin;
    above = sh.border_above;
  }
  return prefix;
}

// Any rules, over the whole row. Returns after the answer is written.
template <typename T>
__device__ void choose_over_row(cg::cluster_group& cluster, Shared& sh, const SampleArgs& a, int64_t row, const Row<T>& r,
                                int top_k, float top_p, float min_p, float u) {
  const int tid = threadIdx.x, rank = (int)cluster.block_rank();
  uint32_t border = 1;       // tokens below it are out,
  uint64_t ties = ~0ull;     // of those at it the first so many are in
  auto one = [](uint32_t) -> uint64_t { return 1; };
  // The sum of f over the cluster's tokens.
  auto sum_of = [&](auto&& f) {
    uint64_t own = 0, all;
    for (int at = tid; at < r.n; at += kThreads) own += f(r.key(at));
    scan_block(own, sh.scan, all);
    if (tid == 0) sh.mass = all;
    cluster.sync();
    all = over_blocks(cluster, sh, [](const Shared& o) { return o.mass; });
    cluster.sync();
    return all;
  };
  if (top_k > 0 && sum_of([](uint32_t key) -> uint64_t { return key != 0; }) > (uint64_t)top_k) {
    uint64_t above;
    border = border_of(cluster, sh, r, (uint64_t)top_k, above, one, 0, 0);
    ties = (uint64_t)top_k - above;
  }
  if (top_p < 1.0f) {
    const uint64_t each = r.weight(border == 1 ? 0 : border), tied = border == 1 ? 0 : sum_of([&](uint32_t key) -> uint64_t { return key == border; });
    const uint64_t less = tied > ties ? (tied - ties) * each : 0;
    auto weight = [&](uint32_t key) { return key >= border ? r.weight(key) : 0; };
    const uint64_t total = sum_of(weight) - less, want = wanted_of(top_p, total);
    uint64_t above;
    const uint32_t at = border_of(cluster, sh, r, want, above, weight, border, less);
    const uint64_t w = r.weight(at), need = (want - above + w - 1) / w;
    if (at > border || need < ties) ties = need;
    border = at;
  }
  // Threads have contiguous tokens from here on, blocks and threads in index order.
  const int each = (r.n + kThreads - 1) / kThreads, begin = min(r.n, tid * each), end = min(r.n, begin + each);
  uint64_t tie0 = 0;  // ties before this thread's
  if (ties != ~0ull) {
    uint64_t own = 0, all;
    for (int at = begin; at < end; at++) own += r.key(at) == border;
    tie0 = scan_block(own, sh.scan, all);
    if (tid == 0) sh.ties = (int)all;
    cluster.sync();
    over_blocks(cluster, sh, [](const Shared& o) { return o.ties; }, rank, all);
    tie0 += all;
  }
  // Calls f(at, weight) for this thread's kept tokens.
  auto each_kept = [&](auto&& f) {
    uint64_t tie = tie0;
    for (int at = begin; at < end; at++) {
      const uint32_t key = r.key(at);
      if (key == 0 || key < border || (key == border && tie++ >= ties)) continue;
      const double share = r.share(key);
      if (key != r.top && min_p > 0.0f && share < (double)min_p) continue;
      if (f(at, (uint64_t)__double2ull_rn(share * kOne))) break;
    }
  };
  uint64_t own = 0, kept = 0, mass, count;
  each_kept([&](int, uint64_t w) {
    own += w;
    kept++;
    return false;
  });
  uint64_t before = scan_block(own, sh.scan, mass);
  scan_block(kept, sh.scan, count);
  if (tid == 0) {
    sh.mass = mass;
    sh.count = (int)count;
  }
  cluster.sync();
  uint64_t blocks_before;
  mass = over_blocks(cluster, sh, [](const Shared& o) { return o.mass; }, rank, blocks_before);
  before += blocks_before;
  count = over_blocks(cluster, sh, [](const Shared& o) { return o.count; });
  cluster.sync();  // the others have read this block's
  const uint64_t target = target_of(u, mass);
  if (before <= target && target < before + own)
    each_kept([&](int at, uint64_t w) {
      before += w;
      if (before <= target) return false;
      answer(a, row, r.first + at, log_share(w, mass), (int)count);
      return true;
    });
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 4) sample_kernel(const __grid_constant__ SampleArgs a, int block_vecs) {
  pdl_launch_dependents();
  pdl_wait();
  constexpr int V = 16 / sizeof(T);
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ Shared sh;
  cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x, lane = tid % 32, blocks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int64_t row = blockIdx.x / (unsigned)blocks;
  const T* in = static_cast<const T*>(a.logits) + row * a.stride;
  const int vocab = (int)a.vocab;
  // A block's part begins at a 16-byte boundary: the first's up to V - 1 elements before the row.
  const int shift = (int)(((uintptr_t)in & 15) / sizeof(T));
  T* x = reinterpret_cast<T*>(smem);
  Row<T> r;
  r.x = x;
  r.first = rank * block_vecs * V - shift;
  r.n = max(0, min(block_vecs * V, (vocab - r.first + V - 1) / V * V));
  if (tid == 0) {
    sh.top = 0;
    sh.listed = 0;
    sh.head = sh.tail = 0;
    sh.first = INT32_MAX;
  }
  sh.near[tid] = 0;
  float own = -INFINITY;  // this thread's largest
  constexpr int kAtOnce = 10;
  for (int v0 = tid; v0 < r.n / V; v0 += kThreads * kAtOnce) {
    uint4 raw[kAtOnce];
#pragma unroll
    for (int i = 0; i < kAtOnce; i++) {
      const int v = v0 + i * kThreads, token = r.first + v * V;
      if (v >= r.n / V) continue;
      if (token >= 0 && token + V <= vocab) {
        raw[i] = __ldcs(reinterpret_cast<const uint4*>(in + token));
      } else {
        T e[V];
#pragma unroll
        for (int j = 0; j < V; j++) e[j] = token + j >= 0 && token + j < vocab ? in[token + j] : from_f32<T>(-INFINITY);
        memcpy(&raw[i], e, 16);
      }
    }
#pragma unroll
    for (int i = 0; i < kAtOnce; i++) {
      const int v = v0 + i * kThreads;
      if (v >= r.n / V) continue;
      *reinterpret_cast<uint4*>(x + v * V) = raw[i];
      T e[V];
      memcpy(e, &raw[i], 16);
#pragma unroll
      for (int j = 0; j < V; j++) own = fmaxf(own, to_f32<T>(e[j]));  // NaN is left out
    }
  }
  __syncthreads();
  const uint32_t warp_top = __reduce_max_sync(0xffffffffu, key_of(own));
  if (lane == 0) atomicMax(&sh.top, warp_top);
  cluster.sync();
  uint32_t top = lane < blocks ? cluster.map_shared_rank(&sh, lane)->top : 0;
  r.top = top = __reduce_max_sync(0xffffffffu, top);
  r.largest = value_of(top);
  Shared* first = cluster.map_shared_rank(&sh, 0);

  const Sampling& how = a.how;
  const float temperature = how.temperature != nullptr ? how.temperature[row] : 1.0f;
  int top_k = how.top_k != nullptr ? max(0, how.top_k[row]) : 0;
  if (top_k >= vocab) top_k = 0;
  const float top_p = how.top_p != nullptr ? how.top_p[row] : 1.0f;
  const float min_p = how.min_p != nullptr ? how.min_p[row] : 0.0f;
  const float u = how.uniform[row];
  const bool p = top_p < 1.0f, m = min_p > 0.0f;
  r.inv = 1.0 / (double)temperature;

  if (top == 0 || !(temperature > 0.0f) || min_p > 1.0f) {  // no token, or the first one alone
    if (top != 0) {
      int least = INT32_MAX;
      for (int at = tid; at < r.n; at += kThreads)
        if (r.key(at) == top) least = min(least, r.first + at);
      least = __reduce_min_sync(0xffffffffu, least);
      if (lane == 0 && least != INT32_MAX) atomicMin(&first->first, least);
    }
    cluster.sync();
    if (rank == 0 && tid == 0) {
      if (top == 0) answer(a, row, -1, -INFINITY, 0);
      else answer(a, row, sh.first, 0.0f, 1);
    }
    return;
  }
  const float per = (float)(1.4426950408889634 * r.inv);  // weights' log2 of a logit
  if ((top_k == 0 && !p && !m) || top_k > kMostK || isinf(r.largest)) {
    choose_over_row(cluster, sh, a, row, r, top_k, top_p, min_p, u);
    return;
  }

  // ---- how far below the largest a token may be and matter
  float far = NAN;  // in logits; NaN: any distance, an infinite one too
  if (top_k > 0) {
    // Bins of an eighth of an octave of the distance, from 2^-16 to 2^16.
    constexpr int kBase = (127 - 16) * 8;
    if (own > -INFINITY) {
      const int bin = (int)(__float_as_uint(r.largest - own) >> 20) - kBase;
      atomicAdd(&sh.near[min(max(bin, 0), kBins - 1)], 1u);
    }
    cluster.sync();
    uint32_t bin_own = 0;
#pragma unroll
    for (int b = 0; b < kMaxBlocks; b++) bin_own += b < blocks ? cluster.map_shared_rank(&sh, b)->near[tid] : 0;
    uint64_t all;
    const uint64_t before = scan_block(bin_own, sh.scan, all);
    if (tid == 0) sh.border_bin = kBins - 1;
    __syncthreads();
    if (before < (uint64_t)top_k && before + bin_own >= (uint64_t)top_k) sh.border_bin = tid;
    __syncthreads();
    if (sh.border_bin < kBins - 1) far = __uint_as_float((uint32_t)(sh.border_bin + kBase + 1) << 20);
  }
  auto log2_weight = [&](float z) { return (z - r.largest) * per; };
  // Calls f(place, logit) for this thread's tokens.
  auto each_token = [&](auto&& f) {
    for (int v = tid; v < r.n / V; v += kThreads) {
      T e[V];
      const uint4 raw = *reinterpret_cast<const uint4*>(x + v * V);
      memcpy(e, &raw, 16);
#pragma unroll
      for (int j = 0; j < V; j++)
        if (const float z = to_f32<T>(e[j]); z > -INFINITY) f(v * V + j, z);
    }
  };
  // min_p's cut may not touch what top_p sums. The margin is what f32 may be off by.
  float low = -INFINITY;  // log2 of a weight
  if (m && !p) low = log2f(min_p) * 1.00001f - 0.001f;
  const bool sums = p && top_k == 0;  // the rest of the row counts in top_p's sum
  if (sums) {
    // Weights in steps of 2^-16 by their log2, the small ones in the last bin.
    each_token([&](int, float z) {
      const float l = log2_weight(z);
      const uint32_t w = __float2uint_rn(exp2f(l + 16.0f));
      if (w != 0) atomicAdd(&sh.near[(int)min(-l, (float)(kLevels - 1))], w);
    });
    cluster.sync();
    // A lane has a bin: enough are those that hold the share and a little more.
    float bin_own = 0.0f;
#pragma unroll
    for (int b = 0; b < kMaxBlocks; b++)
      if (b < blocks && lane < kLevels) bin_own += (float)cluster.map_shared_rank(&sh, b)->near[lane];
    float upto = bin_own;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const float y = __shfl_up_sync(0xffffffffu, upto, off);
      if (lane >= off) upto += y;
    }
    const float whole = __shfl_sync(0xffffffffu, upto, 31);
    const unsigned enough = __ballot_sync(0xffffffffu, upto >= (top_p + 0.002f) * whole);
    low = -(float)min(enough != 0 ? __ffs(enough) : kLevels, kLevels - 1);
  }
  uint64_t head = 0, tail = 0;
  each_token([&](int place, float z) {
    const float l = log2_weight(z);
    if (!(r.largest - z >= far) && !(l < low)) {
      const int at = atomicAdd(&sh.listed, 1);
      if (at < kListed) sh.list_at[at] = (uint16_t)place;
    } else if (sums) {
      tail += l < kExact ? __float2uint_rn(exp2f(l + 44.0f)) : r.weight(key_of(z));
    }
  });
  __syncthreads();
  const int listed = min(sh.listed, kListed);
  for (int i = tid; i < listed; i += kThreads) {
    const uint32_t key = r.key(sh.list_at[i]);
    const uint64_t w = r.weight(key);
    sh.list_key[i] = key;
    sh.list_weight[i] = w;
    head += w;
  }
  if (sums) {
    uint64_t all;
    scan_block(head, sh.scan, all);
    if (tid == 0) sh.head = all;
    scan_block(tail, sh.scan, all);
    if (tid == 0) sh.tail = all;
  }
  cluster.sync();
  // ---- whether the lists hold what matters
  uint64_t before_block;
  const int total = (int)over_blocks(cluster, sh, [](const Shared& o) { return o.listed; }, rank, before_block);
  const bool over = over_blocks(cluster, sh, [](const Shared& o) { return o.listed > kListed; }) != 0;
  if (sums) {
    head = over_blocks(cluster, sh, [](const Shared& o) { return o.head; });
    tail = over_blocks(cluster, sh, [](const Shared& o) { return o.tail; });
  }
  if (over || total > kSorted || (sums && head < wanted_of(top_p, head + tail))) {
    cluster.sync();  // the lists have been read
    choose_over_row(cluster, sh, a, row, r, top_k, top_p, min_p, u);
    return;
  }
  // ---- the first block sorts and decides, over its part of the row
  uint64_t* by = reinterpret_cast<uint64_t*>(cluster.map_shared_rank(smem, 0));
  uint64_t* with = by + kSorted;
  const int n2 = power_of_two(total);
  for (int i = tid; i < listed; i += kThreads) {
    by[before_block + i] = (uint64_t)sh.list_key[i] << 32 | (uint32_t)~(r.first + (int)sh.list_at[i]);
    with[before_block + i] = sh.list_weight[i];
  }
  if (rank == 0)
    for (int i = total + tid; i < n2; i += kThreads) by[i] = with[i] = 0;
  cluster.sync();
  if (rank != 0) return;
  by = reinterpret_cast<uint64_t*>(smem);
  with = by + kSorted;
  sort_block(by, with, n2);
  int kept = top_k > 0 ? min(top_k, total) : total;
  // Threads have contiguous places; `upto` is what lies before a thread's.
  const int each = (n2 + kThreads - 1) / kThreads, begin = min(n2, tid * each), end = min(n2, begin + each);
  if (p) {
    uint64_t sum = 0, all;
    for (int i = begin; i < end; i++)
      if (i < kept) sum += with[i];
    const uint64_t upto = scan_block(sum, sh.scan, all), want = wanted_of(top_p, all + tail);
    if (tid == 0) sh.count = kept;
    __syncthreads();
    if (upto < want && upto + sum >= want) {
      uint64_t run = upto;
      for (int i = begin; i < end && i < kept; i++) {
        run += with[i];
        if (run >= want) {
          sh.count = i + 1;
          break;
        }
      }
    }
    __syncthreads();
    kept = sh.count;
  }
  if (m) {
    int in = 0;
    for (int i = begin; i < end && i < kept; i++) {
      const uint32_t key = (uint32_t)(by[i] >> 32);
      in += key == top || r.share(key) >= (double)min_p;
    }
    uint64_t all;
    scan_block((uint64_t)in, sh.scan, all);
    kept = (int)all;
  }
  // The kept ones in index order.
  const int k2 = power_of_two(kept);
  __syncthreads();
  for (int i = tid; i < k2; i += kThreads) {
    by[i] = i < kept ? by[i] & 0xffffffffu : 0;  // the complement of the token
    with[i] = i < kept ? with[i] : 0;
  }
  sort_block(by, with, k2);
  const int per_thread = (k2 + kThreads - 1) / kThreads, from = min(k2, tid * per_thread), to = min(k2, from + per_thread);
  uint64_t sum = 0, mass;
  for (int i = from; i < to; i++) sum += with[i];
  uint64_t run = scan_block(sum, sh.scan, mass);
  const uint64_t target = target_of(u, mass);
  if (run <= target && target < run + sum)
    for (int i = from; i < to; i++) {
      run += with[i];
      if (run > target) {
        answer(a, row, (int)~(uint32_t)by[i], log_share(with[i], mass), kept);
        break;
      }
    }
}

template <typename T>
cudaError_t launch_type(const SampleArgs& a, cudaStream_t stream, bool pdl) {
  constexpr int V = 16 / sizeof(T);
  // The fewest blocks whose part of a row is 40 KB at most, so that four of them share an SM.
  const int64_t vecs = (a.vocab + 2 * V - 2) / V;
  int blocks = 1;
  while (blocks < kMaxBlocks && (vecs + blocks - 1) / blocks * 16 > 40960) blocks *= 2;
  const int64_t block_vecs = (vecs + blocks - 1) / blocks < 1 ? 1 : (vecs + blocks - 1) / blocks;
  const int bytes = block_vecs * 16 > kSorted * 16 ? (int)block_vecs * 16 : kSorted * 16;
  constexpr int most = (int)(kMaxSampleVocab / kMaxBlocks + V) * (int)sizeof(T);
  if (cudaError_t e = allow_smem<sample_kernel<T>>(most > kSorted * 16 ? most : kSorted * 16); e != cudaSuccess) return e;
  if (blocks > 8)
    if (cudaError_t e = cudaFuncSetAttribute(sample_kernel<T>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        e != cudaSuccess)
      return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.n * blocks));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = (size_t)bytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)blocks;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, sample_kernel<T>, a, (int)block_vecs);
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
