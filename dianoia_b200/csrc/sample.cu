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
// Their weights and keys go to the first block's shared memory, which sorts them
// and decides alone while the others leave. top_p alone may keep any number of
// tokens: all weights go into a histogram by their log2, whose border bin's
// tokens are the ones that are sorted; without a rule but the temperature there
// is nothing to sort. Then every block knows what it keeps, and the one that the
// random number falls to looks for the token. Where more tokens matter than the
// lists hold (thousands of top_k, many ties) the border is found eight bits of the
// key at a time over all of the row in the cluster's shared memory.
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
constexpr int kSteps = 1024;      // bins of top_p's histogram,
constexpr float kPerOctave = 32;  // so many to an octave of weights

// The cluster's barrier counts whole warps: lanes that leave a loop a turn late
// would be counted as there, their additions still to come (seen as sums that
// lacked a few tokens). The block's own barrier waits for every thread.
__device__ __forceinline__ void sync_all(cg::cluster_group& cluster) {
  __syncthreads();
  __syncwarp();
  cluster.sync();
}

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
  // A histogram's sums in three parts of 15 bits, which shared memory adds by
  // itself (64-bit additions are loops there); the share's border tokens over it.
  union {
    uint32_t part[3][kSteps];
    uint64_t sorted[kSteps];
  };
  uint32_t near[kBins];
  uint32_t list_key[kListed];
  uint16_t list_at[kListed];
  uint64_t scan[kWarps];  // of this block alone, as the next two
  uint64_t mass, border, rest;
  uint32_t top, most, least;
  int listed, ties, count, first;
  int border_bin, look_begin, look_end, look_last;
  uint64_t look_before;
  uint64_t border_above;
};

__device__ __forceinline__ void add_to_bin(Shared& sh, int bin, uint64_t w) {
  const uint32_t low = (uint32_t)w & 0x7fff, mid = (uint32_t)(w >> 15) & 0x7fff, high = (uint32_t)(w >> 30);
  if (low != 0) atomicAdd(&sh.part[0][bin], low);
  if (mid != 0) atomicAdd(&sh.part[1][bin], mid);
  if (high != 0) atomicAdd(&sh.part[2][bin], high);
}
__device__ __forceinline__ uint64_t bin_sum(const Shared& sh, int bin) {
  return sh.part[0][bin] + ((uint64_t)sh.part[1][bin] << 15) + ((uint64_t)sh.part[2][bin] << 30);
}

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
  double inv, per256;       // 1 / temperature; of a logit, in 256ths of an octave of weights
  const double* powers;     // 2^(i / 256)
  uint32_t top;

  __device__ __forceinline__ uint32_t key(int at) const { return key_of(to_f32<T>(x[at])); }
  // exp((x - largest) / temperature), 0 for what is no token.
  __device__ __forceinline__ double share(uint32_t key) const {
    if (key == top) return 1.0;
    if (key == 0 || isinf(largest)) return 0.0;
    return exp(((double)value_of(key) - (double)largest) * inv);
  }
  // The same in steps of 2^-44: 2^t with t in 256ths, the whole ones' part from
  // `powers`, and the power series of 2^(r / 256) about 0 for the rest: |r| <= 1/2
  // leaves (ln2 / 512)^5 / 5! = 2^-54 of it out. A few keys side by side: a chain
  // of f64 operations is long, and their number is what a row without cuts costs
  // (11 a token; a series for all of 2^f took 17, and 256 rows 163 us for 121).
  template <int N>
  __device__ __forceinline__ void weights(const uint32_t (&key)[N], uint64_t (&w)[N]) const {
    constexpr double kSeries[5] = {1.0, 0.0027076061740622863, 3.665565596910106e-06, 3.308302680541371e-09, 2.239395190875157e-12};
    constexpr double kWhole = 6755399441055744.0;  // 1.5 2^52: the whole part of a sum lands in the low bits
    double t[N], n[N], r[N], y[N];
#pragma unroll
    for (int i = 0; i < N; i++) {
      t[i] = ((double)value_of(key[i]) - (double)largest) * per256;
      n[i] = t[i] + kWhole;
      r[i] = t[i] - (n[i] - kWhole);
      y[i] = kSeries[4];
    }
#pragma unroll
    for (int k = 3; k >= 0; k--)
#pragma unroll
      for (int i = 0; i < N; i++) y[i] = fma(y[i], r[i], kSeries[k]);
#pragma unroll
    for (int i = 0; i < N; i++) {
      // 2^(44 + n / 256) by the exponent; then the nearest whole number by 2^52.
      const int whole = __double2loint(n[i]);
      y[i] *= powers[whole & 255];
      y[i] = __hiloint2double(__double2hiint(y[i]) + ((whole >> 8) + 44) * (1 << 20), __double2loint(y[i]));
      w[i] = (uint64_t)__double_as_longlong(y[i] + 4503599627370496.0) & 0xfffffffffffffull;
      if (!(t[i] > -46.0 * 256) || key[i] == 0) w[i] = 0;
      if (key[i] == top) w[i] = (uint64_t)1 << 44;
    }
  }
  __device__ __forceinline__ uint64_t weight(uint32_t key) const {
    const uint32_t keys[1] = {key};
    uint64_t w[1];
    weights(keys, w);
    return w[0];
  }
  // Calls f(place, key, weight) for places at0, at0 + step, .. below end, in order.
  template <typename F>
  __device__ __forceinline__ void each_weight(int at0, int end, int step, F&& f) const {
    constexpr int N = 4;
    for (int at = at0; at < end; at += N * step) {
      uint32_t k[N];
      uint64_t w[N];
#pragma unroll
      for (int i = 0; i < N; i++) k[i] = at + i * step < end ? key(at + i * step) : 0;
      weights(k, w);
#pragma unroll
      for (int i = 0; i < N; i++)
        if (k[i] != 0) f(at + i * step, k[i], w[i]);
    }
  }
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
template <bool WITH>
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
          if constexpr (WITH) {
            const uint64_t w = with[lo];
            with[lo] = with[hi];
            with[hi] = w;
          }
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

// Of the histograms that the cluster's blocks have in the first `bins` of theirs
// (a power of two; `more` at the last bin besides), the bin in which the sum over
// the bins before and with it, and `base`, comes to want(whole sum); above: the sum
// before it. Every block sums a part of the bins over the blocks.
template <typename F>
__device__ int border_bin(cg::cluster_group& cluster, Shared& sh, int bins, uint64_t base, uint64_t more, int less_at,
                          uint64_t less, F&& want_of, uint64_t& want, uint64_t& above) {
  const int tid = threadIdx.x, lane = tid % 32, blocks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int share = bins / blocks, per = max(1, share / kThreads), first = rank * share + tid * per;
  uint64_t own[kSteps / kThreads], sum = 0, all;
#pragma unroll
  for (int i = 0; i < kSteps / kThreads; i++) {
    own[i] = 0;
    if (i >= per || tid * per + i >= share) continue;
    const int bin = first + i;
    // All blocks' at once: loads behind conditions would wait for one another.
    uint32_t parts[kMaxBlocks][3];
#pragma unroll
    for (int b = 0; b < kMaxBlocks; b++)
#pragma unroll
      for (int j = 0; j < 3; j++) parts[b][j] = cluster.map_shared_rank(&sh, min(b, blocks - 1))->part[j][bin];
#pragma unroll
    for (int b = 0; b < kMaxBlocks; b++)
      if (b < blocks) own[i] += parts[b][0] + ((uint64_t)parts[b][1] << 15) + ((uint64_t)parts[b][2] << 30);
    own[i] += bin == bins - 1 ? more : 0;
    own[i] -= bin == less_at ? less : 0;
    sum += own[i];
  }
  uint64_t run = scan_block(sum, sh.scan, all);
  if (tid == 0) sh.mass = all;
  sync_all(cluster);
  const uint64_t part = lane < blocks ? cluster.map_shared_rank(&sh, lane)->mass : 0;
  uint64_t upto = part;
#pragma unroll
  for (int off = 1; off < kMaxBlocks; off <<= 1) {
    const uint64_t y = __shfl_up_sync(0xffffffffu, upto, off);
    if (lane >= off) upto += y;
  }
  want = want_of(__shfl_sync(0xffffffffu, upto, kMaxBlocks - 1));
  const uint64_t before = base + upto - part;
  const int owner = __ffs(__ballot_sync(0xffffffffu, lane < blocks && before < want && before + part >= want)) - 1;
  run += __shfl_sync(0xffffffffu, before, rank);
  if (owner == rank) {
#pragma unroll
    for (int i = 0; i < kSteps / kThreads; i++) {
      if (run < want && run + own[i] >= want) {
        sh.border_bin = first + i;
        sh.border_above = run;
      }
      run += own[i];
    }
  }
  sync_all(cluster);
  const Shared* other = cluster.map_shared_rank(&sh, max(owner, 0));
  above = other->border_above;
  return other->border_bin;
}

// The largest key from which on f (counts or weights) sum to at least `want`
// over the row, eight bits at a time, and the sum of the keys above it. `f`
// gives a key's part of the sum; `less` of the sum is left out at key `at_key`.
// All blocks of the cluster come to the same.
template <typename T, typename F>
__device__ uint32_t border_of(cg::cluster_group& cluster, Shared& sh, const Row<T>& r, uint64_t want, uint64_t& above, F&& f,
                              uint32_t at_key, uint64_t less) {
  const int tid = threadIdx.x;
  uint32_t prefix = 0;
  above = 0;
  for (int shift = 24; shift >= 0; shift -= 8) {
    auto inside = [&](uint32_t key) { return shift == 24 || key >> 8 >> shift == prefix; };
    for (int i = 0; i < 3; i++) sh.part[i][tid] = 0;
    __syncthreads();
    for (int at = tid; at < r.n; at += kThreads) {
      const uint32_t key = r.key(at);
      if (key != 0 && inside(key)) add_to_bin(sh, 255 - (key >> shift & 255), f(key));  // large keys first
    }
    sync_all(cluster);
    const int less_at = less != 0 && inside(at_key) ? 255 - (int)(at_key >> shift & 255) : -1;
    uint64_t same;
    const int bin = border_bin(cluster, sh, kBins, above, 0, less_at, less, [&](uint64_t) { return want; }, same, above);
    prefix = prefix << 8 | (uint32_t)(255 - bin);
    sync_all(cluster);  // the border has been read
  }
  return prefix;
}

// Finds the token where the random number falls: among this thread's contiguous
// ones for one thread of the cluster's, which its block's first warp then looks at
// together, with that thread's `last`. before: the kept mass before a thread's,
// own: its own.
template <typename T, typename F>
__device__ void look_among(Shared& sh, const SampleArgs& a, int64_t row, const Row<T>& r, uint64_t before, uint64_t own,
                           int begin, int end, int last, uint64_t mass, uint64_t target, int count, F&& kept) {
  const bool mine = before <= target && target < before + own;
  if (mine) {
    sh.look_begin = begin;
    sh.look_end = end;
    sh.look_last = last;
    sh.look_before = before;
  }
  if (__syncthreads_or(mine) == 0 || threadIdx.x >= 32) return;
  const int lane = threadIdx.x;
  before = sh.look_before;
  end = sh.look_end;
  last = sh.look_last;
  for (int at0 = sh.look_begin; at0 < end; at0 += 32) {
    const int at = at0 + lane;
    const uint32_t key = at < end ? r.key(at) : 0;
    const uint64_t w = key != 0 && kept(key, at, last) ? r.weight(key) : 0;
    uint64_t upto = w;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const uint64_t y = __shfl_up_sync(0xffffffffu, upto, off);
      if (lane >= off) upto += y;
    }
    const unsigned past = __ballot_sync(0xffffffffu, before + upto > target);
    if (past != 0) {
      if (lane == __ffs(past) - 1) answer(a, row, r.first + at, log_share(w, mass), count);
      return;
    }
    before += __shfl_sync(0xffffffffu, upto, 31);
  }
}

// The token among those whose keys are above `border`, the first `ties` of those
// at it, less what min_p leaves out. Returns after the answer is written.
template <typename T>
__device__ void choose_by_border(cg::cluster_group& cluster, Shared& sh, const SampleArgs& a, int64_t row, const Row<T>& r,
                                 uint32_t border, uint64_t ties, float min_p, float u) {
  const int tid = threadIdx.x, rank = (int)cluster.block_rank();
  // Threads have contiguous tokens, blocks and threads in index order.
  const int each = (r.n + kThreads - 1) / kThreads, begin = min(r.n, tid * each), end = min(r.n, begin + each);
  uint64_t all;
  int last = INT32_MAX;  // the place of this thread's last tie that is in
  if (ties != ~0ull) {
    uint64_t own = 0;
    for (int at = begin; at < end; at++) own += r.key(at) == border;
    uint64_t before = scan_block(own, sh.scan, all), of_blocks;
    if (tid == 0) sh.ties = (int)all;
    sync_all(cluster);
    over_blocks(cluster, sh, [](const Shared& o) { return o.ties; }, rank, of_blocks);
    before += of_blocks;
    if (before >= ties) {
      last = -1;
    } else if (before + own > ties) {
      for (int at = begin; at < end; at++)
        if (r.key(at) == border && before++ < ties) last = at;
    }
  }
  auto kept = [&](uint32_t key, int at, int last) {
    return key != 0 && (key > border || (key == border && at <= last)) &&
           (key == r.top || !(min_p > 0.0f) || r.share(key) >= (double)min_p);
  };
  uint64_t own = 0, count = 0;
  r.each_weight(begin, end, 1, [&](int at, uint32_t key, uint64_t w) {
    const bool in = kept(key, at, last);
    own += in ? w : 0;
    count += in;
  });
  uint64_t counts;
  scan_block(count, sh.scan, counts);
  uint64_t before = scan_block(own, sh.scan, all);
  if (tid == 0) {
    sh.mass = all;
    sh.count = (int)counts;
  }
  sync_all(cluster);
  uint64_t of_blocks;
  const uint64_t mass = over_blocks(cluster, sh, [](const Shared& o) { return o.mass; }, rank, of_blocks);
  counts = over_blocks(cluster, sh, [](const Shared& o) { return o.count; });
  sync_all(cluster);  // the others have read this block's
  before += of_blocks;
  look_among(sh, a, row, r, before, own, begin, end, last, mass, target_of(u, mass), (int)counts, kept);
}

// Any rules, over the whole row. Returns after the answer is written.
template <typename T>
__device__ void choose_over_row(cg::cluster_group& cluster, Shared& sh, const SampleArgs& a, int64_t row, const Row<T>& r,
                                int top_k, float top_p, float min_p, float u) {
  const int tid = threadIdx.x;
  uint32_t border = 1;    // tokens below it are out,
  uint64_t ties = ~0ull;  // of those at it the first so many are in
  // The sum of f over the cluster's tokens.
  auto sum_of = [&](auto&& f) {
    uint64_t own = 0, all;
    for (int at = tid; at < r.n; at += kThreads) own += f(r.key(at));
    scan_block(own, sh.scan, all);
    if (tid == 0) sh.mass = all;
    sync_all(cluster);
    all = over_blocks(cluster, sh, [](const Shared& o) { return o.mass; });
    sync_all(cluster);
    return all;
  };
  if (top_k > 0 && sum_of([](uint32_t key) -> uint64_t { return key != 0; }) > (uint64_t)top_k) {
    uint64_t above;
    border = border_of(cluster, sh, r, (uint64_t)top_k, above, [](uint32_t) -> uint64_t { return 1; }, 0, 0);
    ties = (uint64_t)top_k - above;
  }
  if (top_p < 1.0f) {
    const uint64_t each = border == 1 ? 0 : r.weight(border);
    const uint64_t tied = border == 1 ? 0 : sum_of([&](uint32_t key) -> uint64_t { return key == border; });
    const uint64_t less = tied > ties ? (tied - ties) * each : 0;
    auto weight = [&](uint32_t key) { return key >= border ? r.weight(key) : 0; };
    const uint64_t total = sum_of(weight) - less, want = wanted_of(top_p, total);
    uint64_t above;
    const uint32_t at = border_of(cluster, sh, r, want, above, weight, border, less);
    const uint64_t w = r.weight(at), need = (want - above + w - 1) / w;
    if (at > border || need < ties) ties = need;
    border = at;
  }
  choose_by_border(cluster, sh, a, row, r, border, ties, min_p, u);
}

// top_p alone.
template <typename T>
__device__ void choose_by_share(cg::cluster_group& cluster, Shared& sh, const SampleArgs& a, int64_t row,
                                const Row<T>& r, float top_p, float u) {
  const int tid = threadIdx.x, rank = (int)cluster.block_rank();
  constexpr int kOwn = kSteps / kThreads;  // bins of a thread
  const float per = (float)(r.per256 / 256);
  auto bin_of = [&](uint32_t key) {
    return key == r.top ? 0 : (int)fminf((r.largest - value_of(key)) * per * kPerOctave, (float)(kSteps - 1));
  };
#pragma unroll
  for (int i = 0; i < 3 * kOwn; i++) sh.part[i / kOwn][tid * kOwn + i % kOwn] = 0;
  if (tid == 0) {
    sh.most = 0;
    sh.least = ~0u;
  }
  __syncthreads();
  uint64_t rest = 0, all;  // of the last bin, where most tokens may be
  r.each_weight(tid, r.n, kThreads, [&](int, uint32_t key, uint64_t w) {
    const int bin = bin_of(key);
    if (bin < kSteps - 1) add_to_bin(sh, bin, w);
    else rest += w;
  });
  scan_block(rest, sh.scan, all);
  if (tid == 0) sh.rest = all;
  sync_all(cluster);
  rest = over_blocks(cluster, sh, [](const Shared& o) { return o.rest; });
  uint64_t want, above;
  const int border_at = border_bin(cluster, sh, kSteps, 0, rest, -1, 0, [&](uint64_t sum) { return wanted_of(top_p, sum); }, want, above);
  // The border bin's tokens in a list, those above it counted.
  uint64_t count = 0, counts, kept_above = 0;
  uint32_t most = 0, least = ~0u;
  for (int at = tid; at < r.n; at += kThreads) {
    const uint32_t key = r.key(at);
    if (key == 0) continue;
    const int bin = bin_of(key);
    count += bin < border_at;
    if (bin != border_at) continue;
    most = max(most, key);
    least = min(least, key);
    const int place = atomicAdd(&sh.listed, 1);
    if (place < kListed) sh.list_at[place] = (uint16_t)at;
  }
  most = __reduce_max_sync(0xffffffffu, most);
  least = __reduce_min_sync(0xffffffffu, least);
  if (tid % 32 == 0) {
    atomicMax(&sh.most, most);
    atomicMin(&sh.least, least);
  }
#pragma unroll
  for (int i = 0; i < kOwn; i++)
    if (tid * kOwn + i < border_at) kept_above += bin_sum(sh, tid * kOwn + i);
  scan_block(count, sh.scan, counts);
  scan_block(kept_above, sh.scan, kept_above);
  const int listed = min(sh.listed, kListed);
  for (int i = tid; i < listed; i += kThreads) sh.list_key[i] = r.key(sh.list_at[i]);
  sync_all(cluster);
  uint64_t before_block;
  const int in_bin = (int)over_blocks(cluster, sh, [](const Shared& o) { return o.listed; }, rank, before_block);
  if (over_blocks(cluster, sh, [](const Shared& o) { return o.listed > kListed; }) != 0 || in_bin > kSteps) {
    uint64_t unused;
    const uint64_t same_top = over_blocks(cluster, sh, [](const Shared& o) { return o.listed > 0 && o.most != o.least; });
    // Keys that differ between blocks: the sums of the listed blocks' keys tell.
    const uint64_t some = over_blocks(cluster, sh, [](const Shared& o) { return o.listed > 0; });
    const uint64_t keys = over_blocks(cluster, sh, [](const Shared& o) { return o.listed > 0 ? (uint64_t)o.most : 0; }, rank, unused);
    const uint32_t key = (uint32_t)(keys / some);
    const uint64_t others = over_blocks(cluster, sh, [&](const Shared& o) { return o.listed > 0 && o.most != key; });
    sync_all(cluster);  // the lists have been read
    if (same_top == 0 && others == 0) {  // ties of one key
      const uint64_t w = r.weight(key);
      choose_by_border(cluster, sh, a, row, r, key, (want - above + w - 1) / w, 0.0f, u);
    } else {
      choose_over_row(cluster, sh, a, row, r, 0, top_p, 0.0f, u);
    }
    return;
  }
  uint64_t* by = cluster.map_shared_rank(&sh, 0)->sorted;  // over what has been read; the row is still needed
  const int n2 = power_of_two(in_bin);
  for (int i = tid; i < listed; i += kThreads)
    by[before_block + i] = (uint64_t)sh.list_key[i] << 32 | (uint32_t)~(r.first + (int)sh.list_at[i]);
  if (rank == 0)
    for (int i = in_bin + tid; i < n2; i += kThreads) by[i] = 0;
  sync_all(cluster);
  if (rank == 0) {
    sort_block<false>(sh.sorted, nullptr, n2);
    const int each = (n2 + kThreads - 1) / kThreads, begin = min(n2, tid * each), end = min(n2, begin + each);
    auto weight_at = [&](int i) { return r.weight((uint32_t)(sh.sorted[i] >> 32)); };
    uint64_t sum = 0;
    for (int i = begin; i < end; i++) sum += weight_at(i);
    uint64_t upto = above + scan_block(sum, sh.scan, all);
    if (upto < want && upto + sum >= want)
      for (int i = begin; i < end; i++) {
        upto += weight_at(i);
        if (upto >= want) {
          sh.border = sh.sorted[i];
          break;
        }
      }
  }
  sync_all(cluster);
  const uint64_t border = cluster.map_shared_rank(&sh, 0)->border;
  auto composite = [&](uint32_t key, int at) { return (uint64_t)key << 32 | (uint32_t)~(r.first + at); };
  uint64_t band = 0, band_count = 0;
  for (int i = tid; i < listed; i += kThreads)
    if (composite(sh.list_key[i], sh.list_at[i]) >= border) {
      band += r.weight(sh.list_key[i]);
      band_count++;
    }
  scan_block(band, sh.scan, all);
  kept_above += all;
  scan_block(band_count, sh.scan, all);
  counts += all;
  if (tid == 0) {
    sh.mass = kept_above;
    sh.count = (int)counts;
  }
  sync_all(cluster);
  uint64_t before;
  const uint64_t mass = over_blocks(cluster, sh, [](const Shared& o) { return o.mass; }, rank, before);
  counts = over_blocks(cluster, sh, [](const Shared& o) { return o.count; });
  sync_all(cluster);  // the others have read this block's
  const uint64_t target = target_of(u, mass);
  if (!(before <= target && target < before + kept_above)) return;  // the whole block
  auto kept = [&](uint32_t key, int at, int) { return composite(key, at) >= border; };
  const int each = (r.n + kThreads - 1) / kThreads, begin = min(r.n, tid * each), end = min(r.n, begin + each);
  uint64_t own = 0;
  r.each_weight(begin, end, 1, [&](int at, uint32_t key, uint64_t w) { own += kept(key, at, 0) ? w : 0; });
  before += scan_block(own, sh.scan, all);
  look_among(sh, a, row, r, before, own, begin, end, 0, mass, target, (int)counts, kept);
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 4) sample_kernel(const __grid_constant__ SampleArgs a, int block_vecs) {
  pdl_launch_dependents();
  pdl_wait();
  constexpr int V = 16 / sizeof(T);
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ Shared sh;
  __shared__ double powers[256];
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
    sh.first = INT32_MAX;
  }
  sh.near[tid] = 0;
  powers[tid] = exp2((double)tid / 256);
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
  sync_all(cluster);
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
  r.per256 = r.inv * (1.4426950408889634 * 256);
  r.powers = powers;

  if (top == 0 || !(temperature > 0.0f) || min_p > 1.0f) {  // no token, or the first one alone
    if (top != 0) {
      int least = INT32_MAX;
      for (int at = tid; at < r.n; at += kThreads)
        if (r.key(at) == top) least = min(least, r.first + at);
      least = __reduce_min_sync(0xffffffffu, least);
      if (lane == 0 && least != INT32_MAX) atomicMin(&first->first, least);
    }
    sync_all(cluster);
    if (rank == 0 && tid == 0) {
      if (top == 0) answer(a, row, -1, -INFINITY, 0);
      else answer(a, row, sh.first, 0.0f, 1);
    }
    return;
  }
  if (top_k > kMostK || isinf(r.largest) || (top_k == 0 && p && m)) {
    choose_over_row(cluster, sh, a, row, r, top_k, top_p, min_p, u);
    return;
  }
  if (top_k == 0 && !m) {
    if (p)
      choose_by_share(cluster, sh, a, row, r, top_p, u);
    else
      choose_by_border(cluster, sh, a, row, r, 1, ~0ull, 0.0f, u);
    return;
  }
  const float per = (float)(r.per256 / 256);

  // ---- how far below the largest a token may be and matter
  float far = NAN;  // in logits; NaN: any distance, an infinite one too
  if (top_k > 0) {
    // Bins of an eighth of an octave of the distance, from 2^-16 to 2^16.
    constexpr int kBase = (127 - 16) * 8;
    if (own > -INFINITY) {
      const int bin = (int)(__float_as_uint(r.largest - own) >> 20) - kBase;
      atomicAdd(&sh.near[min(max(bin, 0), kBins - 1)], 1u);
    }
    sync_all(cluster);
    uint32_t bin_own = 0, of_block[kMaxBlocks];
#pragma unroll
    for (int b = 0; b < kMaxBlocks; b++) of_block[b] = cluster.map_shared_rank(&sh, min(b, blocks - 1))->near[tid];
#pragma unroll
    for (int b = 0; b < kMaxBlocks; b++) bin_own += b < blocks ? of_block[b] : 0;
    uint64_t all;
    const uint64_t before = scan_block(bin_own, sh.scan, all);
    if (tid == 0) sh.border_bin = kBins - 1;
    __syncthreads();
    if (before < (uint64_t)top_k && before + bin_own >= (uint64_t)top_k) sh.border_bin = tid;
    __syncthreads();
    if (sh.border_bin < kBins - 1) far = __uint_as_float((uint32_t)(sh.border_bin + kBase + 1) << 20);
  }
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
  each_token([&](int place, float z) {
    if (!(r.largest - z >= far) && !((z - r.largest) * per < low)) {
      const int at = atomicAdd(&sh.listed, 1);
      if (at < kListed) sh.list_at[at] = (uint16_t)place;
    }
  });
  __syncthreads();
  const int listed = min(sh.listed, kListed);
  for (int i = tid; i < listed; i += kThreads) sh.list_key[i] = r.key(sh.list_at[i]);
  sync_all(cluster);
  // ---- whether the lists hold what matters
  uint64_t before_block;
  const int total = (int)over_blocks(cluster, sh, [](const Shared& o) { return o.listed; }, rank, before_block);
  const bool over = over_blocks(cluster, sh, [](const Shared& o) { return o.listed > kListed; }) != 0;
  if (over || total > kSorted) {
    sync_all(cluster);  // the lists have been read
    choose_over_row(cluster, sh, a, row, r, top_k, top_p, min_p, u);
    return;
  }
  // ---- the first block sorts and decides, over its part of the row
  uint64_t* by = reinterpret_cast<uint64_t*>(cluster.map_shared_rank(smem, 0));
  uint64_t* with = by + kSorted;
  const int n2 = power_of_two(total);
  for (int i = tid; i < listed; i += kThreads) {
    by[before_block + i] = (uint64_t)sh.list_key[i] << 32 | (uint32_t)~(r.first + (int)sh.list_at[i]);
    with[before_block + i] = r.weight(sh.list_key[i]);
  }
  if (rank == 0)
    for (int i = total + tid; i < n2; i += kThreads) by[i] = with[i] = 0;
  sync_all(cluster);
  if (rank != 0) return;
  by = reinterpret_cast<uint64_t*>(smem);
  with = by + kSorted;
  sort_block<true>(by, with, n2);
  int kept = top_k > 0 ? min(top_k, total) : total;
  // Threads have contiguous places; `upto` is what lies before a thread's.
  const int each = (n2 + kThreads - 1) / kThreads, begin = min(n2, tid * each), end = min(n2, begin + each);
  if (p) {
    uint64_t sum = 0, all;
    for (int i = begin; i < end; i++)
      if (i < kept) sum += with[i];
    const uint64_t upto = scan_block(sum, sh.scan, all), want = wanted_of(top_p, all);
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
  sort_block<true>(by, with, k2);
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
