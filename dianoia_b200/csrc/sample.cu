// The choice of a token from a row of logits (dn_sample).
//
// w_v = exp((x_v - max) / T) as whole steps of 2^-44 (64 bits hold the sum of
// 2^19 of them), so that sums have no rounding and no order. The kept tokens
// are a prefix of the row ordered by logit, equal ones by index: top_k cuts it
// by count, top_p by the sum of weights, min_p by the weight itself. Logits map
// to ordered 32-bit keys.
//
// Bytes-bound for many rows, latency for few. Few rows: a cluster of blocks holds
// one in its shared memory (38 KB a block of a 151936-token row of f32 over 16
// blocks), every token read once. Many rows: a block of 1024 threads has one to
// itself and goes over it a few times, in L2 (148 rows of f32 are 90 MB of its 126):
// the cluster's barriers, a microsecond each and more with other rows beside, cost
// 256 rows more than that (top_k 240 us, top_p 570). Both run the same steps: the
// largest logit, then the few tokens that can matter:
//  - top_k: the threads' own largest logits, one for each 37 tokens or so, in a
//    histogram of their distance from the largest one: at least k tokens are as
//    near as the k-th of these;
//  - min_p: the weight says it.
// Their weights and keys go to the first block's shared memory, which cuts them by
// histograms of their keys' bytes and decides alone while the others leave. top_p
// alone may keep any number of tokens: f32 sums by steps of 1.5 octaves of the
// weights tell where its border is to a step or two, whose weights go into a
// histogram (shared memory adds fewer than two lanes a clock: all weights in one
// took 15 of 38 us), and the border bin's tokens are the ones that the first block
// cuts; without a rule but the temperature there is nothing to cut. Then the place
// that the random number falls to is looked for by sums of blocks, warps, segments.
// Where more tokens matter than the lists hold (thousands of top_k, many ties) the
// border is found eight bits of the key at a time over all of the row.
//
// Measured at 151936 f32 logits, one row / 256 rows, us: the largest alone 5 / 51,
// no rules 13 / 116, min_p 11 / 73 to 94, top_k 17 / 88, top_k with top_p 21 / 102,
// top_p alone 33 / 227; reading 256 rows takes 24. A row without rules is bound by
// its f64 weights (30 of 54 us on an SM: about 11 operations at 64 a clock and the
// conversions), top_p by four passes and the cuts, of 114 us with a row on every
// SM: 8 the maximum, 20 the steps, 16 to 25 the bins, 42 the weights with the band, 7
// the cuts. 256 rows are 1.7 to an SM, so the last ones run on 108 of 148 SMs; two
// blocks of 512 threads to an SM instead, all rows at once, were slower (top_k 111,
// top_p 362: 156 MB do not stay in L2).
#include <algorithm>
#include <cfloat>

#include <cooperative_groups.h>

#include "dn_common.cuh"
#include "dn_launch.h"
#include "elem.cuh"
#include "kernel_smem.h"

namespace dn {
namespace {

namespace cg = cooperative_groups;

constexpr int kMaxBlocks = 16;  // of a cluster
constexpr int kGathered = 2048;  // tokens that the first block gathers
constexpr int kMostK = 1536;    // top_k up to which the histogram is asked
constexpr int kBins = 256;
constexpr int kNears = 512;     // bins of distances: 32 to an octave, from 2^-8 to 2^8 of a logit
constexpr int kDepths = 16;       // steps of weights that top_p's border is looked for in,
constexpr float kDepth = 1.5f;    // so many octaves each,
constexpr float kDeepest = 31.0f;  // and the last of them that any weight is in: 2^-46 of the largest

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

// WHOLE: a block to a row, which stays in memory; else a cluster, its parts in
// shared memory.
template <bool WHOLE>
struct Form {
  static constexpr int kThreads = WHOLE ? 1024 : 256, kWarps = kThreads / 32;
  static constexpr int kListed = WHOLE ? kGathered : 512;  // tokens that a block lists
  static constexpr int kTops = WHOLE ? 4 : 1;            // largest logits that a thread has
  static constexpr int kNear = WHOLE ? 2048 : 1024;      // tokens of top_p's border that the first block gathers
};

// What the blocks of a cluster read of one another.
template <bool WHOLE>
struct Shared {
  static constexpr int kWarps = Form<WHOLE>::kWarps, kListed = Form<WHOLE>::kListed;
  // A histogram's sums in three parts of 15 bits, which shared memory adds by
  // itself (64-bit additions are loops there).
  uint32_t part[3][kBins];
  uint64_t gathered[Form<WHOLE>::kNear];
  uint32_t near[kNears];
  uint32_t list_key[kListed];
  typename std::conditional<WHOLE, uint32_t, uint16_t>::type list_at[kListed];
  uint64_t scan[kWarps];  // of this block alone, as the next two
  uint64_t mass, border, above, rest;
  float octave[kDepths + 1];
  uint32_t top, most, least;
  int listed, ties, count, first;
  int border_bin, band_first, band_last, place;
  uint64_t border_above;
};

template <bool W>
__device__ __forceinline__ void add_to_bin(Shared<W>& sh, int bin, uint64_t w) {
  const uint32_t low = (uint32_t)w & 0x7fff, mid = (uint32_t)(w >> 15) & 0x7fff, high = (uint32_t)(w >> 30);
  if (low != 0) atomicAdd(&sh.part[0][bin], low);
  if (mid != 0) atomicAdd(&sh.part[1][bin], mid);
  if (high != 0) atomicAdd(&sh.part[2][bin], high);
}
template <bool W>
__device__ __forceinline__ uint64_t bin_sum(const Shared<W>& sh, int bin) {
  return sh.part[0][bin] + ((uint64_t)sh.part[1][bin] << 15) + ((uint64_t)sh.part[2][bin] << 30);
}

// The sum over the cluster's blocks of f(what a block shares), the same in every
// lane; the blocks before `upto` in `before`. A lane asks a block.
template <bool W, typename F>
__device__ __forceinline__ uint64_t over_blocks(cg::cluster_group& cluster, Shared<W>& sh, F&& f, int upto, uint64_t& before) {
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
template <bool W, typename F>
__device__ __forceinline__ uint64_t over_blocks(cg::cluster_group& cluster, Shared<W>& sh, F&& f) {
  uint64_t before;
  return over_blocks(cluster, sh, f, 0, before);
}

__device__ __forceinline__ float power2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The whole part of 0 <= x < 2^23: by an addition, which four times as many lanes
// do as a conversion.
__device__ __forceinline__ int whole_part(float x) { return __float_as_int(__fadd_rd(x, 8388608.0f)) & 0x7fffff; }

template <typename T>
struct Row {
  const T* x;     // this block's part of the row, in shared memory or where the caller has it
  int n, first;   // its elements (some before the row's begin or past its end hold -inf), the token of the first
  float largest, lowest;  // logits below `lowest` have weights of 2^-46 and less
  bool steep;             // there is no such f32: neighbours of `largest` may be below
  double inv, per256;     // 1 / temperature; of a logit, in 256ths of an octave of weights
  const double* powers;   // 2^(44 + i / 256)

  __device__ __forceinline__ float logit(int at) const { return to_f32<T>(x[at]); }
  __device__ __forceinline__ uint32_t key(int at) const { return key_of(logit(at)); }
  // exp((z - largest) / temperature), 0 for what is no token.
  __device__ __forceinline__ double share(float z) const {
    if (z == largest) return 1.0;
    if (!(z > -INFINITY) || isinf(largest)) return 0.0;
    return exp(((double)z - (double)largest) * inv);
  }
  // The same in steps of 2^-44: 2^t with t in 256ths, the whole ones' part from
  // `powers`, and the power series of 2^(r / 256) about 0 for the rest: |r| <= 1/2
  // leaves (ln2 / 512)^5 / 5! = 2^-54 of it out. A few logits side by side: a chain
  // of f64 operations is long, and their number, 11 a token, is what a row without
  // cuts costs. What is no token is raised to `lowest` with the rest of that.
  template <int N>
  __device__ __forceinline__ void weights(const float (&z)[N], uint64_t (&w)[N]) const {
    constexpr double kSeries[5] = {1.0, 0.0027076061740622863, 3.665565596910106e-06, 3.308302680541371e-09, 2.239395190875157e-12};
    constexpr double kWhole = 6755399441055744.0;  // 1.5 2^52: the whole part of a sum lands in the low bits
    double t[N], n[N], r[N], y[N];
    if (isinf(largest)) {
#pragma unroll
      for (int i = 0; i < N; i++) w[i] = z[i] == largest ? (uint64_t)1 << 44 : 0;
      return;
    }
#pragma unroll
    for (int i = 0; i < N; i++) t[i] = ((double)fmaxf(z[i], lowest) - (double)largest) * per256;
    if (steep)
#pragma unroll
      for (int i = 0; i < N; i++) t[i] = z[i] > -INFINITY ? fmax(((double)z[i] - (double)largest) * per256, -46.0 * 256) : -46.0 * 256;
#pragma unroll
    for (int i = 0; i < N; i++) {
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
      // The octaves by the exponent; then the nearest whole number by 2^52.
      const int whole = __double2loint(n[i]);
      y[i] *= powers[whole & 255];
      y[i] = __hiloint2double(__double2hiint(y[i]) + (whole & ~255) * 4096, __double2loint(y[i]));
      w[i] = (uint64_t)__double_as_longlong(y[i] + 4503599627370496.0) & 0xfffffffffffffull;
    }
  }
  __device__ __forceinline__ uint64_t weight(float z) const {
    const float one[1] = {z};
    uint64_t w[1];
    weights(one, w);
    return w[0];
  }
  // Elements of the 16 bytes that begin at place `at`, of this part's alone; -inf
  // for the others. Where the caller has the row, places begin `shift` before it
  // at a 16-byte boundary.
  static constexpr int V = 16 / sizeof(T);
  __device__ __forceinline__ uint4 vector(int at, int end) const {
    if (at >= 0 && at + V <= end) return *reinterpret_cast<const uint4*>(x + at);
    T e[V];
#pragma unroll
    for (int j = 0; j < V; j++) e[j] = at + j >= 0 && at + j < end ? x[at + j] : from_f32<T>(-INFINITY);
    uint4 raw;
    memcpy(&raw, e, 16);
    return raw;
  }
  __device__ __forceinline__ int shift() const { return (int)(((uintptr_t)x & 15) / sizeof(T)); }
  // Calls f(place, logit) for all of this part's tokens; for places outside, too, with -inf.
  template <bool W, typename F>
  __device__ __forceinline__ void each_logit(F&& f) const {
    constexpr int kThreads = Form<W>::kThreads;
    if constexpr (W) {
      // From L2: 48 bytes a thread on the way, as single elements 16.
      constexpr int N = 3;
      const int step = kThreads * V;
      for (int at = (int)threadIdx.x * V - shift(); at < n; at += N * step) {
        uint4 raw[N];
#pragma unroll
        for (int i = 0; i < N; i++) raw[i] = vector(at + i * step, n);
#pragma unroll
        for (int i = 0; i < N; i++) {
          T e[V];
          memcpy(e, &raw[i], 16);
#pragma unroll
          for (int j = 0; j < V; j++) f(at + i * step + j, to_f32<T>(e[j]));
        }
      }
    } else {
      constexpr int N = 4;
      for (int at = threadIdx.x; at < n; at += N * kThreads) {
        float z[N];
#pragma unroll
        for (int i = 0; i < N; i++) z[i] = at + i * kThreads < n ? logit(at + i * kThreads) : -INFINITY;
#pragma unroll
        for (int i = 0; i < N; i++) f(at + i * kThreads, z[i]);
      }
    }
  }
};

// The sum of s over the threads before this one, and over all of them in `all`.
template <bool W>
__device__ __forceinline__ uint64_t scan_block(uint64_t s, Shared<W>& sh, uint64_t& all) {
  uint64_t* warps = sh.scan;
  constexpr int kWarps = Form<W>::kWarps;
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
  if constexpr (W) {
    all = warps[lane];
    before = lane < warp ? all : 0;
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) {
      all += __shfl_xor_sync(0xffffffffu, all, off);
      before += __shfl_xor_sync(0xffffffffu, before, off);
    }
  } else {
#pragma unroll
    for (int w = 0; w < kWarps; w++) {
      if (w < warp) before += warps[w];
      all += warps[w];
    }
  }
  return before + up - s;
}

// The largest of n keys of shift + 8 bits from which on the parts sum to at least
// `want`, a byte at a time, and the sum above it; within a block.
template <bool W, typename K, typename F>
__device__ uint32_t list_border(Shared<W>& sh, int n, int shift, uint64_t want, uint64_t& above, K&& key_at, F&& part_at) {
  constexpr int kThreads = Form<W>::kThreads;
  const int tid = threadIdx.x;
  uint32_t prefix = 0;
  above = 0;
  for (; shift >= 0; shift -= 8) {
    for (int i = tid; i < 3 * kBins; i += kThreads) sh.part[i / kBins][i % kBins] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += kThreads) {
      const uint32_t key = key_at(i);
      if (key >> 8 >> shift == prefix) add_to_bin(sh, 255 - (key >> shift & 255), part_at(i));
    }
    __syncthreads();
    const uint64_t own = tid < kBins ? bin_sum(sh, tid) : 0;
    uint64_t all;
    const uint64_t before = above + scan_block(own, sh, all);
    if (before < want && before + own >= want) {
      sh.border_bin = tid;
      sh.border_above = before;
    }
    __syncthreads();
    prefix = prefix << 8 | (uint32_t)(255 - sh.border_bin);
    above = sh.border_above;
  }
  return prefix;
}

struct Gathered {
  uint64_t weight;
  uint32_t key, token;
};

// A border among listed tokens: larger keys are in, and those at `key` up to `token`.
struct Border {
  uint32_t key, token;
  __device__ __forceinline__ bool in(uint32_t k, uint32_t t) const { return k > key || (k == key && t <= token); }
};

constexpr uint32_t kLastToken = 0xffffff;  // three bytes of token; kLastToken - token orders them down

// Where the first tokens of n, by key and token, come to `want` by part_of(i)
// (0 for what is out, else the same for equal keys).
template <bool W, typename K, typename I, typename F>
__device__ Border cut_list(Shared<W>& sh, int n, uint64_t want, K&& key_at, I&& token_at, F&& part_at) {
  const int tid = threadIdx.x;
  uint64_t above, unused, own = 0, tied, each = 0;
  Border b{0, ~0u};
  b.key = list_border(sh, n, 24, want, above, key_at, part_at);
  for (int i = tid; i < n; i += Form<W>::kThreads)
    if (key_at(i) == b.key && part_at(i) != 0) {
      own++;
      each = part_at(i);
    }
  scan_block(own, sh, tied);
  if (own != 0) sh.border_above = each;  // all the same
  __syncthreads();
  each = sh.border_above;
  __syncthreads();
  const uint64_t need = (want - above + each - 1) / each;
  if (need < tied)
    b.token = kLastToken - list_border(
                               sh, n, 16, need, unused, [&](int i) { return kLastToken - token_at(i); },
                               [&](int i) -> uint64_t { return key_at(i) == b.key && part_at(i) != 0; });
  return b;
}

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

// Of the histograms that the cluster's blocks have, the bin in which the sum over
// the bins before and with it, and `base`, comes to `want`, which is asked of
// the sum over all bins; above: the sum before it. -1 where none does. `less` is
// left out at bin less_at. A block sums its part of the bins, as many lanes to a bin
// as there are blocks; all of them come to the same.
template <bool W, typename F>
__device__ int border_bin(cg::cluster_group& cluster, Shared<W>& sh, uint64_t base, int less_at, uint64_t less, F&& want_of,
                          uint64_t& want, uint64_t& above) {
  const int tid = threadIdx.x, lane = tid % 32, blocks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int bin = (rank * kBins + tid) / blocks;  // of the first kBins threads
  uint64_t own = tid < kBins ? bin_sum(*cluster.map_shared_rank(&sh, tid % blocks), bin) : 0, all;
  for (int off = 1; off < blocks; off <<= 1) own += __shfl_xor_sync(0xffffffffu, own, off);
  own -= bin == less_at ? less : 0;
  const bool speaks = tid % blocks == 0 && tid < kBins;
  const uint64_t run = scan_block(speaks ? own : 0, sh, all);
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
  const uint64_t mine = __shfl_sync(0xffffffffu, before, rank) + run;
  if (owner == rank && speaks && mine < want && mine + own >= want) {
    sh.border_bin = bin;
    sh.border_above = mine;
  }
  sync_all(cluster);
  if (owner < 0) return -1;
  const auto* other = cluster.map_shared_rank(&sh, owner);
  above = other->border_above;
  return other->border_bin;
}

// The largest key from which on f (counts or weights) sum to at least `want`
// over the row, eight bits at a time, and the sum of the keys above it. `f`
// gives a key's part of the sum; `less` of the sum is left out at key `at_key`.
// All blocks of the cluster come to the same.
template <bool W, typename T, typename F>
__device__ uint32_t border_of(cg::cluster_group& cluster, Shared<W>& sh, const Row<T>& r, uint64_t want, uint64_t& above, F&& f,
                              uint32_t at_key, uint64_t less) {
  constexpr int kThreads = Form<W>::kThreads;
  const int tid = threadIdx.x;
  uint32_t prefix = 0;
  above = 0;
  for (int shift = 24; shift >= 0; shift -= 8) {
    auto inside = [&](uint32_t key) { return shift == 24 || key >> 8 >> shift == prefix; };
    for (int i = tid; i < 3 * kBins; i += kThreads) sh.part[i / kBins][i % kBins] = 0;
    __syncthreads();
    for (int at = tid; at < r.n; at += kThreads) {
      const uint32_t key = r.key(at);
      if (key != 0 && inside(key)) add_to_bin(sh, 255 - (key >> shift & 255), f(key));  // large keys first
    }
    sync_all(cluster);
    const int less_at = less != 0 && inside(at_key) ? 255 - (int)(at_key >> shift & 255) : -1;
    uint64_t same;
    const int bin = border_bin(cluster, sh, above, less_at, less, [&](uint64_t) { return want; }, same, above);
    prefix = prefix << 8 | (uint32_t)(255 - bin);
    sync_all(cluster);  // the border has been read
  }
  return prefix;
}

// Segments of this block's part of the row, in index order: a warp has a run of
// tokens, cut into up to 32 segments of whole chunks of 128, which its lanes read
// side by side.
template <bool W, typename T>
struct Segments {
  static constexpr int kChunk = 128;
  int run, size, base, last;  // tokens of a warp, of a segment; this warp's run
  __device__ __forceinline__ explicit Segments(const Row<T>& r) {
    run = ((r.n + Form<W>::kWarps - 1) / Form<W>::kWarps + kChunk - 1) / kChunk * kChunk;
    size = (run + 32 * kChunk - 1) / (32 * kChunk) * kChunk;
    base = (int)threadIdx.x / 32 * run;
    last = min(r.n, base + run);
  }
  // The thread that has the segment of a place.
  __device__ __forceinline__ int lane_of(int at) const { return at / run * 32 + at % run / size; }
  // f(place, logit, weight) gives a token's part of the sum; a lane gets the sum
  // over its segment.
  template <bool WEIGHTS, typename F>
  __device__ __forceinline__ uint64_t sums(const Row<T>& r, F&& f) const {
    const int lane = threadIdx.x % 32;
    uint64_t mine = 0;
    constexpr int N = 4;
    for (int s = 0; base + s * size < last; s++) {
      const int begin = base + s * size, end = min(last, begin + size);
      uint64_t sum = 0;
      for (int at = begin + lane; at - lane < end; at += 32 * N) {
        float z[N];
        uint64_t w[N] = {};
#pragma unroll
        for (int i = 0; i < N; i++) z[i] = at + i * 32 < end ? r.logit(at + i * 32) : -INFINITY;
        if constexpr (WEIGHTS) r.weights(z, w);
#pragma unroll
        for (int i = 0; i < N; i++) sum += at + i * 32 < end ? f(at + i * 32, z[i], w[i]) : 0;
      }
#pragma unroll
      for (int off = 16; off >= 1; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
      if (lane == s) mine = sum;
    }
    return mine;
  }
  // The place up to which the parts sum to more than `target`, `before` of them
  // before this lane's segment, `mine` in it: for the one warp that has it, in
  // place and weight; false for the others.
  template <bool WEIGHTS, typename F>
  __device__ __forceinline__ bool find(const Row<T>& r, uint64_t before, uint64_t mine, uint64_t target, F&& f, int& place,
                                       uint64_t& part) const {
    const int lane = threadIdx.x % 32;
    const unsigned here = __ballot_sync(0xffffffffu, before <= target && target < before + mine);
    if (here == 0) return false;
    const int s = __ffs(here) - 1, begin = base + s * size, end = min(last, begin + size);
    before = __shfl_sync(0xffffffffu, before, s);
    for (int at0 = begin; at0 < end; at0 += 32) {
      const int at = at0 + lane;
      const float z = at < end ? r.logit(at) : -INFINITY;
      const uint64_t own = at < end ? f(at, z, WEIGHTS ? r.weight(z) : 0) : 0;
      uint64_t upto = own;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const uint64_t y = __shfl_up_sync(0xffffffffu, upto, off);
        if (lane >= off) upto += y;
      }
      const unsigned past = __ballot_sync(0xffffffffu, before + upto > target);
      if (past != 0) {
        place = at0 + __ffs(past) - 1;
        part = __shfl_sync(0xffffffffu, own, __ffs(past) - 1);
        return true;
      }
      before += __shfl_sync(0xffffffffu, upto, 31);
    }
    return false;
  }
};

// The answer from the tokens of which kept(logit, token) says that they are, where
// `before` is the kept mass of the blocks before this one.
template <bool W, typename T, typename F>
__device__ void find_token(Shared<W>& sh, const SampleArgs& a, int64_t row, const Row<T>& r, const Segments<W, T>& segments,
                           uint64_t before, uint64_t mine, uint64_t mass, float u, int count, F&& kept) {
  int place;
  uint64_t weight;
  if (segments.template find<true>(r, before, mine, target_of(u, mass),
                                   [&](int at, float z, uint64_t w) { return kept(z, r.first + at) ? w : 0; }, place, weight) &&
      threadIdx.x % 32 == 0)
    answer(a, row, r.first + place, log_share(weight, mass), count);
}

// The token among those whose logits are above `border`, the first `ties` of those
// at it (~0: all), less what min_p leaves out. Returns after the answer is written.
template <bool W, typename T>
__device__ void choose_by_border(cg::cluster_group& cluster, Shared<W>& sh, const SampleArgs& a, int64_t row, const Row<T>& r,
                                 float border, uint64_t ties, float min_p, float u) {
  const int tid = threadIdx.x, rank = (int)cluster.block_rank();
  const Segments<W, T> segments(r);
  uint64_t all, of_blocks;
  int last = border > -INFINITY ? INT32_MAX : INT32_MIN;  // the last token at the border that is in
  if (ties != ~0ull) {
    auto tied = [&](int, float z, uint64_t) -> uint64_t { return z == border; };
    const uint64_t mine = segments.template sums<false>(r, tied);
    uint64_t before = scan_block(mine, sh, all), part;
    if (tid == 0) {
      sh.ties = (int)all;
      sh.place = INT32_MAX;
    }
    sync_all(cluster);
    over_blocks(cluster, sh, [](const auto& o) { return o.ties; }, rank, of_blocks);
    int place;
    if (segments.template find<false>(r, before + of_blocks, mine, ties - 1, tied, place, part) && tid % 32 == 0)
      sh.place = r.first + place;
    sync_all(cluster);
    const int lane = tid % 32;
    last = lane < (int)cluster.num_blocks() ? cluster.map_shared_rank(&sh, lane)->place : INT32_MAX;
    last = __reduce_min_sync(0xffffffffu, last);
  }
  // Logits that min_p surely lets in, and that it surely does not; in f64 between.
  const float cut = min_p > 0.0f ? (float)((double)r.largest + log((double)min_p) / r.inv) : -INFINITY;
  const float in_from = min_p > 0.0f ? cut + fabsf(cut) * 1e-6f + fabsf(r.largest) * 1e-6f : -INFINITY;
  const float out_to = min_p > 0.0f ? cut - fabsf(cut) * 1e-6f - fabsf(r.largest) * 1e-6f : -INFINITY;
  auto kept = [&](float z, int token) {
    return (z > border || (z == border && token <= last)) &&
           (z >= in_from || z == r.largest || (z >= out_to && r.share(z) >= (double)min_p));
  };
  uint64_t counts, count = 0;
  const uint64_t mine = segments.template sums<true>(r, [&](int at, float z, uint64_t w) {
    const bool in = kept(z, r.first + at);
    count += in;
    return in ? w : 0;
  });
  scan_block(count, sh, counts);
  uint64_t before = scan_block(mine, sh, all);
  if (tid == 0) {
    sh.mass = all;
    sh.count = (int)counts;
  }
  sync_all(cluster);
  const uint64_t mass = over_blocks(cluster, sh, [](const auto& o) { return o.mass; }, rank, of_blocks);
  counts = over_blocks(cluster, sh, [](const auto& o) { return o.count; });
  sync_all(cluster);  // the others have read this block's
  find_token(sh, a, row, r, segments, before + of_blocks, mine, mass, u, (int)counts, kept);
}

// Any rules, over the whole row. Returns after the answer is written.
template <bool W, typename T>
__device__ void choose_over_row(cg::cluster_group& cluster, Shared<W>& sh, const SampleArgs& a, int64_t row, const Row<T>& r,
                                int top_k, float top_p, float min_p, float u) {
  constexpr int kThreads = Form<W>::kThreads;
  const int tid = threadIdx.x;
  uint32_t border = 1;    // tokens below it are out,
  uint64_t ties = ~0ull;  // of those at it the first so many are in
  // The sum of f over the cluster's tokens.
  auto sum_of = [&](auto&& f) {
    uint64_t own = 0, all;
    for (int at = tid; at < r.n; at += kThreads) own += f(r.key(at));
    scan_block(own, sh, all);
    if (tid == 0) sh.mass = all;
    sync_all(cluster);
    all = over_blocks(cluster, sh, [](const auto& o) { return o.mass; });
    sync_all(cluster);
    return all;
  };
  if (top_k > 0 && sum_of([](uint32_t key) -> uint64_t { return key != 0; }) > (uint64_t)top_k) {
    uint64_t above;
    border = border_of(cluster, sh, r, (uint64_t)top_k, above, [](uint32_t) -> uint64_t { return 1; }, 0, 0);
    ties = (uint64_t)top_k - above;
  }
  if (top_p < 1.0f) {
    const uint64_t each = border == 1 ? 0 : r.weight(value_of(border));
    const uint64_t tied = border == 1 ? 0 : sum_of([&](uint32_t key) -> uint64_t { return key == border; });
    const uint64_t less = tied > ties ? (tied - ties) * each : 0;
    auto weight = [&](uint32_t key) { return key >= border ? r.weight(value_of(key)) : 0; };
    const uint64_t total = sum_of(weight) - less, want = wanted_of(top_p, total);
    uint64_t above;
    const uint32_t at = border_of(cluster, sh, r, want, above, weight, border, less);
    const uint64_t w = r.weight(value_of(at)), need = (want - above + w - 1) / w;
    if (at > border || need < ties) ties = need;
    border = at;
  }
  choose_by_border(cluster, sh, a, row, r, border == 1 ? -INFINITY : value_of(border), ties, min_p, u);
}

// top_p alone.
template <bool W, typename T>
__device__ void choose_by_share(cg::cluster_group& cluster, Shared<W>& sh, const SampleArgs& a, int64_t row, const Row<T>& r,
                                float top_p, float u, uint8_t* smem) {
  constexpr int kThreads = Form<W>::kThreads, kWarps = Form<W>::kWarps, kListed = Form<W>::kListed;
  const int tid = threadIdx.x, lane = tid % 32, blocks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const float per = (float)(r.per256 / 256);
  // How far a token lies below the largest, in steps of kDepth octaves of weights.
  const float per_step = per / kDepth;
  auto depth_of = [&](float z) { return z == r.largest ? 0.0f : z > -INFINITY ? (r.largest - z) * per_step : INFINITY; };
  // ---- the sums to each step, and of all
  {
    float sum[kDepths] = {}, whole = 0.0f;
    if constexpr (W) {
      // A column of shared memory to a thread, with its sums of each step: 20 us of
      // 152 thousand tokens where 16 comparisons a token took 53.
      float* column = reinterpret_cast<float*>(smem) + tid;
#pragma unroll
      for (int i = 0; i < kDepths; i++) column[i * kThreads] = 0.0f;
      r.template each_logit<W>([&](int, float z) {
        const float d = depth_of(z), w = power2(-kDepth * d);
        whole += w;
        if (d < (float)kDepths) column[whole_part(d) * kThreads] += w;
      });
#pragma unroll
      for (int i = 0; i < kDepths; i++) sum[i] = column[i * kThreads] + (i > 0 ? sum[i > 0 ? i - 1 : 0] : 0.0f);
    } else {
      r.template each_logit<W>([&](int, float z) {
        const float d = depth_of(z), w = power2(-kDepth * d);
        whole += w;
#pragma unroll
        for (int i = 0; i < kDepths; i++)
          if (d < (float)(i + 1)) sum[i] += w;
      });
    }
    float mine = 0.0f;
#pragma unroll
    for (int i = 0; i <= kDepths; i++) {
      float x = i < kDepths ? sum[i < kDepths ? i : 0] : whole;
#pragma unroll
      for (int off = 16; off >= 1; off >>= 1) x += __shfl_xor_sync(0xffffffffu, x, off);
      if (lane == i) mine = x;
    }
    constexpr int kRow = kDepths + 1;
    static_assert(kWarps * kRow <= 3 * kBins, "the histogram's place holds the warps' sums");
    float* warps = reinterpret_cast<float*>(sh.part);
    if (lane < kRow) warps[tid / 32 * kRow + lane] = mine;
    __syncthreads();
    if (tid < kRow) {
      float x = 0.0f;
#pragma unroll
      for (int w = 0; w < kWarps; w++) x += warps[w * kRow + tid];
      sh.octave[tid] = x;
    }
  }
  if (tid == 0) {
    sh.most = 0;
    sh.least = ~0u;
  }
  sync_all(cluster);
  float upto = 0.0f, of_block[kMaxBlocks];
#pragma unroll
  for (int b = 0; b < kMaxBlocks; b++) of_block[b] = cluster.map_shared_rank(&sh, min(b, blocks - 1))->octave[min(lane, kDepths)];
#pragma unroll
  for (int b = 0; b < kMaxBlocks; b++) upto += b < blocks ? of_block[b] : 0.0f;
  const float whole = __shfl_sync(0xffffffffu, upto, kDepths);
  // The border lies from step `near` to `far`, whatever f32 sums may be off by.
  const unsigned enough = __ballot_sync(0xffffffffu, lane < kDepths && upto >= (top_p + 0.001f) * whole);
  const unsigned short_of = __ballot_sync(0xffffffffu, lane < kDepths && upto <= (top_p - 0.001f) * whole);
  const float near = (float)__popc(short_of), far = enough != 0 ? (float)__ffs(enough) : kDeepest;
  const float base_sum = short_of != 0 ? __shfl_sync(0xffffffffu, upto, __popc(short_of) - 1) : 0.0f;
  const float per_bin = (float)kBins / (far - near);
  // ---- the bins of those steps, in units of 2^-16 of the first one's weights
  if (tid < kBins) sh.part[0][tid] = 0;
  if (tid == 0) {
    sh.band_first = 0;
    sh.band_last = kBins - 1;
  }
  __syncthreads();
  r.template each_logit<W>([&](int, float z) {
    const float d = depth_of(z);
    if (d >= near && d < far)
      atomicAdd(&sh.part[0][min(whole_part((d - near) * per_bin), kBins - 1)], __float2uint_rn(power2(kDepth * (near - d) + 16.0f)));
  });
  sync_all(cluster);
  uint64_t all;
  {
    uint32_t of_block[kMaxBlocks];
    uint64_t own = 0;
#pragma unroll
    for (int b = 0; b < (W ? 1 : kMaxBlocks); b++) of_block[b] = cluster.map_shared_rank(&sh, min(b, blocks - 1))->part[0][tid % kBins];
#pragma unroll
    for (int b = 0; b < (W ? 1 : kMaxBlocks); b++) own += b < blocks && tid < kBins ? of_block[b] : 0;
    const uint64_t before = scan_block(own, sh, all);
    const float unit = power2(-16.0f - kDepth * near), from = base_sum + (float)before * unit, to = base_sum + (float)(before + own) * unit;
    const float less = (top_p - 2e-5f) * whole, more = (top_p + 2e-5f) * whole;
    if (tid < kBins && from <= less && less < to) sh.band_first = tid;
    if (tid < kBins && from < more && more <= to) sh.band_last = tid;
  }
  __syncthreads();
  // The band in logits, a little wider than what f32 rounds its ends by; what it
  // holds is checked below.
  const float high_step = near + (float)sh.band_first / per_bin, low_step = near + (float)(sh.band_last + 1) / per_bin;
  auto at_step = [&](float step) { return r.largest - step / per_step; };
  const float wider = (fabsf(r.largest) + low_step / per_step) * 1e-6f;
  const float high = high_step > 0.0f ? at_step(high_step) + wider : INFINITY;
  const float low = low_step < kDeepest ? at_step(low_step) - wider : -FLT_MAX;
  // ---- all weights: those above the band by segments, the band's tokens in a list
  uint64_t count = 0, counts, rest = 0;
  uint32_t most = 0, least = ~0u;
  const Segments<W, T> segments(r);
  uint64_t mine = segments.template sums<true>(r, [&](int at, float z, uint64_t w) -> uint64_t {
    if (z > high) {
      count++;
      return w;
    }
    if (!(z >= low)) {
      rest += w;
      return 0;
    }
    const uint32_t key = key_of(z);
    most = max(most, key);
    least = min(least, key);
    const int place = atomicAdd(&sh.listed, 1);
    if (place < kListed) sh.list_at[place] = at;
    return 0;
  });
  most = __reduce_max_sync(0xffffffffu, most);
  least = __reduce_min_sync(0xffffffffu, least);
  if (lane == 0) {
    atomicMax(&sh.most, most);
    atomicMin(&sh.least, least);
  }
  uint64_t above;
  scan_block(count, sh, counts);
  scan_block(mine, sh, above);
  scan_block(rest, sh, rest);
  if (tid == 0) {
    sh.above = above;
    sh.rest = rest;
  }
  const int listed = min(sh.listed, kListed);
  for (int i = tid; i < listed; i += kThreads) sh.list_key[i] = r.key(sh.list_at[i]);
  sync_all(cluster);
  uint64_t before_block;
  const int in_band = (int)over_blocks(cluster, sh, [](const auto& o) { return o.listed; }, rank, before_block);
  const uint64_t base = over_blocks(cluster, sh, [](const auto& o) { return o.above; });
  rest = over_blocks(cluster, sh, [](const auto& o) { return o.rest; });
  if (over_blocks(cluster, sh, [](const auto& o) { return o.listed > kListed; }) != 0 || in_band > Form<W>::kNear) {
    uint64_t unused;
    const uint64_t several = over_blocks(cluster, sh, [](const auto& o) { return o.listed > 0 && o.most != o.least; });
    // Keys that differ between blocks: their mean is not all of theirs.
    const uint64_t some = over_blocks(cluster, sh, [](const auto& o) { return o.listed > 0; });
    const uint64_t keys = over_blocks(cluster, sh, [](const auto& o) { return o.listed > 0 ? (uint64_t)o.most : 0; }, rank, unused);
    const uint32_t key = (uint32_t)(keys / some);
    const uint64_t others = over_blocks(cluster, sh, [&](const auto& o) { return o.listed > 0 && o.most != key; });
    sync_all(cluster);  // the lists have been read
    const uint64_t w = r.weight(value_of(key)), want = wanted_of(top_p, base + in_band * w + rest);
    if (several == 0 && others == 0 && base < want && want <= base + in_band * w)  // ties of one key
      choose_by_border(cluster, sh, a, row, r, value_of(key), (want - base + w - 1) / w, 0.0f, u);
    else
      choose_over_row(cluster, sh, a, row, r, 0, top_p, 0.0f, u);
    return;
  }
  uint64_t* to = cluster.map_shared_rank(&sh, 0)->gathered;
  for (int i = tid; i < listed; i += kThreads)
    to[before_block + i] = (uint64_t)sh.list_key[i] << 32 | (uint32_t)(r.first + (int)sh.list_at[i]);
  sync_all(cluster);
  if (rank == 0) {
    auto key_at = [&](int i) { return (uint32_t)(sh.gathered[i] >> 32); };
    auto weight_at = [&](int i) { return r.weight(value_of(key_at(i))); };
    uint64_t band = 0;
    for (int i = tid; i < in_band; i += kThreads) band += weight_at(i);
    scan_block(band, sh, band);
    const uint64_t want = wanted_of(top_p, base + band + rest);
    Border b{0, 0};  // not in the band after all
    if (base < want && want <= base + band)
      b = cut_list(sh, in_band, want - base, key_at, [&](int i) { return (uint32_t)sh.gathered[i]; }, weight_at);
    if (tid == 0) sh.border = (uint64_t)b.key << 32 | b.token;
  }
  sync_all(cluster);
  const uint64_t packed = cluster.map_shared_rank(&sh, 0)->border;
  const Border border{(uint32_t)(packed >> 32), (uint32_t)packed};
  if (border.key == 0) {
    choose_over_row(cluster, sh, a, row, r, 0, top_p, 0.0f, u);
    return;
  }
  // The band's kept tokens count in their segments. (A lane that looked through the
  // list for its own took a third of the time.)
  static_assert(Form<W>::kNear >= kThreads, "the gathered ones' place holds a sum for each segment");
  sh.gathered[tid] = 0;
  __syncthreads();
  uint64_t band_count = 0;
  for (int i = tid; i < listed; i += kThreads) {  // no more than were gathered
    const int at = (int)sh.list_at[i];
    if (!border.in(sh.list_key[i], (uint32_t)(r.first + at))) continue;
    atomicAdd(reinterpret_cast<unsigned long long*>(&sh.gathered[segments.lane_of(at)]), r.weight(value_of(sh.list_key[i])));
    band_count++;
  }
  scan_block(band_count, sh, all);
  counts += all;
  mine += sh.gathered[tid];
  uint64_t before = scan_block(mine, sh, all), of_blocks;
  if (tid == 0) {
    sh.mass = all;
    sh.count = (int)counts;
  }
  sync_all(cluster);
  const uint64_t mass = over_blocks(cluster, sh, [](const auto& o) { return o.mass; }, rank, of_blocks);
  counts = over_blocks(cluster, sh, [](const auto& o) { return o.count; });
  sync_all(cluster);  // the others have read this block's
  find_token(sh, a, row, r, segments, before + of_blocks, mine, mass, u, (int)counts,
             [&](float z, int token) { return border.in(key_of(z), (uint32_t)token); });
}

template <typename T, bool W>
__global__ void __launch_bounds__(Form<W>::kThreads, W ? 1 : 4) sample_kernel(const __grid_constant__ SampleArgs a, int block_vecs) {
  constexpr int kThreads = Form<W>::kThreads, kListed = Form<W>::kListed, kTops = Form<W>::kTops;
  pdl_launch_dependents();
  pdl_wait();
  constexpr int V = 16 / sizeof(T);
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ Shared<W> sh;
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
  r.x = W ? in : x;
  r.first = W ? 0 : rank * block_vecs * V - shift;
  r.n = W ? vocab : max(0, min(block_vecs * V, (vocab - r.first + V - 1) / V * V));
  if (tid == 0) {
    sh.top = 0;
    sh.listed = 0;
    sh.first = INT32_MAX;
  }
  if (tid < kBins) powers[tid] = exp2(44.0 + (double)tid / 256);
  for (int i = tid; i < kNears; i += kThreads) sh.near[i] = 0;
  // The row's vectors that this block has, from the one with the row's first element on.
  const int first_token = W ? -shift : r.first, vecs = W ? (vocab + shift + V - 1) / V : r.n / V;
  float tops[kTops];  // this thread's largest
#pragma unroll
  for (int i = 0; i < kTops; i++) tops[i] = -INFINITY;
  constexpr int kAtOnce = W ? 8 : 10;
  for (int v0 = tid; v0 < vecs; v0 += kThreads * kAtOnce) {
    uint4 raw[kAtOnce];
#pragma unroll
    for (int i = 0; i < kAtOnce; i++) {
      const int v = v0 + i * kThreads, token = first_token + v * V;
      if (v >= vecs) continue;
      if (token >= 0 && token + V <= vocab) {
        // Only once of a cluster's row; the others go over theirs again.
        raw[i] = W ? *reinterpret_cast<const uint4*>(in + token) : __ldcs(reinterpret_cast<const uint4*>(in + token));
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
      if (v >= vecs) continue;
      if constexpr (!W) *reinterpret_cast<uint4*>(x + v * V) = raw[i];
      T e[V];
      memcpy(e, &raw[i], 16);
#pragma unroll
      for (int j = 0; j < V; j++) tops[j % kTops] = fmaxf(tops[j % kTops], to_f32<T>(e[j]));  // NaN is left out
    }
  }
  float own = tops[0];
#pragma unroll
  for (int i = 1; i < kTops; i++) own = fmaxf(own, tops[i]);
  __syncthreads();
  const uint32_t warp_top = __reduce_max_sync(0xffffffffu, key_of(own));
  if (lane == 0) atomicMax(&sh.top, warp_top);
  sync_all(cluster);
  uint32_t top = lane < blocks ? cluster.map_shared_rank(&sh, lane)->top : 0;
  top = __reduce_max_sync(0xffffffffu, top);
  r.largest = value_of(top);
  Shared<W>* first = cluster.map_shared_rank(&sh, 0);

  const Sampling& how = a.how;
  const float temperature = how.temperature != nullptr ? how.temperature[row] : 1.0f;
  int top_k = how.top_k != nullptr ? max(0, how.top_k[row]) : 0;
  if (top_k >= vocab) top_k = 0;
  const float top_p = how.top_p != nullptr ? how.top_p[row] : 1.0f;
  const float min_p = how.min_p != nullptr ? how.min_p[row] : 0.0f;
  const float u = how.uniform[row];
  const bool p = top_p < 1.0f, m = min_p > 0.0f;
  r.inv = fmax(1.0 / (double)temperature, 1e-30);
  r.per256 = r.inv * (1.4426950408889634 * 256);
  r.lowest = (float)((double)r.largest - 46.0 * 256 / r.per256);
  const double octaves = ((double)r.largest - (double)r.lowest) * r.per256 / 256;
  r.steep = !(octaves > 45.5 && octaves < 64.0);
  r.powers = powers;

  if (top == 0 || !(temperature > 0.0f) || min_p > 1.0f) {  // no token, or the first one alone
    if (top != 0) {
      int least = INT32_MAX;
      r.template each_logit<W>([&](int at, float z) {
        if (z == r.largest) least = min(least, r.first + at);
      });
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
      choose_by_share(cluster, sh, a, row, r, top_p, u, smem);
    else
      choose_by_border(cluster, sh, a, row, r, -INFINITY, ~0ull, 0.0f, u);
    return;
  }
  const float per = (float)(r.per256 / 256);

  // ---- how far below the largest a token may be and matter
  float far = NAN;  // in logits; NaN: any distance, an infinite one too
  if (top_k > 0) {
    constexpr int kBase = (127 - 8) * 32, kPer = W ? 1 : kNears / kThreads;
#pragma unroll
    for (int i = 0; i < kTops; i++)
      if (tops[i] > -INFINITY) {
        const int bin = (int)(__float_as_uint(r.largest - tops[i]) >> 18) - kBase;
        atomicAdd(&sh.near[min(max(bin, 0), kNears - 1)], 1u);
      }
    sync_all(cluster);
    uint32_t near[kPer], mine = 0, of_block[kMaxBlocks][kPer];
#pragma unroll
    for (int b = 0; b < (W ? 1 : kMaxBlocks); b++)
#pragma unroll
      for (int i = 0; i < kPer; i++)
        of_block[b][i] = cluster.map_shared_rank(&sh, min(b, blocks - 1))->near[(tid * kPer + i) % kNears];
#pragma unroll
    for (int i = 0; i < kPer; i++) {
      near[i] = 0;
#pragma unroll
      for (int b = 0; b < (W ? 1 : kMaxBlocks); b++) near[i] += b < blocks && tid * kPer < kNears ? of_block[b][i] : 0;
      mine += near[i];
    }
    uint64_t all;
    uint64_t before = scan_block(mine, sh, all);
    if (tid == 0) sh.border_bin = kNears - 1;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kPer; i++) {
      if (before < (uint64_t)top_k && before + near[i] >= (uint64_t)top_k) sh.border_bin = tid * kPer + i;
      before += near[i];
    }
    __syncthreads();
    if (sh.border_bin < kNears - 1) far = __uint_as_float((uint32_t)(sh.border_bin + kBase + 1) << 18);
  }
  // min_p's cut may not touch what top_p sums. The margin is what f32 may be off by.
  float low = -INFINITY;  // log2 of a weight
  if (m && !p) low = log2f(min_p) * 1.00001f - 0.001f;
  r.template each_logit<W>([&](int place, float z) {
    if (z > -INFINITY && !(r.largest - z >= far) && !((z - r.largest) * per < low)) {
      const int at = atomicAdd(&sh.listed, 1);
      if (at < kListed) sh.list_at[at] = place;
    }
  });
  __syncthreads();
  const int listed = min(sh.listed, kListed);
  for (int i = tid; i < listed; i += kThreads) sh.list_key[i] = r.key(sh.list_at[i]);
  sync_all(cluster);
  // ---- whether the lists hold what matters
  uint64_t before_block;
  const int total = (int)over_blocks(cluster, sh, [](const auto& o) { return o.listed; }, rank, before_block);
  const bool over = over_blocks(cluster, sh, [](const auto& o) { return o.listed > kListed; }) != 0;
  if (over || total > kGathered) {
    sync_all(cluster);  // the lists have been read
    choose_over_row(cluster, sh, a, row, r, top_k, top_p, min_p, u);
    return;
  }
  // ---- the first block cuts and decides, over its part of the row
  Gathered* list = reinterpret_cast<Gathered*>(cluster.map_shared_rank(smem, 0));
  for (int i = tid; i < listed; i += kThreads)
    list[before_block + i] = Gathered{r.weight(value_of(sh.list_key[i])), sh.list_key[i], (uint32_t)(r.first + (int)sh.list_at[i])};
  sync_all(cluster);
  if (rank != 0) return;
  list = reinterpret_cast<Gathered*>(smem);
  auto key_at = [&](int i) { return list[i].key; };
  auto token_at = [&](int i) { return list[i].token; };
  Border border{0, ~0u};
  if (top_k > 0 && total > top_k) border = cut_list(sh, total, top_k, key_at, token_at, [](int) -> uint64_t { return 1; });
  auto part_at = [&](int i) { return border.in(list[i].key, list[i].token) ? list[i].weight : 0; };
  auto sum_kept = [&](uint64_t& count) {
    uint64_t sum = 0, some = 0;
    for (int i = tid; i < total; i += kThreads) {
      const uint64_t w = part_at(i);
      sum += w;
      some += border.in(list[i].key, list[i].token);
    }
    scan_block(some, sh, count);
    scan_block(sum, sh, sum);
    return sum;
  };
  uint64_t kept, mass = sum_kept(kept);
  if (p) {
    Border by_share = cut_list(sh, total, wanted_of(top_p, mass), key_at, token_at, part_at);
    if (by_share.key == border.key) by_share.token = min(by_share.token, border.token);  // top_k's cut among equals stays
    border = by_share;
    mass = sum_kept(kept);
  }
  if (m) {  // these are the last ones, but for the largest
    __syncthreads();
    for (int i = tid; i < total; i += kThreads)
      if (const uint32_t key = list[i].key; key != top && !(r.share(value_of(key)) >= (double)min_p)) list[i].key = 0;
    if (border.key == 0) border.key = 1;
    __syncthreads();
    mass = sum_kept(kept);
  }
  uint64_t unused;
  const uint32_t token = kLastToken - list_border(
                                          sh, total, 16, target_of(u, mass) + 1, unused,
                                          [&](int i) { return kLastToken - list[i].token; }, part_at);
  for (int i = tid; i < total; i += kThreads)
    if (list[i].token == token) answer(a, row, (int)token, log_share(list[i].weight, mass), (int)kept);
}

// From so many rows on a row is one block's: 49 rows are more than the 32 or so
// clusters of 16 blocks that the GPU runs at once.
constexpr int64_t kMany = 49;

template <typename T, bool W>
cudaError_t launch_form(const SampleArgs& a, int blocks, int block_vecs, int bytes, cudaStream_t stream, bool pdl) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.n * blocks));
  cfg.blockDim = dim3(Form<W>::kThreads);
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
  return cudaLaunchKernelEx(&cfg, sample_kernel<T, W>, a, block_vecs);
}

template <typename T>
cudaError_t launch_type(const SampleArgs& a, cudaStream_t stream, bool pdl) {
  constexpr int V = 16 / sizeof(T);
  if (a.n >= kMany) {
    // The gathered tokens, or the columns of top_p's steps.
    constexpr int bytes = std::max(kGathered * 16, kDepths * Form<true>::kThreads * (int)sizeof(float));
    if (cudaError_t e = allow_smem<sample_kernel<T, true>>(bytes); e != cudaSuccess) return e;
    return launch_form<T, true>(a, 1, 0, bytes, stream, pdl);
  }
  // The fewest blocks whose part of a row is 40 KB at most, so that four of them share an SM.
  const int64_t vecs = (a.vocab + 2 * V - 2) / V;
  int blocks = 1;
  while (blocks < kMaxBlocks && (vecs + blocks - 1) / blocks * 16 > 40960) blocks *= 2;
  const int64_t block_vecs = (vecs + blocks - 1) / blocks < 1 ? 1 : (vecs + blocks - 1) / blocks;
  const int bytes = block_vecs * 16 > kGathered * 16 ? (int)block_vecs * 16 : kGathered * 16;
  constexpr int most = (int)(kMaxSampleVocab / kMaxBlocks + V) * (int)sizeof(T);
  if (cudaError_t e = allow_smem<sample_kernel<T, false>>(most > kGathered * 16 ? most : kGathered * 16); e != cudaSuccess)
    return e;
  if (blocks > 8)
    if (cudaError_t e = cudaFuncSetAttribute(sample_kernel<T, false>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        e != cudaSuccess)
      return e;
  return launch_form<T, false>(a, blocks, (int)block_vecs, bytes, stream, pdl);
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
