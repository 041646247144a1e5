// Attention over a paged cache for a batch whose sequences share a prefix
// (dn_paged_attention): out = softmax(scale q . k) v over the positions a
// query sees, the shared ones read once for every query of the batch.
// paged_attention.cuh says how the work is divided and joined.
#include "paged_attention.cuh"

namespace dn {

using namespace paged;

namespace {

// ------------------------------------------------------- the f32 arithmetic
//
// Any type, head size up to 256 and alignment; f32 caches first of all, whose
// products the tensor cores would round. Bound by the keys' bytes for the few
// rows of a decode step (a block holds a sequence's rows, at most 8, and reads
// its keys for them, the prefix's too), so nothing goes through shared memory: a warp's lanes
// lie along the head (V dimensions each, 32 V more on), and a step of 32 / RT
// keys is 32 / RT whole rows loaded at once for RT rows of queries. The 32
// partial products of a lane are summed over the lanes by halves (31
// exchanges for 32 sums), which leaves lane l with the score of key l / RT for
// row l % RT; each probability goes back to all lanes for the values. A block's
// 4 warps take steps in turn and are joined once at the end.
// Measured: 7 sequences of 680 keys, 8 kv heads of 128, 2 heads a group, window
// 600: 12.6 us with the join (46 us with tiles in shared memory, where a block's
// 16 rows were mostly empty). What it costs where rows are many or a 16-bit cache
// is not the tensor cores': a prompt of 2048 f32 tokens (16 heads of 128) 884 us;
// 32 chat sequences of a bf16 cache that starts 8 bytes off a 16-byte boundary
// 80 us, 2 bytes off (element by element) 278 us, where the tensor cores take 24.
constexpr int kSimtThreads = 128;
constexpr int kSimtWarps = kSimtThreads / kLanes;
constexpr float kSlack = 8.0f;  // log2 units a score may pass the running base

template <typename T, int V, int NU, int RT>
__global__ void __launch_bounds__(kSimtThreads) attention_simt_kernel(const __grid_constant__ Params p) {
  pdl_launch_dependents();
  pdl_wait();
  constexpr int kStep = kLanes / RT;  // keys
  constexpr int kTile = kSimtWarps * kStep;
  constexpr int kWidth = kLanes * V * NU;
  __shared__ float os[kSimtWarps][RT][kWidth];
  __shared__ float2 ml[kSimtWarps][RT];
  Work w;
  if (!find_work(p, w)) return;
  const int warp = threadIdx.x / kLanes, lane = threadIdx.x % kLanes;
  const int hd = (int)p.a.cache.hd;
  // What each row sees (lane l: row l % RT).
  const int my_row = lane % RT;
  int low = 0, high = -1;
  if (my_row < w.rows) sees(p, w, (w.row0 + my_row) / p.group, low, high);
  const bool any = high >= low;
  const int all_low = __reduce_max_sync(0xffffffffu, any ? low : 0);
  const int all_high = __reduce_min_sync(0xffffffffu, any ? high : INT32_MAX);
  const int any_low = __reduce_min_sync(0xffffffffu, any ? low : INT32_MAX);
  const int any_high = __reduce_max_sync(0xffffffffu, any ? high : -1);
  int begin, end;
  slice_keys(p, w, any_low, any_high, kTile, begin, end);

  float q[RT][NU][V], acc[RT][NU][V], m = -INFINITY, l = 0.0f;  // m, l: of row my_row, this lane's keys
#pragma unroll
  for (int r = 0; r < RT; r++) {
    int t, head;
    out_index(p, w, r < w.rows ? r : 0, t, head);
    const T* src = static_cast<const T*>(p.a.q) + t * p.a.q_stride + (int64_t)head * hd;
#pragma unroll
    for (int u = 0; u < NU; u++)
#pragma unroll
      for (int e = 0; e < V; e++) {
        const int d = (u * kLanes + lane) * V + e;
        q[r][u][e] = r < w.rows && d < hd ? to_f32<T>(src[d]) : 0.0f;
        acc[r][u][e] = 0.0f;
      }
  }
  const T* keys = static_cast<const T*>(p.a.cache.keys);
  const T* vals = static_cast<const T*>(p.a.cache.values);
  // Lane k looks key k of a step up, a step ahead.
  auto look_up = [&](int k) { return lane < kStep && k + lane < end ? entry_at(p, w, k + lane) : -1; };
  int entry = look_up(begin + warp * kStep);
  for (int k0 = begin + warp * kStep; k0 < end; k0 += kTile) {
    const int64_t mine = lane < kStep ? row_at(p, w, entry, k0 + lane, any_low, end) : -1;
    entry = look_up(k0 + kTile);
    const unsigned there = __ballot_sync(0xffffffffu, mine >= 0);
    float s[kLanes];
#pragma unroll
    for (int i = 0; i < kLanes; i++) s[i] = 0.0f;
#pragma unroll
    for (int k = 0; k < kStep; k++) {
      const int64_t at = __shfl_sync(0xffffffffu, mine, k);
#pragma unroll
      for (int u = 0; u < NU; u++) {
        const int d = (u * kLanes + lane) * V;
        float x[V] = {};
        if (at >= 0 && d < hd) load_run<T, V>(keys + at + d, x);
#pragma unroll
        for (int r = 0; r < RT; r++)
#pragma unroll
          for (int e = 0; e < V; e++) s[k * RT + r] = fmaf(q[r][u][e], x[e], s[k * RT + r]);
      }
    }
#pragma unroll
    for (int half = kLanes / 2; half >= 1; half >>= 1) {
      const bool upper = (lane & half) != 0;
#pragma unroll
      for (int i = 0; i < half; i++) {
        const float keep = upper ? s[i + half] : s[i], give = upper ? s[i] : s[i + half];
        s[i] = keep + __shfl_xor_sync(0xffffffffu, give, half);
      }
    }
    const int key = k0 + lane / RT;
    const bool seen = (there >> (lane / RT) & 1u) != 0 && key >= low && key <= high;
    const float x = seen ? s[0] * p.scale_log2 : -INFINITY;
    if (__any_sync(0xffffffffu, x > m + kSlack)) {  // a new base: the row's maximum so far
      float top = x;
#pragma unroll
      for (int off = RT; off < kLanes; off <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
      const float next = fmaxf(m, top), keep = next == -INFINITY ? 1.0f : exp2_fast(m - next);
      m = next;
      l *= keep;
#pragma unroll
      for (int r = 0; r < RT; r++) {
        const float f = __shfl_sync(0xffffffffu, keep, r);
#pragma unroll
        for (int u = 0; u < NU; u++)
#pragma unroll
          for (int e = 0; e < V; e++) acc[r][u][e] *= f;
      }
    }
    // -0: not seen. (A key that is seen counts, however small its weight.)
    const float pr = seen ? exp2_fast(x - (m == -INFINITY ? 0.0f : m)) : -0.0f;
    l += pr;
    const bool all = there == (kStep == 32 ? 0xffffffffu : (1u << kStep) - 1) && k0 >= all_low &&
                     k0 + kStep - 1 <= all_high;
#pragma unroll
    for (int k = 0; k < kStep; k++) {
      const int64_t at = __shfl_sync(0xffffffffu, mine, k);
      float y[NU][V] = {};
#pragma unroll
      for (int u = 0; u < NU; u++) {
        const int d = (u * kLanes + lane) * V;
        if (at >= 0 && d < hd) load_run<T, V>(vals + at + d, y[u]);
      }
#pragma unroll
      for (int r = 0; r < RT; r++) {
        const float f = __shfl_sync(0xffffffffu, pr, k * RT + r);
        if (!all && __float_as_int(f) < 0) continue;  // a key that the row does not see adds nothing, infinite or not
#pragma unroll
        for (int u = 0; u < NU; u++)
#pragma unroll
          for (int e = 0; e < V; e++) acc[r][u][e] = fmaf(f, y[u][e], acc[r][u][e]);
      }
    }
  }
  // Joined: the lanes' sums of a row, then the warps' results.
#pragma unroll
  for (int off = RT; off < kLanes; off <<= 1) l += __shfl_xor_sync(0xffffffffu, l, off);
  if (high < low) l = 0.0f;
  if (lane < RT) ml[warp][lane] = make_float2(m, l);
#pragma unroll
  for (int r = 0; r < RT; r++)
#pragma unroll
    for (int u = 0; u < NU; u++) store_run<float, V>(&os[warp][r][(u * kLanes + lane) * V], acc[r][u]);
  __syncthreads();
  for (int i = threadIdx.x; i < w.rows * hd; i += kSimtThreads) {
    const int r = i / hd, d = i % hd;
    float top = -INFINITY, sum = 0.0f, o = 0.0f;
#pragma unroll
    for (int k = 0; k < kSimtWarps; k++) top = fmaxf(top, ml[k][r].x);
    const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll
    for (int k = 0; k < kSimtWarps; k++) {
      const float2 part = ml[k][r];
      if (part.y == 0.0f) continue;
      const float f = exp2_fast(part.x - base);
      sum += part.y * f;
      o += os[k][r][d] * f;
    }
    int t, head;
    const int64_t row = out_index(p, w, r, t, head);
    if (p.direct) {
      static_cast<T*>(p.a.out)[t * p.a.out_stride + (int64_t)head * hd + d] = from_f32<T>(sum == 0.0f ? 0.0f : o / sum);
    } else {
      const int64_t to = slice_index(p, w) * (p.a.n * p.a.heads) + row;
      if (d == 0) p.ml[to] = make_float2(top, sum);
      p.acc[to * hd + d] = o;
    }
  }
}

// ------------------------------------------------------------------ the join

constexpr int kJoinThreads = 128;

// One warp for each (token, head): its lanes take a slice's maximum and sum
// each, then four (V) or one dimension each of every slice's values.
template <typename T, int V>
__global__ void __launch_bounds__(kJoinThreads) attention_join_kernel(const __grid_constant__ Params p) {
  pdl_launch_dependents();
  pdl_wait();
  const int64_t rows = p.a.n * p.a.heads;
  const int64_t row = (int64_t)blockIdx.x * (kJoinThreads / kLanes) + threadIdx.x / kLanes;
  if (row >= rows) return;
  constexpr int kRuns = kMaxPagedHd / (kLanes * V);
  const int lane = threadIdx.x % kLanes, hd = (int)p.a.cache.hd;
  const int t = (int)((uint32_t)row / (uint32_t)p.a.heads), head = (int)((uint32_t)row % (uint32_t)p.a.heads);
  // Whether the token belongs to a sequence.
  const bool covered = t >= seq_start(p, 0) && t < seq_start(p, (int)p.a.cache.sequences);
  const int slices = p.slices;
  const float2 first = lane < slices ? p.ml[lane * rows + row] : make_float2(-INFINITY, 0.0f);
  float m = first.x;
  for (int i = lane + kLanes; i < slices; i += kLanes) m = fmaxf(m, p.ml[i * rows + row].x);
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
  const float base = m == -INFINITY ? 0.0f : m;
  float l = 0.0f, acc[kRuns][V] = {};
  for (int i0 = 0; i0 < slices; i0 += kLanes) {
    float2 ml = first;
    if (i0 > 0) ml = i0 + lane < slices ? p.ml[(i0 + lane) * rows + row] : make_float2(-INFINITY, 0.0f);
    const float mine = ml.y == 0.0f ? 0.0f : exp2_fast(ml.x - base);
    l += ml.y * mine;
    const unsigned held = __ballot_sync(0xffffffffu, ml.y != 0.0f);  // (a slice with l = 0 may hold anything)
    const int count = min(kLanes, slices - i0);
    constexpr int kAtOnce = 8;
    for (int i = 0; i < count; i += kAtOnce) {
      float x[kAtOnce][kRuns][V];
#pragma unroll
      for (int k = 0; k < kAtOnce; k++) {
        const float* a = p.acc + ((i0 + min(i + k, count - 1)) * rows + row) * hd;
#pragma unroll
        for (int u = 0; u < kRuns; u++) {
          const int d = (u * kLanes + lane) * V;
          if (d < hd) load_run<float, V>(a + d, x[k][u]);
        }
      }
#pragma unroll
      for (int k = 0; k < kAtOnce; k++) {
        const float f = __shfl_sync(0xffffffffu, mine, (i + k) % kLanes);
        if (i + k >= count || (held >> (i + k) & 1u) == 0) continue;
#pragma unroll
        for (int u = 0; u < kRuns; u++)
#pragma unroll
          for (int e = 0; e < V; e++) acc[u][e] += x[k][u][e] * f;
      }
    }
  }
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) l += __shfl_xor_sync(0xffffffffu, l, off);
  if (!covered) return;
  T* out = static_cast<T*>(p.a.out) + t * p.a.out_stride + (int64_t)head * hd;
#pragma unroll
  for (int u = 0; u < kRuns; u++) {
    const int d = (u * kLanes + lane) * V;
    if (d >= hd) continue;
#pragma unroll
    for (int e = 0; e < V; e++) acc[u][e] = l == 0.0f ? 0.0f : acc[u][e] / l;
    if (p.runs) {
      store_run<T, V>(out + d, acc[u]);
    } else {
#pragma unroll
      for (int e = 0; e < V; e++) out[d + e] = from_f32<T>(acc[u][e]);
    }
  }
}

// ------------------------------------------------------------------ the host

// Whether the tensor-core kernel takes a cache: 16-bit elements whose rows are
// whole, aligned runs of 16 bytes.
bool mma_cache(const PagedCache& c) {
  return c.type != kF32 && (((uintptr_t)c.keys | (uintptr_t)c.values) & 15) == 0 && (c.page_stride | c.hd) % 8 == 0;
}

// Limits up to which sequences read the prefix for themselves: keys of the
// longest, and of the prefix, once for each sequence. Measured with and without
// (us; 8 kv heads of 128, 2 heads a group, bf16, 16 own keys): 2 sequences
// behind 64 keys 6.7 and 8.2, 8 behind 256 10.8 and 13.5, 16 behind 512 12.3
// and 13.8, 32 behind 256 15.8 and 17.1; past the limits 16 behind 1024 18.1
// and 14.4, 32 behind 512 19.5 and 19.2, though 8 behind 1024 11.6 and 13.8.
// One or two sequences of 320 to 512 keys lose 0.1 to 0.8 by it.
constexpr int64_t kSoloKeys = 512;
constexpr int64_t kSoloReads = 8192;

// Least keys of a slice: of the thin kernel, the f32 one, and a wide block of
// two groups and of one. Over 35 batches (16 to 192 sequences behind 700 to 8192
// keys, heads of 64 and 128) a least of 384 takes the same time as 512, 1% more
// than 256, and 2% and 7% less than 128 and 768, in the geometric mean; single
// batches differ more (32 chat sequences and 24 of drafts: 23.6 and 22.1 us with
// 384, 21.9 and 27.3 with 256, 24.8 and 23.1 with 512). With 256-wide heads 29 us
// with 128, 32 with 256.
constexpr int kThinLeast = 256, kSimtLeast = 128, kWide2Least = 384, kWide1Least = 128;

// How the work is divided, from sizes that the host knows.
Params plan(const PagedCache& c, int64_t heads, int64_t n, int64_t prefix, int64_t max_length) {
  Params p{};
  p.group = (int)(heads / c.kv_heads);
  const int64_t rows = n * p.group, seqs = c.sequences > 1 ? c.sequences : 1;
  const bool wide = mma_cache(c) && c.page_size % 16 == 0 && c.pages > 0;
  // Short sequences in all: each reads the prefix for itself, from L2, which
  // saves the second launch that joins two parts. The page list then changes at
  // `prefix`, which no copy may span: 16 keys of a thin block, a wide one's box.
  p.own_wide = wide && rows > kWideFrom * seqs;
  p.solo = prefix > 0 && prefix % (p.own_wide ? wide_box(c.page_size) : 16) == 0 && max_length <= kSoloKeys &&
           c.sequences * prefix <= kSoloReads;
  if (p.solo) prefix = 0;
  p.prefix_wide = wide && prefix > 0 && rows > kWideFrom;
  // 8 rows to a thin block where a sequence's rows, and the whole batch's on
  // the prefix, are that few; else 16.
  const bool few = rows <= 8 * seqs && (prefix == 0 || p.prefix_wide || rows <= 8);
  p.thin_rows = few ? 8 : 16;
  if (!mma_cache(c)) {
    // Rows of a block of the f32 kernel: a sequence's, at most 8.
    const int64_t each = (rows + seqs - 1) / seqs;
    p.thin_rows = each <= 1 ? 1 : each <= 2 ? 2 : each <= 4 ? 4 : 8;
  }
  p.prefix_rows = p.prefix_wide ? kWideRows : p.thin_rows;
  p.own_rows = p.own_wide ? kWideRows : p.thin_rows;
  p.own_rows_log2 = 31 - __builtin_clz((unsigned)p.own_rows);
  const int64_t tiles = (rows + p.prefix_rows - 1) / p.prefix_rows;
  p.prefix_tiles = prefix > 0 ? (int)tiles : 0;
  p.own_slots = (int)(rows / p.own_rows + c.sequences);
  // A part's keys are split as long as blocks are wanting (four thin or f32
  // blocks to an SM, one wide) and a slice keeps its least keys: shorter ones
  // cost the join more than they save the slices.
  const int wide_least = wide_groups(c.hd) == 2 ? kWide2Least : kWide1Least;
  p.prefix_least = p.prefix_wide ? wide_least : mma_cache(c) ? kThinLeast : kSimtLeast;
  p.own_least = p.own_wide ? wide_least : mma_cache(c) ? kThinLeast : kSimtLeast;
  auto splits = [&](int64_t blocks, int64_t keys, bool on_wide, int64_t least_keys) {
    const int64_t want = on_wide ? 148 / (blocks > 0 ? blocks : 1) : (4 * 148 + blocks - 1) / (blocks > 0 ? blocks : 1);
    const int64_t most = (keys + least_keys - 1) / least_keys, least = want < most ? want : most;
    return (int)(least > 1 ? least : 1);
  };
  p.prefix_splits = prefix > 0 ? splits(tiles * c.kv_heads, prefix, p.prefix_wide, p.prefix_least) : 0;
  const int64_t own = max_length > prefix ? max_length - prefix : 1;
  p.own_splits = splits((int64_t)p.own_slots * c.kv_heads, own, p.own_wide, p.own_least);
  p.slices = p.prefix_splits + p.own_splits;
  p.direct = p.slices == 1;
  return p;
}

// The tensor-core kernels on the parts that are theirs; the thin one runs
// beside the wide one, whose blocks leave it half of each SM.
cudaError_t launch_mma(const Params& p, cudaStream_t stream, bool pdl) {
  const bool wide = p.prefix_wide || p.own_wide;
  if (wide) {
    Params part = p;
    if (!p.prefix_wide) part.prefix_tiles = 0;
    if (!p.own_wide) part.own_slots = 0;
    if (cudaError_t e = launch_attention_wide(part, stream, pdl); e != cudaSuccess) return e;
  }
  Params part = p;
  part.beside = wide;
  if (p.prefix_wide) part.prefix_tiles = 0;
  if (p.own_wide) part.own_slots = 0;
  if (part.prefix_tiles == 0 && part.own_slots == 0) return cudaSuccess;
  return launch_attention_thin(part, stream, pdl || wide);
}

template <typename T, int V, int NU>
cudaError_t launch_simt_rows(const Params& p, cudaStream_t stream, bool pdl) {
  const dim3 grid = attention_grid(p);
  switch (p.own_rows) {
    case 1: return launch_ex(attention_simt_kernel<T, V, NU, 1>, grid, kSimtThreads, 0, stream, pdl, p);
    case 2: return launch_ex(attention_simt_kernel<T, V, NU, 2>, grid, kSimtThreads, 0, stream, pdl, p);
    case 4: return launch_ex(attention_simt_kernel<T, V, NU, 4>, grid, kSimtThreads, 0, stream, pdl, p);
    default: return launch_ex(attention_simt_kernel<T, V, NU, 8>, grid, kSimtThreads, 0, stream, pdl, p);
  }
}

template <typename T>
cudaError_t launch_simt(const Params& p, cudaStream_t stream, bool pdl) {
  const PagedCache& c = p.a.cache;
  const bool runs = (((uintptr_t)c.keys | (uintptr_t)c.values) & (4 * sizeof(T) - 1)) == 0 &&
                    (c.page_stride | c.hd) % 4 == 0;
  if (!runs) return launch_simt_rows<T, 1, 8>(p, stream, pdl);
  return c.hd <= 128 ? launch_simt_rows<T, 4, 1>(p, stream, pdl) : launch_simt_rows<T, 4, 2>(p, stream, pdl);
}

template <typename T>
cudaError_t launch_type(const Params& p, cudaStream_t stream, bool pdl) {
  const PagedCache& c = p.a.cache;
  const cudaError_t e = mma_cache(c) ? launch_mma(p, stream, pdl) : launch_simt<T>(p, stream, pdl);
  if (e != cudaSuccess || p.direct) return e;
  const int64_t warps = p.a.n * p.a.heads, per = kJoinThreads / kLanes;
  const dim3 grid((unsigned)((warps + per - 1) / per));
  return c.hd % 4 == 0 ? launch_ex(attention_join_kernel<T, 4>, grid, kJoinThreads, 0, stream, true, p)
                       : launch_ex(attention_join_kernel<T, 1>, grid, kJoinThreads, 0, stream, true, p);
}

}  // namespace

int64_t paged_attention_workspace(const PagedCache& c, int64_t heads, int64_t n, int64_t prefix,
                                  int64_t max_length) {
  const Params p = plan(c, heads, n, prefix, max_length);
  return p.slices * n * heads * (c.hd + 2) * (int64_t)sizeof(float) + 16;
}

cudaError_t launch_paged_attention(const PagedAttentionArgs& a, cudaStream_t stream, bool pdl) {
  if (a.n <= 0 || a.cache.sequences <= 0) return cudaSuccess;  // no sequence: no token belongs to one
  Params p = plan(a.cache, a.heads, a.n, a.prefix, a.max_length);
  p.a = a;
  p.status = a.status;
  p.page_shift = -1;
  for (int s = 0; s <= 20; s++)
    if (a.cache.page_size == (int64_t)1 << s) p.page_shift = s;
  p.runs = (((uintptr_t)a.q | (uintptr_t)a.out) & 15) == 0 &&
           ((a.q_stride | a.out_stride | a.cache.hd) * elem_size(a.cache.type)) % 16 == 0;
  p.pairs = (((uintptr_t)a.q | (uintptr_t)a.out) & 3) == 0 && (a.q_stride | a.out_stride) % 2 == 0;
  // A scale of 0 is taken as the least normal number: the exponents still come
  // out equal, and a masked score's minus infinity stays one.
  p.scale_log2 = a.scale == 0.0f ? 1.17549435e-38f : a.scale * kLog2e;
  const int64_t rows = p.slices * a.n * a.heads;
  p.ml = static_cast<float2*>(a.workspace);
  p.acc = reinterpret_cast<float*>(p.ml + (rows + 1) / 2 * 2);
  switch (a.cache.type) {
    case kF32: return launch_type<float>(p, stream, pdl);
    case kF16: return launch_type<__half>(p, stream, pdl);
    default: return launch_type<__nv_bfloat16>(p, stream, pdl);
  }
}

}  // namespace dn
