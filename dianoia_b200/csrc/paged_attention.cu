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
// Any type, head size up to 256 and alignment. A block of 4 warps takes 16
// rows; each tile of 32 keys is brought to shared memory as f32 for all of
// them. Warp w owns rows 4 w .. 4 w + 3: lane j scores key j for each (f32
// FMAs along the head), the tile's maximum and sum are warp reductions, and
// for the values lane j owns dimensions 4 j .. 4 j + 3 (and 128 more on).
constexpr int kSimtThreads = 128;
constexpr int kSimtKeys = 32;
constexpr int kWarpRows = 4;

// Floats of a row of keys, values or queries in shared memory: 16-byte
// aligned, and eight rows apart by 16 bytes of banks.
__host__ __device__ constexpr int simt_pitch(int hd) { return (hd + 31) / 32 * 32 + 4; }

template <typename T, int V>
__global__ void __launch_bounds__(kSimtThreads) attention_simt_kernel(const __grid_constant__ Params p) {
  pdl_launch_dependents();
  pdl_wait();
  extern __shared__ float smem[];
  const int hd = (int)p.a.cache.hd, pitch = simt_pitch(hd);
  float* qs = smem;                            // [kSimtRows][pitch]
  float* ks = qs + kSimtRows * pitch;          // [kSimtKeys][pitch]
  float* vs = ks + kSimtKeys * pitch;          // [kSimtKeys][pitch]
  float* ps = vs + kSimtKeys * pitch;          // [4 warps][kSimtKeys][kWarpRows]
  __shared__ int row_low[kSimtRows], row_high[kSimtRows], span[2];
  __shared__ int key_page[kSimtKeys];
  Work w;
  if (!find_work(p, w)) return;
  const int tid = threadIdx.x, warp = tid / kLanes, lane = tid % kLanes;
  if (tid < kSimtRows) {
    int low = 0, high = -1;
    if (tid < w.rows) {
      const int t = (w.row0 + tid) / p.group;
      sees(p, w, t, low, high);
    }
    row_low[tid] = low;
    row_high[tid] = high;
    const bool any = high >= low;
    const int lo = __reduce_min_sync(0xffffu, any ? low : INT32_MAX);
    const int hi = __reduce_max_sync(0xffffu, any ? high : -1);
    if (tid == 0) {
      span[0] = lo;
      span[1] = hi;
    }
  }
  for (int i = tid; i < kSimtRows * pitch; i += kSimtThreads) {
    const int r = i / pitch, d = i % pitch;
    float x = 0.0f;
    if (r < w.rows && d < hd) {
      int t, head;
      out_index(p, w, r, t, head);
      x = to_f32<T>(static_cast<const T*>(p.a.q)[t * p.a.q_stride + (int64_t)head * hd + d]);
    }
    qs[i] = x;
  }
  __syncthreads();
  int begin, end;
  slice_keys(p, w, span[0], span[1], kSimtKeys, begin, end);

  float m[kWarpRows], l[kWarpRows], acc[kWarpRows][2][4];
#pragma unroll
  for (int r = 0; r < kWarpRows; r++) {
    m[r] = -INFINITY;
    l[r] = 0.0f;
#pragma unroll
    for (int u = 0; u < 2; u++)
#pragma unroll
      for (int e = 0; e < 4; e++) acc[r][u][e] = 0.0f;
  }
  const int row_base = warp * kWarpRows;
  int low[kWarpRows], high[kWarpRows];
#pragma unroll
  for (int r = 0; r < kWarpRows; r++) {
    low[r] = row_low[row_base + r];
    high[r] = row_high[row_base + r];
  }
  for (int k0 = begin; k0 < end; k0 += kSimtKeys) {
    __syncthreads();  // the last tile is read
    if (tid < kSimtKeys) key_page[tid] = k0 + tid < end ? page_of(p, w, k0 + tid) : -1;
    __syncthreads();
    const int runs = pitch / V;
    for (int i = tid; i < kSimtKeys * runs; i += kSimtThreads) {
      const int j = i / runs, d = i % runs * V;
      float x[V] = {}, y[V] = {};
      if (key_page[j] >= 0 && d < hd) {
        const int slot = (k0 + j) % (int)p.a.cache.page_size;
        const int64_t at = key_page[j] * p.a.cache.page_stride +
                           ((int64_t)w.head * p.a.cache.page_size + slot) * hd + d;
        load_run<T, V>(static_cast<const T*>(p.a.cache.keys) + at, x);
        load_run<T, V>(static_cast<const T*>(p.a.cache.values) + at, y);
      }
#pragma unroll
      for (int e = 0; e < V; e++) {
        ks[j * pitch + d + e] = x[e];
        vs[j * pitch + d + e] = y[e];
      }
    }
    __syncthreads();
    // Scores of key `lane` for the warp's rows.
    float s[kWarpRows] = {};
    const float4* kv = reinterpret_cast<const float4*>(ks + lane * pitch);
    for (int d = 0; d < (hd + 3) / 4; d++) {
      const float4 k = kv[d];
#pragma unroll
      for (int r = 0; r < kWarpRows; r++) {
        const float4 q = reinterpret_cast<const float4*>(qs + (row_base + r) * pitch)[d];
        s[r] = fmaf(q.x, k.x, s[r]);
        s[r] = fmaf(q.y, k.y, s[r]);
        s[r] = fmaf(q.z, k.z, s[r]);
        s[r] = fmaf(q.w, k.w, s[r]);
      }
    }
    const bool there = key_page[lane] >= 0;
    float pr[kWarpRows];
    bool all = true;  // every row that sees a key of the tile sees all of it
#pragma unroll
    for (int r = 0; r < kWarpRows; r++) {
      const bool seen = there && k0 + lane >= low[r] && k0 + lane <= high[r];
      const float x = seen ? s[r] * p.scale_log2 : -INFINITY;
      float top = x;
#pragma unroll
      for (int off = 16; off >= 1; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
      const float next = fmaxf(m[r], top);
      const float base = next == -INFINITY ? 0.0f : next;
      const float keep = exp2_fast(m[r] - base);
      pr[r] = seen ? exp2_fast(x - base) : 0.0f;
      m[r] = next;
      l[r] = l[r] * keep + pr[r];  // a lane's share; summed over the lanes at the end
#pragma unroll
      for (int u = 0; u < 2; u++)
#pragma unroll
        for (int e = 0; e < 4; e++) acc[r][u][e] *= keep;
      all = all && (seen || high[r] < low[r]);  // (a row that sees nothing has only zeros to add)
    }
    float4* pw = reinterpret_cast<float4*>(ps) + warp * kSimtKeys;
    pw[lane] = make_float4(pr[0], pr[1], pr[2], pr[3]);
    __syncwarp();
    const bool fast = __all_sync(0xffffffffu, all);
    for (int j = 0; j < kSimtKeys; j++) {
      const float4 q = pw[j];
      const float pj[kWarpRows] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int u = 0; u < 2; u++) {
        const int d = 4 * lane + 128 * u;
        if (d >= hd) break;
        const float4 v = *reinterpret_cast<const float4*>(vs + j * pitch + d);
        const float ve[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int r = 0; r < kWarpRows; r++)
#pragma unroll
          for (int e = 0; e < 4; e++) {
            // A key that a row does not see adds nothing, infinite or not.
            if (fast || pj[r] != 0.0f) acc[r][u][e] = fmaf(pj[r], ve[e], acc[r][u][e]);
          }
      }
    }
    __syncwarp();
  }
#pragma unroll
  for (int r = 0; r < kWarpRows; r++) {
    float sum = l[r];
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    if (row_base + r >= w.rows) continue;
    int t, head;
    const int64_t row = out_index(p, w, row_base + r, t, head);
    if (p.direct) {
      const float inv = sum > 0.0f ? 1.0f / sum : sum == 0.0f ? 0.0f : sum;  // NaN stays
      T* out = static_cast<T*>(p.a.out) + t * p.a.out_stride + (int64_t)head * hd;
#pragma unroll
      for (int u = 0; u < 2; u++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const int d = 4 * lane + 128 * u + e;
          if (d < hd) out[d] = from_f32<T>(sum == 0.0f ? 0.0f : acc[r][u][e] * inv);
        }
    } else {
      const int64_t at = slice_index(p, w) * (p.a.n * p.a.heads) + row;
      if (lane == 0) p.ml[at] = make_float2(m[r], sum);
#pragma unroll
      for (int u = 0; u < 2; u++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const int d = 4 * lane + 128 * u + e;
          if (d < hd) p.acc[at * hd + d] = acc[r][u][e];
        }
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
  if (p.a.q_start != nullptr && seq_of(p, t) < 0) return;
  const int slices = p.slices;
  float m = -INFINITY;
  for (int i = lane; i < slices; i += kLanes) m = fmaxf(m, p.ml[i * rows + row].x);
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
  const float base = m == -INFINITY ? 0.0f : m;
  float l = 0.0f, acc[kRuns][V] = {};
  for (int i0 = 0; i0 < slices; i0 += kLanes) {
    const float2 ml = i0 + lane < slices ? p.ml[(i0 + lane) * rows + row] : make_float2(-INFINITY, 0.0f);
    const float mine = ml.y == 0.0f ? 0.0f : exp2_fast(ml.x - base);
    l += ml.y * mine;
    unsigned left = __ballot_sync(0xffffffffu, ml.y != 0.0f);  // (a slice with l = 0 may hold anything)
    const int count = min(kLanes, slices - i0);
#pragma unroll 4
    for (int i = 0; i < count; i++) {
      const float f = __shfl_sync(0xffffffffu, mine, i);
      const float* a = p.acc + ((i0 + i) * rows + row) * hd;
      if ((left >> i & 1u) == 0) continue;
#pragma unroll
      for (int u = 0; u < kRuns; u++) {
        const int d = (u * kLanes + lane) * V;
        if (d >= hd) continue;
        float x[V];
        load_run<float, V>(a + d, x);
#pragma unroll
        for (int e = 0; e < V; e++) acc[u][e] += x[e] * f;
      }
    }
  }
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) l += __shfl_xor_sync(0xffffffffu, l, off);
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

constexpr int64_t kSoloKeys = 512;    // of the longest sequence
constexpr int64_t kSoloReads = 8192;  // keys of the prefix, once for each sequence

// How the work is divided, from sizes that the host knows.
Params plan(const PagedCache& c, int64_t heads, int64_t n, int64_t prefix, int64_t max_length) {
  Params p{};
  p.group = (int)(heads / c.kv_heads);
  const int64_t rows = n * p.group, seqs = c.sequences > 1 ? c.sequences : 1;
  const bool wide = mma_cache(c) && c.page_size % 16 == 0 && c.pages > 0;
  // Short sequences in all: each reads the prefix for itself, from L2, which
  // saves the second launch that joins two parts.
  p.solo = prefix > 0 && prefix % 16 == 0 && max_length <= kSoloKeys && c.sequences * prefix <= kSoloReads;
  if (p.solo) prefix = 0;
  p.prefix_wide = wide && prefix > 0 && rows > kWideFrom;
  p.own_wide = wide && rows > kWideFrom * seqs;
  // 8 rows to a thin block where a sequence's rows, and the whole batch's on
  // the prefix, are that few; else 16.
  const bool few = rows <= 8 * seqs && (prefix == 0 || p.prefix_wide || rows <= 8);
  p.thin_rows = mma_cache(c) ? few ? 8 : 16 : kSimtRows;
  p.prefix_rows = p.prefix_wide ? kWideRows : p.thin_rows;
  p.own_rows = p.own_wide ? kWideRows : p.thin_rows;
  p.own_rows_log2 = 31 - __builtin_clz((unsigned)p.own_rows);
  p.min_slice = 128;
  const int64_t tiles = (rows + p.prefix_rows - 1) / p.prefix_rows;
  p.prefix_tiles = prefix > 0 ? (int)tiles : 0;
  p.own_slots = (int)(rows / p.own_rows + c.sequences);
  // A part's keys are split as long as blocks are wanting and a slice keeps
  // min_slice keys: two thin blocks to an SM, one wide.
  auto splits = [&](int64_t blocks, int64_t keys, bool on_wide) {
    const int64_t want = on_wide ? 148 / (blocks > 0 ? blocks : 1) : (2 * 148 + blocks - 1) / (blocks > 0 ? blocks : 1);
    const int64_t most = (keys + p.min_slice - 1) / p.min_slice, least = want < most ? want : most;
    return (int)(least > 1 ? least : 1);
  };
  p.prefix_splits = prefix > 0 ? splits(tiles * c.kv_heads, prefix, p.prefix_wide) : 0;
  const int64_t own = max_length > prefix ? max_length - prefix : 1;
  p.own_splits = splits((int64_t)p.own_slots * c.kv_heads, own, p.own_wide);
  p.prefix_slices = p.prefix_splits * (p.prefix_wide ? wide_groups(c.hd) : 1);
  p.slices = p.prefix_slices + p.own_splits * (p.own_wide ? wide_groups(c.hd) : 1);
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

template <typename T, int V>
cudaError_t launch_simt(const Params& p, cudaStream_t stream, bool pdl) {
  const size_t smem = ((kSimtRows + 2 * kSimtKeys) * (size_t)simt_pitch((int)p.a.cache.hd) +
                       kSimtThreads / kLanes * kSimtKeys * kWarpRows) * sizeof(float);
  if (cudaError_t e = cudaFuncSetAttribute(attention_simt_kernel<T, V>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                           (int)smem);
      e != cudaSuccess)
    return e;
  return launch_ex(attention_simt_kernel<T, V>, attention_grid(p), kSimtThreads, smem, stream, pdl, p);
}

template <typename T>
cudaError_t launch_type(const Params& p, cudaStream_t stream, bool pdl) {
  constexpr int V = 16 / sizeof(T);
  const PagedCache& c = p.a.cache;
  const bool runs = (((uintptr_t)c.keys | (uintptr_t)c.values) & 15) == 0 && (c.page_stride | c.hd) % V == 0;
  cudaError_t e = mma_cache(c) ? launch_mma(p, stream, pdl)
                  : runs       ? launch_simt<T, V>(p, stream, pdl)
                               : launch_simt<T, 1>(p, stream, pdl);
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
  if (a.n <= 0) return cudaSuccess;
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
