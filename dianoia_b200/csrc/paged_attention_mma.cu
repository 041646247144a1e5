// The paged attention's tensor-core kernel for 16-bit caches (f16, bf16).
//
// Scores S = Q K^T and outputs O = P V as m16n8k16 products with f32
// accumulators, the softmax between them in registers: a lane holds the same
// two rows of S, P and O throughout, so P goes from the scores' fragments into
// the values' product without leaving the warp. P is rounded to the cache's
// type there (the products take 16-bit operands); its sum l is of the f32
// values. Keys and values come to shared memory by 16-byte asynchronous copies,
// a row's 16-byte chunk c at chunk c ^ (row & 7), so that the fragment loads
// meet no bank twice.
//
// Thin blocks (16 rows: the heads of one group of a decode step) are bound by
// the keys' bytes. Each of the 4 warps streams its own 16 keys of every 64
// through a ring of kStages buffers and keeps its own maximum, sum and output;
// they are joined once at the end, so that no block barrier stands in the loop.
// Wide blocks (64 rows: the whole batch on the shared prefix, long chunks of
// queries) give each warp 16 rows and share tiles of 64 keys, so that a key is
// brought once for 64 rows.
#include "paged_attention.cuh"

namespace dn {

using namespace paged;

namespace {

constexpr int kThreads = 128;
constexpr int kWarps = kThreads / kLanes;
constexpr int kStep = 16;      // keys of a warp's step in a thin block
constexpr int kTile = 64;      // keys of a tile: kWarps steps, or a wide block's
constexpr int kStages = 3;

template <typename T>
struct Pair;
template <>
struct Pair<__half> {
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    uint32_t u;
    memcpy(&u, &h, 4);
    return u;
  }
  // Whether either half is an infinity or a NaN.
  static __device__ __forceinline__ bool unbounded(uint32_t u) {
    return (u & 0x7c00u) == 0x7c00u || (u & 0x7c000000u) == 0x7c000000u;
  }
};
template <>
struct Pair<__nv_bfloat16> {
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    uint32_t u;
    memcpy(&u, &h, 4);
    return u;
  }
  static __device__ __forceinline__ bool unbounded(uint32_t u) {
    return (u & 0x7f80u) == 0x7f80u || (u & 0x7f800000u) == 0x7f800000u;
  }
};

// Two elements of a query or an output; `pairs`: every row is 4-byte aligned.
template <typename T>
__device__ __forceinline__ uint32_t load_pair(const T* p, bool pairs) {
  if (pairs) return *reinterpret_cast<const uint32_t*>(p);
  const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
  return h[0] | (uint32_t)h[1] << 16;
}
template <typename T>
__device__ __forceinline__ void store_pair(T* p, uint32_t v, bool pairs) {
  if (pairs) {
    *reinterpret_cast<uint32_t*>(p) = v;
  } else {
    uint16_t* h = reinterpret_cast<uint16_t*>(p);
    h[0] = (uint16_t)v;
    h[1] = (uint16_t)(v >> 16);
  }
}

__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __half) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __nv_bfloat16) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}

// 16 bytes to shared memory, zeros where `there` is false.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Byte offset of 16-byte chunk c of row r in a tile of rows of HDP elements.
template <int HDP>
__device__ __forceinline__ uint32_t chunk_at(int r, int c) {
  return (uint32_t)(r * HDP * 2 + ((c ^ (r & 7)) << 4));
}

// One warp's rows: fragments of Q, the running maximum and sum and O. Lane
// (g, i) = (lane / 4, lane % 4) holds rows g and g + 8, columns 2 i, 2 i + 1
// of each 8-wide tile.
template <typename T, int HDP>
struct Rows {
  static constexpr bool kQInRegs = HDP <= 128;
  uint32_t q[kQInRegs ? HDP / 16 : 1][4];
  uint32_t q_smem;  // where they are otherwise
  float o[HDP / 8][4];
  float m[2], l[2];
  int low[2], high[2];  // the positions that rows g, g + 8 see
  int all_low, all_high;  // that every row of the warp sees
  int any_low, any_high;  // that some row sees

  __device__ __forceinline__ void init(const Params& p, const Work& w, int row_base, char* smem, int lane) {
    const int hd = (int)p.a.cache.hd;
    int lo = 0, hi = -1;
    const int r = row_base + lane;
    if (lane < 16 && r < w.rows) {
      const int t = (w.row0 + r) / p.group;
      sees(p, w.prefix ? seq_of(p, t) : w.seq, t, lo, hi);
    }
    const bool mine = lane < 16 && r < w.rows, any = hi >= lo;
    all_low = __reduce_max_sync(0xffffffffu, mine ? any ? lo : INT32_MAX : 0);
    all_high = __reduce_min_sync(0xffffffffu, mine ? hi : INT32_MAX);
    any_low = __reduce_min_sync(0xffffffffu, any ? lo : INT32_MAX);
    any_high = __reduce_max_sync(0xffffffffu, any ? hi : -1);
    const T* src[2];
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const int row = lane / 4 + 8 * h;
      low[h] = __shfl_sync(0xffffffffu, lo, row);
      high[h] = __shfl_sync(0xffffffffu, hi, row);
      m[h] = -INFINITY;
      l[h] = 0.0f;
      src[h] = nullptr;
      if (row_base + row < w.rows) {
        int t, head;
        out_index(p, w, row_base + row, t, head);
        src[h] = static_cast<const T*>(p.a.q) + t * p.a.q_stride + (int64_t)head * hd;
      }
    }
#pragma unroll
    for (int j = 0; j < HDP / 8; j++)
#pragma unroll
      for (int e = 0; e < 4; e++) o[j][e] = 0.0f;
    q_smem = smem_u32(smem);
#pragma unroll
    for (int k = 0; k < HDP / 16; k++) {
      uint32_t f[4];
#pragma unroll
      for (int u = 0; u < 4; u++) {  // row g + 8 (u & 1), columns 8 (u >> 1) + 2 i
        const int d = 16 * k + 8 * (u >> 1) + 2 * (lane % 4);
        f[u] = src[u & 1] != nullptr && d < hd ? load_pair(src[u & 1] + d, p.pairs) : 0u;
      }
      if constexpr (kQInRegs) {
#pragma unroll
        for (int u = 0; u < 4; u++) q[k][u] = f[u];
      } else {
        *reinterpret_cast<uint4*>(smem + k * 512 + lane * 16) = make_uint4(f[0], f[1], f[2], f[3]);
      }
    }
  }

  // Scores of NT * 8 keys at rows `row` .. of the key tile at `keys`.
  template <int NT>
  __device__ __forceinline__ void scores(float (&s)[NT][4], uint32_t keys, int row, int lane) {
#pragma unroll
    for (int j = 0; j < NT; j++)
#pragma unroll
      for (int e = 0; e < 4; e++) s[j][e] = 0.0f;
#pragma unroll
    for (int k = 0; k < HDP / 16; k++) {
      uint32_t a[4];
      if constexpr (kQInRegs) {
#pragma unroll
        for (int u = 0; u < 4; u++) a[u] = q[k][u];
      } else {
        asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                     : "=r"(a[0]), "=r"(a[1]), "=r"(a[2]), "=r"(a[3])
                     : "r"(q_smem + k * 512 + lane * 16));
      }
#pragma unroll
      for (int j = 0; j < NT; j += 2) {
        uint32_t b[4];  // keys 8 j .. 8 j + 15: (k low, k high) of each eight
        const int r = row + 8 * j + (lane & 7) + ((lane >> 4) << 3), c = 2 * k + ((lane >> 3) & 1);
        ldsm4(b, keys + chunk_at<HDP>(r, c));
        mma(s[j], a, b[0], b[1], T());
        mma(s[j + 1], a, b[2], b[3], T());
      }
    }
  }

  // Scores to probabilities against the new running maximum; O and l scaled
  // to it. Keys k0 .. : masked by what each row sees unless `all`.
  template <int NT>
  __device__ __forceinline__ void softmax(float (&s)[NT][4], int k0, bool all, uint64_t there, float scale, int lane) {
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int j = 0; j < NT; j++)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        float x = s[j][e] * scale;
        if (!all) {
          const int at = 8 * j + 2 * (lane % 4) + (e & 1), h = e >> 1;
          const bool seen = (there >> at & 1) != 0 && k0 + at >= low[h] && k0 + at <= high[h];
          x = seen ? x : -INFINITY;
        }
        s[j][e] = x;
        top[e >> 1] = fmaxf(top[e >> 1], x);
      }
    float base[2], keep[2];
    bool moved = false;
#pragma unroll
    for (int h = 0; h < 2; h++) {
      top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
      top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 2));
      const float next = fmaxf(m[h], top[h]);
      base[h] = next == -INFINITY ? 0.0f : next;
      keep[h] = exp2f(m[h] - base[h]);
      moved = moved || next != m[h];
      m[h] = next;
    }
    if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
      for (int j = 0; j < HDP / 8; j++)
#pragma unroll
        for (int e = 0; e < 4; e++) o[j][e] *= keep[e >> 1];
      l[0] *= keep[0];
      l[1] *= keep[1];
    }
#pragma unroll
    for (int j = 0; j < NT; j++)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        s[j][e] = exp2f(s[j][e] - base[e >> 1]);
        l[e >> 1] += s[j][e];  // a lane's share of the row's sum
      }
  }

  // O += P V for 16 keys at rows `row` .. of the value tile.
  __device__ __forceinline__ void values(const float (&s0)[4], const float (&s1)[4], uint32_t vals, int row, int lane) {
    const uint32_t a[4] = {Pair<T>::pack(s0[0], s0[1]), Pair<T>::pack(s0[2], s0[3]), Pair<T>::pack(s1[0], s1[1]),
                           Pair<T>::pack(s1[2], s1[3])};
    const int r = row + (lane & 15);
#pragma unroll
    for (int j = 0; j < HDP / 8; j += 2) {
      uint32_t b[4];
      ldsm4_t(b, vals + chunk_at<HDP>(r, j + (lane >> 4)));
      mma(o[j], a, b[0], b[1], T());
      mma(o[j + 1], a, b[2], b[3], T());
    }
  }

  // The same where a value that some row does not see is not finite: a
  // product with probability 0 would be NaN, so such terms are left out.
  __device__ __forceinline__ void values_guarded(const float (&s0)[4], const float (&s1)[4], const char* vals, int row,
                                              int lane) {
#pragma unroll 1
    for (int k = 0; k < 16; k++) {
      const int from = (lane & ~3) | ((k % 8) / 2);
      const float x0 = k % 2 ? k < 8 ? s0[1] : s1[1] : k < 8 ? s0[0] : s1[0];
      const float x1 = k % 2 ? k < 8 ? s0[3] : s1[3] : k < 8 ? s0[2] : s1[2];
      const float p0 = __shfl_sync(0xffffffffu, x0, from), p1 = __shfl_sync(0xffffffffu, x1, from);
      const float r0 = to_f32<T>(from_f32<T>(p0)), r1 = to_f32<T>(from_f32<T>(p1));
#pragma unroll
      for (int j = 0; j < HDP / 8; j++) {
        const T* v = reinterpret_cast<const T*>(vals + chunk_at<HDP>(row + k, j)) + 2 * (lane % 4);
        const float v0 = to_f32<T>(v[0]), v1 = to_f32<T>(v[1]);
        if (p0 != 0.0f) {
          o[j][0] = fmaf(r0, v0, o[j][0]);
          o[j][1] = fmaf(r0, v1, o[j][1]);
        }
        if (p1 != 0.0f) {
          o[j][2] = fmaf(r1, v0, o[j][2]);
          o[j][3] = fmaf(r1, v1, o[j][3]);
        }
      }
    }
  }

  __device__ __forceinline__ void finish() {
#pragma unroll
    for (int h = 0; h < 2; h++) {
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
    }
  }
};

// Whether any of `rows` rows of a value tile holds an infinity or a NaN.
template <typename T, int HDP>
__device__ __forceinline__ bool any_unbounded(const char* vals, int rows, int lane) {
  bool bad = false;
  for (int i = lane; i < rows * HDP / 8; i += kLanes) {
    const uint4 v = *reinterpret_cast<const uint4*>(vals + i * 16);
    bad = bad || Pair<T>::unbounded(v.x) || Pair<T>::unbounded(v.y) || Pair<T>::unbounded(v.z) || Pair<T>::unbounded(v.w);
  }
  return __any_sync(0xffffffffu, bad);
}

// Element offset of a position's row of its kv head in the pools, or -1.
__device__ __forceinline__ int64_t row_at(const Params& p, const Work& w, int pos, int low, int end) {
  if (pos < low || pos >= end) return -1;
  const int page = page_of(p, w, pos);
  if (page < 0) return -1;
  const int size = (int)p.a.cache.page_size;
  return page * p.a.cache.page_stride + ((int64_t)w.head * size + pos % size) * p.a.cache.hd;
}

// A finished row (running maximum and sum m, l) of the block to its place.
template <typename T>
struct Sink {
  const Params& p;
  const Work& w;
  __device__ __forceinline__ void pair(int r, int d, float x, float y, float m, float l) const {
    int t, head;
    const int64_t row = out_index(p, w, r, t, head);
    const int hd = (int)p.a.cache.hd;
    if (p.direct) {
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      T* out = static_cast<T*>(p.a.out) + t * p.a.out_stride + (int64_t)head * hd + d;
      store_pair(out, l == 0.0f ? 0u : Pair<T>::pack(x * inv, y * inv), p.pairs);
    } else {
      const int64_t at = slice_index(p, w) * (p.a.n * p.a.heads) + row;
      if (d == 0) p.ml[at] = make_float2(m, l);
      *reinterpret_cast<float2*>(p.acc + at * hd + d) = make_float2(x, y);
    }
  }
};

template <typename T, int HDP>
__device__ void thin_block(const Params& p, const Work& w, char* smem) {
  constexpr int kBuf = kStep * HDP * 2;  // bytes of a step's keys, and of its values
  constexpr int kChunks = HDP / 8;
  const int warp = threadIdx.x / kLanes, lane = threadIdx.x % kLanes;
  const int hd = (int)p.a.cache.hd;
  const T* keys = static_cast<const T*>(p.a.cache.keys);
  const T* vals = static_cast<const T*>(p.a.cache.values);
  char* ring = smem + warp * kStages * 2 * kBuf;
  Rows<T, HDP> rows;
  rows.init(p, w, 0, smem + kWarps * kStages * 2 * kBuf, lane);
  __syncthreads();
  int begin, end;
  slice_keys(p, w, rows.any_low, rows.any_high, kTile, begin, end);
  if (hd < HDP) {  // the columns that no copy writes are zeros
    for (int i = lane; i < kStages * 2 * kStep * kChunks; i += kLanes)
      if (i % kChunks * 8 >= hd)
        *reinterpret_cast<uint4*>(ring + i / kChunks / kStep * kBuf + chunk_at<HDP>(i / kChunks % kStep, i % kChunks)) =
            make_uint4(0, 0, 0, 0);
    __syncwarp();
  }
  const int first = begin + warp * kStep;
  const int steps = first < end ? (end - first + kTile - 1) / kTile : 0;
  // Lane l < 16 looks up the step's key l, one step ahead of its copy.
  int64_t at = lane < kStep && steps > 0 ? row_at(p, w, first + lane, rows.any_low, end) : -1;
  uint32_t there[kStages];  // which of a buffer's keys are there
  auto issue = [&](int step, uint32_t& mask) {
    if (step < steps) {
      char* buf = ring + step % kStages * 2 * kBuf;
      const uint32_t kb = smem_u32(buf), vb = kb + kBuf;
      mask = __ballot_sync(0xffffffffu, at >= 0) & 0xffffu;
#pragma unroll
      for (int i = 0; i < kStep * kChunks / kLanes; i++) {
        const int idx = i * kLanes + lane, r = idx / kChunks, c = idx % kChunks;
        const int64_t from = __shfl_sync(0xffffffffu, at, r);
        if (c * 8 < hd) {
          const int64_t e = from >= 0 ? from + c * 8 : 0;
          copy16(kb + chunk_at<HDP>(r, c), keys + e, from >= 0);
          copy16(vb + chunk_at<HDP>(r, c), vals + e, from >= 0);
        }
      }
      at = lane < kStep && step + 1 < steps ? row_at(p, w, first + (step + 1) * kTile + lane, rows.any_low, end) : -1;
    }
    copy_commit();
  };
#pragma unroll
  for (int s = 0; s < kStages - 1; s++) issue(s, there[s]);
  for (int step = 0; step < steps; step += kStages) {
#pragma unroll
    for (int b = 0; b < kStages; b++) {
      if (step + b >= steps) break;
      copy_wait<kStages - 2>();
      __syncwarp();
      issue(step + b + kStages - 1, there[(b + kStages - 1) % kStages]);
      const char* buf = ring + (step + b) % kStages * 2 * kBuf;
      const uint32_t kb = smem_u32(buf), vb = kb + kBuf;
      const int k0 = first + (step + b) * kTile;
      float s[2][4];
      rows.template scores<2>(s, kb, 0, lane);
      const bool all = there[b] == 0xffffu && k0 >= rows.all_low && k0 + kStep - 1 <= rows.all_high;
      rows.template softmax<2>(s, k0, all, there[b], p.scale_log2, lane);
      // Where rows see different keys, one row's value must not reach another's sum as 0 * infinity.
      if (!all && any_unbounded<T, HDP>(buf + kBuf, kStep, lane))
        rows.values_guarded(s[0], s[1], buf + kBuf, 0, lane);
      else
        rows.values(s[0], s[1], vb, 0, lane);
      __syncwarp();
    }
  }
  copy_wait<0>();
  rows.finish();
  __syncthreads();
  // The four warps' parts, through shared memory.
  constexpr int kPitch = HDP + 8;
  float* os = reinterpret_cast<float*>(smem);                     // [kWarps][16][kPitch]
  float2* ml = reinterpret_cast<float2*>(os + kWarps * 16 * kPitch);  // [kWarps][16]
#pragma unroll
  for (int h = 0; h < 2; h++) {
    const int r = lane / 4 + 8 * h;
    if (lane % 4 == 0) ml[warp * 16 + r] = make_float2(rows.m[h], rows.l[h]);
#pragma unroll
    for (int j = 0; j < HDP / 8; j++)
      *reinterpret_cast<float2*>(os + (warp * 16 + r) * kPitch + 8 * j + 2 * (lane % 4)) =
          make_float2(rows.o[j][2 * h], rows.o[j][2 * h + 1]);
  }
  __syncthreads();
  const Sink<T> sink{p, w};
  for (int i = threadIdx.x; i < w.rows * (HDP / 2); i += kThreads) {
    const int r = i / (HDP / 2), d = i % (HDP / 2) * 2;
    if (d >= hd) continue;
    float m = -INFINITY;
#pragma unroll
    for (int k = 0; k < kWarps; k++) m = fmaxf(m, ml[k * 16 + r].x);
    const float base = m == -INFINITY ? 0.0f : m;
    float l = 0.0f, x = 0.0f, y = 0.0f;
#pragma unroll
    for (int k = 0; k < kWarps; k++) {
      const float2 q = ml[k * 16 + r];
      const float f = exp2f(q.x - base);
      const float2 v = *reinterpret_cast<const float2*>(os + (k * 16 + r) * kPitch + d);
      if (q.y == 0.0f) continue;
      l += q.y * f;
      x += v.x * f;
      y += v.y * f;
    }
    sink.pair(r, d, x, y, m, l);
  }
}

template <typename T, int HDP>
__device__ void wide_block(const Params& p, const Work& w, char* smem) {
  constexpr int kBuf = kTile * HDP * 2;
  constexpr int kChunks = HDP / 8;
  constexpr int kDepth = HDP <= 128 ? kStages : 2;
  const int warp = threadIdx.x / kLanes, lane = threadIdx.x % kLanes;
  const int hd = (int)p.a.cache.hd;
  const T* keys = static_cast<const T*>(p.a.cache.keys);
  const T* vals = static_cast<const T*>(p.a.cache.values);
  __shared__ int span[kWarps][2];
  Rows<T, HDP> rows;
  rows.init(p, w, warp * 16, smem + kDepth * 2 * kBuf + warp * (HDP / 16) * 512, lane);
  if (lane == 0) {
    span[warp][0] = rows.any_low;
    span[warp][1] = rows.any_high;
  }
  __syncthreads();
  int low = span[0][0], high = span[0][1];
#pragma unroll
  for (int k = 1; k < kWarps; k++) {
    low = min(low, span[k][0]);
    high = max(high, span[k][1]);
  }
  int begin, end;
  slice_keys(p, w, low, high, kTile, begin, end);
  if (hd < HDP)
    for (int i = threadIdx.x; i < kDepth * 2 * kTile * kChunks; i += kThreads)
      if (i % kChunks * 8 >= hd)
        *reinterpret_cast<uint4*>(smem + i / kChunks / kTile * kBuf + chunk_at<HDP>(i / kChunks % kTile, i % kChunks)) =
            make_uint4(0, 0, 0, 0);
  const int tiles = begin < end ? (end - begin + kTile - 1) / kTile : 0;
  // Warp w copies keys 16 w .. 16 w + 15 of a tile; lane l < 16 looks up key l.
  __shared__ uint32_t there[kDepth][kWarps];
  auto issue = [&](int tile) {
    if (tile < tiles) {
      char* buf = smem + tile % kDepth * 2 * kBuf;
      const uint32_t kb = smem_u32(buf), vb = kb + kBuf;
      const int64_t at = lane < 16 ? row_at(p, w, begin + tile * kTile + warp * 16 + lane, low, end) : -1;
      const uint32_t mask = __ballot_sync(0xffffffffu, at >= 0);
      if (lane == 0) there[tile % kDepth][warp] = mask;
#pragma unroll
      for (int i = 0; i < 16 * kChunks / kLanes; i++) {
        const int idx = i * kLanes + lane, r = idx / kChunks, c = idx % kChunks;
        const int64_t from = __shfl_sync(0xffffffffu, at, r);
        if (c * 8 < hd) {
          const int64_t e = from >= 0 ? from + c * 8 : 0;
          copy16(kb + chunk_at<HDP>(warp * 16 + r, c), keys + e, from >= 0);
          copy16(vb + chunk_at<HDP>(warp * 16 + r, c), vals + e, from >= 0);
        }
      }
    }
    copy_commit();
  };
#pragma unroll
  for (int s = 0; s < kDepth - 1; s++) issue(s);
  for (int tile = 0; tile < tiles; tile++) {
    copy_wait<kDepth - 2>();
    __syncthreads();  // the tile is there, and the buffer of the one before it is read
    issue(tile + kDepth - 1);
    const int b = tile % kDepth;
    const char* buf = smem + b * 2 * kBuf;
    const uint32_t kb = smem_u32(buf), vb = kb + kBuf;
    const int k0 = begin + tile * kTile;
    if (k0 > rows.any_high || k0 + kTile <= rows.any_low) continue;
    uint64_t mask = 0;
#pragma unroll
    for (int k = 0; k < kWarps; k++) mask |= (uint64_t)(there[b][k] & 0xffffu) << (16 * k);
    float s[kTile / 8][4];
    rows.template scores<kTile / 8>(s, kb, 0, lane);
    const bool all = mask == ~0ull && k0 >= rows.all_low && k0 + kTile - 1 <= rows.all_high;
    rows.template softmax<kTile / 8>(s, k0, all, mask, p.scale_log2, lane);
    if (!all && any_unbounded<T, HDP>(buf + kBuf, kTile, lane)) {
#pragma unroll
      for (int k = 0; k < kTile / 16; k++) rows.values_guarded(s[2 * k], s[2 * k + 1], buf + kBuf, 16 * k, lane);
    } else {
#pragma unroll
      for (int k = 0; k < kTile / 16; k++) rows.values(s[2 * k], s[2 * k + 1], vb, 16 * k, lane);
    }
  }
  copy_wait<0>();
  rows.finish();
  const Sink<T> sink{p, w};
#pragma unroll
  for (int h = 0; h < 2; h++) {
    const int r = warp * 16 + lane / 4 + 8 * h;
    if (r >= w.rows) continue;
#pragma unroll
    for (int j = 0; j < HDP / 8; j++) {
      const int d = 8 * j + 2 * (lane % 4);
      if (d < hd) sink.pair(r, d, rows.o[j][2 * h], rows.o[j][2 * h + 1], rows.m[h], rows.l[h]);
    }
  }
}

template <typename T, int HDP>
__global__ void __launch_bounds__(kThreads) attention_mma_kernel(const __grid_constant__ Params p) {
  pdl_launch_dependents();
  pdl_wait();
  extern __shared__ __align__(128) char smem[];
  Work w;
  if (!find_work(p, w)) return;
  if ((w.prefix ? p.prefix_rows : p.own_rows) == kThinRows)
    thin_block<T, HDP>(p, w, smem);
  else
    wide_block<T, HDP>(p, w, smem);
}

template <typename T, int HDP>
cudaError_t launch_size(const Params& p, cudaStream_t stream, bool pdl) {
  constexpr int kDepth = HDP <= 128 ? kStages : 2;
  constexpr int kQ = HDP <= 128 ? 0 : HDP / 16 * 512;  // a warp's query fragments
  constexpr int thin = kWarps * kStages * 2 * kStep * HDP * 2 + kQ;
  constexpr int join = kWarps * 16 * ((HDP + 8) * 4 + 8);
  constexpr int wide = kDepth * 2 * kTile * HDP * 2 + kWarps * kQ;
  constexpr int smem = thin > wide ? (thin > join ? thin : join) : (wide > join ? wide : join);
  if (cudaError_t e = cudaFuncSetAttribute(attention_mma_kernel<T, HDP>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                           smem);
      e != cudaSuccess)
    return e;
  return launch_ex(attention_mma_kernel<T, HDP>, p, attention_grid(p), kThreads, smem, stream, pdl);
}

template <typename T>
cudaError_t launch_heads(const Params& p, cudaStream_t stream, bool pdl) {
  if (p.a.cache.hd <= 64) return launch_size<T, 64>(p, stream, pdl);
  if (p.a.cache.hd <= 128) return launch_size<T, 128>(p, stream, pdl);
  return launch_size<T, 256>(p, stream, pdl);
}

}  // namespace

namespace paged {

cudaError_t launch_attention_mma(const Params& p, cudaStream_t stream, bool pdl) {
  return p.a.cache.type == kF16 ? launch_heads<__half>(p, stream, pdl) : launch_heads<__nv_bfloat16>(p, stream, pdl);
}

}  // namespace paged
}  // namespace dn
