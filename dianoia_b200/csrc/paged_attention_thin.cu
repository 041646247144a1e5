// The paged attention's kernel for few rows of queries on 16-bit caches: the
// heads of one group of a decode step, a small batch on the shared prefix.
//
// Bound by the keys' and values' bytes; what it must not spend is
// instructions. So the products are taken with the keys as the wide side:
// S^T = K Q^T (16 keys x 8 rows) and O^T = V^T P^T (16 dimensions x 8 rows)
// with m16n8k16 and f32 accumulators, so that 8 rows cost 8 rows' work, and a
// step of 16 keys of 128 dimensions takes 16 products. P^T comes from S^T's
// layout by an 8 x 8 transpose in registers. The softmax keeps the base it has
// (kLift below the maximum of the time, pair16.cuh) until a score passes that
// maximum by kSlack, so most steps exchange nothing between lanes; what is
// stored is exact for any base.
//
// Each of a block's 4 warps streams its own 16 keys of every 64 through a ring
// of kStages buffers, so that no block barrier stands in the loop; the warps'
// results are joined once at the end. Where 16 keys lie in one page (page
// sizes that are multiples of 16) one lane brings them by tiled TMA copies of
// 16 x 64 elements (one bulk copy a row, which needs no tensor map, brought 3.1
// TB/s where these brought 4.3); for other page sizes the lanes copy 16 bytes
// each. Both leave chunk c of key r's 64 elements at chunk
// c ^ (r & 7), which the fragment loads read without a bank conflict.
// Measured: 192 sequences of 540 keys on average, 8 kv heads of 128, 4 heads a
// group, bf16: 69 us, 5.9 TB/s of keys and values. Two buffers a warp and three
// blocks to an SM stream faster than three and two (69 against 79 us): a block
// is mostly latency (finding its sequence, its pages, its first keys: 3 us).
#include "dn_tmap.h"
#include "paged_attention.cuh"
#include "pair16.cuh"

namespace dn {

using namespace paged;

namespace {

constexpr int kThreads = 128;
constexpr int kWarps = kThreads / kLanes;
constexpr int kStep = 16;             // keys of a warp's step
constexpr int kTile = kWarps * kStep;  // keys of the block's

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
__device__ __forceinline__ uint32_t transposed(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}

// 16 bytes to shared memory, zeros where `there` is false.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
// One arrival on `bar` once the thread's copies so far are done.
__device__ __forceinline__ void copy_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

struct alignas(64) Maps {
  CUtensorMap keys, values;
};

template <int HDP>
struct Shape {
  static constexpr int kPanels = HDP / 64;                // 64 elements wide
  static constexpr int kPanel = kStep * 128;              // bytes of a panel of a step
  static constexpr int kBuf = kPanels * kPanel;           // a step's keys; as many again its values
  static constexpr int kStages = 2;
  static constexpr int kRing = kStages * 2 * kBuf;        // a warp's
};

// Bytes of a block's rings, which the warps' results take over at the end.
constexpr int smem_tiles(int hdp, int nt) {
  const int ring = kWarps * 2 * 2 * kStep * hdp * 2, join = kWarps * 8 * nt * ((hdp + 4) * 4 + 8);
  return ring > join ? ring : join;
}

// Byte offset of 16-byte chunk c (8 elements) of key r of a step.
__device__ __forceinline__ uint32_t chunk_at(int r, int c) {
  return (uint32_t)((c >> 3) * (kStep * 128) + r * 128 + (((c ^ r) & 7) << 4));
}

// A block of NT * 8 rows of one kv head on a slice of one part's keys. Lane
// (g, i) = (lane / 4, lane % 4) holds, of each 8 rows, rows 2 i and 2 i + 1:
// their scores of keys g and g + 8, their outputs of dimensions g and g + 8 of
// each 16, and their base m and sum l.
template <typename T, int HDP, int NT, bool TMA>
__device__ __forceinline__ void thin_block(const Params& p, const Maps& maps, const Work& w, char* smem,
                                           uint64_t* bars) {
  using S = Shape<HDP>;
  constexpr int kRows = 8 * NT;
  constexpr float kLift = Pair<T>::kLift, kSlack = Pair<T>::kSlack;
  const int warp = threadIdx.x / kLanes, lane = threadIdx.x % kLanes;
  const int hd = (int)p.a.cache.hd;
  char* ring = smem + warp * S::kRing;
  uint64_t* full = bars + warp * S::kStages;
  if (lane == 0) {
    for (int i = 0; i < S::kStages; i++) mbar_init(&full[i], TMA ? 1 : kLanes);
    fence_mbar_init();
  }

  // What each row sees, and the queries' fragments.
  int lo = 0, hi = -1;
  if (lane < w.rows) {
    const int t = (w.row0 + lane) / p.group;
    sees(p, w, t, lo, hi);
  }
  // (Rows that see nothing take part unmasked; their results are dropped.)
  const bool any = hi >= lo;
  const int all_low = __reduce_max_sync(0xffffffffu, any ? lo : 0);
  const int all_high = __reduce_min_sync(0xffffffffu, any ? hi : INT32_MAX);
  const int any_low = __reduce_min_sync(0xffffffffu, any ? lo : INT32_MAX);
  const int any_high = __reduce_max_sync(0xffffffffu, any ? hi : -1);
  int begin, end;
  slice_keys(p, w, any_low, any_high, kTile, begin, end);
  const int first = begin + warp * kStep;
  const int steps = first < end ? (end - first + kTile - 1) / kTile : 0;

  if (!TMA && hd < HDP)  // the columns that no copy writes are zeros
    for (int i = lane; i < S::kStages * 2 * kStep * (HDP - hd) / 8; i += kLanes) {
      const int c = hd / 8 + i % ((HDP - hd) / 8), r = i / ((HDP - hd) / 8);
      *reinterpret_cast<uint4*>(ring + r / kStep * S::kBuf + chunk_at(r % kStep, c)) = make_uint4(0, 0, 0, 0);
    }
  __syncwarp();

  // The entry of a step's page (TMA), or of lane l's key l % 16, is on its way
  // one step ahead of the copies.
  const int panels = (hd + 63) / 64;
  uint32_t there[S::kStages];  // which of a buffer's keys are there
  int entry = -1;
  auto look_up = [&](int step) {
    const int k0 = first + step * kTile;
    if (step < steps) entry = entry_at(p, w, TMA ? k0 : k0 + lane % kStep);
  };
  auto issue = [&](int step, int b) {
    if (step >= steps) return;
    char* kb = ring + b * 2 * S::kBuf;
    char* vb = kb + S::kBuf;
    if constexpr (TMA) {
      const int k0 = first + step * kTile;
      // A page that is not there is one past the last, which reads as zeros.
      const int found = page_of(p, entry), page = found >= 0 ? found : (int)p.a.cache.pages;
      const int slot = k0 - entry_of(p, k0) * (int)p.a.cache.page_size;
      there[b] = found >= 0 ? 0xffffu : 0u;
      if (lane == 0) mbar_arrive_expect_tx(&full[b], (uint32_t)panels * 2 * S::kPanel);
      __syncwarp();
      if (lane < 2 * panels) {  // a copy a lane: the panels of the keys, then of the values
        const int c = lane < panels ? lane : lane - panels;
        tma_load_4d((lane < panels ? kb : vb) + c * S::kPanel, lane < panels ? &maps.keys : &maps.values, 64 * c, slot,
                    w.head, page, &full[b]);
      }
    } else {
      const int64_t at = row_at(p, w, entry, first + step * kTile + lane % kStep, any_low, end);
      there[b] = __ballot_sync(0xffffffffu, at >= 0) & 0xffffu;
      const T* keys = static_cast<const T*>(p.a.cache.keys);
      const T* vals = static_cast<const T*>(p.a.cache.values);
#pragma unroll 4
      for (int i = lane; i < kStep * HDP / 8; i += kLanes) {
        const int r = i / (HDP / 8), c = i % (HDP / 8);
        const int64_t from = __shfl_sync(0xffffffffu, at, r);
        if (c * 8 < hd) {
          const int64_t e = from >= 0 ? from + c * 8 : 0;
          copy16(smem_u32(kb) + chunk_at(r, c), keys + e, from >= 0);
          copy16(smem_u32(vb) + chunk_at(r, c), vals + e, from >= 0);
        }
      }
      copy_arrive(&full[b]);
    }
    look_up(step + 1);
  };
  look_up(0);
#pragma unroll
  for (int s = 0; s < S::kStages; s++) issue(s, s);

  int low[NT][2], high[NT][2];
  float m[NT][2], l[NT][2], o[NT][HDP / 16][4];
  uint32_t q[NT][HDP / 16][2];
#pragma unroll
  for (int n = 0; n < NT; n++) {
#pragma unroll
    for (int h = 0; h < 2; h++) {
      low[n][h] = __shfl_sync(0xffffffffu, lo, 8 * n + 2 * (lane % 4) + h);
      high[n][h] = __shfl_sync(0xffffffffu, hi, 8 * n + 2 * (lane % 4) + h);
      m[n][h] = -INFINITY;
      l[n][h] = 0.0f;
    }
    const T* src = nullptr;
    const int row = 8 * n + lane / 4;
    if (row < w.rows) {
      int t, head;
      out_index(p, w, row, t, head);
      src = static_cast<const T*>(p.a.q) + t * p.a.q_stride + (int64_t)head * hd;
    }
#pragma unroll
    for (int k = 0; k < HDP / 16; k++) {
#pragma unroll
      for (int u = 0; u < 2; u++) {
        const int d = 16 * k + 8 * u + 2 * (lane % 4);
        q[n][k][u] = src != nullptr && d < hd ? load_pair(src + d, p.pairs) : 0u;
      }
#pragma unroll
      for (int e = 0; e < 4; e++) o[n][k][e] = 0.0f;
    }
  }

  bool live = true;
  int step = 0;
  for (int base = 0; base < steps && live; base += S::kStages) {
#pragma unroll
    for (int b = 0; b < S::kStages; b++) {
      step = base + b;
      if (step >= steps) break;
      live = __all_sync(0xffffffffu, wait_phase(&full[b], (step / S::kStages) & 1, p.status, kStatusTmaTimeout));
      if (!live) break;
      const char* buf = ring + b * 2 * S::kBuf;
      const uint32_t kb = smem_u32(buf), vb = kb + S::kBuf;
      const int k0 = first + step * kTile;

      // S^T: two chains of accumulators, of even and odd slices of the head.
      float s[NT][4], s2[NT][4];
#pragma unroll
      for (int n = 0; n < NT; n++)
#pragma unroll
        for (int e = 0; e < 4; e++) s[n][e] = s2[n][e] = 0.0f;
#pragma unroll
      for (int k = 0; k < HDP / 16; k++) {
        // Heads of 129 to 192 have a panel that no copy writes: what stands there
        // may be NaN, which the queries' zeros would pass on.
        if (HDP > 128 && 16 * k >= hd) continue;
        uint32_t a[4];
        ldsm4(a, kb + chunk_at(lane & 15, 2 * k + (lane >> 4)));
#pragma unroll
        for (int n = 0; n < NT; n++) mma(k % 2 ? s2[n] : s[n], a, q[n][k][0], q[n][k][1], T());
      }
      const bool all = there[b] == 0xffffu && k0 >= all_low && k0 + kStep - 1 <= all_high;
      bool past = false;
#pragma unroll
      for (int n = 0; n < NT; n++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          float x = (s[n][e] + s2[n][e]) * p.scale_log2;
          if (!all) {
            const int j = lane / 4 + 8 * (e >> 1), h = e & 1;
            const bool seen = (there[b] >> j & 1u) != 0 && k0 + j >= low[n][h] && k0 + j <= high[n][h];
            x = seen ? x : -INFINITY;
          }
          s[n][e] = x;
        }
#pragma unroll
      for (int n = 0; n < NT; n++)
#pragma unroll
        for (int h = 0; h < 2; h++) past = past || fmaxf(s[n][h], s[n][2 + h]) - m[n][h] > kSlack + kLift;
      if (__any_sync(0xffffffffu, past)) {  // new bases: kLift below the rows' maxima so far
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
          for (int h = 0; h < 2; h++) {
            float top = fmaxf(s[n][h], s[n][2 + h]);
#pragma unroll
            for (int off = 4; off <= 16; off <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
            const float next = fmaxf(m[n][h], top - kLift);
            const float keep = next == -INFINITY ? 1.0f : exp2_fast(m[n][h] - next);
            m[n][h] = next;
            l[n][h] *= keep;
#pragma unroll
            for (int k = 0; k < HDP / 16; k++) {
              o[n][k][h] *= keep;
              o[n][k][2 + h] *= keep;
            }
          }
      }
      uint32_t pf[NT][2];
#pragma unroll
      for (int n = 0; n < NT; n++) {
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const float base_m = m[n][e & 1] == -INFINITY ? 0.0f : m[n][e & 1];
          s[n][e] = exp2_fast(s[n][e] - base_m);
          l[n][e & 1] += s[n][e];  // a lane's share of the row's sum
        }
        pf[n][0] = transposed(Pair<T>::pack(s[n][0], s[n][1]));
        pf[n][1] = transposed(Pair<T>::pack(s[n][2], s[n][3]));
      }
      // Where rows see different keys, one row's value must not reach
      // another's sum as 0 * infinity: then terms are added one by one.
      bool bad = false;
      if (!all)
        for (int i = lane; i < kStep * 8 * panels; i += kLanes) bad = bad || unbounded16<T>(buf + S::kBuf + i * 16);
      if (__any_sync(0xffffffffu, bad)) {
#pragma unroll 1
        for (int j = 0; j < kStep; j++) {
#pragma unroll
          for (int n = 0; n < NT; n++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
              const float x = __shfl_sync(0xffffffffu, j < 8 ? s[n][h] : s[n][2 + h], j % 8 * 4 + lane % 4);
              const float r = to_f32<T>(from_f32<T>(x));
              // (A key that the row sees counts, however small its weight.)
              if ((there[b] >> j & 1u) == 0 || k0 + j < low[n][h] || k0 + j > high[n][h]) continue;
#pragma unroll
              for (int k = 0; k < HDP / 16; k++)
#pragma unroll
                for (int u = 0; u < 2; u++) {
                  const T v = reinterpret_cast<const T*>(buf + S::kBuf + chunk_at(j, 2 * k + u))[lane / 4];
                  o[n][k][2 * u + h] = fmaf(r, to_f32<T>(v), o[n][k][2 * u + h]);
                }
            }
        }
      } else {
#pragma unroll
        for (int k = 0; k < HDP / 16; k++) {
          if (HDP > 128 && 16 * k >= hd) continue;
          uint32_t a[4];
          ldsm4_t(a, vb + chunk_at((lane & 7) + (lane >> 4) * 8, 2 * k + ((lane >> 3) & 1)));
#pragma unroll
          for (int n = 0; n < NT; n++) mma(o[n][k], a, pf[n][0], pf[n][1], T());
        }
      }
      __syncwarp();  // the buffer is read: its next copy may start
      issue(step + S::kStages, b);
    }
  }
  if (!live)  // copies on their way into this step's buffer and the ones after it
    for (int i = step; i < min(steps, step + S::kStages); i++) mbar_land(&full[i % S::kStages], (i / S::kStages) & 1);
#pragma unroll
  for (int n = 0; n < NT; n++)
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
      for (int off = 4; off <= 16; off <<= 1) l[n][h] += __shfl_xor_sync(0xffffffffu, l[n][h], off);

#pragma unroll
  for (int n = 0; n < NT; n++)
#pragma unroll
    for (int h = 0; h < 2; h++)
      if (high[n][h] < low[n][h]) {
        m[n][h] = -INFINITY;
        l[n][h] = 0.0f;
      }

  // The four warps' parts, through shared memory.
  __syncthreads();
  constexpr int kOut = HDP + 4;
  float* os = reinterpret_cast<float*>(smem);                          // [kWarps][kRows][kOut]
  float2* ml = reinterpret_cast<float2*>(os + kWarps * kRows * kOut);  // [kWarps][kRows]
#pragma unroll
  for (int n = 0; n < NT; n++)
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const int r = 8 * n + 2 * (lane % 4) + h;
      if (lane < 4) ml[warp * kRows + r] = make_float2(m[n][h], l[n][h]);
      if (r < w.rows)
#pragma unroll
        for (int k = 0; k < HDP / 16; k++) {
          os[(warp * kRows + r) * kOut + 16 * k + lane / 4] = o[n][k][h];
          os[(warp * kRows + r) * kOut + 16 * k + 8 + lane / 4] = o[n][k][2 + h];
        }
    }
  __syncthreads();
  for (int i = threadIdx.x; i < w.rows * (HDP / 2); i += kThreads) {
    const int r = i / (HDP / 2), d = i % (HDP / 2) * 2;
    if (d >= hd) continue;
    float top = -INFINITY;
#pragma unroll
    for (int k = 0; k < kWarps; k++) top = fmaxf(top, ml[k * kRows + r].x);
    const float base = top == -INFINITY ? 0.0f : top;
    float sum = 0.0f, x = 0.0f, y = 0.0f;
#pragma unroll
    for (int k = 0; k < kWarps; k++) {
      const float2 part = ml[k * kRows + r];
      if (part.y == 0.0f) continue;  // (a NaN goes on)
      const float f = exp2_fast(part.x - base);
      const float2 v = *reinterpret_cast<const float2*>(os + (k * kRows + r) * kOut + d);
      sum += part.y * f;
      x += v.x * f;
      y += v.y * f;
    }
    int t, head;
    const int64_t row = out_index(p, w, r, t, head);
    if (p.direct) {
      const float inv = 1.0f / sum;
      T* out = static_cast<T*>(p.a.out) + t * p.a.out_stride + (int64_t)head * hd + d;
      store_pair(out, sum == 0.0f ? 0u : Pair<T>::pack(x * inv, y * inv), p.pairs);
    } else {
      const int64_t to = slice_index(p, w) * (p.a.n * p.a.heads) + row;
      if (d == 0) p.ml[to] = make_float2(top, sum);
      *reinterpret_cast<float2*>(p.acc + to * hd + d) = make_float2(x, y);
    }
  }
}

template <typename T, int HDP, int NT, bool TMA>
__global__ void __launch_bounds__(kThreads)
    attention_thin_kernel(const __grid_constant__ Params p, const __grid_constant__ Maps maps) {
  pdl_launch_dependents();
  // Beside the wide kernel, whose start already followed the inputs, there is
  // nothing to wait for but its end, before this grid's: one block does.
  if (!p.beside) pdl_wait();
  extern __shared__ __align__(1024) char smem[];
  // (No static shared memory: it would be rounded up to this alignment.)
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + smem_tiles(HDP, NT));
  Work w;
  if (find_work(p, w)) thin_block<T, HDP, NT, TMA>(p, maps, w, smem, bars);
  if (p.beside && blockIdx.x == 0 && blockIdx.y == 0) pdl_wait();
}

template <typename T, int HDP, int NT, bool TMA>
cudaError_t launch_copies(const Params& p, const Maps& maps, cudaStream_t stream, bool pdl) {
  static_assert(smem_tiles(HDP, NT) >= kWarps * Shape<HDP>::kRing, "rings");
  constexpr int smem = smem_tiles(HDP, NT) + kWarps * Shape<HDP>::kStages * 8;
  if (cudaError_t e = allow_smem<attention_thin_kernel<T, HDP, NT, TMA>>(smem); e != cudaSuccess) return e;
  return launch_ex(attention_thin_kernel<T, HDP, NT, TMA>, attention_grid(p), kThreads, smem, stream, pdl, p, maps);
}

template <typename T, int HDP>
cudaError_t launch_rows(const Params& p, cudaStream_t stream, bool pdl) {
  const PagedCache& c = p.a.cache;
  Maps maps{};
  const bool tma = c.page_size % kStep == 0 && c.pages > 0;
  if (tma && !(encode_tmap_pages(&maps.keys, c.keys, c.type == kBF16, c.hd, c.page_size, c.kv_heads, c.pages,
                                 c.page_stride, kStep) &&
               encode_tmap_pages(&maps.values, c.values, c.type == kBF16, c.hd, c.page_size, c.kv_heads, c.pages,
                                 c.page_stride, kStep)))
    return cudaErrorInvalidValue;
  if (p.thin_rows == 8)
    return tma ? launch_copies<T, HDP, 1, true>(p, maps, stream, pdl) : launch_copies<T, HDP, 1, false>(p, maps, stream, pdl);
  return tma ? launch_copies<T, HDP, 2, true>(p, maps, stream, pdl) : launch_copies<T, HDP, 2, false>(p, maps, stream, pdl);
}

template <typename T>
cudaError_t launch_heads(const Params& p, cudaStream_t stream, bool pdl) {
  if (p.a.cache.hd <= 64) return launch_rows<T, 64>(p, stream, pdl);
  if (p.a.cache.hd <= 128) return launch_rows<T, 128>(p, stream, pdl);
  return launch_rows<T, 256>(p, stream, pdl);
}

}  // namespace

namespace paged {

cudaError_t launch_attention_thin(const Params& p, cudaStream_t stream, bool pdl) {
  return p.a.cache.type == kF16 ? launch_heads<__half>(p, stream, pdl) : launch_heads<__nv_bfloat16>(p, stream, pdl);
}

}  // namespace paged
}  // namespace dn
