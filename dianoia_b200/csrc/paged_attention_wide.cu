// The paged attention's kernel for many rows of queries on 16-bit caches: the
// whole batch on the shared prefix, long chunks of a sequence's queries.
//
// 128 rows of one kv head share every key, so the products are the bound:
// S = Q K^T and O += P V on the 5th-generation tensor cores (tcgen05, f32
// accumulators in TMEM). A block runs three parts at once:
//   warp 4 brings tiles of 64 keys and their values by tiled TMA copies;
//   warp 5 issues the products: S of tile i + 1 while tile i is in softmax;
//   warps 0 .. 3 hold a row of S each thread: they read it from TMEM, keep the
//   row's base and sum, and write P (16-bit) over it, which the tensor cores
//   read from there as the first operand of P V.
// S is doubled in TMEM so that the tensor cores and the softmax overlap. A
// base moves only when a score passes it by kSlack (P then stays below 2^8),
// so O is rescaled in TMEM in the first tiles and hardly ever after. Where rows
// of the block see different keys of a tile and a value there is not finite,
// that tile's P V is added term by term instead (0 * infinity would be NaN).
#include <type_traits>

#include "dn_tmap.h"
#include "paged_attention.cuh"
#include "pair16.cuh"

namespace dn {

using namespace paged;

namespace {

constexpr int kRows = kWideRows;
constexpr int kKeys = 64;       // of a tile
constexpr int kRowThreads = 128;
constexpr int kThreads = 192;
constexpr float kSlack = 8.0f;  // log2 units a score may pass the running base

struct alignas(64) Maps {
  CUtensorMap keys, values;
};

template <int HDP>
struct Shape {
  static constexpr int kPanels = HDP / 64;
  static constexpr int kQPanel = kRows * 128;       // bytes: 64 elements of every row
  static constexpr int kPanel = kKeys * 128;        // of every key of a tile
  static constexpr int kTileBytes = kPanels * kPanel;
  static constexpr int kStages = HDP <= 128 ? 3 : 2;
  static constexpr int kQ = kPanels * kQPanel;
  static constexpr int kSmem = kQ + kStages * 2 * kTileBytes;
  static constexpr uint32_t kCols = HDP <= 128 ? 256 : 512;  // of TMEM: S twice, then O
};

struct Bars {
  uint64_t k_full[3], k_empty[3], v_full[3], v_empty[3], s_full[2], p_full[2];
  // Of even and odd tiles: a row thread may pass over a tile's, and the parity
  // of a barrier tells two phases in a row apart, not three.
  uint64_t o_done[2];
};

// Shared-memory operand, 128-byte swizzled; `lead` is the stride between
// panels (used where the 64 contiguous elements are the operand's rows).
__device__ __forceinline__ uint64_t desc(uint32_t addr, uint32_t lead) {
  return (uint64_t)((addr >> 4) & 0x3FFF) | ((uint64_t)(lead >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// f32 accumulator, A and B both of the element type; `b_rows`: B's 64
// contiguous elements run along its N.
constexpr uint32_t idesc(bool bf16, int n, bool b_rows) {
  return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((b_rows ? 1u : 0u) << 16) |
         ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kRows >> 4) << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(id), "r"(add)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t id, uint32_t add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(id), "r"(add)
      : "memory");
}
__device__ __forceinline__ void commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// 32 columns of the thread's lane; the values are there after wait_ld.
__device__ __forceinline__ void ld32(uint32_t addr, float (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, "
      "%11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, "
      "%28, %29, %30, %31}, [%32];"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]),
        "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]),
        "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]),
        "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void wait_ld(float (&v)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]),
                 "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]),
                 "+f"(v[15]), "+f"(v[16]), "+f"(v[17]), "+f"(v[18]), "+f"(v[19]), "+f"(v[20]), "+f"(v[21]),
                 "+f"(v[22]), "+f"(v[23]), "+f"(v[24]), "+f"(v[25]), "+f"(v[26]), "+f"(v[27]), "+f"(v[28]),
                 "+f"(v[29]), "+f"(v[30]), "+f"(v[31])
               :
               : "memory");
}
__device__ __forceinline__ void st32(uint32_t addr, const uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(addr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]),
      "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]),
      "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
      : "memory");
}
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// The rows' part. Row `r` of the block is the thread's.
template <typename T, int HDP>
__device__ __forceinline__ void softmax_rows(const Params& p, const Work& w, char* smem, Bars& bars, uint32_t* skip,
                                             uint32_t tmem, int begin, int tiles, int low, int high, int all_low,
                                             int all_high) {
  using S = Shape<HDP>;
  const int r = threadIdx.x, lane = r % kLanes;
  const uint32_t mine = tmem + ((uint32_t)(r / kLanes * 32) << 16);
  const uint32_t out_cols = mine + 2 * kKeys;
  const int hd = (int)p.a.cache.hd;
  float m = -INFINITY, l = 0.0f;
  // Lanes 0 .. 3 know which 16 keys of the next tile have a page.
  auto look_up = [&](int tile) {
    return lane < kKeys / 16 && tile < tiles && page_of(p, w, begin + tile * kKeys + 16 * lane) >= 0;
  };
  bool next_there = look_up(0);
  bool live = true;
  for (int i = 0; i < tiles; i++) {
    const unsigned there = __ballot_sync(0xffffffffu, next_there);
    next_there = look_up(i + 1);
    const int k0 = begin + i * kKeys;
    const uint32_t cols = mine + (uint32_t)(i & 1) * kKeys;
    live = __all_sync(0xffffffffu, mbar_wait_bounded(&bars.s_full[i & 1], (i >> 1) & 1, p.status, kStatusMmaTimeout));
    if (!live) break;
    fence_after();
    float s[2][32];
    ld32(cols, s[0]);
    ld32(cols + 32, s[1]);
    wait_ld(s[0]);
    wait_ld(s[1]);
    const bool all = there == 0xfu && k0 >= all_low && k0 + kKeys - 1 <= all_high;  // the same in every row
    if (!all) {
#pragma unroll
      for (int j = 0; j < kKeys; j++) {
        const bool seen = (there >> (j / 16) & 1u) != 0 && k0 + j >= low && k0 + j <= high;
        s[j / 32][j % 32] = seen ? s[j / 32][j % 32] * p.scale_log2 : -INFINITY;
      }
    } else {
#pragma unroll
      for (int j = 0; j < kKeys; j++) s[j / 32][j % 32] *= p.scale_log2;
    }
    float top4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
    for (int j = 0; j < kKeys; j++) top4[j % 4] = fmaxf(top4[j % 4], s[j / 32][j % 32]);
    const float top = fmaxf(fmaxf(top4[0], top4[1]), fmaxf(top4[2], top4[3]));
    bool waited = false;
    if (__any_sync(0xffffffffu, top > m + kSlack)) {
      const float next = fmaxf(m, top);
      const float keep = next == -INFINITY ? 1.0f : exp2_fast(m - next);
      m = next;
      l *= keep;
      if (i > 0) {
        live = __all_sync(0xffffffffu, mbar_wait_bounded(&bars.o_done[(i - 1) & 1], ((i - 1) >> 1) & 1, p.status, kStatusMmaTimeout));
        if (!live) break;
        waited = true;
        fence_after();
#pragma unroll 1
        for (int c = 0; c < HDP; c += 32) {
          float o[32];
          ld32(out_cols + c, o);
          wait_ld(o);
          uint32_t u[32];
#pragma unroll
          for (int e = 0; e < 32; e++) u[e] = __float_as_uint(o[e] * keep);
          st32(out_cols + c, u);
        }
        wait_st();
      }
    }
    const float base = m == -INFINITY ? 0.0f : m;
    uint32_t pk[32];
    float sum4[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < kKeys; j += 2) {
      const float x = exp2_fast(s[j / 32][j % 32] - base), y = exp2_fast(s[j / 32][j % 32 + 1] - base);
      s[j / 32][j % 32] = x;
      s[j / 32][j % 32 + 1] = y;
      sum4[j / 2 % 4] += x + y;
      pk[j / 2] = Pair<T>::pack(x, y);
    }
    l += (sum4[0] + sum4[1]) + (sum4[2] + sum4[3]);
    if (!all) {
      // The values have to be looked at, and may have to be added here.
      char* vals = smem + S::kQ + (i % S::kStages) * 2 * S::kTileBytes + S::kTileBytes;
      live = __all_sync(0xffffffffu, mbar_wait_bounded(&bars.v_full[i % S::kStages], (i / S::kStages) & 1, p.status,
                                                       kStatusTmaTimeout));
      bool bad = false;
      for (int c = lane; c < S::kTileBytes / 16; c += kLanes) bad = bad || unbounded16<T>(vals + c * 16);
      bad = __any_sync(0xffffffffu, bad);  // every warp finds the same
      if (r == 0) skip[i & 1] = bad ? 1u : 0u;
      if (bad) {
        if (i > 0 && !waited)
          live = __all_sync(0xffffffffu, mbar_wait_bounded(&bars.o_done[(i - 1) & 1], ((i - 1) >> 1) & 1, p.status, kStatusMmaTimeout));
        fence_after();
        float pr[kKeys];  // indexed at run time: in local memory, here only
#pragma unroll
        for (int j = 0; j < kKeys; j++) pr[j] = to_f32<T>(from_f32<T>(s[j / 32][j % 32]));
#pragma unroll 1
        for (int c = 0; c < HDP; c += 32) {
          float o[32];
          ld32(out_cols + c, o);
          wait_ld(o);
          if (i == 0)
#pragma unroll
            for (int e = 0; e < 32; e++) o[e] = 0.0f;
#pragma unroll 1
          for (int j = 0; j < kKeys; j++) {
            if (pr[j] != 0.0f)
#pragma unroll
              for (int e = 0; e < 32; e++) {
                const int d = c + e;
                const T v = reinterpret_cast<const T*>(vals + d / 64 * S::kPanel + j * 128 +
                                                       (((d % 64 / 8) ^ (j & 7)) << 4))[d % 8];
                o[e] = fmaf(pr[j], to_f32<T>(v), o[e]);
              }
          }
          uint32_t u[32];
#pragma unroll
          for (int e = 0; e < 32; e++) u[e] = __float_as_uint(o[e]);
          __syncwarp();
          st32(out_cols + c, u);
        }
      }
    } else if (r == 0) {
      skip[i & 1] = 0;
    }
    st32(cols, pk);
    wait_st();
    fence_before();
    mbar_arrive(&bars.p_full[i & 1]);
  }
  if (tiles > 0 && live) {
    live = __all_sync(0xffffffffu,
                      mbar_wait_bounded(&bars.o_done[(tiles - 1) & 1], ((tiles - 1) >> 1) & 1, p.status, kStatusMmaTimeout));
    fence_after();
  }
  // The row's result.
  int t = 0, head = 0;
  const bool there = r < w.rows;
  const int64_t row = there ? out_index(p, w, r, t, head) : 0;
  const int64_t to = slice_index(p, w) * (p.a.n * p.a.heads) + row;
  if (high < low) {  // a row that sees nothing took part unmasked
    m = -INFINITY;
    l = 0.0f;
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  if (there && !p.direct) p.ml[to] = make_float2(m, l);
  if (tiles == 0 && !p.direct) return;  // the join reads no values of a row with l = 0
#pragma unroll 1
  for (int c = 0; c < HDP; c += 32) {
    float o[32];
    if (tiles > 0) {
      ld32(out_cols + c, o);
      wait_ld(o);
    } else {
#pragma unroll
      for (int e = 0; e < 32; e++) o[e] = 0.0f;
    }
    if (!there) continue;
    if (p.direct) {
      T* out = static_cast<T*>(p.a.out) + t * p.a.out_stride + (int64_t)head * hd;
#pragma unroll
      for (int e = 0; e < 32; e += 2)
        if (c + e < hd)
          store_pair(out + c + e, l == 0.0f ? 0u : Pair<T>::pack(o[e] * inv, o[e + 1] * inv), p.pairs);
    } else {
#pragma unroll
      for (int e = 0; e < 32; e += 4)
        if (c + e < hd)
          *reinterpret_cast<float4*>(p.acc + to * hd + c + e) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
    }
  }
}

template <typename T, int HDP>
__global__ void __launch_bounds__(kThreads)
    attention_wide_kernel(const __grid_constant__ Params p, const __grid_constant__ Maps maps, int box) {
  using S = Shape<HDP>;
  pdl_wait();
  pdl_launch_dependents();  // after the wait: what starts now may read this kernel's inputs
  extern __shared__ __align__(1024) char smem[];
  __shared__ Bars bars;
  __shared__ uint32_t tmem_at, skip[2];
  __shared__ int span[kRowThreads / kLanes][4];
  Work w;
  if (!find_work(p, w)) return;
  const int tid = threadIdx.x, warp = tid / kLanes, lane = tid % kLanes;
  const int hd = (int)p.a.cache.hd;
  if (warp == 5) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_at)),
                 "r"(S::kCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (tid == kRowThreads) {
    for (int i = 0; i < S::kStages; i++) {
      mbar_init(&bars.k_full[i], 1);
      mbar_init(&bars.k_empty[i], 1);
      mbar_init(&bars.v_full[i], 1);
      mbar_init(&bars.v_empty[i], 1);
    }
    for (int i = 0; i < 2; i++) {
      mbar_init(&bars.s_full[i], 1);
      mbar_init(&bars.p_full[i], kRowThreads);
      mbar_init(&bars.o_done[i], 1);
    }
    fence_mbar_init();
  }
  int low = 0, high = -1;
  if (tid < kRowThreads) {
    const bool mine = tid < w.rows;
    if (mine) sees(p, w, (w.row0 + tid) / p.group, low, high);
    const bool any = high >= low;
    const int all_lo = __reduce_max_sync(0xffffffffu, any ? low : 0);
    const int all_hi = __reduce_min_sync(0xffffffffu, any ? high : INT32_MAX);
    const int any_lo = __reduce_min_sync(0xffffffffu, any ? low : INT32_MAX);
    const int any_hi = __reduce_max_sync(0xffffffffu, any ? high : -1);
    if (lane == 0) {
      span[warp][0] = all_lo;
      span[warp][1] = all_hi;
      span[warp][2] = any_lo;
      span[warp][3] = any_hi;
    }
    // Row tid of Q: chunk c of 8 elements at chunk c ^ (row & 7) of its panel.
    const T* src = nullptr;
    if (mine) {
      int t, head;
      out_index(p, w, tid, t, head);
      src = static_cast<const T*>(p.a.q) + t * p.a.q_stride + (int64_t)head * hd;
    }
#pragma unroll 4
    for (int c = 0; c < HDP / 8; c++) {
      uint32_t v[4];
#pragma unroll
      for (int u = 0; u < 4; u++) v[u] = src != nullptr && 8 * c < hd ? load_pair(src + 8 * c + 2 * u, p.pairs) : 0u;
      *reinterpret_cast<uint4*>(smem + c / 8 * S::kQPanel + tid * 128 + (((c ^ tid) & 7) << 4)) =
          make_uint4(v[0], v[1], v[2], v[3]);
    }
    fence_proxy_async_smem();
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = tmem_at;
  int all_low = span[0][0], all_high = span[0][1], any_low = span[0][2], any_high = span[0][3];
#pragma unroll
  for (int i = 1; i < kRowThreads / kLanes; i++) {
    all_low = max(all_low, span[i][0]);
    all_high = min(all_high, span[i][1]);
    any_low = min(any_low, span[i][2]);
    any_high = max(any_high, span[i][3]);
  }
  int begin, end;
  slice_keys(p, w, any_low, any_high, kKeys, begin, end);
  const int tiles = (end - begin + kKeys - 1) / kKeys;

  if (warp < 4) {
    softmax_rows<T, HDP>(p, w, smem, bars, skip, tmem, begin, tiles, low, high, all_low, all_high);
  } else if (warp == 4) {
    const int panels = (hd + 63) / 64, groups = kKeys / box;
    auto look_up = [&](int tile) {
      int page = -1;
      if (lane < groups && tile < tiles) page = page_of(p, w, begin + tile * kKeys + lane * box);
      return page >= 0 ? page : (int)p.a.cache.pages;  // one past the last reads as zeros
    };
    int next = look_up(0);
    for (int i = 0; i < tiles; i++) {
      const int s = i % S::kStages, page = next;
      next = look_up(i + 1);
      char* kb = smem + S::kQ + s * 2 * S::kTileBytes;
      bool live = true;
#pragma unroll
      for (int kv = 0; kv < 2; kv++) {
        uint64_t* full = kv ? &bars.v_full[s] : &bars.k_full[s];
        if (i >= S::kStages)
          live = live && mbar_wait_bounded(kv ? &bars.v_empty[s] : &bars.k_empty[s], (i / S::kStages - 1) & 1,
                                           p.status, kStatusMmaTimeout);
        live = __all_sync(0xffffffffu, live);
        if (!live) break;
        if (lane == 0) mbar_arrive_expect_tx(full, (uint32_t)(panels * S::kPanel));
        for (int g = 0; g < groups; g++) {
          const int pg = __shfl_sync(0xffffffffu, page, g);
          const int pos = begin + i * kKeys + g * box, slot = pos - entry_of(p, pos) * (int)p.a.cache.page_size;
          if (lane == 0)
            for (int c = 0; c < panels; c++)
              tma_load_4d(kb + kv * S::kTileBytes + c * S::kPanel + g * box * 128, kv ? &maps.values : &maps.keys,
                          64 * c, slot, w.head, pg, full);
        }
      }
      if (!live) break;
    }
  } else {
    constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
    constexpr uint32_t kQk = idesc(kBf16, kKeys, false), kPv = idesc(kBf16, HDP, true);
    const uint32_t q = smem_u32(smem);
    const int steps = (hd + 15) / 16;
    auto pv = [&](int i) {
      const int s = i % S::kStages;
      if (!mbar_wait_bounded(&bars.p_full[i & 1], (i >> 1) & 1, p.status, kStatusMmaTimeout) ||
          !mbar_wait_bounded(&bars.v_full[s], (i / S::kStages) & 1, p.status, kStatusTmaTimeout))
        return false;
      fence_after();
      if (skip[i & 1] == 0) {
        const uint32_t v = q + S::kQ + s * 2 * S::kTileBytes + S::kTileBytes;
        for (int k = 0; k < kKeys / 16; k++)
          mma_ts(tmem + 2 * kKeys, tmem + (uint32_t)(i & 1) * kKeys + 8 * k, desc(v + k * 2048, S::kPanel), kPv,
                 i > 0 || k > 0 ? 1u : 0u);
      }
      commit(&bars.o_done[i & 1]);
      commit(&bars.v_empty[s]);
      return true;
    };
    if (elect_one()) {
      for (int i = 0; i < tiles; i++) {
        const int s = i % S::kStages;
        // S's buffer is free once the P V of two tiles ago has read P there.
        if (i >= 2 && !mbar_wait_bounded(&bars.o_done[i & 1], ((i - 2) >> 1) & 1, p.status, kStatusMmaTimeout)) break;
        if (!mbar_wait_bounded(&bars.k_full[s], (i / S::kStages) & 1, p.status, kStatusTmaTimeout)) break;
        fence_after();
        const uint32_t k = q + S::kQ + s * 2 * S::kTileBytes;
        for (int c = 0; c < steps; c++)
          mma_ss(tmem + (uint32_t)(i & 1) * kKeys, desc(q + c / 4 * S::kQPanel + c % 4 * 32, 16),
                 desc(k + c / 4 * S::kPanel + c % 4 * 32, 16), kQk, c > 0 ? 1u : 0u);
        commit(&bars.s_full[i & 1]);
        commit(&bars.k_empty[s]);
        if (i > 0 && !pv(i - 1)) break;
        if (i == tiles - 1) pv(i);
      }
    }
    __syncwarp();
  }
  fence_before();
  __syncthreads();
  if (warp == 5) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(S::kCols) : "memory");
  }
}

template <typename T, int HDP>
cudaError_t launch_size(const Params& p, cudaStream_t stream, bool pdl) {
  const PagedCache& c = p.a.cache;
  const int box = c.page_size % 64 == 0 ? 64 : c.page_size % 32 == 0 ? 32 : 16;
  Maps maps{};
  if (!(encode_tmap_pages(&maps.keys, c.keys, c.type == kBF16, c.hd, c.page_size, c.kv_heads, c.pages, c.page_stride,
                          box) &&
        encode_tmap_pages(&maps.values, c.values, c.type == kBF16, c.hd, c.page_size, c.kv_heads, c.pages,
                          c.page_stride, box)))
    return cudaErrorInvalidValue;
  if (cudaError_t e = cudaFuncSetAttribute(attention_wide_kernel<T, HDP>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                           Shape<HDP>::kSmem);
      e != cudaSuccess)
    return e;
  return launch_ex(attention_wide_kernel<T, HDP>, attention_grid(p), kThreads, Shape<HDP>::kSmem, stream, pdl, p, maps,
                   box);
}

template <typename T>
cudaError_t launch_heads(const Params& p, cudaStream_t stream, bool pdl) {
  if (p.a.cache.hd <= 64) return launch_size<T, 64>(p, stream, pdl);
  if (p.a.cache.hd <= 128) return launch_size<T, 128>(p, stream, pdl);
  return launch_size<T, 256>(p, stream, pdl);
}

}  // namespace

namespace paged {

cudaError_t launch_attention_wide(const Params& p, cudaStream_t stream, bool pdl) {
  return p.a.cache.type == kF16 ? launch_heads<__half>(p, stream, pdl) : launch_heads<__nv_bfloat16>(p, stream, pdl);
}

}  // namespace paged
}  // namespace dn
