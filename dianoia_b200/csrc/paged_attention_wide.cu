// The paged attention's kernel for many rows of queries on 16-bit caches: the
// whole batch on the shared prefix, long chunks of a sequence's queries.
//
// 128 rows of one kv head share every key, so operations are the bound, not
// bytes: S = Q K^T and O += P V go to the 5th-generation tensor cores (tcgen05,
// f32 accumulators in TMEM). A block runs two parts at once:
//   a warp for each group brings the group's tiles of 128 keys and their values
//   by tiled TMA copies, a copy a lane, and issues its products;
//   two groups of 4 warps (one for heads over 128 wide) take the even and the
//   odd tiles, a row of S each thread: they read it from TMEM 64 keys (a half)
//   at a time, keep the row's base and sum, and write P (16-bit) over it, which
//   the tensor cores read from there as the first operand of P V. Each group
//   has an O of its own, so the groups do not wait for one another until the
//   first takes the second's result in, through shared memory, at the end.
// A group's S, P and O follow one another; while one group is in softmax the
// tensor cores serve the other. (S by halves, one ahead, leaves a group no gap
// between them but takes products of N = 64 and twice the commits: 121 us
// where whole tiles took 117, on 192 sequences behind 8192 keys; joining the
// groups here instead of in the join kernel made that 113.) A base, set
// kLift below a maximum, moves only when a score passes that by kSlack (both
// pair16.cuh), so O is rescaled in TMEM in the first tiles and hardly ever
// after. Where rows of the block see different keys of a half and a value there
// is not finite, that half's P V is added term by term instead (0 * infinity
// would be NaN).
// Measured: 768 rows on 8192 keys of 8 kv heads of 128, bf16, in 45 us alone
// (570 TFLOP/s); a group's tile takes some 5500 cycles, 3300 of them softmax
// (the exponentials' unit for half of that, with both groups in step) and 2150
// the way from the last P through P V, its commit and the next S.
#include <type_traits>

#include "dn_tmap.h"
#include "paged_attention.cuh"
#include "pair16.cuh"

namespace dn {

using namespace paged;

namespace {

constexpr int kRows = kWideRows;
constexpr int kHalf = 64;         // keys of a half, which one P V takes
constexpr int kKeys = 2 * kHalf;  // of a tile, which one S takes
constexpr int kRowThreads = 128;  // of a group
constexpr int kScores = 2;        // tiles of S in TMEM
constexpr int kHalves = 2 * kScores;

struct alignas(64) Maps {
  CUtensorMap keys, values;
};

template <int HDP>
struct Shape {
  static constexpr int kPanels = HDP / 64;
  // With two groups, three warps to a quarter of the SM: 128 registers leave a
  // warp of an 8-row thin block (128) its place in the quarter's 16384 (not of a
  // 16-row one, which takes 168 of heads of 65 to 128 and waits for wide blocks
  // to end).
  static constexpr int kRegs = wide_groups(HDP) == 2 ? 128 : 168;
  static constexpr int kQPanel = kRows * 128;  // bytes: 64 elements of every row
  static constexpr int kKPanel = kKeys * 128;  // of every key of a tile
  static constexpr int kVPanel = kHalf * 128;  // of every value of a half
  static constexpr int kGroups = wide_groups(HDP);
  static constexpr int kThreads = kGroups * (kRowThreads + kLanes);
  static constexpr int kK = kPanels * kQPanel;              // where the keys start
  static constexpr int kV = kK + kGroups * kPanels * kKPanel;  // one tile of keys a group, and of values
  static constexpr int kSmem = kV + kGroups * 2 * kPanels * kVPanel;
  static constexpr uint32_t kCols = 512;  // of TMEM: S, then each group's O
  static_assert(kScores * kKeys + kGroups * HDP <= 512, "TMEM");
};

// Tile i has barriers i % kScores, half j = 2 i, 2 i + 1 of it j % kHalves
// (o_done: its P V is done). A thread may pass over phases, and a parity tells
// two phases in a row apart, not three: S of a group's tile is there only once
// P V of its tile before is done, so whoever waits for a half of either knows
// the phase before it past.
struct Bars {
  uint64_t k_full[2], v_full[2], s_full[kScores], p_full[kHalves], o_done[kHalves];  // k, v: a group's
  uint64_t second;  // the second group's results are in shared memory
};

// What stands in shared memory behind the tiles.
template <int HDP>
struct Control {
  Bars bars;
  uint32_t tmem_at, skip[kHalves];
  int span[Shape<HDP>::kGroups * kRowThreads / kLanes][4];
  float2 second[Shape<HDP>::kGroups == 2 ? kRowThreads : 1];  // its rows' m and l
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

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// Two f32 operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "add.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

// A group's part, of tiles group, group + kGroups, ...; `halves` in all of the
// block; row `r` of the block is the thread's.
template <typename T, int HDP>
__device__ __forceinline__ void softmax_rows(const Params& p, const Work& w, char* smem, Bars& bars, float2* second, uint32_t* skip,
                                             uint32_t tmem, int begin, int halves, int group, int low, int high,
                                             int all_low, int all_high) {
  using S = Shape<HDP>;
  constexpr float kLift = Pair<T>::kLift, kSlack = Pair<T>::kSlack;
  const int r = threadIdx.x % kRowThreads, lane = r % kLanes;
  const uint32_t mine = tmem + ((uint32_t)(r / kLanes * 32) << 16);
  const uint32_t out_cols = mine + kScores * kKeys + (uint32_t)(group * HDP);
  const int hd = (int)p.a.cache.hd, tiles = (halves + 1) / 2;
  const float scale = fabsf(p.scale_log2);
  float m = -INFINITY, l = 0.0f;
  // Lanes 0 .. 7 know which 16 keys of the next tile have a page.
  auto look_up = [&](int tile) {
    return lane < kKeys / 16 && tile < tiles ? entry_at(p, w, begin + tile * kKeys + 16 * lane) : -1;
  };
  int next_entry = look_up(group);
  bool live = true;
  auto done = [&](int j) {
    return __all_sync(0xffffffffu, wait_phase(&bars.o_done[j % kHalves], (j / kHalves) & 1, p.status,
                                                     kStatusMmaTimeout));
  };
  int last = -1;  // the group's last half
  for (int i = group; i < tiles && live; i += S::kGroups) {
    const unsigned tile_there = __ballot_sync(0xffffffffu, page_of(p, next_entry) >= 0);
    next_entry = look_up(i + S::kGroups);
    live = __all_sync(0xffffffffu, wait_phase(&bars.s_full[i % kScores], (i / kScores) & 1, p.status,
                                                     kStatusMmaTimeout));
    if (!live) break;
    fence_after();
#pragma unroll 1
    for (int h = 0; h < 2; h++) {
      const int j = 2 * i + h, k0 = begin + j * kHalf;
      if (j >= halves) break;
      const uint32_t cols = mine + (uint32_t)(j % kHalves) * kHalf;
      const unsigned there = tile_there >> (4 * h) & 0xfu;
      float s[2][32];
      ld32(cols, s[0]);
      ld32(cols + 32, s[1]);
      wait_ld(s[0]);
      wait_ld(s[1]);
      const bool all = there == 0xfu && k0 >= all_low && k0 + kHalf - 1 <= all_high;  // the same in every row
      if (p.scale_log2 < 0.0f) {
#pragma unroll
        for (int e = 0; e < kHalf; e++) s[e / 32][e % 32] = -s[e / 32][e % 32];
      }
      if (!all) {
#pragma unroll
        for (int e = 0; e < kHalf; e++) {
          const bool seen = (there >> (e / 16) & 1u) != 0 && k0 + e >= low && k0 + e <= high;
          if (!seen) s[e / 32][e % 32] = -INFINITY;
        }
      }
      float top4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int e = 0; e < kHalf; e += 2)
        top4[e / 2 % 4] = max3(top4[e / 2 % 4], s[e / 32][e % 32], s[e / 32][e % 32 + 1]);
      const float top = fmaxf(fmaxf(top4[0], top4[1]), fmaxf(top4[2], top4[3])) * scale;
      bool waited = last < 0;
      if (__any_sync(0xffffffffu, top - m > kSlack + kLift)) {
        const float next = fmaxf(m, top - kLift);
        const float keep = next == -INFINITY ? 1.0f : exp2_fast(m - next);
        m = next;
        l *= keep;
        if (last >= 0) {
          live = done(last);
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
      float2 sums[2] = {};
#pragma unroll
      for (int e = 0; e < kHalf; e += 2) {
        float2 x = fma2(make_float2(s[e / 32][e % 32], s[e / 32][e % 32 + 1]), make_float2(scale, scale),
                        make_float2(-base, -base));
        x.x = exp2_fast(x.x);
        x.y = exp2_fast(x.y);
        s[e / 32][e % 32] = x.x;
        s[e / 32][e % 32 + 1] = x.y;
        sums[e / 2 % 2] = add2(sums[e / 2 % 2], x);
        pk[e / 2] = Pair<T>::pack(x.x, x.y);
      }
      l += (sums[0].x + sums[0].y) + (sums[1].x + sums[1].y);
      if (!all) {
        // The values have to be looked at, and may have to be added here.
        char* vals = smem + S::kV + (2 * group + h) * S::kPanels * S::kVPanel;
        live = __all_sync(0xffffffffu, wait_phase(&bars.v_full[group], (i / S::kGroups) & 1, p.status,
                                                  kStatusTmaTimeout));
        if (!live) break;
        bool bad = false;
        const int copied = (hd + 63) / 64 * S::kVPanel;  // the head's panels: nothing writes the others
        for (int c = lane; c < copied / 16; c += kLanes) bad = bad || unbounded16<T>(vals + c * 16);
        bad = __any_sync(0xffffffffu, bad);  // every warp finds the same
        if (r == 0) skip[j % kHalves] = bad ? 1u : 0u;
        if (bad) {
          if (!waited) live = done(last);
          if (!live) break;
          fence_after();
          float pr[kHalf];  // indexed at run time: in local memory, here only
#pragma unroll
          for (int e = 0; e < kHalf; e++) {
            // -0: not seen. (A key that is seen counts, however small its weight.)
            const bool seen = (there >> (e / 16) & 1u) != 0 && k0 + e >= low && k0 + e <= high;
            pr[e] = seen ? to_f32<T>(from_f32<T>(s[e / 32][e % 32])) : -0.0f;
          }
#pragma unroll 1
          for (int c = 0; c < hd; c += 32) {
            float o[32];
            ld32(out_cols + c, o);
            wait_ld(o);
            if (last < 0)
#pragma unroll
              for (int e = 0; e < 32; e++) o[e] = 0.0f;
#pragma unroll 1
            for (int k = 0; k < kHalf; k++) {
              if (__float_as_int(pr[k]) >= 0)
#pragma unroll
                for (int e = 0; e < 32; e++) {
                  const int d = c + e;
                  const T v = reinterpret_cast<const T*>(vals + d / 64 * S::kVPanel + k * 128 +
                                                         (((d % 64 / 8) ^ (k & 7)) << 4))[d % 8];
                  o[e] = fmaf(pr[k], to_f32<T>(v), o[e]);
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
        skip[j % kHalves] = 0;
      }
      st32(cols, pk);
      wait_st();
      fence_before();
      mbar_arrive(&bars.p_full[j % kHalves]);
      last = j;
    }
  }
  if (last >= 0 && live) {
    done(last);
    fence_after();
  }
  if (high < low) {  // a row that sees nothing took part unmasked
    m = -INFINITY;
    l = 0.0f;
  }
  // The second group's result goes to the first through the second's own keys'
  // and values' places: 4 columns at a time, chunk c of row r at c ^ r.
  constexpr int kPart = HDP / 8;  // chunks in the keys' place; as many in the values'
  auto place = [&](int chunk) {
    char* at = smem + (chunk < kPart ? S::kK + S::kPanels * S::kKPanel : S::kV + 2 * S::kPanels * S::kVPanel);
    return reinterpret_cast<float4*>(at + r * (kPart * 16) + ((chunk ^ r) & (kPart - 1)) * 16);
  };
  float keep_first = 1.0f, keep_second = 0.0f;
  if constexpr (S::kGroups == 2) {
    if (group == 1) {
      if (last >= 0) {
#pragma unroll 1
        for (int c = 0; c < HDP; c += 32) {
          float o[32];
          ld32(out_cols + c, o);
          wait_ld(o);
#pragma unroll
          for (int e = 0; e < 32; e += 4) *place((c + e) / 4) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
        }
      }
      second[r] = make_float2(m, l);
      mbar_arrive(&bars.second);
      return;
    }
    live = __all_sync(0xffffffffu, wait_phase(&bars.second, 0, p.status, kStatusMmaTimeout));
    const float2 other = second[r];
    if (live && other.y != 0.0f) {
      const float top = fmaxf(m, other.x), base = top == -INFINITY ? 0.0f : top;
      keep_first = exp2_fast(m - base);
      keep_second = exp2_fast(other.x - base);
      l = (l == 0.0f ? 0.0f : l * keep_first) + other.y * keep_second;
      m = top;
    }
  }
  // The row's result.
  int t = 0, head = 0;
  const bool mine_row = r < w.rows;
  const int64_t row = mine_row ? out_index(p, w, r, t, head) : 0;
  const int64_t to = slice_index(p, w) * (p.a.n * p.a.heads) + row;
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  if (mine_row && !p.direct) p.ml[to] = make_float2(m, l);
  if (last < 0 && !p.direct) return;  // the join reads no values of a row with l = 0
#pragma unroll 1
  for (int c = 0; c < HDP; c += 32) {
    float o[32];
    if (last >= 0) {
      ld32(out_cols + c, o);
      wait_ld(o);
    } else {
#pragma unroll
      for (int e = 0; e < 32; e++) o[e] = 0.0f;
    }
    if (keep_second != 0.0f) {
#pragma unroll
      for (int e = 0; e < 32; e += 4) {
        const float4 v = *place((c + e) / 4);
        o[e] = o[e] * keep_first + v.x * keep_second;
        o[e + 1] = o[e + 1] * keep_first + v.y * keep_second;
        o[e + 2] = o[e + 2] * keep_first + v.z * keep_second;
        o[e + 3] = o[e + 3] * keep_first + v.w * keep_second;
      }
    }
    if (mine_row && p.direct) {
      T* out = static_cast<T*>(p.a.out) + t * p.a.out_stride + (int64_t)head * hd;
#pragma unroll
      for (int e = 0; e < 32; e += 2)
        if (c + e < hd)
          store_pair(out + c + e, l == 0.0f ? 0u : Pair<T>::pack(o[e] * inv, o[e + 1] * inv), p.pairs);
    } else if (mine_row) {
#pragma unroll
      for (int e = 0; e < 32; e += 4)
        if (c + e < hd)
          *reinterpret_cast<float4*>(p.acc + to * hd + c + e) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
    }
    __syncwarp();  // the next load takes whole warps
  }
}

template <typename T, int HDP>
__global__ void __maxnreg__(Shape<HDP>::kRegs)
    attention_wide_kernel(const __grid_constant__ Params p, const __grid_constant__ Maps maps, int box) {
  using S = Shape<HDP>;
  pdl_wait();
  pdl_launch_dependents();  // after the wait: what starts now may read this kernel's inputs
  extern __shared__ __align__(1024) char smem[];
  // No static shared memory: it would be rounded up to the tiles' alignment,
  // and a thin block would no longer fit beside this one.
  Control<HDP>& ctl = *reinterpret_cast<Control<HDP>*>(smem + S::kSmem);
  Bars& bars = ctl.bars;
  uint32_t* const skip = ctl.skip;
  constexpr int kRowWarps = S::kGroups * kRowThreads / kLanes;
  auto& span = ctl.span;
  Work w;
  if (!find_work(p, w)) return;
  const int tid = threadIdx.x, warp = tid / kLanes, lane = tid % kLanes;
  const int hd = (int)p.a.cache.hd;
  if (warp == kRowWarps) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&ctl.tmem_at)),
                 "r"(S::kCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (tid == kRowWarps * kLanes) {
    for (int i = 0; i < S::kGroups; i++) {
      mbar_init(&bars.k_full[i], 1);
      mbar_init(&bars.v_full[i], 1);
    }
    for (int i = 0; i < kScores; i++) mbar_init(&bars.s_full[i], 1);
    mbar_init(&bars.second, kRowThreads);
    for (int i = 0; i < kHalves; i++) {
      mbar_init(&bars.p_full[i], kRowThreads);
      mbar_init(&bars.o_done[i], 1);
    }
    fence_mbar_init();
  }
  int low = 0, high = -1;
  if (warp < kRowWarps) {
    const int r = tid % kRowThreads;
    if (r < w.rows) sees(p, w, (w.row0 + r) / p.group, low, high);
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
    // Q, a run of lanes for each row: chunk c of 8 elements of row r at chunk
    // c ^ (r & 7) of its panel.
    constexpr int kChunks = HDP / 8, kAtOnce = kLanes / kChunks > 0 ? kLanes / kChunks : 1;
#pragma unroll 4
    for (int row = warp * kAtOnce + lane / kChunks; row < kRows; row += kRowWarps * kAtOnce) {
      const int c = lane % kChunks;
      uint4 v = make_uint4(0, 0, 0, 0);
      if (row < w.rows && 8 * c < hd) {
        int t, head;
        out_index(p, w, row, t, head);
        const T* src = static_cast<const T*>(p.a.q) + t * p.a.q_stride + (int64_t)head * hd + 8 * c;
        if (p.runs) {
          v = *reinterpret_cast<const uint4*>(src);
        } else {
          v = make_uint4(load_pair(src, p.pairs), load_pair(src + 2, p.pairs), load_pair(src + 4, p.pairs),
                         load_pair(src + 6, p.pairs));
        }
      }
      *reinterpret_cast<uint4*>(smem + c / 8 * S::kQPanel + row * 128 + (((c ^ row) & 7) << 4)) = v;
    }
    fence_proxy_async_smem();
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = ctl.tmem_at;
  int all_low = span[0][0], all_high = span[0][1], any_low = span[0][2], any_high = span[0][3];
#pragma unroll
  for (int i = 1; i < kRowWarps; i++) {
    all_low = max(all_low, span[i][0]);
    all_high = min(all_high, span[i][1]);
    any_low = min(any_low, span[i][2]);
    any_high = max(any_high, span[i][3]);
  }
  int begin, end;
  slice_keys(p, w, any_low, any_high, kHalf, begin, end);
  const int halves = (end - begin + kHalf - 1) / kHalf, tiles = (halves + 1) / 2;

  if (warp < kRowWarps) {
    softmax_rows<T, HDP>(p, w, smem, bars, ctl.second, skip, tmem, begin, halves, tid / kRowThreads, low, high, all_low, all_high);
  } else {
    const int group = warp - kRowWarps;
    // One copy a lane: panel c of the keys (values) g * box .. of a tile, all
    // of one page, whose entry is on its way a tile ahead. (One lane issuing
    // them all took 300 cycles a copy; a third warp for both groups' copies
    // was the bound, 3300 cycles a tile.)
    const int panels = (hd + 63) / 64, groups = kHalf / box;  // of a half
    const int g = lane / S::kPanels, c = lane % S::kPanels, half = g / groups;
    const uint32_t row0 = (uint32_t)(g % groups * box * 128);
    char* const k_at = smem + S::kK + group * S::kPanels * S::kKPanel + c * S::kKPanel + half * kHalf * 128 + row0;
    char* const v_at = smem + S::kV + (2 * group + half) * S::kPanels * S::kVPanel + c * S::kVPanel + row0;
    const bool mine = half < 2 && c < panels;
    auto look_up = [&](int tile) {
      return mine && tile < tiles ? entry_at(p, w, begin + tile * kKeys + g * box) : -1;
    };
    // The page of the lane's keys; one past the last reads as zeros.
    auto page_at = [&](int entry) {
      const int page = page_of(p, entry);
      return page >= 0 ? page : (int)p.a.cache.pages;
    };
    auto slot_at = [&](int tile) {
      const int pos = begin + tile * kKeys + g * box;
      return pos - entry_of(p, pos) * (int)p.a.cache.page_size;
    };
    auto load = [&](const CUtensorMap* map, char* dst, int tile, int page, int slot, uint64_t* full) {
      const int parts = min(2, halves - 2 * tile);
      if (lane == 0) mbar_arrive_expect_tx(full, (uint32_t)(parts * panels * S::kVPanel));
      __syncwarp();
      if (mine && half < parts) tma_load_4d(dst, map, 64 * c, slot, w.head, page, full);
    };
    constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
    constexpr uint32_t kQk = idesc(kBf16, kKeys, false), kPv = idesc(kBf16, HDP, true);
    // Operands' descriptors; the address field counts 16 bytes, so an offset adds.
    const uint32_t q = smem_u32(smem);
    const uint64_t q_desc = desc(q, 16), k_desc = desc(q + S::kK + group * S::kPanels * S::kKPanel, 16),
                   v_desc = desc(q + S::kV + group * 2 * S::kPanels * S::kVPanel, S::kVPanel);
    const int steps = (hd + 15) / 16;
    const uint32_t out = tmem + kScores * kKeys + (uint32_t)(group * HDP);
    const bool leader = elect_one();
    auto wait = [&](uint64_t* bar, int phase, uint32_t bits) {
      return __all_sync(0xffffffffu, wait_phase(bar, phase & 1, p.status, bits));
    };
    int page = page_at(look_up(group)), slot = slot_at(group), next = look_up(group + S::kGroups);
    if (group < tiles) load(&maps.keys, k_at, group, page, slot, &bars.k_full[group]);
    bool live = true;
    int last = -1;  // the group's last half
    int keys = group, tile = -1;  // the last tiles whose keys, and whose S and values, were asked for
    for (int i = group; i < tiles && live; i += S::kGroups) {
      const int turn = i / S::kGroups, page_k = page_at(next), slot_k = slot_at(i + S::kGroups);
      next = look_up(i + 2 * S::kGroups);
      // S's place, and the values', are free once P V of the group's last tile is done.
      if (last >= 0) live = wait(&bars.o_done[last % kHalves], last / kHalves, kStatusMmaTimeout);
      live = live && wait(&bars.k_full[group], turn, kStatusTmaTimeout);
      if (!live) break;
      fence_after();
      if (leader) {
#pragma unroll
        for (int e = 0; e < HDP / 16; e++)
          if (e < steps)
            mma_ss(tmem + (uint32_t)(i % kScores) * kKeys, q_desc + (uint32_t)((e / 4 * S::kQPanel + e % 4 * 32) >> 4),
                   k_desc + (uint32_t)((e / 4 * S::kKPanel + e % 4 * 32) >> 4), kQk, e > 0 ? 1u : 0u);
        commit(&bars.s_full[i % kScores]);
      }
      __syncwarp();
      load(&maps.values, v_at, i, page, slot, &bars.v_full[group]);
      // S is there: its keys' place is free.
      live = wait(&bars.s_full[i % kScores], i / kScores, kStatusMmaTimeout);
      if (live && i + S::kGroups < tiles) {
        keys = i + S::kGroups;
        load(&maps.keys, k_at, keys, page_k, slot_k, &bars.k_full[group]);
      }
      page = page_k;
      slot = slot_k;
      for (int j = 2 * i; j < min(2 * i + 2, halves) && live; j++) {
        live = wait(&bars.v_full[group], turn, kStatusTmaTimeout) &&
               wait(&bars.p_full[j % kHalves], j / kHalves, kStatusMmaTimeout);
        if (!live) break;
        fence_after();
        if (leader) {
          if (skip[j % kHalves] == 0) {
            const uint64_t v = v_desc + (uint32_t)(j % 2 * S::kPanels * S::kVPanel >> 4);
            const uint32_t pr = tmem + (uint32_t)(j % kHalves) * kHalf;
#pragma unroll
            for (int e = 0; e < kHalf / 16; e++)
              mma_ts(out, pr + 8 * e, v + (uint32_t)(e * 2048 >> 4), kPv, e > 0 || last >= 0 ? 1u : 0u);
          }
          commit(&bars.o_done[j % kHalves]);
        }
        __syncwarp();
        last = j;
      }
    }
    // Nothing is in flight when the block goes, given up or not.
    if (!live) {
      mbar_land(&bars.k_full[group], keys / S::kGroups & 1);
      if (tile >= 0) {
        mbar_land(&bars.v_full[group], tile / S::kGroups & 1);
        mbar_land(&bars.s_full[tile % kScores], tile / kScores & 1);
      }
    }
    if (last >= 0) mbar_land(&bars.o_done[last % kHalves], last / kHalves & 1);
    __syncwarp();
  }
  fence_before();
  __syncthreads();
  if (warp == kRowWarps) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(S::kCols) : "memory");
  }
}

template <typename T, int HDP>
cudaError_t launch_size(const Params& p, cudaStream_t stream, bool pdl) {
  const PagedCache& c = p.a.cache;
  const int box = wide_box(c.page_size);
  Maps maps{};
  if (!(encode_tmap_pages(&maps.keys, c.keys, c.type == kBF16, c.hd, c.page_size, c.kv_heads, c.pages, c.page_stride,
                          box) &&
        encode_tmap_pages(&maps.values, c.values, c.type == kBF16, c.hd, c.page_size, c.kv_heads, c.pages,
                          c.page_stride, box)))
    return cudaErrorInvalidValue;
  constexpr int smem = Shape<HDP>::kSmem + (int)sizeof(Control<HDP>);
  if (cudaError_t e = allow_smem<attention_wide_kernel<T, HDP>>(smem); e != cudaSuccess) return e;
  return launch_ex(attention_wide_kernel<T, HDP>, attention_grid(p), Shape<HDP>::kThreads, smem, stream, pdl, p, maps,
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
