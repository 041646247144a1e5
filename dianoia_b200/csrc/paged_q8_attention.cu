// Attention over an 8-bit paged cache (dn_paged_q8_attention).
//
// Per query row, over the positions it sees:
//   x_j = scale s_kj (q . k_j),  p_j = 2^(log2e x_j - m),
//   out = sum_j (p_j s_vj) v_j / sum_j p_j,
// with the keys' and values' rows as the integers they are kept as: a row's
// scale leaves the sum over its values.
//
// Bytes-bound at a few rows a sequence: 2 (hd + 4) bytes a position and kv
// head, 23 bytes a clock and SM. So the matrix instructions take the keys (and
// the values' dims) as their wide side, S^T = K Q^T and O^T = V^T P^T with 8
// query rows to a tile, and the integers become bf16 on the way from shared
// memory to registers, four operations a pair: a byte of seven bits and a sign
// is 128 + low and 128 + 128 sign (bit patterns with bf16's exponent), one less
// the other, exactly. bf16's 8 bits hold them whole, and its range any weight
// p s; queries and weights of more bits go in two or three bf16 parts, each the
// rounding of what the ones before leave.
//
// A block takes a slice of the keys of one tile of rows (tokens of a sequence
// times the heads of a kv head); its four warps take every fourth chunk of 16
// keys and bring them themselves, by 16-byte asynchronous copies into a ring
// of their own, the rows found through the page table a chunk ahead. The base m
// of a row's softmax is set kSlack (log2) above its largest score so far and
// stands until a score passes it, which keeps the common path free of
// reductions: weights stay at most 1, and bf16 weights and f32 sums lose
// nothing by being 2^-kSlack of that. The warps join in shared memory, slices through the
// workspace in a second launch that is already waiting (programmatic launch).
#include "dn_common.cuh"
#include "dn_launch.h"
#include "elem.cuh"
#include "kernel_smem.h"
#include "pair16.cuh"

namespace dn {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kRun = 16;  // keys of a product; pages of whole runs are copied as such
constexpr float kSlack = 8.0f;
constexpr int kJoinWarps = 8;

// Parts of a query, and of a weight (bf16's one part alone would be the
// largest error of all: 2.3e-3 of a random batch's outputs against 1.7e-3, which
// is the outputs' own rounding).
template <typename T>
struct Parts {
  static constexpr int query = 3, weight = 3;
};
template <>
struct Parts<__half> {
  static constexpr int query = 2, weight = 2;
};
template <>
struct Parts<__nv_bfloat16> {
  static constexpr int query = 1, weight = 2;
};

// How the launch divides the batch; the same in both kernels.
struct Split {
  int rows;      // of a tile: 8, 16 or 32
  int slices;    // of a tile, at most
  int slice;     // keys of each but the last, a multiple of 64
  int most;      // slices that a call with a window may have at most
  int64_t tiles;
};

struct Work {
  int seq, first, count;  // the sequence, its first token, its tokens
  int row0, rows;         // the tile's first row of the sequence's, rows left from there
  int begin, end;         // keys that some row may see, begin a multiple of kRun
  int slices;             // in use
  int length;
};

// The tile's work; called by whole warps. Sequence s owns the tiles from
// q_start[s] group / rows + s on: at least as many as it needs, some of them idle.
__device__ __forceinline__ Work find_work(const PagedQ8AttentionArgs& a, const Split& d, int64_t tile, int group) {
  Work w;
  int64_t local;
  if (a.q_start == nullptr) {
    const int per = (group + d.rows - 1) / d.rows;
    w.seq = (int)(tile / per);
    local = tile % per;
    w.first = w.seq;
    w.count = 1;
  } else {
    const int lane = threadIdx.x % 32;
    int lo = 0, hi = (int)a.cache.sequences;
    while (hi - lo > 1) {  // 32 ways at a time
      const int step = (hi - lo + 31) / 32, at = lo + lane * step;
      const bool before = at < hi && (int64_t)a.q_start[at] * group / d.rows + at <= tile;
      const int k = max(1, __popc(__ballot_sync(0xffffffffu, before)));
      lo += (k - 1) * step;
      hi = min(hi, lo + step);
    }
    w.seq = lo;
    w.first = a.q_start[lo];
    w.count = max(0, a.q_start[lo + 1] - w.first);
    local = tile - ((int64_t)w.first * group / d.rows + lo);
  }
  const int64_t rows = (int64_t)w.count * group, row0 = local * d.rows;
  w.rows = local < 0 || row0 >= rows ? 0 : (int)min64(rows - row0, d.rows);
  w.row0 = (int)min64(row0, INT32_MAX);
  w.begin = w.end = 0;
  w.slices = 1;
  w.length = 0;
  if (w.rows == 0) return w;
  w.length = a.lengths[w.seq];
  // Positions of the tile's first and last tokens.
  const int64_t first = (int64_t)w.length - w.count + w.row0 / group;
  const int64_t last = (int64_t)w.length - w.count + (w.row0 + w.rows - 1) / group;
  const int64_t most = a.cache.table_stride * a.cache.page_size;
  w.end = (int)(last + 1 < 0 ? 0 : min64(last + 1, most));
  const int64_t low = a.window > 0 ? first - a.window + 1 : 0;
  w.begin = low > 0 ? (int)(min64(low, most) / kRun * kRun) : 0;
  if (w.end > w.begin) w.slices = min(d.slices, (w.end - w.begin + d.slice - 1) / d.slice);
  return w;
}

__device__ __forceinline__ void cp16(void* dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp4(void* dst, const void* src, bool there) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(there ? 4 : 0) : "memory");
}

__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// An 8 x 8 matrix of 16-bit elements, a row's pair to a lane, transposed.
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// Bytes 0 and 2 of x, as int8, to bf16; bytes 1 and 3 do not count. `bits` is
// kExponent in a register: with two literals the compiler takes two operations
// for each of these.
constexpr uint32_t kExponent = 0x43004300u;
__device__ __forceinline__ uint32_t widened(uint32_t x, uint32_t bits) {
  uint32_t low, sign;
  asm("lop3.b32 %0, %1, 0x007f007f, %2, 0xea;" : "=r"(low) : "r"(x), "r"(bits));   // x & mask | bits
  asm("lop3.b32 %0, %1, 0x00800080, %2, 0xea;" : "=r"(sign) : "r"(x), "r"(bits));
  __nv_bfloat162 l, s;
  memcpy(&l, &low, 4);
  memcpy(&s, &sign, 4);
  l = __hsub2(l, s);
  uint32_t y;
  memcpy(&y, &l, 4);
  return y;
}

__device__ __forceinline__ float power2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float2 unpacked(uint32_t x) {
  return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
}

// Bytes [HD / 8 * g, ...) of a row; HD / 8 of them.
template <int WORDS>
__device__ __forceinline__ void load_words(const uint8_t* p, uint32_t (&w)[WORDS]) {
  if constexpr (WORDS == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x, w[1] = v.y;
  } else {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
  }
}

// Where 16-byte part `part` of row `row` lies in a chunk: in lines of 128 bytes,
// turned so that the eight lanes that read at once (keys: two rows' four parts;
// values: four even or odd rows' two parts) meet eight different places of the
// line.
template <int HD>
__host__ __device__ constexpr int turn_of(int row) {
  return HD == 64 ? row & 6 : (row & 6) ^ (row & 1) << 2;
}
template <int HD>
__device__ __forceinline__ int place(int row, int part) {
  return ((row * (HD / 16) + part) ^ turn_of<HD>(row)) * 16;
}

template <int HD, int NT, int PARTS>
struct Smem {
  // A warp's ring: chunks of kKeys keys and values, kStages of them.
  static constexpr int kKeys = HD == 256 ? 16 : 32, kStages = HD == 64 ? 4 : HD == 128 ? 2 : 3;
  static constexpr int kChunk = kKeys * HD;  // bytes of a chunk's keys, or values
  static constexpr int kRing = kWarps * kStages * 2 * kChunk;
  static constexpr int kJoin = kWarps * NT * 8 * HD * 4;  // the warps' sums, over the ring
  static constexpr int kScales = kRing > kJoin ? kRing : kJoin;
  static constexpr int kMasks = kScales + kWarps * kStages * 2 * kKeys * 4;
  static constexpr int kStats = kMasks + kWarps * kStages * 4;
  static constexpr int kQueries = (kStats + kWarps * NT * 8 * 2 * 4 + 15) / 16 * 16;
  static constexpr int kBytes = kQueries + PARTS * NT * (HD / 16) * 32 * 8;
};

template <typename T, int HD, int NT, int BLOCKS>
__global__ void __launch_bounds__(kThreads, BLOCKS)
    paged_q8_attention_kernel(const __grid_constant__ PagedQ8AttentionArgs a, const Split d) {
  constexpr int PARTS = Parts<T>::query, WPARTS = Parts<T>::weight, R = NT * 8;
  // The tensor cores cut their sums off (2^-23 of each, one way), which f32
  // results would show: there each chunk's sums begin at 0 and are added here.
  constexpr bool kFine = std::is_same<T, float>::value;
  using S = Smem<HD, NT, PARTS>;
  constexpr int STAGES = S::kStages, KEYS = S::kKeys, STEPS = HD / 16;
  extern __shared__ __align__(128) uint8_t smem[];
  pdl_launch_dependents();
  pdl_wait();
  const PagedQ8Cache& c = a.cache;
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32, g = lane / 4, t = lane % 4;
  const int hd = (int)c.hd, page_size = (int)c.page_size, group = (int)(a.heads / c.kv_heads);
  const int kv = (int)(blockIdx.x % (unsigned)c.kv_heads);
  const int slice = (int)(blockIdx.x / (unsigned)c.kv_heads % (unsigned)d.slices);
  const int64_t tile = blockIdx.x / (unsigned)c.kv_heads / (unsigned)d.slices;
  const Work w = find_work(a, d, tile, group);
  if (w.rows == 0 || slice >= w.slices) return;
  const int begin = w.begin + slice * d.slice;
  const int end = slice + 1 == w.slices ? w.end : min(w.end, begin + d.slice);

  // ---- the ring: this lane's row of a chunk, its page a chunk ahead
  uint8_t* ring = smem + warp * STAGES * 2 * S::kChunk;
  float* scales = reinterpret_cast<float*>(smem + S::kScales) + warp * STAGES * 2 * KEYS;
  uint32_t* masks = reinterpret_cast<uint32_t*>(smem + S::kMasks) + warp * STAGES;
  if (hd != HD) {  // parts that no copy writes
    for (int at = lane * 16; at < STAGES * 2 * S::kChunk; at += 32 * 16)
      *reinterpret_cast<uint4*>(ring + at) = make_uint4(0, 0, 0, 0);
    __syncwarp();
  }
  const int32_t* table = c.table + (int64_t)w.seq * c.table_stride;
  // Pages of whole runs of 16: LANES lanes copy a run, as one run of bytes. Else
  // a row's parts are copied from where the lane that follows it says.
  const bool runs = page_size % kRun == 0;
  constexpr int LANES = KEYS == 32 ? 16 : 32, COPIES = KEYS * HD / 16 / 32;
  const int row = lane % KEYS, in_run = row % kRun;
  int pos = begin + warp * KEYS + row;  // of the next chunk to issue
  int entry = pos / page_size, slot = pos - entry * page_size;
  const int entry_step = kWarps * KEYS / page_size, slot_step = kWarps * KEYS - entry_step * page_size;
  auto page_at = [&]() { return pos - (runs ? in_run : 0) < end ? table[entry] : -1; };
  int page = page_at();
  const int parts = hd / 16;
  const uint32_t per_part = 65536u / (uint32_t)parts + 1;  // x per_part / 65536 is x / parts, for x below 512
  const int first_to = place<HD>(lane / 16 * (KEYS == 32 ? kRun : 1) + lane % 16 / (HD / 16), lane % LANES % (HD / 16));
  auto issue = [&](int stage) {
    const bool held = page >= 0 && page < c.pages, there = held && pos < end;
    const int64_t scale_at = there ? page * c.scale_stride + (int64_t)kv * page_size + slot : 0;
    const uint32_t mask = __ballot_sync(0xffffffffu, there);
    uint8_t* keys = ring + stage * 2 * S::kChunk;
    uint8_t* values = keys + S::kChunk;
    if (runs) {
      const int64_t at = held ? page * c.page_stride + ((int64_t)kv * page_size + (slot - in_run)) * hd : 0;
      const int8_t* from_keys = c.keys + at + lane % LANES * 16;
      const int8_t* from_values = c.values + at + lane % LANES * 16;
      if (hd == HD) {
#pragma unroll
        for (int i = 0; i < COPIES; i++) {  // LANES * 16 / HD rows on each time
          const int to = (first_to ^ turn_of<HD>(i * (LANES * 16 / HD)) * 16) + i * LANES * 16;
          cp16(keys + to, from_keys + i * LANES * 16, held);
          cp16(values + to, from_values + i * LANES * 16, held);
        }
      } else {
#pragma unroll
        for (int i = 0; i < COPIES; i++) {
          const int which = lane % LANES + i * LANES, r = (int)(which * per_part >> 16);
          if (r < kRun) {
            const int to = place<HD>(r + (KEYS == 32 ? lane / 16 * kRun : 0), which - r * parts);
            cp16(keys + to, from_keys + i * LANES * 16, held);
            cp16(values + to, from_values + i * LANES * 16, held);
          }
        }
      }
    } else {
      const int64_t at = there ? page * c.page_stride + ((int64_t)kv * page_size + slot) * hd : -1;
#pragma unroll
      for (int i = 0; i < COPIES; i++) {
        const int which = lane + 32 * i, r = (int)(which * per_part >> 16), part = which - r * parts;
        const int64_t from = __shfl_sync(0xffffffffu, at, r % KEYS);
        if (r < KEYS) {
          const int to = place<HD>(r, part);
          const int64_t src = from >= 0 ? from + part * 16 : 0;
          cp16(keys + to, c.keys + src, from >= 0);
          cp16(values + to, c.values + src, from >= 0);
        }
      }
    }
    if constexpr (KEYS == 32) {
      cp4(scales + stage * 2 * KEYS + lane, c.key_scales + scale_at, there);
      cp4(scales + stage * 2 * KEYS + KEYS + lane, c.value_scales + scale_at, there);
    } else {
      cp4(scales + stage * 2 * KEYS + lane, (lane < KEYS ? c.key_scales : c.value_scales) + scale_at, there);
    }
    if (lane == 0) masks[stage] = mask;
    pos += kWarps * KEYS;
    entry += entry_step;
    slot += slot_step;
    if (slot >= page_size) {
      slot -= page_size;
      entry++;
    }
    page = page_at();
  };
  const int mine = end - begin - warp * KEYS, chunks = mine > 0 ? (mine + kWarps * KEYS - 1) / (kWarps * KEYS) : 0;
#pragma unroll
  for (int s = 0; s < STAGES; s++) {
    if (s < chunks) issue(s);
    asm volatile("cp.async.commit_group;" ::: "memory");
  }

  // ---- the queries, as the products take them: of step i lane (g, t) holds
  // row g's dims 64 (i / 4) + 16 t + 4 (i % 4) .. + 3, the even ones first as
  // the keys' words give them
  uint2* queries = reinterpret_cast<uint2*>(smem + S::kQueries);
  for (int at = tid; at < NT * STEPS * 32; at += kThreads) {
    const int l = at % 32, i = at / 32 % STEPS, nt = at / 32 / STEPS, r = nt * 8 + l / 4;
    const int dim = i / 4 * 64 + l % 4 * 16 + i % 4 * 4;
    const int token = w.first + (w.row0 + r) / group, head = kv * group + (w.row0 + r) % group;
    float x[4] = {};
    if (r < w.rows && dim < hd && token >= 0 && token < a.n) {
      const T* src = static_cast<const T*>(a.q) + (int64_t)token * a.q_stride + (int64_t)head * hd + dim;
#pragma unroll
      for (int e = 0; e < 4; e++) x[e] = to_f32<T>(src[e]);
    }
#pragma unroll
    for (int p = 0; p < PARTS; p++) {
      const uint2 b = make_uint2(Pair<__nv_bfloat16>::pack(x[0], x[2]), Pair<__nv_bfloat16>::pack(x[1], x[3]));
      queries[(p * NT + nt) * STEPS * 32 + i * 32 + l] = b;
      const float2 lo = unpacked(b.x), hi = unpacked(b.y);
      x[0] -= lo.x, x[2] -= lo.y, x[1] -= hi.x, x[3] -= hi.y;
    }
  }
  __syncthreads();
  constexpr bool kHeld = PARTS * NT * STEPS * 2 <= 32;  // in registers
  uint2 held[kHeld ? PARTS * NT * STEPS : 1];
  if constexpr (kHeld)
#pragma unroll
    for (int i = 0; i < PARTS * NT * STEPS; i++) held[i] = queries[i * 32 + lane];

  // Positions that this lane's rows (2 t and 2 t + 1 of each eight) see, and what all of the tile's see.
  int high[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; nt++)
#pragma unroll
    for (int e = 0; e < 2; e++) high[nt][e] = w.length - w.count + (w.row0 + nt * 8 + 2 * t + e) / group;
  const int64_t window = a.window;
  const int all_high = w.length - w.count + w.row0 / group;
  const int64_t all_low = window > 0 ? (int64_t)w.length - w.count + (w.row0 + w.rows - 1) / group - window + 1 : 0;
  const float factor = a.scale * 1.4426950408889634f;

  float acc[NT][STEPS][4], m[NT][2], sum[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; nt++) {
    m[nt][0] = m[nt][1] = -INFINITY;
    sum[nt][0] = sum[nt][1] = 0.0f;
#pragma unroll
    for (int i = 0; i < STEPS; i++) acc[nt][i][0] = acc[nt][i][1] = acc[nt][i][2] = acc[nt][i][3] = 0.0f;
  }

  // Where this lane's words lie: its two keys' parts (the second 8 rows on), its values' (keys 2 t and 2 t + 1; 8 rows on).
  const int key_at[2] = {place<HD>(g, t), place<HD>(g, (t + 4) % (HD / 16))};
  const int value_at[2] = {HD == 64 ? place<HD>(2 * t, g / 2) + g % 2 * 8 : place<HD>(2 * t, g),
                           HD == 64 ? place<HD>(2 * t + 1, g / 2) + g % 2 * 8 : place<HD>(2 * t + 1, g)};

  uint32_t bits;
  asm volatile("mov.b32 %0, %1;" : "=r"(bits) : "n"(kExponent));
  int stage = 0;
  for (int chunk = 0; chunk < chunks; chunk++) {
    asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
    __syncwarp();
#pragma unroll 1
    for (int run = 0; run < KEYS / kRun; run++) {
      const uint8_t* keys = ring + stage * 2 * S::kChunk + run * kRun * HD;
      const uint8_t* values = keys + S::kChunk;

      // Scores: rows 2 t, 2 t + 1 of keys g (0, 1) and g + 8 (2, 3).
      float s[NT][4], less[NT][4];  // `less`: of the queries' parts but the first
#pragma unroll
      for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int e = 0; e < 4; e++) s[nt][e] = less[nt][e] = 0.0f;
#pragma unroll
      for (int block = 0; block < HD / 64; block++) {
        uint32_t k0[4], k1[4];
        load_words<4>(keys + key_at[block % 2] + block / 2 * 128, k0);
        load_words<4>(keys + key_at[block % 2] + block / 2 * 128 + 8 * HD, k1);
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const uint32_t f[4] = {widened(k0[j], bits), widened(k1[j], bits), widened(k0[j] >> 8, bits),
                                 widened(k1[j] >> 8, bits)};
          const int i = block * 4 + j;
#pragma unroll
          for (int p = 0; p < PARTS; p++)
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
              const int at = (p * NT + nt) * STEPS + i;
              uint2 b;
              if constexpr (kHeld) b = held[at]; else b = queries[at * 32 + lane];
              mma16816(p == 0 ? s[nt] : less[nt], f, b.x, b.y);
            }
        }
      }
      const float* sc = scales + stage * 2 * KEYS + run * kRun;
      const float ks0 = sc[g] * factor, ks1 = sc[g + 8] * factor, vs0 = sc[KEYS + g], vs1 = sc[KEYS + g + 8];
      const int first = begin + (chunk * kWarps + warp) * KEYS + run * kRun;
      const uint32_t mask = masks[stage] >> run * kRun & 0xffffu;
      const bool whole = mask == 0xffffu && first + kRun - 1 <= all_high && first >= all_low;
      bool past = false;
#pragma unroll
      for (int nt = 0; nt < NT; nt++) {
#pragma unroll
        for (int e = 0; e < 4; e++) s[nt][e] = (PARTS > 1 ? s[nt][e] + less[nt][e] : s[nt][e]) * (e < 2 ? ks0 : ks1);
        if (!whole) {
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const int key = g + (e >= 2 ? 8 : 0), at = first + key, hi = high[nt][e & 1];
            const bool sees = (mask >> key & 1u) != 0 && at <= hi && (window == 0 || (int64_t)at > hi - window);
            s[nt][e] = sees ? s[nt][e] : -INFINITY;
          }
        }
        past |= fmaxf(s[nt][0], s[nt][2]) > m[nt][0] || fmaxf(s[nt][1], s[nt][3]) > m[nt][1];
      }
      if (__any_sync(0xffffffffu, past)) {
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
          for (int e = 0; e < 2; e++) {
            float top = fmaxf(s[nt][e], s[nt][e + 2]);
#pragma unroll
            for (int off = 4; off <= 16; off <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
            if (!(top > m[nt][e])) continue;  // the same in the row's lanes
            top += kSlack;
            const float fade = power2(m[nt][e] - top);
            m[nt][e] = top;
            sum[nt][e] *= fade;
#pragma unroll
            for (int i = 0; i < STEPS; i++) {
              acc[nt][i][e] *= fade;
              acc[nt][i][e + 2] *= fade;
            }
          }
      }
      // Weights, as the second product takes them: keys down, rows across.
      uint32_t b[WPARTS][NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; nt++) {
        const float m0 = m[nt][0] == -INFINITY ? 0.0f : m[nt][0], m1 = m[nt][1] == -INFINITY ? 0.0f : m[nt][1];
        const float p0 = power2(s[nt][0] - m0), p1 = power2(s[nt][1] - m1), p2 = power2(s[nt][2] - m0), p3 = power2(s[nt][3] - m1);
        sum[nt][0] += p0 + p2;
        sum[nt][1] += p1 + p3;
        float x0 = p0 * vs0, x1 = p1 * vs0, x2 = p2 * vs1, x3 = p3 * vs1;
        if (!whole) {  // an unseen value's scale does not count, whatever it is
          x0 = s[nt][0] == -INFINITY ? 0.0f : x0;
          x1 = s[nt][1] == -INFINITY ? 0.0f : x1;
          x2 = s[nt][2] == -INFINITY ? 0.0f : x2;
          x3 = s[nt][3] == -INFINITY ? 0.0f : x3;
        }
#pragma unroll
        for (int p = 0; p < WPARTS; p++) {
          const uint32_t lo = Pair<__nv_bfloat16>::pack(x0, x1), hi = Pair<__nv_bfloat16>::pack(x2, x3);
          b[p][nt][0] = transposed(lo);
          b[p][nt][1] = transposed(hi);
          const float2 l = unpacked(lo), h = unpacked(hi);
          x0 -= l.x, x1 -= l.y, x2 -= h.x, x3 -= h.y;
        }
      }
      // Values: lane (g, t) holds dims HD / 8 g .. of keys 2 t, 2 t + 1, 2 t + 8, 2 t + 9.
      constexpr int WORDS = HD == 64 ? 2 : 4;
#pragma unroll
      for (int half = 0; half < (HD == 256 ? 2 : 1); half++) {
        uint32_t v[4][WORDS];
#pragma unroll
        for (int j = 0; j < 4; j++) {
          load_words<WORDS>(values + value_at[j % 2] + j / 2 * 8 * HD + half * 128, v[j]);
        }
#pragma unroll
        for (int word = 0; word < WORDS; word++)
#pragma unroll
          for (int two = 0; two < 2; two++) {  // dims 2 two and 2 two + 1 of the word: rows g and g + 8
            const uint32_t s0 = two == 0 ? 0x4400u : 0x6622u, s1 = two == 0 ? 0x5511u : 0x7733u;
            const uint32_t f[4] = {
                widened(__byte_perm(v[0][word], v[1][word], s0), bits), widened(__byte_perm(v[0][word], v[1][word], s1), bits),
                widened(__byte_perm(v[2][word], v[3][word], s0), bits), widened(__byte_perm(v[2][word], v[3][word], s1), bits)};
            const int i = half * 8 + word * 2 + two;
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
              float fresh[4] = {};
#pragma unroll
              for (int p = WPARTS - 1; p >= 0; p--) mma16816(kFine ? fresh : acc[nt][i], f, b[p][nt][0], b[p][nt][1]);
              if constexpr (kFine)
#pragma unroll
                for (int e = 0; e < 4; e++) acc[nt][i][e] += fresh[e];
            }
          }
      }
    }
    __syncwarp();
    if (chunk + STAGES < chunks) issue(stage);
    asm volatile("cp.async.commit_group;" ::: "memory");
    stage = stage + 1 == STAGES ? 0 : stage + 1;
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");

  // ---- the warps join
  float* stats = reinterpret_cast<float*>(smem + S::kStats);  // [warp][row][base, sum]
  float* sums = reinterpret_cast<float*>(smem);               // [warp][row][dim], over the ring
  __syncthreads();
#pragma unroll
  for (int nt = 0; nt < NT; nt++)
#pragma unroll
    for (int e = 0; e < 2; e++) {
      float total = sum[nt][e];
#pragma unroll
      for (int off = 4; off <= 16; off <<= 1) total += __shfl_xor_sync(0xffffffffu, total, off);
      const int r = nt * 8 + 2 * t + e;
      if (g == 0) {
        stats[(warp * R + r) * 2] = m[nt][e];
        stats[(warp * R + r) * 2 + 1] = total;
      }
      float* to = sums + (warp * R + r) * HD;
#pragma unroll
      for (int i = 0; i < STEPS; i++) {
        // Step i's dims: two of this lane's run of 16 (8 where HD is 64) in its half.
        const int dim = HD == 64 ? g * 8 + i * 2 : i / 8 * 128 + g * 16 + i % 8 * 2;
        *reinterpret_cast<float2*>(to + dim) = make_float2(acc[nt][i][e], acc[nt][i][e + 2]);
      }
    }
  __syncthreads();
  const bool alone = w.slices == 1;
  float* part = static_cast<float*>(a.workspace) + ((tile * c.kv_heads + kv) * d.slices + slice) * (int64_t)(R * (HD + 2));
  for (int at = tid; at < w.rows * (HD / 4); at += kThreads) {
    const int r = at / (HD / 4), dim = at % (HD / 4) * 4;
    float top = -INFINITY, total = 0.0f;
#pragma unroll
    for (int i = 0; i < kWarps; i++) top = fmaxf(top, stats[(i * R + r) * 2]);
    const float base = top == -INFINITY ? 0.0f : top;
    float o[4] = {};
#pragma unroll
    for (int i = 0; i < kWarps; i++) {
      const float fade = power2(stats[(i * R + r) * 2] - base);
      total += stats[(i * R + r) * 2 + 1] * fade;
      const float4 v = *reinterpret_cast<const float4*>(sums + (i * R + r) * HD + dim);
      o[0] += v.x * fade, o[1] += v.y * fade, o[2] += v.z * fade, o[3] += v.w * fade;
    }
    if (!alone) {
      if (dim == 0) *reinterpret_cast<float2*>(part + R * HD + r * 2) = make_float2(top, total);
      *reinterpret_cast<float4*>(part + r * HD + dim) = make_float4(o[0], o[1], o[2], o[3]);
    } else if (dim < hd) {
      const int token = w.first + (w.row0 + r) / group, head = kv * group + (w.row0 + r) % group;
      if (token < 0 || token >= a.n) continue;
      T* out = static_cast<T*>(a.out) + (int64_t)token * a.out_stride + (int64_t)head * hd + dim;
#pragma unroll
      for (int e = 0; e < 4; e++) out[e] = from_f32<T>(total == 0.0f ? 0.0f : o[e] / total);
    }
  }
}

// The slices of a row, a block: its warps take every kJoinWarps-th.
template <typename T, int HD>
__global__ void __launch_bounds__(kJoinWarps * 32)
    paged_q8_join_kernel(const __grid_constant__ PagedQ8AttentionArgs a, const Split d) {
  pdl_launch_dependents();
  __shared__ float sums[kJoinWarps][HD], totals[kJoinWarps];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int kvh = (int)a.cache.kv_heads, group = (int)(a.heads / kvh), hd = (int)a.cache.hd;
  const int r = (int)(blockIdx.x % (unsigned)d.rows), kv = (int)(blockIdx.x / (unsigned)d.rows % (unsigned)kvh);
  const int64_t tile = blockIdx.x / (unsigned)d.rows / (unsigned)kvh;
  pdl_wait();
  const Work w = find_work(a, d, tile, group);
  if (r >= w.rows || w.slices == 1) return;
  const int64_t step = d.rows * (HD + 2);
  const float* part = static_cast<const float*>(a.workspace) + (tile * kvh + kv) * d.slices * step;
  const float2* stats = reinterpret_cast<const float2*>(part + d.rows * HD + r * 2);
  float top = -INFINITY;
  for (int i = lane; i < w.slices; i += 32) top = fmaxf(top, stats[i * step / 2].x);
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
  const float base = top == -INFINITY ? 0.0f : top;
  constexpr int N = HD > 128 ? HD / 128 : 1;
  float o[N][4] = {}, total = 0.0f;
#pragma unroll 8
  for (int i = warp; i < w.slices; i += kJoinWarps) {
    const float2 st = stats[i * step / 2];
    const float fade = power2(st.x - base);
    total += st.y * fade;
#pragma unroll
    for (int j = 0; j < N; j++) {
      const int dim = (j * 32 + lane) * 4;
      if (dim < HD) {
        const float4 v = *reinterpret_cast<const float4*>(part + i * step + r * HD + dim);
        o[j][0] += v.x * fade, o[j][1] += v.y * fade, o[j][2] += v.z * fade, o[j][3] += v.w * fade;
      }
    }
  }
#pragma unroll
  for (int j = 0; j < N; j++) {
    const int dim = (j * 32 + lane) * 4;
    if (dim < HD) *reinterpret_cast<float4*>(&sums[warp][dim]) = make_float4(o[j][0], o[j][1], o[j][2], o[j][3]);
  }
  if (lane == 0) totals[warp] = total;
  __syncthreads();
  const int token = w.first + (w.row0 + r) / group, head = kv * group + (w.row0 + r) % group;
  if (token < 0 || token >= a.n) return;
  T* out = static_cast<T*>(a.out) + (int64_t)token * a.out_stride + (int64_t)head * hd;
  for (int dim = threadIdx.x; dim < hd; dim += kJoinWarps * 32) {
    float x = 0.0f, all = 0.0f;
#pragma unroll
    for (int i = 0; i < kJoinWarps; i++) {
      x += sums[i][dim];
      all += totals[i];
    }
    out[dim] = from_f32<T>(all == 0.0f ? 0.0f : x / all);
  }
}

// ------------------------------------------------------------------ the host

constexpr int kMinSlice = 256;          // keys
constexpr int64_t kBlocks = 148 * 3 * 4;  // a few turns of what is resident

int padded_hd(int64_t hd) { return hd <= 64 ? 64 : hd <= 128 ? 128 : 256; }

Split split_of(const PagedQ8Cache& c, int64_t heads, int64_t n, int64_t max_length, int64_t window, bool ragged) {
  const int64_t group = heads / c.kv_heads, seqs = c.sequences < 1 ? 1 : c.sequences;
  const int64_t each = (n + seqs - 1) / seqs * group;
  Split d;
  d.rows = each <= 8 ? 8 : each <= 16 || padded_hd(c.hd) == 256 ? 16 : 32;
  d.tiles = ragged ? n * group / d.rows + c.sequences : c.sequences * ((group + d.rows - 1) / d.rows);
  // Keys that a tile may see.
  int64_t keys = max_length < 1 ? 1 : max_length;
  if (window > 0 && window + d.rows < keys) keys = window + d.rows;
  int64_t slices = (kBlocks + d.tiles * c.kv_heads - 1) / (d.tiles * c.kv_heads < 1 ? 1 : d.tiles * c.kv_heads);
  const int64_t most = (keys + kMinSlice - 1) / kMinSlice;
  slices = slices < most ? slices : most;
  d.most = (int)slices;
  const int64_t step = 64, slice = ((keys + slices - 1) / slices + step - 1) / step * step;
  d.slice = (int)slice;
  d.slices = (int)((keys + slice - 1) / slice);
  return d;
}

int64_t split_bytes(const PagedQ8Cache& c, const Split& d) {
  return d.most == 1 ? 16 : d.tiles * c.kv_heads * d.most * d.rows * (padded_hd(c.hd) + 2) * 4;
}

template <auto KERNEL>
cudaError_t launch(int64_t blocks, int threads, int smem, const PagedQ8AttentionArgs& a, const Split& d, cudaStream_t stream,
                   bool pdl) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl ? 1 : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, KERNEL, a, d);
}

template <typename T, int HD, int NT, int BLOCKS>
cudaError_t launch_tile(const PagedQ8AttentionArgs& a, const Split& d, cudaStream_t stream, bool pdl) {
  constexpr int smem = Smem<HD, NT, Parts<T>::query>::kBytes;
  if (cudaError_t e = allow_smem<paged_q8_attention_kernel<T, HD, NT, BLOCKS>>(smem); e != cudaSuccess) return e;
  if (cudaError_t e = launch<paged_q8_attention_kernel<T, HD, NT, BLOCKS>>(d.tiles * a.cache.kv_heads * d.slices, kThreads, smem,
                                                                           a, d, stream, pdl);
      e != cudaSuccess || d.slices == 1)
    return e;
  return launch<paged_q8_join_kernel<T, HD>>(d.tiles * a.cache.kv_heads * d.rows, kJoinWarps * 32, 0, a, d, stream, true);
}

template <typename T>
cudaError_t launch_type(const PagedQ8AttentionArgs& a, const Split& d, cudaStream_t stream, bool pdl) {
  switch (padded_hd(a.cache.hd)) {
    case 64:
      return d.rows == 8    ? launch_tile<T, 64, 1, 3>(a, d, stream, pdl)
             : d.rows == 16 ? launch_tile<T, 64, 2, 3>(a, d, stream, pdl)
                            : launch_tile<T, 64, 4, 2>(a, d, stream, pdl);
    case 128:
      return d.rows == 8    ? launch_tile<T, 128, 1, 3>(a, d, stream, pdl)
             : d.rows == 16 ? launch_tile<T, 128, 2, 3>(a, d, stream, pdl)
                            : launch_tile<T, 128, 4, 2>(a, d, stream, pdl);
    default:
      return d.rows == 8 ? launch_tile<T, 256, 1, 2>(a, d, stream, pdl) : launch_tile<T, 256, 2, 2>(a, d, stream, pdl);
  }
}

}  // namespace

int64_t paged_q8_attention_workspace(const PagedQ8Cache& c, int64_t heads, int64_t n, int64_t max_length) {
  // For either form of the queries, and every window: fewer keys are split
  // into at most as many slices, before their lengths are rounded up.
  int64_t bytes = 16;
  for (const bool ragged : {false, true}) {
    const Split d = split_of(c, heads, n, max_length, 0, ragged);
    const int64_t need = split_bytes(c, d);
    bytes = need > bytes ? need : bytes;
  }
  return bytes;
}

cudaError_t launch_paged_q8_attention(const PagedQ8AttentionArgs& a, cudaStream_t stream, bool pdl) {
  if (a.n <= 0 || a.cache.sequences <= 0) return cudaSuccess;
  const Split d = split_of(a.cache, a.heads, a.n, a.max_length, a.window, a.q_start != nullptr);
  switch (a.type) {
    case kF32: return launch_type<float>(a, d, stream, pdl);
    case kF16: return launch_type<__half>(a, d, stream, pdl);
    default: return launch_type<__nv_bfloat16>(a, d, stream, pdl);
  }
}

}  // namespace dn
