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
// The batch's work is divided on the device, by the lengths that it has: a pair
// (a tile of rows, a kv head) is a row of units of 64 keys, the pairs of all
// sequences one after another, and every block of one turn of the GPU takes an
// equal share of the units, whole pairs and parts of them. A block's four warps
// take every fourth chunk of 32 keys and bring it themselves, by 16-byte
// asynchronous copies into a ring of their own, the rows found through the page
// table a chunk ahead. (Warps that each took a share of their own were slower:
// one sequence of 131072 keys 58 us against 41, everyone at another place of the
// code and many more parts to join.) The base m of a row's softmax is set kSlack (log2)
// above its largest score so far and stands until a score passes it, which keeps
// the common path free of reductions: weights stay at most 1, and bf16 weights
// and f32 sums lose nothing by being 2^-kSlack of that. The parts of a pair join
// through the workspace in a second launch that is already waiting (programmatic
// launch).
//
// Measured, device time and share of a copy's 6.5 TB/s: 64 sequences of up to 16384
// positions, 32 heads on 8 of 128, bf16: 204 us, 83 %; f16 215 us; f32 at half the
// sequences 124 us, 68 %; 64 heads on 4 (16 rows a tile) 163 us, 52 %. One sequence
// of 131072, 28 heads on 4: 39 us, 54 %, of which the join 5. Prompts run too, though
// this is made for decode steps: 2048 bf16 tokens of 16 heads on 8 in 250 us.
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
constexpr int kCuts = 4;  // that a block of the second launch looks at
constexpr int kSms = 148;
constexpr int64_t kWhole = 256;  // batches whose sequences are said to be no longer are not split

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

constexpr int kUnit = 64;  // keys
// What a pair costs beside its keys, in units: its queries, the first copies'
// way through the page table, the join. It comes before the keys. A border
// between two blocks that would leave the first of them fewer than kLeast units
// of keys, or the second, is at the pair's begin or end instead.
// 32 sequences of up to 4096 keys: 67 us without it (short sequences' pairs fill
// some blocks and keep the others waiting).
constexpr int kCost = 4, kLeast = 2;

// A sequence's share of the batch: `tiles` tiles of its rows, each of them with
// every kv head `units` units (as many as its longest tile needs).
struct Share {
  int first, count, length;  // the sequence's first token, its tokens, its positions
  int64_t tiles, units;
};

template <int R>
__device__ __forceinline__ Share share_of(const PagedQ8AttentionArgs& a, int seq, int group) {
  Share s;
  s.first = a.q_start != nullptr ? a.q_start[seq] : seq;
  s.count = a.q_start != nullptr ? min(max(0, a.q_start[seq + 1] - s.first), (int)a.n) : 1;
  s.length = a.lengths[seq];
  s.tiles = ((int64_t)s.count * group + R - 1) / R;
  int64_t keys = min64(s.length, a.cache.table_stride * a.cache.page_size);
  // A tile's window and its other tokens, from a multiple of kRun on.
  if (a.window > 0) keys = min64(keys, a.window + (R - 1) / group + 1 + kRun);
  s.units = kCost + (keys <= 0 ? 0 : (keys + kUnit - 1) / kUnit);
  return s;
}

// Where a border at unit `at` of a pair of `units` comes to be.
__device__ __forceinline__ int64_t border_at(int64_t at, int64_t units) {
  return at < kCost + kLeast ? 0 : units - at < kLeast ? units : at;
}

// A pair that is split: its parts are what the block before left in its second
// place, and this block and those up to `last` in their first.
struct Cut {
  int rows;  // 0: no pair begins to be split here
  int first, row0, kv, last;
};

constexpr int64_t kMaxBlocks = kSms * 4;

// Behind the parts: two places a block, [row][dim] sums and [row] base and total.
__device__ __forceinline__ Cut* cuts_of(const PagedQ8AttentionArgs& a, int rows, int hd) {
  return reinterpret_cast<Cut*>(static_cast<float*>(a.workspace) + kMaxBlocks * 2 * rows * (hd + 2));
}

// The dim at place p of a row of sums, which lie as the products' lanes hold
// them: step p / 16's pair of dims of lane group p % 16 / 2.
template <int HD>
__device__ __forceinline__ int dim_of(int p) {
  const int i = p / 16, g = p % 16 / 2;
  return (HD == 64 ? g * 8 + i * 2 : i / 8 * 128 + g * 16 + i % 8 * 2) + p % 2;
}

// a / b for a >= 0, b > 0, by the short division where that is enough.
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
  return ((a | b) >> 32) == 0 ? (int64_t)((uint32_t)a / (uint32_t)b) : a / b;
}

__device__ __forceinline__ void cp16(void* dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp4(void* dst, const void* src, bool there) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(there ? 4 : 0) : "memory");
}

__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// An 8 x 8 matrix of 16-bit elements, a row's pair to a lane, transposed.
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
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
  static constexpr int kRow = HD + 4;                      // floats: the lanes' pairs meet all banks
  static constexpr int kJoin = kWarps * NT * 8 * kRow * 4;  // the warps' sums, over the ring
  static constexpr int kScales = kRing > kJoin ? kRing : kJoin;
  static constexpr int kMasks = kScales + kWarps * kStages * 2 * kKeys * 4;
  static constexpr int kStats = kMasks + kWarps * kStages * 4;
  static constexpr int kQueries = (kStats + kWarps * NT * 8 * 2 * 4 + 15) / 16 * 16;
  static constexpr int kBytes = kQueries + PARTS * NT * (HD / 16) * 32 * 8;
};

// EXACT: rows of HD values in pages of whole runs.
template <typename T, int HD, int NT, int BLOCKS, bool EXACT>
__global__ void __launch_bounds__(kThreads, BLOCKS)
    paged_q8_attention_kernel(const __grid_constant__ PagedQ8AttentionArgs a, const int split) {
  constexpr int PARTS = Parts<T>::query, WPARTS = Parts<T>::weight, R = NT * 8;
  // The tensor cores cut their sums off (2^-23 of each, one way), which f32
  // results would show: there each chunk's sums begin at 0 and are added here.
  constexpr bool kFine = std::is_same<T, float>::value;
  using S = Smem<HD, NT, PARTS>;
  constexpr int STAGES = S::kStages, KEYS = S::kKeys, STEPS = HD / 16;
  constexpr int RUNS = NT == 1 ? KEYS / kRun : 1;  // taken together: independent products while others are under way
  constexpr uint32_t kAll = RUNS == 2 ? 0xffffffffu : 0xffffu;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int64_t sums_of[kWarps], found_at;
  __shared__ int found;
  pdl_launch_dependents();
  pdl_wait();
  const PagedQ8Cache& c = a.cache;
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32, g = lane / 4, t = lane % 4;
  const int hd = EXACT ? HD : (int)c.hd, page_size = (int)c.page_size, group = (int)(a.heads / c.kv_heads), kvh = (int)c.kv_heads;

  // ---- the block's units, and the sequence that the first one belongs to
  const int seqs = (int)c.sequences, each = (seqs + kThreads - 1) / kThreads;
  int64_t own = 0;
  for (int i = tid * each; i < min(seqs, (tid + 1) * each); i++) {
    const Share s = share_of<R>(a, i, group);
    own += s.tiles * s.units * kvh;
  }
  int64_t before = own;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, before, off);
    if (lane >= off) before += y;
  }
  if (lane == 31) sums_of[warp] = before;
  __syncthreads();
  int64_t total = 0;
#pragma unroll
  for (int i = 0; i < kWarps; i++) {
    if (i < warp) before += sums_of[i];
    total += sums_of[i];
  }
  before -= own;
  const int64_t blocks = min64(gridDim.x, total), block = blockIdx.x;
  Cut* cut = &cuts_of(a, R, HD)[block];
  if (block >= blocks) {
    if (split != 0 && tid == 0) cut->rows = 0;
    return;
  }
  int64_t at = quotient(block * total, blocks);
  const int64_t stop = quotient((block + 1) * total, blocks);
  if (at >= before && at < before + own) {
    int64_t start = before;
    int seq = tid * each;
    for (;; seq++) {
      const Share s = share_of<R>(a, seq, group);
      const int64_t size = s.tiles * s.units * kvh;
      if (at < start + size) break;
      start += size;
    }
    found = seq;
    found_at = start;
  }
  __syncthreads();
  int seq = found;
  int64_t seq_at = found_at;
  // Four values of a query at once.
  const bool wide_q = ((uintptr_t)a.q & (4 * sizeof(T) - 1)) == 0 && a.q_stride % 4 == 0;
  bool opening = true;  // the block's first pair
  while (at < stop) {
    const Share sh = share_of<R>(a, seq, group);
    const int64_t pair_units = sh.units, seq_units = sh.tiles * pair_units * kvh;
    if (at >= seq_at + seq_units) {
      seq_at += seq_units;
      seq++;
      continue;
    }
    const int64_t pair = quotient(at - seq_at, pair_units), pair_at = seq_at + pair * pair_units;
    const int64_t tile = quotient(pair, kvh);
    const int kv = (int)(pair - tile * kvh);
    const int row0 = (int)(tile * R), rows = (int)min64((int64_t)sh.count * group - row0, R);
    int64_t from = 0, to = pair_units;
    if (split != 0) {
      if (opening) {
        from = border_at(at - pair_at, pair_units);
        // The first border inside a pair tells the second launch of it.
        const bool inside = from > 0 && from < pair_units;
        const bool first_border = inside && border_at(quotient((block - 1) * total, blocks) - pair_at, pair_units) == 0;
        if (tid == 0) {
          cut->rows = first_border ? rows : 0;
          if (first_border) {
            const int64_t pair_end = pair_at + pair_units, last = (pair_end * blocks - 1) / total;
            cut->first = sh.first;
            cut->row0 = row0;
            cut->kv = kv;
            cut->last = (int)(border_at(quotient(last * total, blocks) - pair_at, pair_units) == pair_units ? last - 1 : last);
          }
        }
      }
      if (stop < pair_at + pair_units) to = border_at(stop - pair_at, pair_units);
    } else if (at > pair_at) {  // a pair belongs to the block that its first unit falls to
      from = to;
    }
    opening = false;
    at = pair_at + pair_units;
    if (from >= to) continue;
    const bool alone = from == 0 && to == pair_units;

    // Positions of the tile's first and last tokens, and the keys of this part.
    const int64_t first_pos = (int64_t)sh.length - sh.count + row0 / group;
    const int64_t last_pos = (int64_t)sh.length - sh.count + (row0 + rows - 1) / group;
    const int64_t most = c.table_stride * page_size;
    const int64_t low = a.window > 0 ? first_pos - a.window + 1 : 0;
    const int64_t pair_begin = low > 0 ? min64(low, most) / kRun * kRun : 0;
    const int64_t pair_end = last_pos + 1 < 0 ? 0 : min64(last_pos + 1, most);
    const int begin = (int)min64(pair_begin + (from > 0 ? from - kCost : 0) * kUnit, most);
    const int end = (int)min64(pair_end, pair_begin + (to - kCost) * kUnit);
    __syncthreads();  // the part before has left shared memory

    // ---- the ring: this lane's row of a chunk, its page a chunk ahead
    uint8_t* ring = smem + warp * STAGES * 2 * S::kChunk;
    float* scales = reinterpret_cast<float*>(smem + S::kScales) + warp * STAGES * 2 * KEYS;
    uint32_t* masks = reinterpret_cast<uint32_t*>(smem + S::kMasks) + warp * STAGES;
    if (hd != HD) {  // parts that no copy writes
      for (int at = lane * 16; at < STAGES * 2 * S::kChunk; at += 32 * 16)
        *reinterpret_cast<uint4*>(ring + at) = make_uint4(0, 0, 0, 0);
      __syncwarp();
    }
    const int32_t* table = c.table + (int64_t)seq * c.table_stride;
    // Where pages have whole runs of 16 rows of HD values, LANES lanes copy a run,
    // as one run of bytes. Else a row's parts are copied from where the lane that
    // follows it says.
    constexpr int LANES = KEYS == 32 ? 16 : 32, COPIES = KEYS * HD / 16 / 32;
    const int row = lane % KEYS, in_run = row % kRun;
    int pos = begin + warp * KEYS + row;  // of the next chunk to issue
    int entry = pos / page_size, slot = pos - entry * page_size;
    const int entry_step = kWarps * KEYS / page_size, slot_step = kWarps * KEYS - entry_step * page_size;
    auto page_at = [&]() { return pos - (EXACT ? in_run : 0) < end ? table[entry] : -1; };
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
      if constexpr (EXACT) {
        const int64_t at = held ? page * c.page_stride + ((int64_t)kv * page_size + (slot - in_run)) * hd : 0;
        const int8_t* from_keys = c.keys + at + lane % LANES * 16;
        const int8_t* from_values = c.values + at + lane % LANES * 16;
#pragma unroll
        for (int i = 0; i < COPIES; i++) {  // LANES * 16 / HD rows on each time
          const int to = (first_to ^ turn_of<HD>(i * (LANES * 16 / HD)) * 16) + i * LANES * 16;
          cp16(keys + to, from_keys + i * LANES * 16, held);
          cp16(values + to, from_values + i * LANES * 16, held);
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
    // ---- the queries, as the products take them: of step i lane (g, t) holds
    // row g's dims 64 (i / 4) + 16 t + 4 (i % 4) .. + 3, the even ones first as
    // the keys' words give them
    auto load_query = [&](int nt, int i, int l, uint2(&to)[PARTS]) {
      const int r = nt * 8 + l / 4, dim = i / 4 * 64 + l % 4 * 16 + i % 4 * 4;
      const int token = sh.first + (row0 + r) / group, head = kv * group + (row0 + r) % group;
      float x[4] = {};
      if (r < rows && dim < hd && token >= 0 && token < a.n) {
        const T* src = static_cast<const T*>(a.q) + (int64_t)token * a.q_stride + (int64_t)head * hd + dim;
        if (wide_q) {
          load_run<T, 4>(src, x);
        } else {
#pragma unroll
          for (int e = 0; e < 4; e++) x[e] = to_f32<T>(src[e]);
        }
      }
#pragma unroll
      for (int p = 0; p < PARTS; p++) {
        to[p] = make_uint2(Pair<__nv_bfloat16>::pack(x[0], x[2]), Pair<__nv_bfloat16>::pack(x[1], x[3]));
        const float2 lo = unpacked(to[p].x), hi = unpacked(to[p].y);
        x[0] -= lo.x, x[2] -= lo.y, x[1] -= hi.x, x[3] -= hi.y;
      }
    };
    uint2* queries = reinterpret_cast<uint2*>(smem + S::kQueries);
    for (int at = tid; at < NT * STEPS * 32; at += kThreads) {
      uint2 x[PARTS];
      load_query(at / 32 / STEPS, at / 32 % STEPS, at % 32, x);
#pragma unroll
      for (int p = 0; p < PARTS; p++) queries[p * NT * STEPS * 32 + at] = x[p];
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
      for (int e = 0; e < 2; e++) high[nt][e] = sh.length - sh.count + (row0 + nt * 8 + 2 * t + e) / group;
    const int64_t window = a.window;
    const int all_high = sh.length - sh.count + row0 / group;
    const int64_t all_low = window > 0 ? (int64_t)sh.length - sh.count + (row0 + rows - 1) / group - window + 1 : 0;
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
    // The first STAGES turns only fill the ring: `issue` and what follows are in
    // the code once, which the instruction cache needs with every warp elsewhere.
#pragma unroll 1
    for (int chunk = -STAGES; chunk < chunks; chunk++) {
     if (chunk >= 0) {
      asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
      __syncwarp();
#pragma unroll 1
      for (int run0 = 0; run0 < KEYS / kRun; run0 += RUNS) {
        const uint8_t* keys = ring + stage * 2 * S::kChunk + run0 * kRun * HD;
        const uint8_t* values = keys + S::kChunk;

        // Scores: rows 2 t, 2 t + 1 of keys g (0, 1) and g + 8 (2, 3). `less`:
        // of the queries' parts but the first; of bf16, of every other step,
        // which leaves a chain of products half as long.
        float s[RUNS][NT][4], less[RUNS][NT][4];
#pragma unroll
        for (int run = 0; run < RUNS; run++)
#pragma unroll
          for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int e = 0; e < 4; e++) s[run][nt][e] = less[run][nt][e] = 0.0f;
#pragma unroll
        for (int block = 0; block < HD / 64; block++) {
          uint32_t k[RUNS][2][4];
#pragma unroll
          for (int run = 0; run < RUNS; run++)
#pragma unroll
            for (int e = 0; e < 2; e++)
              load_words<4>(keys + key_at[block % 2] + block / 2 * 128 + (run * kRun + e * 8) * HD, k[run][e]);
#pragma unroll
          for (int j = 0; j < 4; j++)
#pragma unroll
            for (int run = 0; run < RUNS; run++) {
              const uint32_t k0 = k[run][0][j], k1 = k[run][1][j];
              const uint32_t f[4] = {widened(k0, bits), widened(k1, bits), widened(k0 >> 8, bits), widened(k1 >> 8, bits)};
              const int i = block * 4 + j;
#pragma unroll
              for (int p = 0; p < PARTS; p++)
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                  const int at = (p * NT + nt) * STEPS + i;
                  uint2 b;
                  if constexpr (kHeld) b = held[at]; else b = queries[at * 32 + lane];
                  mma16816((PARTS > 1 ? p > 0 : i % 2 != 0) ? less[run][nt] : s[run][nt], f, b.x, b.y);
                }
            }
        }
        const float* sc = scales + stage * 2 * KEYS + run0 * kRun;
        const int first = begin + (chunk * kWarps + warp) * KEYS + run0 * kRun;
        const uint32_t mask = masks[stage] >> run0 * kRun & kAll;
        const bool whole = mask == kAll && first + RUNS * kRun - 1 <= all_high && first >= all_low;
        bool past = false;
#pragma unroll
        for (int run = 0; run < RUNS; run++) {
          const float ks[2] = {sc[run * kRun + g] * factor, sc[run * kRun + g + 8] * factor};
#pragma unroll
          for (int nt = 0; nt < NT; nt++) {
            float(&x)[4] = s[run][nt];
#pragma unroll
            for (int e = 0; e < 4; e++) x[e] = (x[e] + less[run][nt][e]) * ks[e / 2];
            if (!whole) {
#pragma unroll
              for (int e = 0; e < 4; e++) {
                const int key = run * kRun + g + e / 2 * 8, at = first + key, hi = high[nt][e & 1];
                const bool sees = (mask >> key & 1u) != 0 && at <= hi && (window == 0 || (int64_t)at > hi - window);
                x[e] = sees ? x[e] : -INFINITY;
              }
            }
            past |= fmaxf(x[0], x[2]) > m[nt][0] || fmaxf(x[1], x[3]) > m[nt][1];
          }
        }
        if (__any_sync(0xffffffffu, past)) {
#pragma unroll
          for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
              float top = fmaxf(s[0][nt][e], s[0][nt][e + 2]);
#pragma unroll
              for (int run = 1; run < RUNS; run++) top = fmaxf(top, fmaxf(s[run][nt][e], s[run][nt][e + 2]));
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
        uint32_t b[RUNS][WPARTS][NT][2];
#pragma unroll
        for (int run = 0; run < RUNS; run++) {
          const float vs[2] = {sc[KEYS + run * kRun + g], sc[KEYS + run * kRun + g + 8]};
#pragma unroll
          for (int nt = 0; nt < NT; nt++) {
            float x[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
              const float base = m[nt][e & 1] == -INFINITY ? 0.0f : m[nt][e & 1];
              const float p = power2(s[run][nt][e] - base);
              sum[nt][e & 1] += p;
              x[e] = p * vs[e / 2];
              // An unseen value's scale does not count, whatever it is.
              if (!whole) x[e] = s[run][nt][e] == -INFINITY ? 0.0f : x[e];
            }
#pragma unroll
            for (int p = 0; p < WPARTS; p++) {
              const uint32_t lo = Pair<__nv_bfloat16>::pack(x[0], x[1]), hi = Pair<__nv_bfloat16>::pack(x[2], x[3]);
              b[run][p][nt][0] = transposed(lo);
              b[run][p][nt][1] = transposed(hi);
              const float2 l = unpacked(lo), h = unpacked(hi);
              x[0] -= l.x, x[1] -= l.y, x[2] -= h.x, x[3] -= h.y;
            }
          }
        }
        // Values: lane (g, t) holds dims HD / 8 g .. of keys 2 t, 2 t + 1, 2 t + 8, 2 t + 9.
        constexpr int WORDS = HD == 64 ? 2 : 4;
#pragma unroll
        for (int half = 0; half < (HD == 256 ? 2 : 1); half++)
#pragma unroll
          for (int run = 0; run < RUNS; run++) {
            uint32_t v[4][WORDS];
#pragma unroll
            for (int j = 0; j < 4; j++)
              load_words<WORDS>(values + value_at[j % 2] + (run * kRun + j / 2 * 8) * HD + half * 128, v[j]);
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
                  for (int p = WPARTS - 1; p >= 0; p--)
                    mma16816(kFine ? fresh : acc[nt][i], f, b[run][p][nt][0], b[run][p][nt][1]);
                  if constexpr (kFine)
#pragma unroll
                    for (int e = 0; e < 4; e++) acc[nt][i][e] += fresh[e];
                }
              }
          }
      }
      __syncwarp();
     }
      if (chunk + STAGES < chunks) issue(stage);
      asm volatile("cp.async.commit_group;" ::: "memory");
      stage = stage + 1 == STAGES ? 0 : stage + 1;
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");

    // ---- out, or to this part's place
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
      for (int e = 0; e < 2; e++)
#pragma unroll
        for (int off = 4; off <= 16; off <<= 1) sum[nt][e] += __shfl_xor_sync(0xffffffffu, sum[nt][e], off);
    float* part = static_cast<float*>(a.workspace) + (block * 2 + (from == 0 ? 1 : 0)) * (int64_t)(R * (HD + 2));
    auto out_row = [&](int r) -> T* {
      const int token = sh.first + (row0 + r) / group, head = kv * group + (row0 + r) % group;
      return token < 0 || token >= a.n ? nullptr : static_cast<T*>(a.out) + (int64_t)token * a.out_stride + (int64_t)head * hd;
    };
    float* stats = reinterpret_cast<float*>(smem + S::kStats);  // [warp][row][base, sum]
    float* sums = reinterpret_cast<float*>(smem);               // [warp][row][place], over the ring
    __syncthreads();
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
      for (int e = 0; e < 2; e++) {
        const int r = nt * 8 + 2 * t + e;
        if (g == 0) {
          stats[(warp * R + r) * 2] = m[nt][e];
          stats[(warp * R + r) * 2 + 1] = sum[nt][e];
        }
        float* to = sums + (warp * R + r) * S::kRow + g * 2;
#pragma unroll
        for (int i = 0; i < STEPS; i++)
          *reinterpret_cast<float2*>(to + i * 16) = make_float2(acc[nt][i][e], acc[nt][i][e + 2]);
      }
    __syncthreads();
    for (int at = tid; at < rows * (HD / 4); at += kThreads) {
      const int r = at / (HD / 4), p = at % (HD / 4) * 4;
      float top = -INFINITY, whole_sum = 0.0f;
#pragma unroll
      for (int i = 0; i < kWarps; i++) top = fmaxf(top, stats[(i * R + r) * 2]);
      const float base = top == -INFINITY ? 0.0f : top;
      float o[4] = {};
#pragma unroll
      for (int i = 0; i < kWarps; i++) {
        const float fade = power2(stats[(i * R + r) * 2] - base);
        whole_sum += stats[(i * R + r) * 2 + 1] * fade;
        const float4 v = *reinterpret_cast<const float4*>(sums + (i * R + r) * S::kRow + p);
        o[0] += v.x * fade, o[1] += v.y * fade, o[2] += v.z * fade, o[3] += v.w * fade;
      }
      if (!alone) {
        if (p == 0) *reinterpret_cast<float2*>(part + R * HD + r * 2) = make_float2(top, whole_sum);
        *reinterpret_cast<float4*>(part + r * HD + p) = make_float4(o[0], o[1], o[2], o[3]);
      } else if (T* out = out_row(r); out != nullptr) {
        const float inv = whole_sum == 0.0f ? 0.0f : 1.0f / whole_sum;
#pragma unroll
        for (int e = 0; e < 4; e++)
          if (const int dim = dim_of<HD>(p + e); dim < hd) out[dim] = from_f32<T>(o[e] * inv);
      }
    }
  }
}

// A row of the pairs that kCuts blocks begin to split: a warp to a pair of few
// parts, all of the block to one of many.
template <typename T, int HD>
__global__ void __launch_bounds__(kJoinWarps * 32)
    paged_q8_join_kernel(const __grid_constant__ PagedQ8AttentionArgs a, const int tile_rows) {
  pdl_launch_dependents();
  constexpr int N = HD > 128 ? HD / 128 : 1, kFew = 8;
  __shared__ float sums[kJoinWarps][HD], totals[kJoinWarps];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, r = (int)blockIdx.y;
  const int group = (int)(a.heads / a.cache.kv_heads), hd = (int)a.cache.hd;
  const int64_t block0 = (int64_t)blockIdx.x * kCuts, step = 2 * tile_rows * (HD + 2);
  pdl_wait();
  const Cut* cuts = cuts_of(a, tile_rows, HD) + block0;
  // Sums of every `by`-th part from `i0` on, under the base of all.
  auto sum_parts = [&](const Cut& cut, int64_t block, int i0, int by, float(&o)[N][4], float& total) {
    // Part 0 lies in the second place of the block before; part i in block + i - 1's first.
    const float* parts = static_cast<const float*>(a.workspace) + (block - 1) * step;
    const int count = (int)(cut.last - block) + 2;
    auto part = [&](int i) { return parts + i * step + (i == 0 ? step / 2 : 0); };
    auto stats = [&](int i) { return *reinterpret_cast<const float2*>(part(i) + tile_rows * HD + r * 2); };
    float top = -INFINITY;
    for (int i = lane; i < count; i += 32) top = fmaxf(top, stats(i).x);
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
    const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll 4
    for (int i = i0; i < count; i += by) {
      const float2 st = stats(i);
      const float fade = power2(st.x - base);
      total += st.y * fade;
#pragma unroll
      for (int j = 0; j < N; j++) {
        const int p = (j * 32 + lane) * 4;
        if (p < HD) {
          const float4 v = *reinterpret_cast<const float4*>(part(i) + r * HD + p);
          o[j][0] += v.x * fade, o[j][1] += v.y * fade, o[j][2] += v.z * fade, o[j][3] += v.w * fade;
        }
      }
    }
  };
  auto out_row = [&](const Cut& cut) -> T* {
    const int token = cut.first + (cut.row0 + r) / group, head = cut.kv * group + (cut.row0 + r) % group;
    return token < 0 || token >= a.n ? nullptr : static_cast<T*>(a.out) + (int64_t)token * a.out_stride + (int64_t)head * hd;
  };
  if (const Cut cut = cuts[warp % kCuts]; warp < kCuts && r < cut.rows && cut.last - (block0 + warp) + 2 <= kFew) {
    float o[N][4] = {}, total = 0.0f;
    sum_parts(cut, block0 + warp, 0, 1, o, total);
    if (T* out = out_row(cut); out != nullptr) {
      const float inv = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
      for (int j = 0; j < N; j++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const int p = (j * 32 + lane) * 4 + e;
          if (const int dim = dim_of<HD>(p); p < HD && dim < hd) out[dim] = from_f32<T>(o[j][e] * inv);
        }
    }
  }
  for (int i = 0; i < kCuts; i++) {
    const Cut cut = cuts[i];
    if (r >= cut.rows || cut.last - (block0 + i) + 2 <= kFew) continue;  // the same in all threads
    float o[N][4] = {}, total = 0.0f;
    sum_parts(cut, block0 + i, warp, kJoinWarps, o, total);
    __syncthreads();  // the pair before has been read
#pragma unroll
    for (int j = 0; j < N; j++) {
      const int p = (j * 32 + lane) * 4;
      if (p < HD) *reinterpret_cast<float4*>(&sums[warp][p]) = make_float4(o[j][0], o[j][1], o[j][2], o[j][3]);
    }
    if (lane == 0) totals[warp] = total;
    __syncthreads();
    T* out = out_row(cut);
    for (int p = threadIdx.x; p < HD; p += kJoinWarps * 32) {
      float x = 0.0f, all = 0.0f;
#pragma unroll
      for (int j = 0; j < kJoinWarps; j++) {
        x += sums[j][p];
        all += totals[j];
      }
      if (const int dim = dim_of<HD>(p); out != nullptr && dim < hd) out[dim] = from_f32<T>(all == 0.0f ? 0.0f : x * (1.0f / all));
    }
  }
}

// ------------------------------------------------------------------ the host

int padded_hd(int64_t hd) { return hd <= 64 ? 64 : hd <= 128 ? 128 : 256; }

// Rows of a tile: those that a sequence has on average, if one tile can hold them.
int tile_rows(const PagedQ8Cache& c, int64_t heads, int64_t n) {
  const int64_t seqs = c.sequences < 1 ? 1 : c.sequences, each = (n + seqs - 1) / seqs * (heads / c.kv_heads);
  return each <= 8 ? 8 : each <= 16 || padded_hd(c.hd) == 256 ? 16 : 32;
}

template <auto KERNEL>
cudaError_t launch(dim3 grid, int threads, int smem, const PagedQ8AttentionArgs& a, int arg, cudaStream_t stream, bool pdl) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl ? 1 : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, KERNEL, a, arg);
}

template <typename T, int HD, int NT, int BLOCKS, bool EXACT>
cudaError_t launch_tile(const PagedQ8AttentionArgs& a, cudaStream_t stream, bool pdl) {
  using S = Smem<HD, NT, Parts<T>::query>;
  constexpr int blocks = kSms * BLOCKS;
  static_assert(blocks <= kMaxBlocks && blocks % kCuts == 0, "the workspace has places for so many");
  if (cudaError_t e = allow_smem<paged_q8_attention_kernel<T, HD, NT, BLOCKS, EXACT>>(S::kBytes); e != cudaSuccess) return e;
  const bool split = a.max_length > kWhole;
  if (cudaError_t e = launch<paged_q8_attention_kernel<T, HD, NT, BLOCKS, EXACT>>(dim3(blocks), kThreads, S::kBytes, a,
                                                                           split ? 1 : 0, stream, pdl);
      e != cudaSuccess || !split)
    return e;
  return launch<paged_q8_join_kernel<T, HD>>(dim3(blocks / kCuts, NT * 8), kJoinWarps * 32, 0, a, NT * 8, stream, true);
}

template <typename T, bool EXACT>
cudaError_t launch_type(const PagedQ8AttentionArgs& a, cudaStream_t stream, bool pdl) {
  // Queries of two and three parts leave registers for 16 rows.
  constexpr int most = Parts<T>::query == 1 ? 4 : 2;
  const int rows = tile_rows(a.cache, a.heads, a.n);
  switch (padded_hd(a.cache.hd)) {
    case 64:
      return rows == 8    ? launch_tile<T, 64, 1, 3, EXACT>(a, stream, pdl)
             : rows == 16 ? launch_tile<T, 64, 2, 3, EXACT>(a, stream, pdl)
                          : launch_tile<T, 64, most, 2, EXACT>(a, stream, pdl);
    case 128:
      return rows == 8    ? launch_tile<T, 128, 1, 3, EXACT>(a, stream, pdl)
             : rows == 16 ? launch_tile<T, 128, 2, 2, EXACT>(a, stream, pdl)
                          : launch_tile<T, 128, most, 2, EXACT>(a, stream, pdl);
    default:
      return rows == 8 ? launch_tile<T, 256, 1, 2, EXACT>(a, stream, pdl) : launch_tile<T, 256, 2, 2, EXACT>(a, stream, pdl);
  }
}

}  // namespace

int64_t paged_q8_attention_workspace(const PagedQ8Cache& c, int64_t heads, int64_t n, int64_t max_length) {
  if (max_length <= kWhole) return 16;
  return kMaxBlocks * (2 * tile_rows(c, heads, n) * (padded_hd(c.hd) + 2) * 4 + (int64_t)sizeof(Cut));
}

cudaError_t launch_paged_q8_attention(const PagedQ8AttentionArgs& a, cudaStream_t stream, bool pdl) {
  if (a.n <= 0 || a.cache.sequences <= 0) return cudaSuccess;
  const bool exact = a.cache.hd == padded_hd(a.cache.hd) && a.cache.page_size % kRun == 0;
  switch (a.type) {
    case kF32: return exact ? launch_type<float, true>(a, stream, pdl) : launch_type<float, false>(a, stream, pdl);
    case kF16: return exact ? launch_type<__half, true>(a, stream, pdl) : launch_type<__half, false>(a, stream, pdl);
    default:
      return exact ? launch_type<__nv_bfloat16, true>(a, stream, pdl) : launch_type<__nv_bfloat16, false>(a, stream, pdl);
  }
}

}  // namespace dn
