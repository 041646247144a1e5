// The pieces that the paged attention's kernels share: how a launch's blocks
// map to work, what a row of queries sees, and where partial results go.
//
// A row is one head's query of one token; the rows of a kv head's group lie
// together, row = token * group + g. The keys a row sees, positions low ..
// high, fall in two parts: the shared prefix (positions below `prefix`, read
// through one page list for the whole batch) and the sequence's own. A block
// takes a tile of rows of one kv head and a slice of one part's keys and
// leaves, for each row, the running maximum m of its scores (in log2 units),
// the sum l of 2^(score - m) and the weighted values acc; the join is
//   m = max m_i, l = sum l_i 2^(m_i - m), out = sum acc_i 2^(m_i - m) / l.
#pragma once

#include "dn_common.cuh"
#include "dn_launch.h"
#include "elem.cuh"
#include "kernel_smem.h"

namespace dn {
namespace paged {

constexpr float kLog2e = 1.4426950408889634f;

struct Params {
  PagedAttentionArgs a;
  int group;            // query heads of a kv head
  int prefix_rows, own_rows;  // rows of a block's tile, by the part (a power of two)
  int own_rows_log2;
  int thin_rows;        // of the tiles of the thin or the f32 kernel
  bool prefix_wide, own_wide;  // which parts the wide kernel takes
  bool beside;          // this launch runs beside the one before it
  int prefix_tiles, prefix_splits;
  int own_slots, own_splits;
  int prefix_least, own_least;  // keys: slices are not made shorter than this
  int slices;           // results of a row
  float* acc;           // [slices][n * heads][hd]
  float2* ml;           // [slices][n * heads]: m, l
  float scale_log2;
  int page_shift;       // log2 of the page size, or -1
  uint32_t* status;     // bounded waits' status word
  bool pairs, runs;     // rows of q and out are 4-byte, 16-byte aligned
  bool solo;            // each sequence reads the prefix for itself
  bool direct;          // one slice in all: blocks write `out` themselves
};

// A block's work: rows row0 .. row0 + rows - 1 of kv head `head`, slice
// `slice` of the part's keys, whose pages are `pages`.
struct Work {
  bool prefix;
  int head, row0, rows, slice, splits;
  int seq, seq_end, length;  // own work: the sequence, its last token + 1, its length
};

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ int seq_start(const Params& p, int s) {
  if (p.a.q_start == nullptr) return s;
  const int v = p.a.q_start[s];
  return v < 0 ? 0 : v > (int)p.a.n ? (int)p.a.n : v;
}

// A bounded wait that first spins without the clock, whose reading takes
// longer than most waits here.
__device__ __forceinline__ bool wait_phase(uint64_t* bar, uint32_t parity, uint32_t* status, uint32_t bits) {
#pragma unroll 1
  for (int i = 0; i < 64; i++)
    if (mbar_try_wait(bar, parity)) return true;
  return mbar_wait_bounded(bar, parity, status, bits);
}

// The sequence that token t belongs to, or -1. A batch of one token a
// sequence is recognized in one round of loads.
__device__ __forceinline__ int seq_of(const Params& p, int t) {
  const int seqs = (int)p.a.cache.sequences;
  if (p.a.q_start == nullptr) return t < seqs ? t : -1;
  if (t < seqs && seq_start(p, t) == t && seq_start(p, t + 1) == t + 1) return t;
  int lo = 0, hi = seqs;  // the last s with seq_start(s) <= t
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (seq_start(p, mid) <= t) lo = mid + 1;
    else hi = mid;
  }
  const int s = lo - 1;
  return s >= 0 && t < seq_start(p, s + 1) ? s : -1;
}

// Positions low .. high of the prefix, or of the sequence's own part, that
// token t sees (high < low: none).
__device__ __forceinline__ void sees(const Params& p, const Work& w, int t, int& low, int& high) {
  low = 0;
  high = -1;
  if (w.prefix) {
    // One token a sequence: one round of loads.
    const int seqs = (int)p.a.cache.sequences, near = min(t, seqs - 1);
    if (near < 0) return;
    const int start = seq_start(p, near), end = seq_start(p, near + 1), length = p.a.lengths[near];
    if (near == t && start == t && end == t + 1) {
      high = length - 1;
    } else {
      const int s = seq_of(p, t);
      if (s < 0) return;
      high = p.a.lengths[s] - (seq_start(p, s + 1) - t);
    }
  } else {
    high = w.length - (w.seq_end - t);
  }
  if (p.a.window > 0) low = max(0, high - (int)p.a.window + 1);
  if (w.prefix) {
    high = min(high, (int)p.a.prefix - 1);
  } else {
    if (!p.solo) low = max(low, (int)p.a.prefix);
    const int held = (int)(p.a.cache.table_stride * p.a.cache.page_size);  // (the prefix needs no table)
    high = min(high, (p.solo ? max(held, (int)p.a.prefix) : held) - 1);
  }
}

// Slots of own work: sequence s has slots first(s) .. first(s + 1) - 1, at
// least its ceil(rows / own_rows); first(sequences) = own_slots at most.
__device__ __forceinline__ int first_slot(const Params& p, int start, int s) {
  return ((start * p.group) >> p.own_rows_log2) + s;
}

// Called by every thread of a block of whole warps.
__device__ __forceinline__ bool find_work(const Params& p, Work& w) {
  int b = blockIdx.x;
  w.head = blockIdx.y;
  const int prefix_blocks = p.prefix_tiles * p.prefix_splits;
  w.prefix = b < prefix_blocks;
  if (w.prefix) {
    w.seq = -1;
    w.splits = p.prefix_splits;
    w.slice = b / p.prefix_tiles;
    w.row0 = b % p.prefix_tiles * p.prefix_rows;
    w.rows = min(p.prefix_rows, (int)p.a.n * p.group - w.row0);
    return w.rows > 0;
  }
  b -= prefix_blocks;
  w.splits = p.own_splits;
  w.slice = b / p.own_slots;
  const int slot = b % p.own_slots;
  const int seqs = (int)p.a.cache.sequences;
  if (p.a.q_start == nullptr && p.group <= p.own_rows) {
    if (slot >= seqs) return false;
    w.seq = slot;
    w.row0 = slot * p.group;
    w.rows = p.group;
    w.seq_end = slot + 1;
    w.length = p.a.lengths[slot];
    return true;
  }
  if (seqs == 0) return false;
  // The last s < seqs with first_slot(s) <= slot: by 32-fold sections, the
  // first of them around where one token a sequence would put it.
  const int lane = threadIdx.x % 32;
  int lo = 0, hi = seqs;  // the answer lies in lo .. hi - 1
  const int guess = (int)((unsigned)(slot * p.own_rows) / (unsigned)(p.own_rows + p.group)) - 16;
  int at = max(0, min(guess, seqs - 32)), step = 1, start, ahead, length;
  for (;;) {
    const int s = at + lane * step;
    start = s < seqs ? seq_start(p, s) : -1;
    length = s < seqs ? p.a.lengths[s] : 0;
    const bool under = s < hi && first_slot(p, start, s) <= slot;
    const unsigned votes = __ballot_sync(0xffffffffu, under);
    const int count = __popc(votes);  // monotone: lanes 0 .. count - 1
    if (count > 0) lo = max(lo, at + (count - 1) * step);
    if (count < 32) hi = min(hi, at + count * step);
    if (hi - lo <= 1) break;
    step = max(1, (hi - lo + 31) / 32);
    at = lo;
  }
  w.seq = lo;
  // Its start, its end and its length: in a lane as a rule, else loaded.
  const int from = (lo - at) / step;
  if (step == 1 && from >= 0 && from < 31) {
    ahead = __shfl_sync(0xffffffffu, start, from + 1);
    start = __shfl_sync(0xffffffffu, start, from);
    length = __shfl_sync(0xffffffffu, length, from);
    if (ahead < 0) ahead = seq_start(p, lo + 1);
  } else {
    start = seq_start(p, lo);
    ahead = seq_start(p, lo + 1);
    length = p.a.lengths[lo];
  }
  w.seq_end = ahead;
  w.length = length;
  const int tile = slot - first_slot(p, start, lo);
  w.row0 = start * p.group + tile * p.own_rows;
  w.rows = min(p.own_rows, w.seq_end * p.group - w.row0);
  return tile >= 0 && w.rows > 0;
}

// A position's entry of the page list (a shift for the usual page sizes: a
// division by a variable takes some twenty instructions).
__device__ __forceinline__ int entry_of(const Params& p, int pos) {
  return p.page_shift >= 0 ? pos >> p.page_shift : pos / (int)p.a.cache.page_size;
}

// The entry of a position's page as it lies in the list, -1 past its end. Not
// looked at here, so that the load may be on its way until page_of is called.
__device__ __forceinline__ int entry_at(const Params& p, const Work& w, int pos) {
  const int entry = entry_of(p, pos);
  const bool shared = w.prefix || (p.solo && pos < (int)p.a.prefix);
  const int* list = shared ? p.a.prefix_pages : p.a.cache.table + (int64_t)w.seq * p.a.cache.table_stride;
  return (shared ? pos < (int)p.a.prefix : entry < (int)p.a.cache.table_stride) ? list[entry] : -1;
}
// The page that an entry names, or -1 where that is none.
__device__ __forceinline__ int page_of(const Params& p, int entry) {
  return entry >= 0 && entry < (int)p.a.cache.pages ? entry : -1;
}

// The slice's keys, begin .. end - 1, of the positions low .. high that the
// tile's rows see between them; slices start at multiples of `tile`.
__device__ __forceinline__ void slice_keys(const Params& p, const Work& w, int low, int high, int tile, int& begin,
                                           int& end) {
  begin = end = 0;
  if (high < low) return;
  const int lo = low / tile * tile, keys = high - lo + 1;
  int per = max((keys + w.splits - 1) / w.splits, w.prefix ? p.prefix_least : p.own_least);
  per = (per + tile - 1) / tile * tile;
  const int64_t b = lo + (int64_t)w.slice * per;
  begin = (int)min((int64_t)high + 1, b);
  end = (int)min((int64_t)high + 1, b + per);
}

// Element offset, in the pools, of the row of position pos of the block's kv
// head, whose entry is `entry`, or -1; seen are positions low .. end - 1.
__device__ __forceinline__ int64_t row_at(const Params& p, const Work& w, int entry, int pos, int low, int end) {
  const int page = page_of(p, entry);
  if (pos < low || pos >= end || page < 0) return -1;
  const int size = (int)p.a.cache.page_size;
  const int slot = p.page_shift >= 0 ? pos & (size - 1) : pos % size;
  return page * p.a.cache.page_stride + ((int64_t)w.head * size + slot) * p.a.cache.hd;
}

// Index of a row of the tile in the workspace: token * heads + head.
__device__ __forceinline__ int64_t out_index(const Params& p, const Work& w, int r, int& token, int& head) {
  const int row = w.row0 + r;
  token = row / p.group;
  head = w.head * p.group + row % p.group;
  return (int64_t)token * p.a.heads + head;
}

// Where a block's result goes among a row's.
__device__ __forceinline__ int slice_index(const Params& p, const Work& w) {
  return w.prefix ? w.slice : p.prefix_splits + w.slice;
}

// Rows of a block of the wide kernel (the thin one: 8 or 16, the f32 one: 1 to 8).
constexpr int kWideRows = 128;
// Rows (of the batch on the prefix, of a sequence on average) past which the
// wide one runs. Measured, thin and wide (us, whole calls; 8 kv heads of 128, 2
// heads a group, bf16): on a prefix of 8192 keys 16 rows 22 and 24, 32 rows 32
// and 26, 64 rows 39 and 29, 128 rows 57 and 33; of 1024 keys 40 rows 14.7 and
// 18.5, 64 rows 15 and 19, 96 rows 21 and 20, 128 rows 22 and 22; rows of 16
// sequences of up to 1024 own keys, 24 rows on average 28 and 28, 32 rows 33 and
// 28, 48 rows 44 and 33; of one sequence of 2048 keys, at most 96 rows, 14 and
// 18. A middle: the long prefix gains from some 20 rows on, the short one from 96.
constexpr int kWideFrom = 32;
constexpr int kLanes = 32;

// Groups of a wide block: two outputs of 128 columns stand in TMEM beside the
// scores, of 256 one.
constexpr int wide_groups(int64_t hd) { return hd <= 128 ? 2 : 1; }

// Keys of a wide block's copy, all of one page: the box must divide the page.
inline int wide_box(int64_t page_size) { return page_size % 64 == 0 ? 64 : page_size % 32 == 0 ? 32 : 16; }

inline dim3 attention_grid(const Params& p) {
  return dim3((unsigned)(p.prefix_tiles * p.prefix_splits + p.own_slots * p.own_splits),
              (unsigned)p.a.cache.kv_heads);
}

template <typename K, typename... Args>
inline cudaError_t launch_ex(K kern, dim3 grid, int threads, size_t smem, cudaStream_t stream, bool pdl,
                             const Args&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl ? 1 : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, args...);
}

// The tensor-core kernels for the caches that mma_cache (paged_attention.cu)
// lets through: few rows of a tile (paged_attention_thin.cu), many
// (paged_attention_wide.cu).
cudaError_t launch_attention_thin(const Params& p, cudaStream_t stream, bool pdl);
cudaError_t launch_attention_wide(const Params& p, cudaStream_t stream, bool pdl);

}  // namespace paged
}  // namespace dn
