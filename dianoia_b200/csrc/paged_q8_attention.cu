// Attention over an 8-bit paged cache (dn_paged_q8_attention).
//
// Per query row: score_j = scale s_kj (q . k_j) over the positions it sees,
// out = sum_j exp(score_j - max) s_vj v_j / sum_j exp(score_j - max), all in
// f32. A block takes one head of one token; its warps take every kWarps-th
// key, a lane eight values of it, and join at the end.
#include "dn_common.cuh"
#include "dn_launch.h"
#include "elem.cuh"

namespace dn {
namespace {

constexpr int kWarps = 4;

template <typename T>
__global__ void __launch_bounds__(kWarps * 32) paged_q8_attention_kernel(const __grid_constant__ PagedQ8AttentionArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  const PagedQ8Cache& c = a.cache;
  const int hd = (int)c.hd, lane = threadIdx.x % 32, warp = threadIdx.x / 32, page_size = (int)c.page_size;
  const int t = (int)(blockIdx.x / (unsigned)a.heads), head = (int)(blockIdx.x % (unsigned)a.heads);
  const int kv = head / (int)(a.heads / c.kv_heads);
  int s = t, high = 0;  // the token's sequence and position
  if (a.q_start == nullptr) {
    high = a.lengths[s] - 1;
  } else {
    if (t >= a.q_start[c.sequences]) return;
    int lo = 0, hi = (int)c.sequences;  // the last sequence that starts at or before t
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (a.q_start[mid] <= t) lo = mid; else hi = mid;
    }
    s = lo;
    high = a.lengths[s] - (a.q_start[s + 1] - t);
  }
  const int64_t most = c.table_stride * page_size;
  int end = high < most ? high + 1 : (int)most;
  int begin = a.window > 0 && high - a.window + 1 > 0 ? (int)(high - a.window + 1) : 0;
  const bool mine = lane * 8 < hd;
  float q[8] = {}, acc[8] = {}, m = -INFINITY, sum = 0.0f;
  if (mine) {
    const T* src = static_cast<const T*>(a.q) + (int64_t)t * a.q_stride + (int64_t)head * hd + lane * 8;
#pragma unroll
    for (int e = 0; e < 8; e++) q[e] = to_f32<T>(src[e]);
  }
  for (int j = begin + warp; j < end; j += kWarps) {
    const int64_t page = c.table[s * c.table_stride + j / page_size];
    if (page < 0 || page >= c.pages) continue;
    const int64_t row = (int64_t)kv * page_size + j % page_size;
    float dot = 0.0f;
    int8_t k[8] = {}, v[8] = {};
    if (mine) {
      const int2 kk = *reinterpret_cast<const int2*>(c.keys + page * c.page_stride + row * hd + lane * 8);
      const int2 vv = *reinterpret_cast<const int2*>(c.values + page * c.page_stride + row * hd + lane * 8);
      memcpy(k, &kk, 8);
      memcpy(v, &vv, 8);
    }
#pragma unroll
    for (int e = 0; e < 8; e++) dot += q[e] * (float)k[e];
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, off);
    const float x = dot * c.key_scales[page * c.scale_stride + row] * a.scale;
    const float vs = c.value_scales[page * c.scale_stride + row];
    const float to = fmaxf(m, x), old = to == -INFINITY ? 0.0f : __expf(m - to), p = to == -INFINITY && x == to ? 0.0f : expf(x - to);
    m = to;
    sum = sum * old + p;
#pragma unroll
    for (int e = 0; e < 8; e++) acc[e] = acc[e] * old + p * vs * (float)v[e];
  }
  __shared__ float part[kWarps][256], tops[kWarps], sums[kWarps];
  if (lane == 0) {
    tops[warp] = m;
    sums[warp] = sum;
  }
  if (mine)
#pragma unroll
    for (int e = 0; e < 8; e++) part[warp][lane * 8 + e] = acc[e];
  __syncthreads();
  float top = -INFINITY, total = 0.0f;
  for (int w = 0; w < kWarps; w++) top = fmaxf(top, tops[w]);
  T* out = static_cast<T*>(a.out) + (int64_t)t * a.out_stride + (int64_t)head * hd;
  for (int w = 0; w < kWarps; w++) total += tops[w] == -INFINITY ? sums[w] : sums[w] * expf(tops[w] - top);
  for (int d = threadIdx.x; d < hd; d += kWarps * 32) {
    float o = 0.0f;
    for (int w = 0; w < kWarps; w++) o += tops[w] == -INFINITY ? part[w][d] : part[w][d] * expf(tops[w] - top);
    out[d] = from_f32<T>(total == 0.0f ? 0.0f : o / total);
  }
}

template <typename T>
cudaError_t launch_type(const PagedQ8AttentionArgs& a, cudaStream_t stream, bool pdl) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.n * a.heads));
  cfg.blockDim = dim3(kWarps * 32);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl ? 1 : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, paged_q8_attention_kernel<T>, a);
}

}  // namespace

int64_t paged_q8_attention_workspace(const PagedQ8Cache&, int64_t, int64_t, int64_t) { return 16; }

cudaError_t launch_paged_q8_attention(const PagedQ8AttentionArgs& a, cudaStream_t stream, bool pdl) {
  if (a.n <= 0) return cudaSuccess;
  switch (a.type) {
    case kF32: return launch_type<float>(a, stream, pdl);
    case kF16: return launch_type<__half>(a, stream, pdl);
    default: return launch_type<__nv_bfloat16>(a, stream, pdl);
  }
}

}  // namespace dn
