// An 8-bit paged cache written and read back (dn_paged_q8_append,
// dn_paged_q8_read).
//
// Append: the head norm and the rotation of paged_append.cu in f32, then a
// row of hd values becomes int8: scale = max |x| / 127,
// q = round_half_away(x (1 / scale)). Read: q scale.
//
// Bytes-bound: every value is read and written once. As in paged_append.cu a
// head belongs to a group of G lanes and a lane holds two runs of V values,
// the halves of a rotation pair, so the rotation needs no exchange; the row's
// largest magnitude is one more shuffle reduction of the group.
#include "dn_common.cuh"
#include "dn_launch.h"
#include "elem.cuh"

namespace dn {
namespace {

constexpr int kThreads = 256;

// The page and slot of a position; -1 where the cache holds none.
__device__ __forceinline__ int64_t page_of(const PagedQ8Cache& c, int seq, int pos, int& slot) {
  if (seq < 0 || seq >= c.sequences || pos < 0) return -1;
  const int entry = pos / (int)c.page_size;
  slot = pos - entry * (int)c.page_size;
  if (entry >= c.table_stride) return -1;
  const int64_t page = c.table[seq * c.table_stride + entry];
  return page >= 0 && page < c.pages ? page : -1;
}

template <int V>
__device__ __forceinline__ void store_q8(int8_t* p, const float (&x)[V], float inv) {
  int q[V];
#pragma unroll
  for (int e = 0; e < V; e++) q[e] = quant_q8_elem(x[e], inv);
  if constexpr (V == 8) {
    *reinterpret_cast<uint2*>(p) = make_uint2(pack4(q[0], q[1], q[2], q[3]), pack4(q[4], q[5], q[6], q[7]));
  } else {
#pragma unroll
    for (int e = 0; e < V; e++) p[e] = (int8_t)q[e];
  }
}

template <typename TI, typename TO, int V, int G, int ITER>
__global__ void __launch_bounds__(kThreads) paged_q8_append_kernel(const __grid_constant__ PagedQ8AppendArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  const int hd = (int)a.cache.hd, heads = (int)a.heads, kvh = (int)a.cache.kv_heads;
  const uint32_t per_token = (uint32_t)(heads + 2 * kvh);
  const int64_t unit = (int64_t)blockIdx.x * (kThreads / G) + threadIdx.x / G;
  if (unit >= a.n * per_token) return;  // whole groups leave together
  const uint32_t t = (uint32_t)(unit / per_token), h = (uint32_t)(unit % per_token);
  const int lane = threadIdx.x % G;
  const unsigned group = G == 32 ? 0xffffffffu : ((1u << G) - 1) << (threadIdx.x % 32 / G * G);
  const bool query = (int)h < heads, value = (int)h >= heads + kvh;

  // A slot's two runs: (s, s + rot / 2) for the rotated pairs, then the rest;
  // of a value, which does not turn, runs 2 s and 2 s + 1.
  const int rot = (int)a.rot, pairs = value ? 0 : rot / 2 / V, slots = hd / V / 2, turned = value ? 0 : rot;
  int first[ITER], second[ITER];
#pragma unroll
  for (int i = 0; i < ITER; i++) {
    const int s = lane + i * G;
    first[i] = s < pairs ? s * V : turned + 2 * (s - pairs) * V;
    second[i] = s < pairs ? first[i] + rot / 2 : first[i] + V;
  }
  const TI* src = query   ? static_cast<const TI*>(a.q) + (int64_t)t * a.q_stride + (int64_t)h * hd
                  : value ? static_cast<const TI*>(a.v) + (int64_t)t * a.v_stride + (int64_t)(h - heads - kvh) * hd
                          : static_cast<const TI*>(a.k) + (int64_t)t * a.k_stride + (int64_t)(h - heads) * hd;
  float p[ITER][V], q[ITER][V];
#pragma unroll
  for (int i = 0; i < ITER; i++) {
#pragma unroll
    for (int e = 0; e < V; e++) p[i][e] = q[i][e] = 0.0f;
    if (lane + i * G < slots) {
      load_run<TI, V>(src + first[i], p[i]);
      load_run<TI, V>(src + second[i], q[i]);
    }
  }
  const int pos = a.pos[t];
  int slot = 0;
  const int64_t page = a.rot > 0 && pos >= a.rope_rows ? -1 : page_of(a.cache, a.seq[t], pos, slot);
  TO* out = static_cast<TO*>(a.q_out) + (int64_t)t * a.q_out_stride + (int64_t)h * hd;
  if (page < 0) {  // the whole group
    const float zero[V] = {};
#pragma unroll
    for (int i = 0; i < ITER; i++)
      if (query && lane + i * G < slots) {
        store_run<TO, V>(out + first[i], zero);
        store_run<TO, V>(out + second[i], zero);
      }
    return;
  }
  const float* w = query ? a.q_norm : value ? nullptr : a.k_norm;
  if (w != nullptr) {
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < ITER; i++)
#pragma unroll
      for (int e = 0; e < V; e++) sum += p[i][e] * p[i][e] + q[i][e] * q[i][e];
#pragma unroll
    for (int off = G / 2; off >= 1; off >>= 1) sum += __shfl_xor_sync(group, sum, off);
    const float r = 1.0f / sqrtf(sum / (float)hd + a.eps);
#pragma unroll
    for (int i = 0; i < ITER; i++) {
      if (lane + i * G >= slots) continue;
      float wx[V], wy[V];
      load_run<float, V>(w + first[i], wx);
      load_run<float, V>(w + second[i], wy);
#pragma unroll
      for (int e = 0; e < V; e++) {
        p[i][e] *= r * wx[e];
        q[i][e] *= r * wy[e];
      }
    }
  }
  const float* turns = a.rope + (int64_t)pos * rot;
#pragma unroll
  for (int i = 0; i < ITER; i++) {
    if (lane + i * G >= pairs) continue;
    float c[V], n[V];
    load_run<float, V>(turns + first[i], c);
    load_run<float, V>(turns + rot / 2 + first[i], n);
#pragma unroll
    for (int e = 0; e < V; e++) {
      const float f = p[i][e], g = q[i][e];
      p[i][e] = f * c[e] - g * n[e];
      q[i][e] = g * c[e] + f * n[e];
    }
  }
  if (query) {
#pragma unroll
    for (int i = 0; i < ITER; i++)
      if (lane + i * G < slots) {
        store_run<TO, V>(out + first[i], p[i]);
        store_run<TO, V>(out + second[i], q[i]);
      }
    return;
  }
  float amax = 0.0f;  // infinite where a value is not finite (fmaxf leaves NaN out)
#pragma unroll
  for (int i = 0; i < ITER; i++)
#pragma unroll
    for (int e = 0; e < V; e++) {
      const float m = fmaxf(fabsf(p[i][e]), fabsf(q[i][e]));
      amax = fmaxf(amax, isnan(p[i][e]) || isnan(q[i][e]) ? INFINITY : m);
    }
#pragma unroll
  for (int off = G / 2; off >= 1; off >>= 1) amax = fmaxf(amax, __shfl_xor_sync(group, amax, off));
  float scale, inv;
  q8_scale(amax, scale, inv);
  if (scale < 1.17549435e-38f) scale = inv = 0.0f;  // 1 / scale would overflow
  const bool bad = isinf(amax);
  const int64_t head = value ? h - heads - kvh : h - heads;
  const int64_t row = head * a.cache.page_size + slot;
  int8_t* dst = (value ? a.cache.values : a.cache.keys) + page * a.cache.page_stride + row * hd;
  float* dst_scale = (value ? a.cache.value_scales : a.cache.key_scales) + page * a.cache.scale_stride + row;
  if (lane == 0) *dst_scale = bad ? NAN : scale;
#pragma unroll
  for (int i = 0; i < ITER; i++) {
    if (lane + i * G >= slots) continue;
    if (bad)
#pragma unroll
      for (int e = 0; e < V; e++) p[i][e] = q[i][e] = 0.0f;
    store_q8<V>(dst + first[i], p[i], bad ? 0.0f : inv);
    store_q8<V>(dst + second[i], q[i], bad ? 0.0f : inv);
  }
}

template <typename TI, typename TO, int V, int G, int ITER>
cudaError_t launch_append(const PagedQ8AppendArgs& a, cudaStream_t stream, bool pdl) {
  const int64_t units = a.n * (a.heads + 2 * a.cache.kv_heads);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((units * G + kThreads - 1) / kThreads));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl ? 1 : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, paged_q8_append_kernel<TI, TO, V, G, ITER>, a);
}

template <typename TI, typename TO>
cudaError_t append_types(const PagedQ8AppendArgs& a, cudaStream_t stream, bool pdl) {
  // Runs of 8 values where sizes, strides and addresses allow 16-byte
  // accesses of each type; else one value at a time.
  const uintptr_t addr = (uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.q_out | (uintptr_t)a.rope |
                         (uintptr_t)a.q_norm | (uintptr_t)a.k_norm;
  const int64_t step = a.q_stride | a.k_stride | a.v_stride | a.q_out_stride | a.rot / 2;
  if ((addr & 15) != 0 || step % 8 != 0) return launch_append<TI, TO, 1, 32, 4>(a, stream, pdl);
  if (a.cache.hd <= 64) return launch_append<TI, TO, 8, 4, 1>(a, stream, pdl);
  if (a.cache.hd <= 128) return launch_append<TI, TO, 8, 8, 1>(a, stream, pdl);
  return launch_append<TI, TO, 8, 16, 1>(a, stream, pdl);
}

template <typename TI>
cudaError_t append_in(const PagedQ8AppendArgs& a, cudaStream_t stream, bool pdl) {
  switch (a.out_type) {
    case kF32: return append_types<TI, float>(a, stream, pdl);
    case kF16: return append_types<TI, __half>(a, stream, pdl);
    default: return append_types<TI, __nv_bfloat16>(a, stream, pdl);
  }
}

// 16 values to a lane, a row to a group of G lanes. WIDE: the outputs take
// 16-byte accesses.
template <typename TO, int G, bool WIDE>
__global__ void __launch_bounds__(kThreads) paged_q8_read_kernel(const __grid_constant__ PagedQ8ReadArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  const int hd = (int)a.cache.hd, kvh = (int)a.cache.kv_heads, lane = threadIdx.x % G;
  const int64_t unit = (int64_t)blockIdx.x * (kThreads / G) + threadIdx.x / G;
  if (unit >= a.n * 2 * kvh || lane * 16 >= hd) return;
  const int64_t t = unit / (2 * kvh);
  const int h = (int)(unit % (2 * kvh));
  const bool value = h >= kvh;
  void* to = value ? a.v_out : a.k_out;
  if (to == nullptr) return;
  const int head = value ? h - kvh : h;
  TO* out = static_cast<TO*>(to) + t * (value ? a.v_stride : a.k_stride) + (int64_t)head * hd + lane * 16;
  int slot = 0;
  const int64_t page = page_of(a.cache, a.seq[t], a.pos[t], slot);
  float x[16] = {};
  if (page >= 0) {
    const int64_t row = (int64_t)head * a.cache.page_size + slot;
    const int4 raw = *reinterpret_cast<const int4*>((value ? a.cache.values : a.cache.keys) + page * a.cache.page_stride +
                                                    row * hd + lane * 16);
    const float scale = (value ? a.cache.value_scales : a.cache.key_scales)[page * a.cache.scale_stride + row];
    int8_t q[16];
    memcpy(q, &raw, 16);
#pragma unroll
    for (int e = 0; e < 16; e++) x[e] = __fmul_rn((float)q[e], scale);
  }
  if constexpr (WIDE) {
    store_run<TO, 16>(out, x);
  } else {
#pragma unroll
    for (int e = 0; e < 16; e++) out[e] = from_f32<TO>(x[e]);
  }
}

template <typename TO, int G, bool WIDE>
cudaError_t launch_read(const PagedQ8ReadArgs& a, cudaStream_t stream, bool pdl) {
  const int64_t units = a.n * 2 * a.cache.kv_heads;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((units * G + kThreads - 1) / kThreads));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl ? 1 : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, paged_q8_read_kernel<TO, G, WIDE>, a);
}

template <typename TO, bool WIDE>
cudaError_t read_group(const PagedQ8ReadArgs& a, cudaStream_t stream, bool pdl) {
  if (a.cache.hd <= 64) return launch_read<TO, 4, WIDE>(a, stream, pdl);
  if (a.cache.hd <= 128) return launch_read<TO, 8, WIDE>(a, stream, pdl);
  return launch_read<TO, 16, WIDE>(a, stream, pdl);
}

template <typename TO>
cudaError_t read_types(const PagedQ8ReadArgs& a, cudaStream_t stream, bool pdl) {
  const bool wide = (((uintptr_t)a.k_out | (uintptr_t)a.v_out) & 15) == 0 && (a.k_stride | a.v_stride) % 8 == 0;
  return wide ? read_group<TO, true>(a, stream, pdl) : read_group<TO, false>(a, stream, pdl);
}

}  // namespace

cudaError_t launch_paged_q8_append(const PagedQ8AppendArgs& a, cudaStream_t stream, bool pdl) {
  if (a.n <= 0) return cudaSuccess;
  switch (a.type) {
    case kF32: return append_in<float>(a, stream, pdl);
    case kF16: return append_in<__half>(a, stream, pdl);
    default: return append_in<__nv_bfloat16>(a, stream, pdl);
  }
}

cudaError_t launch_paged_q8_read(const PagedQ8ReadArgs& a, cudaStream_t stream, bool pdl) {
  if (a.n <= 0) return cudaSuccess;
  switch (a.type) {
    case kF32: return read_types<float>(a, stream, pdl);
    case kF16: return read_types<__half>(a, stream, pdl);
    default: return read_types<__nv_bfloat16>(a, stream, pdl);
  }
}

}  // namespace dn
