// An 8-bit paged cache written and read back (dn_paged_q8_append,
// dn_paged_q8_read).
//
// Append: the head norm and the rotation of paged_append.cu in f32, then a
// row of hd values becomes int8: scale = max |x| / 127,
// q = round_half_away(x (1 / scale)). Read: q scale.
//
// Bytes-bound: every value is read and written once. As in paged_append.cu a
// head belongs to a group of G lanes and a lane holds two runs of V values, the
// halves of a rotation pair, so the rotation needs no exchange; the row's largest
// magnitude is one more shuffle reduction of the group. What a lane waits for is a
// chain, position, page and turns, store: for long prompts a group has four heads
// (two of f32) in flight over it.
// Measured: 16384 tokens of 32 + 8 + 8 heads of 128 bf16 values appended in 95 us
// (4.0 TB/s in and out; one head a group 107), their keys and values read back in
// 26 us (3.9 TB/s); 8000 tokens of 16 + 8 + 8 heads from f32 in 45 us.
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

// NaN where either is one.
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

// quant_q8_elem of a row's own values: |x| inv is at most 127 and a rounding, and
// finite, so nothing is left to clamp.
template <int V>
__device__ __forceinline__ void store_q8(int8_t* p, const float (&x)[V], float inv) {
  int q[V];
#pragma unroll
  for (int e = 0; e < V; e++) {
    const float t = __fmul_rn(x[e], inv);
    q[e] = __float2int_rz(__fadd_rn(t, copysignf(0.5f, t)));
  }
  if constexpr (V == 8) {
    auto four = [&](int e) {
      return __byte_perm(__byte_perm(q[e], q[e + 1], 0x0040), __byte_perm(q[e + 2], q[e + 3], 0x0040), 0x5410);
    };
    *reinterpret_cast<uint2*>(p) = make_uint2(four(0), four(4));
  } else {
#pragma unroll
    for (int e = 0; e < V; e++) p[e] = (int8_t)q[e];
  }
}

// A run of V elements as it was read: 16 bytes at a time, or the one element.
template <typename T, int V>
struct Run {
  static constexpr int kWords = V * (int)sizeof(T) / 16;
  uint4 w[kWords];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < kWords; i++) w[i] = make_uint4(0, 0, 0, 0);
  }
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < kWords; i++) w[i] = __ldcs(reinterpret_cast<const uint4*>(p) + i);
  }
  __device__ __forceinline__ void unpack(float (&x)[V]) const {
#pragma unroll
    for (int i = 0; i < kWords; i++) {
      T e[16 / sizeof(T)];
      memcpy(e, &w[i], 16);
#pragma unroll
      for (int k = 0; k < (int)(16 / sizeof(T)); k++) x[i * (16 / (int)sizeof(T)) + k] = to_f32<T>(e[k]);
    }
  }
};
template <typename T>
struct Run<T, 1> {
  float x0;
  __device__ __forceinline__ void clear() { x0 = 0.0f; }
  __device__ __forceinline__ void load(const T* p) { x0 = to_f32<T>(*p); }
  __device__ __forceinline__ void unpack(float (&x)[1]) const { x[0] = x0; }
};

// U heads of one kind (queries, keys or values) of a token to a group, which U
// divides.
template <typename TI, typename TO, int V, int G, int ITER, int U>
__global__ void __launch_bounds__(kThreads, U == 1 ? 4 : U == 2 ? 3 : 2) paged_q8_append_kernel(const __grid_constant__ PagedQ8AppendArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  const int hd = (int)a.cache.hd, q_units = (int)a.heads / U, kv_units = (int)a.cache.kv_heads / U;
  const uint32_t per_token = (uint32_t)(q_units + 2 * kv_units), unit = blockIdx.x * (kThreads / G) + threadIdx.x / G;
  const uint32_t t = unit / per_token;  // units fit 31 bits
  if (t >= a.n) return;                 // whole groups leave together
  // What follows hangs on these: first of all.
  const int pos = a.pos[t], seq = a.seq[t];
  const int lane = threadIdx.x % G, j = (int)(unit - t * per_token);
  const unsigned group = G == 32 ? 0xffffffffu : ((1u << G) - 1) << (threadIdx.x % 32 / G * G);
  const bool query = j < q_units, value = j >= q_units + kv_units;
  const int head = (query ? j : value ? j - q_units - kv_units : j - q_units) * U;
  const TI* src = (query   ? static_cast<const TI*>(a.q) + t * a.q_stride
                   : value ? static_cast<const TI*>(a.v) + t * a.v_stride
                           : static_cast<const TI*>(a.k) + t * a.k_stride) +
                  head * hd;

  // A slot's two runs: (s, s + rot / 2) for the rotated pairs, then the rest; of
  // a value, which does not turn, runs 2 s and 2 s + 1.
  const int rot = (int)a.rot, pairs = value ? 0 : rot / 2 / V, slots = hd / V / 2, turned = value ? 0 : rot;
  int first[ITER], second[ITER];
#pragma unroll
  for (int i = 0; i < ITER; i++) {
    const int s = lane + i * G;
    first[i] = s < pairs ? s * V : turned + 2 * (s - pairs) * V;
    second[i] = s < pairs ? first[i] + rot / 2 : first[i] + V;
  }
  Run<TI, V> x[U][ITER], y[U][ITER];
#pragma unroll
  for (int u = 0; u < U; u++)
#pragma unroll
    for (int i = 0; i < ITER; i++) {
      x[u][i].clear();
      y[u][i].clear();
      if (lane + i * G >= slots) continue;
      x[u][i].load(src + u * hd + first[i]);
      y[u][i].load(src + u * hd + second[i]);
    }
  // The token's turns, beside its page.
  const bool turns = pos >= 0 && pos < a.rope_rows;
  float c[ITER][V], n[ITER][V];
  const float* table = a.rope + (int64_t)pos * rot;
#pragma unroll
  for (int i = 0; i < ITER; i++) {
    if (!turns || lane + i * G >= pairs) continue;
    load_run<float, V>(table + first[i], c[i]);
    load_run<float, V>(table + rot / 2 + first[i], n[i]);
  }
  int slot = 0;
  const int64_t page = rot > 0 && !turns ? -1 : page_of(a.cache, seq, pos, slot);
  TO* out = static_cast<TO*>(a.q_out) + t * a.q_out_stride + head * hd;
  if (page < 0) {  // the whole group
    const float zero[V] = {};
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
      for (int i = 0; i < ITER; i++)
        if (query && lane + i * G < slots) {
          store_run<TO, V>(out + u * hd + first[i], zero);
          store_run<TO, V>(out + u * hd + second[i], zero);
        }
    return;
  }
  const float* w = query ? a.q_norm : value ? nullptr : a.k_norm;
  // Head u in f32, normalized and turned.
  auto head_of = [&](int u, float(&p)[ITER][V], float(&q)[ITER][V]) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < ITER; i++) {
      x[u][i].unpack(p[i]);
      y[u][i].unpack(q[i]);
    }
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
#pragma unroll
    for (int i = 0; i < ITER; i++) {
      if (lane + i * G >= pairs) continue;
#pragma unroll
      for (int e = 0; e < V; e++) {
        const float f = p[i][e], g = q[i][e];
        p[i][e] = f * c[i][e] - g * n[i][e];
        q[i][e] = g * c[i][e] + f * n[i][e];
      }
    }
  };
  if (query) {
#pragma unroll
    for (int u = 0; u < U; u++) {
      float p[ITER][V], q[ITER][V];
      head_of(u, p, q);
#pragma unroll
      for (int i = 0; i < ITER; i++)
        if (lane + i * G < slots) {
          store_run<TO, V>(out + u * hd + first[i], p[i]);
          store_run<TO, V>(out + u * hd + second[i], q[i]);
        }
    }
    return;
  }
  const int page_size = (int)a.cache.page_size;
  const int64_t row = (int64_t)head * page_size + slot;
  int8_t* dst = (value ? a.cache.values : a.cache.keys) + page * a.cache.page_stride + row * hd;
  float* dst_scale = (value ? a.cache.value_scales : a.cache.key_scales) + page * a.cache.scale_stride + row;
#pragma unroll
  for (int u = 0; u < U; u++) {
    float p[ITER][V], q[ITER][V];
    head_of(u, p, q);
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < ITER; i++)
#pragma unroll
      for (int e = 0; e < V; e++) amax = max_nan(amax, max_nan(fabsf(p[i][e]), fabsf(q[i][e])));
#pragma unroll
    for (int off = G / 2; off >= 1; off >>= 1) amax = max_nan(amax, __shfl_xor_sync(group, amax, off));
    float scale, inv;
    q8_scale(amax, scale, inv);
    if (scale < 1.17549435e-38f) scale = inv = 0.0f;  // 1 / scale would overflow
    const bool bad = !(amax < INFINITY);
    if (lane == 0) dst_scale[u * page_size] = bad ? NAN : scale;
#pragma unroll
    for (int i = 0; i < ITER; i++) {
      if (lane + i * G >= slots) continue;
      if (bad)
#pragma unroll
        for (int e = 0; e < V; e++) p[i][e] = q[i][e] = 0.0f;
      int8_t* to = dst + (int64_t)u * page_size * hd;
      store_q8<V>(to + first[i], p[i], bad ? 0.0f : inv);
      store_q8<V>(to + second[i], q[i], bad ? 0.0f : inv);
    }
  }
}

template <typename TI, typename TO, int V, int G, int ITER, int U>
cudaError_t launch_units(const PagedQ8AppendArgs& a, cudaStream_t stream, bool pdl) {
  const int64_t units = a.n * ((a.heads + 2 * a.cache.kv_heads) / U);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((units * G + kThreads - 1) / kThreads));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl ? 1 : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, paged_q8_append_kernel<TI, TO, V, G, ITER, U>, a);
}

template <typename TI, typename TO, int G>
cudaError_t launch_append(const PagedQ8AppendArgs& a, cudaStream_t stream, bool pdl) {
  // Several heads a group, where that leaves every SM its 2048 threads and the
  // groups of a warp queries or none: else one head (12 + 4 + 4 heads of 96, 16384
  // tokens: 52 us with one, 76 with four).
  constexpr int U = sizeof(TI) == 4 ? 2 : 4;
  const int64_t threads = a.n * (a.heads + 2 * a.cache.kv_heads) * G;
  return a.heads % (U * 32 / G) == 0 && a.cache.kv_heads % U == 0 && threads >= (int64_t)U * 148 * 2048
             ? launch_units<TI, TO, 8, G, 1, U>(a, stream, pdl)
             : launch_units<TI, TO, 8, G, 1, 1>(a, stream, pdl);
}

template <typename TI, typename TO>
cudaError_t append_types(const PagedQ8AppendArgs& a, cudaStream_t stream, bool pdl) {
  // Runs of 8 values where sizes, strides and addresses allow 16-byte
  // accesses of each type; else one value at a time.
  const uintptr_t addr = (uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.q_out | (uintptr_t)a.rope |
                         (uintptr_t)a.q_norm | (uintptr_t)a.k_norm;
  const int64_t step = a.q_stride | a.k_stride | a.v_stride | a.q_out_stride | a.rot / 2;
  if ((addr & 15) != 0 || step % 8 != 0) return launch_units<TI, TO, 1, 32, 4, 1>(a, stream, pdl);
  if (a.cache.hd <= 64) return launch_append<TI, TO, 4>(a, stream, pdl);
  if (a.cache.hd <= 128) return launch_append<TI, TO, 8>(a, stream, pdl);
  return launch_append<TI, TO, 16>(a, stream, pdl);
}

template <typename TI>
cudaError_t append_in(const PagedQ8AppendArgs& a, cudaStream_t stream, bool pdl) {
  switch (a.out_type) {
    case kF32: return append_types<TI, float>(a, stream, pdl);
    case kF16: return append_types<TI, __half>(a, stream, pdl);
    default: return append_types<TI, __nv_bfloat16>(a, stream, pdl);
  }
}

// 16 values to a lane, U rows of a token (its keys, then its values) to a group
// of G lanes. WIDE: the outputs take 16-byte accesses.
template <typename TO, int G, bool WIDE, int U>
__global__ void __launch_bounds__(kThreads) paged_q8_read_kernel(const __grid_constant__ PagedQ8ReadArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  const int hd = (int)a.cache.hd, kvh = (int)a.cache.kv_heads, lane = threadIdx.x % G;
  const uint32_t per_token = (uint32_t)(2 * kvh + U - 1) / U;
  const int64_t unit = (int64_t)blockIdx.x * (kThreads / G) + threadIdx.x / G;
  if (unit >= a.n * per_token || lane * 16 >= hd) return;
  const int64_t t = (uint32_t)unit / per_token;  // units fit 31 bits
  const int h0 = (int)((uint32_t)unit % per_token) * U;
  int slot = 0;
  const int64_t page = page_of(a.cache, a.seq[t], a.pos[t], slot);
  int4 raw[U];
  float scale[U];
#pragma unroll
  for (int u = 0; u < U; u++) {
    raw[u] = make_int4(0, 0, 0, 0);
    scale[u] = 0.0f;
    const int h = h0 + u;
    const bool value = h >= kvh;
    if (page < 0 || h >= 2 * kvh || (value ? a.v_out : a.k_out) == nullptr) continue;
    const int64_t row = (int64_t)(value ? h - kvh : h) * a.cache.page_size + slot;
    raw[u] = __ldcs(reinterpret_cast<const int4*>((value ? a.cache.values : a.cache.keys) + page * a.cache.page_stride +
                                                  row * hd + lane * 16));
    scale[u] = (value ? a.cache.value_scales : a.cache.key_scales)[page * a.cache.scale_stride + row];
  }
#pragma unroll
  for (int u = 0; u < U; u++) {
    const int h = h0 + u;
    const bool value = h >= kvh;
    void* to = value ? a.v_out : a.k_out;
    if (h >= 2 * kvh || to == nullptr) continue;
    TO* out = static_cast<TO*>(to) + t * (value ? a.v_stride : a.k_stride) + (int64_t)(value ? h - kvh : h) * hd + lane * 16;
    int8_t q[16];
    memcpy(q, &raw[u], 16);
    float x[16];
#pragma unroll
    for (int e = 0; e < 16; e++) x[e] = __fmul_rn((float)q[e], scale[u]);
    if constexpr (WIDE) {
      store_run<TO, 16>(out, x);
    } else {
#pragma unroll
      for (int e = 0; e < 16; e++) out[e] = from_f32<TO>(x[e]);
    }
  }
}

template <typename TO, int G, bool WIDE, int U>
cudaError_t launch_rows(const PagedQ8ReadArgs& a, cudaStream_t stream, bool pdl) {
  const int64_t units = a.n * ((2 * a.cache.kv_heads + U - 1) / U);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((units * G + kThreads - 1) / kThreads));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl ? 1 : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, paged_q8_read_kernel<TO, G, WIDE, U>, a);
}

template <typename TO, int G, bool WIDE>
cudaError_t launch_read(const PagedQ8ReadArgs& a, cudaStream_t stream, bool pdl) {
  // Four rows a group, once that leaves every SM its 2048 threads twice.
  return a.n * 2 * a.cache.kv_heads * G >= (int64_t)8 * 148 * 2048 ? launch_rows<TO, G, WIDE, 4>(a, stream, pdl)
                                                                   : launch_rows<TO, G, WIDE, 1>(a, stream, pdl);
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
