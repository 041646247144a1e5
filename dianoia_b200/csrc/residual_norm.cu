// What stands between two blocks of a layer (dn_residual_norm): the norm after
// a block, its gate and residual scale, the residual add, the norm before the
// next block.
//
// Per row:  b = post y / sqrt(mean(y^2) + eps)  (or y),
//           x' = x + scale g b,  h = pre x' / sqrt(mean(x'^2) + eps),
// all in f32, each result rounded once.
//
// Bytes-bound: y and x in, x' and h out, once each; the two sums need the
// whole row, so a CTA keeps its row in registers between them (runs of 8
// values a thread, 16-byte accesses) and each sum costs one barrier.
// Measured: 16384 rows of 4096, bf16 over an f32 stream, with a post norm and a
// gate in 132 us (6.1 TB/s in and out; a copy does 6.5), 8000 rows of 2048 in f32
// 47 us; 16 rows of 2048 in 2.7 us.
#include "dn_common.cuh"
#include "dn_launch.h"
#include "elem.cuh"
#include "kernel_smem.h"

namespace dn {
namespace {

constexpr int V = 8;
constexpr int kMaxThreads = 512;

// The sum over the block, the same in every thread; `red` has a float a warp,
// and is not in use by another sum.
__device__ __forceinline__ float block_sum(float s, float* red) {
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
  if (threadIdx.x % 32 == 0) red[threadIdx.x / 32] = s;
  __syncthreads();
  const int warps = (int)blockDim.x / 32;
  s = (int)threadIdx.x % 32 < warps ? red[threadIdx.x % 32] : 0.0f;
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
  return s;
}

__device__ __forceinline__ float inv_rms(float sum, const ResidualNormArgs& a) {
  return 1.0f / sqrtf(sum / (float)a.cols + a.eps);
}

// A row to a CTA of up to THREADS threads, I runs of V values to a thread; rows,
// columns and addresses allow 16-byte accesses. BLOCKS: CTAs that an SM is to hold.
template <typename TY, typename TX, int I, int THREADS, int BLOCKS>
__global__ void __launch_bounds__(THREADS, BLOCKS) residual_norm_kernel(const __grid_constant__ ResidualNormArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  __shared__ float red[2][32];
  const int64_t row = blockIdx.x;
  const int cols = (int)a.cols, step = (int)blockDim.x * V, first = (int)threadIdx.x * V;
  const TY* y = static_cast<const TY*>(a.y) + row * a.y_stride;
  const TY* g = static_cast<const TY*>(a.gate) + row * a.gate_stride;
  const TX* x = static_cast<const TX*>(a.x) + row * a.x_stride;
  float b[I][V], s[I][V];
#pragma unroll
  for (int i = 0; i < I; i++) {
    const int at = first + i * step;
#pragma unroll
    for (int e = 0; e < V; e++) b[i][e] = s[i][e] = 0.0f;
    if (at < cols) {
      load_run<TY, V>(y + at, b[i]);
      load_run<TX, V>(x + at, s[i]);
    }
  }
  float r = 1.0f;
  if (a.post != nullptr) {
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < I; i++)
#pragma unroll
      for (int e = 0; e < V; e++) sum += b[i][e] * b[i][e];
    r = inv_rms(block_sum(sum, red[0]), a);
  }
  TX* x_out = static_cast<TX*>(a.x_out) + row * a.x_out_stride;
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < I; i++) {
    const int at = first + i * step;
    if (at >= cols) continue;
    float w[V];
    if (a.post != nullptr) {
      load_run<float, V>(a.post + at, w);
#pragma unroll
      for (int e = 0; e < V; e++) b[i][e] *= r * w[e];
    }
    if (a.gate != nullptr) {
      load_run<TY, V>(g + at, w);
#pragma unroll
      for (int e = 0; e < V; e++) b[i][e] *= w[e];
    }
#pragma unroll
    for (int e = 0; e < V; e++) {
      s[i][e] += a.scale * b[i][e];
      sum += s[i][e] * s[i][e];
    }
    store_run<TX, V>(x_out + at, s[i]);
  }
  if (a.pre == nullptr) return;
  r = inv_rms(block_sum(sum, red[1]), a);
  TY* h = static_cast<TY*>(a.h) + row * a.h_stride;
#pragma unroll
  for (int i = 0; i < I; i++) {
    const int at = first + i * step;
    float w[V] = {};
    if (at < cols) load_run<float, V>(a.pre + at, w);
#pragma unroll
    for (int e = 0; e < V; e++) s[i][e] *= r * w[e];
    if (a.h != nullptr && at < cols) store_run<TY, V>(h + at, s[i]);
    if (a.qa == nullptr) continue;
    // A block's 32 values lie in four lanes, all of them inside the row or none.
    float amax = 0.0f;
#pragma unroll
    for (int e = 0; e < V; e++) amax = fmaxf(amax, fabsf(s[i][e]));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    if (at >= cols) continue;
    float scale, inv;
    q8_scale(amax, scale, inv);
    int q[V];
#pragma unroll
    for (int e = 0; e < V; e++) q[e] = quant_q8_elem(s[i][e], inv);
    uint8_t* block = a.qa + row * a.qa_stride + at / kBlock * kQABytes;
    uint32_t* to = reinterpret_cast<uint32_t*>(block + at % kBlock);
    to[0] = pack4(q[0], q[1], q[2], q[3]);
    to[1] = pack4(q[4], q[5], q[6], q[7]);
    if (at % kBlock == 0) *reinterpret_cast<float*>(block + kBlock) = scale;
  }
}

// Any alignment, a value at a time; the row's x' stays in shared memory.
template <typename TY, typename TX>
__global__ void __launch_bounds__(kMaxThreads) residual_norm_any_kernel(const __grid_constant__ ResidualNormArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  extern __shared__ float s[];
  __shared__ float red[2][32];
  const int64_t row = blockIdx.x;
  const int cols = (int)a.cols, threads = (int)blockDim.x, tid = (int)threadIdx.x;
  const TY* y = static_cast<const TY*>(a.y) + row * a.y_stride;
  const TY* g = static_cast<const TY*>(a.gate) + row * a.gate_stride;
  const TX* x = static_cast<const TX*>(a.x) + row * a.x_stride;
  float r = 1.0f, sum = 0.0f;
  if (a.post != nullptr) {
    for (int at = tid; at < cols; at += threads) {
      const float v = to_f32<TY>(y[at]);
      sum += v * v;
    }
    r = inv_rms(block_sum(sum, red[0]), a);
  }
  TX* x_out = static_cast<TX*>(a.x_out) + row * a.x_out_stride;
  sum = 0.0f;
  for (int at = tid; at < cols; at += threads) {  // a thread's own values, from here on
    float b = to_f32<TY>(y[at]);
    if (a.post != nullptr) b *= r * a.post[at];
    if (a.gate != nullptr) b *= to_f32<TY>(g[at]);
    const float v = to_f32<TX>(x[at]) + a.scale * b;
    sum += v * v;
    s[at] = v;
    x_out[at] = from_f32<TX>(v);
  }
  if (a.pre == nullptr) return;
  r = inv_rms(block_sum(sum, red[1]), a);
  TY* h = static_cast<TY*>(a.h) + row * a.h_stride;
  for (int at = tid; at - tid % 32 < cols; at += threads) {
    const float v = at < cols ? s[at] * (r * a.pre[at]) : 0.0f;
    if (a.h != nullptr && at < cols) h[at] = from_f32<TY>(v);
    if (a.qa == nullptr) continue;  // cols % 32 == 0: whole warps hold whole blocks
    float amax = fabsf(v);
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, off));
    float scale, inv;
    q8_scale(amax, scale, inv);
    uint8_t* block = a.qa + row * a.qa_stride + at / kBlock * kQABytes;
    block[at % kBlock] = (uint8_t)(int8_t)quant_q8_elem(v, inv);
    if (at % kBlock == 0) *reinterpret_cast<float*>(block + kBlock) = scale;
  }
}

template <auto KERNEL>
cudaError_t launch_rows(const ResidualNormArgs& a, int threads, int smem, cudaStream_t stream, bool pdl) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)a.rows);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl ? 1 : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, KERNEL, a);
}

template <typename TY, typename TX>
cudaError_t launch_types(const ResidualNormArgs& a, cudaStream_t stream, bool pdl) {
  const uintptr_t addr = (uintptr_t)a.y | (uintptr_t)a.post | (uintptr_t)a.gate | (uintptr_t)a.x | (uintptr_t)a.x_out |
                         (uintptr_t)a.pre | (uintptr_t)a.h;
  const int64_t steps = a.y_stride | a.gate_stride | a.x_stride | a.x_out_stride | a.h_stride | a.cols;
  if ((addr & 15) != 0 || steps % V != 0) {
    if (cudaError_t e = allow_smem<residual_norm_any_kernel<TY, TX>>((int)kMaxResidualCols * 4); e != cudaSuccess)
      return e;
    const int threads = a.cols >= kMaxThreads ? kMaxThreads : (int)(a.cols + 31) / 32 * 32;
    return launch_rows<residual_norm_any_kernel<TY, TX>>(a, threads, (int)a.cols * 4, stream, pdl);
  }
  // Two runs a thread from 2048 values on, five CTAs of 256 threads to an SM: 16384
  // rows of 4096 values, bf16 over f32, in 134 us (148 with 512 threads of one run,
  // 144 where the compiler takes the registers of four CTAs). From 4096 on 512
  // threads: 8192 rows of 8192 in 130 us against 161.
  const int64_t runs = a.cols / V;
  auto threads = [&](int64_t i) { return (int)((runs + i - 1) / i + 31) / 32 * 32; };
  if (runs <= 256) return launch_rows<residual_norm_kernel<TY, TX, 1, 256, 1>>(a, threads(1), 0, stream, pdl);
  if (runs <= 512) return launch_rows<residual_norm_kernel<TY, TX, 2, 256, 5>>(a, threads(2), 0, stream, pdl);
  if (runs <= 1024) return launch_rows<residual_norm_kernel<TY, TX, 2, 512, 1>>(a, threads(2), 0, stream, pdl);
  if (runs <= 2048) return launch_rows<residual_norm_kernel<TY, TX, 4, 512, 1>>(a, threads(4), 0, stream, pdl);
  return launch_rows<residual_norm_kernel<TY, TX, 8, 512, 1>>(a, threads(8), 0, stream, pdl);
}

template <typename TY>
cudaError_t launch_in(const ResidualNormArgs& a, cudaStream_t stream, bool pdl) {
  switch (a.x_type) {
    case kF32: return launch_types<TY, float>(a, stream, pdl);
    case kF16: return launch_types<TY, __half>(a, stream, pdl);
    default: return launch_types<TY, __nv_bfloat16>(a, stream, pdl);
  }
}

}  // namespace

cudaError_t launch_residual_norm(const ResidualNormArgs& a, cudaStream_t stream, bool pdl) {
  if (a.rows <= 0 || a.cols <= 0) return cudaSuccess;
  switch (a.type) {
    case kF32: return launch_in<float>(a, stream, pdl);
    case kF16: return launch_in<__half>(a, stream, pdl);
    default: return launch_in<__nv_bfloat16>(a, stream, pdl);
  }
}

}  // namespace dn
