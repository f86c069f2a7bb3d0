// qw_distill.cu -- distillation from a teacher's top logits, loss and gradient:
// with p = softmax(t / T) over a row's valid teacher entries (ids below V) and
// q = softmax(z / T) over its V logits,
//   loss = w T^2 sum_j p_j (log p_j - log q_{i_j}),   dz = w T (q - sum_j p_j e_{i_j}).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../include/qw_qmm.h"
#include "qw_internal.h"
#include "qw_ptx.cuh"

namespace qw {

namespace {

constexpr int kThreads = 512;
constexpr int kTopMax = 1024;  // teacher entries per row

template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f32(float v) { return v; }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ __half from_f32(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ float from_f32(float v) { return v; }

__device__ __forceinline__ float load_value(const DistillArgs& p, int64_t i) {
  if (p.values_dtype == QW_F16) return to_f32(reinterpret_cast<const __half*>(p.values)[i]);
  if (p.values_dtype == QW_BF16) return to_f32(reinterpret_cast<const __nv_bfloat16*>(p.values)[i]);
  return reinterpret_cast<const float*>(p.values)[i];
}

template <typename F>
__device__ float block_reduce(float v, float* red, F f) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if (threadIdx.x % 32 == 0) red[threadIdx.x / 32] = v;
  __syncthreads();
  v = red[0];
  for (int i = 1; i < kThreads / 32; ++i) v = f(v, red[i]);
  return v;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) distill_rows_kernel(DistillArgs p) {
  __shared__ float red[kThreads / 32];
  __shared__ float prob[kTopMax];
  __shared__ uint32_t ids[kTopMax];
  const int64_t m = blockIdx.x;
  const int64_t V = p.V;
  const T* z = reinterpret_cast<const T*>(p.logits) + m * V;
  T* dz = p.dlogits ? reinterpret_cast<T*>(p.dlogits) + m * V : nullptr;
  const float w = p.weights ? p.weights[m] : 1.f;
  const float temp = p.temperature ? *p.temperature : 1.f;
  const float inv = 1.f / temp;
  const int tid = threadIdx.x;
  auto mx = [](float a, float b) { return fmaxf(a, b); };
  auto add = [](float a, float b) { return a + b; };
  // teacher
  float tmax = -INFINITY;
  for (int j = tid; j < p.k; j += kThreads) {
    const uint32_t id = p.idx[m * p.k + j];
    ids[j] = (int64_t)id < V ? id : 0xFFFFFFFFu;
    prob[j] = (int64_t)id < V ? load_value(p, m * p.k + j) : -INFINITY;
    tmax = fmaxf(tmax, prob[j]);
  }
  tmax = block_reduce(tmax, red, mx);
  float tsum = 0.f;
  for (int j = tid; j < p.k; j += kThreads) tsum += prob[j] == -INFINITY ? 0.f : expf((prob[j] - tmax) * inv);
  tsum = block_reduce(tsum, red, add);
  if (w == 0.f || tmax == -INFINITY) {  // no weight, or nothing to learn from
    if (tid == 0) p.loss[m] = 0.f;
    if (dz)
      for (int64_t v = tid; v < V; v += kThreads) dz[v] = from_f32<T>(0.f);
    return;
  }
  // student
  float zmax = -INFINITY;
  for (int64_t v = tid; v < V; v += kThreads) zmax = fmaxf(zmax, to_f32(z[v]));
  zmax = block_reduce(zmax, red, mx);
  float zsum = 0.f;
  for (int64_t v = tid; v < V; v += kThreads) {
    const float x = to_f32(z[v]);
    zsum += x == -INFINITY ? 0.f : expf((x - zmax) * inv);
  }
  zsum = block_reduce(zsum, red, add);
  const float shift = (tmax - zmax) * inv + (logf(tsum) - logf(zsum));  // log-normaliser of p over that of q
  float part = 0.f;
  for (int j = tid; j < p.k; j += kThreads) {
    const float t = prob[j];
    const float pj = t == -INFINITY ? 0.f : expf((t - tmax) * inv) / tsum;
    if (pj > 0.f) {
      const float zj = to_f32(z[ids[j]]);
      part += zj == -INFINITY ? INFINITY : pj * ((t - zj) * inv - shift);
    }
    prob[j] = pj;
  }
  part = block_reduce(part, red, add);
  if (tid == 0) p.loss[m] = w * temp * temp * part;
  if (!dz) return;
  const float c = w * temp;
  for (int64_t v = tid; v < V; v += kThreads) {
    const float x = to_f32(z[v]);
    float q = x == -INFINITY ? 0.f : expf((x - zmax) * inv) / zsum;
    for (int j = 0; j < p.k; ++j)
      if (ids[j] == (uint32_t)v) q -= prob[j];
    dz[v] = from_f32<T>(c * q);
  }
}

}  // namespace

int distill_max_top() { return kTopMax; }

cudaError_t launch_distill(const DistillArgs& p, cudaStream_t stream) {
  if (p.M == 0) return cudaSuccess;
  if (p.dtype == QW_F16) distill_rows_kernel<__half><<<(unsigned)p.M, kThreads, 0, stream>>>(p);
  else if (p.dtype == QW_BF16) distill_rows_kernel<__nv_bfloat16><<<(unsigned)p.M, kThreads, 0, stream>>>(p);
  else distill_rows_kernel<float><<<(unsigned)p.M, kThreads, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace qw
