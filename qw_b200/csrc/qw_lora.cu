// qw_lora.cu -- low-rank adapters beside a quantized projection, many at once:
// row m of x takes adapter idx[m] (none when idx[m] >= L),
//   y[m] += s (x[m] A^T) B^T,            A [R, K], B [N, R], s the adapter's scale
// and the gradient of that term:
//   h = s x A^T, g = s dy B, dA = g^T x, dB = dy^T h, dx = g A
// with the sums over the rows of each adapter.
#include <cuda_fp16.h>

#include "qw_internal.h"
#include "qw_ptx.cuh"

namespace qw {

namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ int64_t adapter_of(const LoraArgs& p, int64_t m) {
  const uint32_t a = p.idx ? p.idx[m] : 0u;
  return (int64_t)a < p.L ? (int64_t)a : -1;
}

// out[m][r] = s sum_i v[m][i] W[r][i] (TRANS: W[i][r]) in fp32, zero without an adapter.
template <bool TRANS>
__global__ void __launch_bounds__(kThreads) shrink_rows_kernel(LoraArgs p, const __half* v, int64_t ld, int64_t len,
                                                               const __half* w, float* out) {
  const int64_t m = blockIdx.x;
  const int64_t a = adapter_of(p, m);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const __half* row = v + m * ld;
  for (int r = warp; r < p.R; r += kThreads / 32) {
    float acc = 0.f;
    if (a >= 0) {
      const __half* wa = w + a * len * p.R;
      for (int64_t i = lane; i < len; i += 32)
        acc += __half2float(row[i]) * __half2float(TRANS ? wa[i * p.R + r] : wa[r * len + i]);
#pragma unroll
      for (int o = 16; o; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
      acc *= p.scales ? p.scales[a] : 1.f;
    }
    if (lane == 0) out[m * p.R + r] = acc;
  }
}

__global__ void __launch_bounds__(kThreads) expand_rows_kernel(LoraArgs p, const float* y32, const float* h,
                                                               const __half* bias, __half* y) {
  const int64_t nb = (p.N + kThreads - 1) / kThreads;
  const int64_t m = blockIdx.x / nb;
  const int64_t n = (blockIdx.x % nb) * kThreads + threadIdx.x;
  if (n >= p.N) return;
  const int64_t a = adapter_of(p, m);
  float acc = y32[m * p.N + n];
  if (a >= 0) {
    const __half* b = reinterpret_cast<const __half*>(p.b) + (a * p.N + n) * p.R;
    for (int r = 0; r < p.R; ++r) acc += h[m * p.R + r] * __half2float(b[r]);
  }
  if (bias) acc += __half2float(bias[n]);
  y[m * p.N + n] = __float2half_rn(acc);
}

__global__ void __launch_bounds__(kThreads) dx_rows_kernel(LoraArgs p, const float* g, __half* dx, bool add) {
  const int64_t nb = (p.K + kThreads - 1) / kThreads;
  const int64_t m = blockIdx.x / nb;
  const int64_t k = (blockIdx.x % nb) * kThreads + threadIdx.x;
  if (k >= p.K) return;
  const int64_t a = adapter_of(p, m);
  if (a < 0 && add) return;
  float acc = add ? __half2float(dx[m * p.K + k]) : 0.f;
  if (a >= 0) {
    const __half* w = reinterpret_cast<const __half*>(p.a) + a * p.R * p.K + k;
    for (int r = 0; r < p.R; ++r) acc += g[m * p.R + r] * __half2float(w[r * p.K]);
  }
  dx[m * p.K + k] = __float2half_rn(acc);
}

// out[a][r][i] (TRANS: out[a][i][r]) = sum over the adapter's rows of t[m][r] v[m][i].
template <bool TRANS>
__global__ void __launch_bounds__(kThreads) outer_rows_kernel(LoraArgs p, const __half* v, int64_t ld, int64_t len,
                                                              const float* t, float* out) {
  const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  const int r = blockIdx.y;
  const int64_t a = blockIdx.z;
  if (i >= len) return;
  float acc = 0.f;
  for (int64_t m = 0; m < p.M; ++m)
    if (adapter_of(p, m) == a) acc += t[m * p.R + r] * __half2float(v[m * ld + i]);
  out[TRANS ? (a * len + i) * p.R + r : (a * p.R + r) * len + i] = acc;
}

}  // namespace

size_t lora_forward_bytes(int64_t M, int64_t N, int64_t R) {
  return (size_t)M * R * sizeof(float) + (size_t)M * N * sizeof(float);
}

cudaError_t launch_lora_shrink(const LoraArgs& p, void* ws, cudaStream_t stream) {
  shrink_rows_kernel<false><<<(unsigned)p.M, kThreads, 0, stream>>>(p, (const __half*)p.x, p.x_ld, p.K,
                                                                    (const __half*)p.a, (float*)ws);
  return cudaGetLastError();
}

float* lora_forward_product(const LoraArgs& p, void* ws) { return (float*)ws + p.M * p.R; }

cudaError_t launch_lora_expand(const LoraArgs& p, void* ws, const void* bias, void* y, cudaStream_t stream) {
  const dim3 grid((unsigned)((p.N + kThreads - 1) / kThreads * p.M));
  expand_rows_kernel<<<grid, kThreads, 0, stream>>>(p, lora_forward_product(p, ws), (const float*)ws,
                                                    (const __half*)bias, (__half*)y);
  return cudaGetLastError();
}

size_t lora_backward_bytes(int64_t M, int64_t N, int64_t K, int64_t R, int64_t L, int sm_count) {
  return (size_t)M * R * 2 * sizeof(float);
}

cudaError_t launch_lora_backward(const LoraArgs& p, const LoraGrads& g, void* ws, int sm_count, cudaStream_t stream) {
  float* h = (float*)ws;
  float* gg = h + p.M * p.R;
  const __half* x = (const __half*)p.x;
  const __half* dy = (const __half*)g.dy;
  if (p.M) {
    shrink_rows_kernel<false><<<(unsigned)p.M, kThreads, 0, stream>>>(p, x, p.x_ld, p.K, (const __half*)p.a, h);
    shrink_rows_kernel<true><<<(unsigned)p.M, kThreads, 0, stream>>>(p, dy, g.dy_ld, p.N, (const __half*)p.b, gg);
  }
  const unsigned kb = (unsigned)((p.K + kThreads - 1) / kThreads), nb = (unsigned)((p.N + kThreads - 1) / kThreads);
  if (g.dx && p.M) dx_rows_kernel<<<(unsigned)(kb * p.M), kThreads, 0, stream>>>(p, gg, (__half*)g.dx, g.add_dx);
  if (g.da && kb)
    outer_rows_kernel<false><<<dim3(kb, p.R, (unsigned)p.L), kThreads, 0, stream>>>(p, x, p.x_ld, p.K, gg, g.da);
  if (g.db && nb)
    outer_rows_kernel<true><<<dim3(nb, p.R, (unsigned)p.L), kThreads, 0, stream>>>(p, dy, g.dy_ld, p.N, h, g.db);
  return cudaGetLastError();
}

}  // namespace qw
