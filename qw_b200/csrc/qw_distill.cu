// qw_distill.cu -- distillation from a teacher's top logits, loss and gradient:
// with p = softmax(t / T) over a row's valid teacher entries (ids below V) and
// q = softmax(z / T) over its V logits,
//   loss = w T^2 sum_j p_j (log p_j - log q_{i_j}),   dz = w T (q - sum_j p_j e_{i_j}).
//
// HBM-bound: z has to be read once and dz written once.  q needs the whole
// row's maximum and sum before the first dz can leave, so a row is held on chip
// in between: a thread-block cluster of up to 8 CTAs per row, each CTA a
// contiguous share of it in registers (kVec 16-byte vectors a thread, 64 KB a
// CTA of 512 threads, two CTAs an SM, so that one row's loads run under
// another's stores).  What a share has beyond that (rows of more than 512 KB)
// is read a second time, from L2.
//   1. every thread issues its loads of z; while they fly, the teacher's k
//      entries are read, their softmax taken by each warp alone, and the z they
//      point at gathered;
//   2. maximum and sum of exponentials by thread, warp and CTA; each CTA then
//      stores (maximum, sum, its part of sum_j p_j (t_j - z_j)) into every CTA
//      of the cluster, and one cluster barrier later every thread has the row's;
//   3. dz = w T q from the registers, then the columns the teacher names are
//      written again by the CTA that owns them, behind a barrier.
// Sums and exponentials are fp32 (ex2.approx, relative error 2^-22); the loss,
// a difference of two log-normalisers, is put together in fp64 from them.
// Rows start at any element: up to 15 bytes before the first 16-byte boundary
// and after the last are single elements of rank 0's and the last rank's
// threads.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../include/qw_qmm.h"
#include "qw_internal.h"
#include "qw_ptx.cuh"

namespace qw {

namespace {

constexpr int kTopMax = 1024;    // teacher entries per row
constexpr int kVec = 8;          // 16-byte vectors a thread holds
constexpr int kClusterMax = 8;   // CTAs per row
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f32(float v) { return v; }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ __half from_f32(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ float from_f32(float v) { return v; }

// The elements of a 16-byte vector as floats, and back.
template <typename T>
struct Vec {
  static constexpr int N = 16 / (int)sizeof(T);
  static __device__ __forceinline__ void load(const uint4& v, float (&f)[N]);
  static __device__ __forceinline__ uint4 pack(const float (&f)[N]);
};
template <>
__device__ __forceinline__ void Vec<__half>::load(const uint4& v, float (&f)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    f[2 * i] = t.x;
    f[2 * i + 1] = t.y;
  }
}
template <>
__device__ __forceinline__ uint4 Vec<__half>::pack(const float (&f)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
template <>
__device__ __forceinline__ void Vec<__nv_bfloat16>::load(const uint4& v, float (&f)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(w[i] << 16);
    f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
template <>
__device__ __forceinline__ uint4 Vec<__nv_bfloat16>::pack(const float (&f)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
template <>
__device__ __forceinline__ void Vec<float>::load(const uint4& v, float (&f)[4]) {
  f[0] = __uint_as_float(v.x), f[1] = __uint_as_float(v.y), f[2] = __uint_as_float(v.z), f[3] = __uint_as_float(v.w);
}
template <>
__device__ __forceinline__ uint4 Vec<float>::pack(const float (&f)[4]) {
  return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
}

__device__ __forceinline__ float load_value(const DistillArgs& p, int64_t i) {
  if (p.values_dtype == QW_F16) return to_f32(reinterpret_cast<const __half*>(p.values)[i]);
  if (p.values_dtype == QW_BF16) return to_f32(reinterpret_cast<const __nv_bfloat16*>(p.values)[i]);
  return reinterpret_cast<const float*>(p.values)[i];
}

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
template <typename F>
__device__ __forceinline__ F warp_sum(F v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// A maximum to subtract: that of values which are all -inf counts as 0.
__device__ __forceinline__ float finite_max(float m) { return m == -INFINITY ? 0.f : m; }

// What a CTA tells its cluster of its share: largest logit, sum of
// exponentials relative to it, and sum_j p_j (t_j - z_j) / T of its columns.
struct Share {
  double gap;
  float max, sum;
};

template <typename T, int TH>
__global__ void __launch_bounds__(TH, 1024 / TH) distill_rows_kernel(const DistillArgs p) {
  using VT = Vec<T>;
  __shared__ uint32_t ids[kTopMax];
  __shared__ float tval[kTopMax];
  __shared__ float zval[kTopMax];  // the logit each entry of this CTA's columns points at
  __shared__ Share warp_share[TH / 32];
  __shared__ Share shares[kClusterMax];
  uint32_t rank, C;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(C));
  const int tid = threadIdx.x, lane = tid % 32;
  const int64_t m = blockIdx.x / C;
  const int64_t V = p.V;
  const T* z = reinterpret_cast<const T*>(p.logits) + m * V;
  T* dz = p.dlogits ? reinterpret_cast<T*>(p.dlogits) + m * V : nullptr;
  const int off = (int)((16 - (reinterpret_cast<uintptr_t>(z) & 15)) & 15) / (int)sizeof(T);
  const int head = off < V ? off : (int)V;
  const int nv = (int)((V - head) / VT::N);
  const int tail = (int)(V - head - (int64_t)nv * VT::N);
  const int v0 = (int)((int64_t)nv * rank / C), v1 = (int)((int64_t)nv * (rank + 1) / C);
  const uint32_t e0 = rank == 0 ? 0u : (uint32_t)(head + v0 * VT::N);
  const uint32_t e1 = rank == C - 1 ? (uint32_t)V : (uint32_t)(head + v1 * VT::N);
  const uint4* zv = reinterpret_cast<const uint4*>(z + head);
  // the single element of this thread, if it has one
  int64_t edge = -1;
  if (rank == 0 && tid < head) edge = tid;
  if (rank == C - 1 && tid >= 32 && tid < 32 + tail) edge = V - tail + (tid - 32);

  uint4 d[kVec];
#pragma unroll
  for (int e = 0; e < kVec; ++e) {
    const int i = v0 + tid + e * TH;
    if (i < v1) d[e] = __ldcg(zv + i);
  }
  const float ze = edge >= 0 ? to_f32(z[edge]) : -INFINITY;

  const float w = p.weights ? p.weights[m] : 1.f;
  const float temp = p.temperature ? *p.temperature : 1.f;
  const float inv = 1.f / temp;
  const float c = inv * kLog2e;
  for (int j = tid; j < p.k; j += TH) {
    const uint32_t id = p.idx[m * p.k + j];
    const bool ok = (int64_t)id < V;
    ids[j] = ok ? id : 0xFFFFFFFFu;
    tval[j] = ok ? load_value(p, m * p.k + j) : -INFINITY;
  }
  __syncthreads();
  float tmax = -INFINITY, tsum = 0.f;
  for (int j = lane; j < p.k; j += 32) tmax = fmaxf(tmax, tval[j]);
  tmax = warp_max(tmax);
  const bool svec = dz && (((reinterpret_cast<uintptr_t>(z) ^ reinterpret_cast<uintptr_t>(dz)) & 15) == 0);
  auto store = [&](int i, const float (&f)[VT::N]) {
    if (svec) {
      reinterpret_cast<uint4*>(dz + head)[i] = VT::pack(f);
    } else {
#pragma unroll
      for (int q = 0; q < VT::N; ++q) dz[head + (int64_t)i * VT::N + q] = from_f32<T>(f[q]);
    }
  };
  if (w == 0.f || tmax == -INFINITY) {  // no weight, or nothing to learn from (the whole cluster takes this branch)
    if (rank == 0 && tid == 0) p.loss[m] = 0.f;
    if (dz) {
      const float zero[VT::N] = {};
      for (int i = v0 + tid; i < v1; i += TH) store(i, zero);
      if (edge >= 0) dz[edge] = from_f32<T>(0.f);
    }
    return;
  }
  for (int j = lane; j < p.k; j += 32) tsum += ex2((tval[j] - tmax) * c);
  tsum = warp_sum(tsum);
  double gap = 0.0;
  for (int j = tid; j < p.k; j += TH) {
    if (ids[j] >= e0 && ids[j] < e1) {
      const float zj = to_f32(z[ids[j]]);
      const float pj = ex2((tval[j] - tmax) * c) / tsum;
      zval[j] = zj;
      if (pj > 0.f) gap += zj == -INFINITY ? (double)INFINITY : (double)pj * ((double)tval[j] - (double)zj);
    }
  }

  // maximum and sum of this thread's, warp's, CTA's and cluster's logits
  float mx = ze;
#pragma unroll
  for (int e = 0; e < kVec; ++e) {
    if (v0 + tid + e * TH < v1) {
      float f[VT::N];
      VT::load(d[e], f);
#pragma unroll
      for (int q = 0; q < VT::N; ++q) mx = fmaxf(mx, f[q]);
    }
  }
  for (int i = v0 + tid + kVec * TH; i < v1; i += TH) {
    float f[VT::N];
    VT::load(__ldcg(zv + i), f);
#pragma unroll
    for (int q = 0; q < VT::N; ++q) mx = fmaxf(mx, f[q]);
  }
  mx = warp_max(mx);
  float sub = finite_max(mx);
  float sum = edge >= 0 ? ex2((ze - sub) * c) : 0.f;
#pragma unroll
  for (int e = 0; e < kVec; ++e) {
    if (v0 + tid + e * TH < v1) {
      float f[VT::N];
      VT::load(d[e], f);
      float part = 0.f;
#pragma unroll
      for (int q = 0; q < VT::N; ++q) part += ex2((f[q] - sub) * c);
      sum += part;
    }
  }
  for (int i = v0 + tid + kVec * TH; i < v1; i += TH) {
    float f[VT::N];
    VT::load(__ldcg(zv + i), f);
    float part = 0.f;
#pragma unroll
    for (int q = 0; q < VT::N; ++q) part += ex2((f[q] - sub) * c);
    sum += part;
  }
  sum = warp_sum(sum);
  gap = warp_sum(gap);
  if (lane == 0) warp_share[tid / 32] = Share{gap, mx, sum};
  __syncthreads();
  if (tid < 32) {
    const Share s = lane < TH / 32 ? warp_share[lane] : Share{0.0, -INFINITY, 0.f};
    const float cm = warp_max(s.max);
    const float cs = warp_sum(s.sum * ex2((finite_max(s.max) - finite_max(cm)) * c));
    const double cg = warp_sum(s.gap);
    if (lane < C) {  // into CTA `lane` of the cluster
      uint32_t to;
      asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(smem_u32(&shares[rank])), "r"((uint32_t)lane));
      asm volatile("st.shared::cluster.v2.b32 [%0], {%1, %2};" ::"r"(to + (uint32_t)offsetof(Share, max)), "f"(cm),
                   "f"(cs)
                   : "memory");
      asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(to), "d"(cg) : "memory");
    }
  }
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  float zmax = -INFINITY, zsum = 0.f;
  for (uint32_t r = 0; r < C; ++r) zmax = fmaxf(zmax, shares[r].max);
  sub = finite_max(zmax);
  for (uint32_t r = 0; r < C; ++r) zsum += shares[r].sum * ex2((finite_max(shares[r].max) - sub) * c);
  if (rank == 0 && tid == 0) {
    double g = 0.0;
    for (uint32_t r = 0; r < C; ++r) g += shares[r].gap;
    // log of p's normaliser over q's; an empty student row (zsum 0) makes it -inf and the loss +inf
    const double norm = ((double)tmax - (double)sub) * inv + log((double)tsum) - log((double)zsum);
    const double kl = isinf(g) ? g : g * inv - norm;
    p.loss[m] = (float)((double)w * temp * temp * kl);
  }
  if (!dz) return;

  const float scale = zsum > 0.f ? w * temp / zsum : (zsum == 0.f ? 0.f : zsum);
#pragma unroll
  for (int e = 0; e < kVec; ++e) {
    const int i = v0 + tid + e * TH;
    if (i < v1) {
      float f[VT::N];
      VT::load(d[e], f);
#pragma unroll
      for (int q = 0; q < VT::N; ++q) f[q] = ex2((f[q] - sub) * c) * scale;
      store(i, f);
    }
  }
  for (int i = v0 + tid + kVec * TH; i < v1; i += TH) {
    float f[VT::N];
    VT::load(__ldcg(zv + i), f);
#pragma unroll
    for (int q = 0; q < VT::N; ++q) f[q] = ex2((f[q] - sub) * c) * scale;
    store(i, f);
  }
  if (edge >= 0) dz[edge] = from_f32<T>(ex2((ze - sub) * c) * scale);
  __syncthreads();
  // the teacher's columns of this CTA: the first entry of an id writes it, with the mass of all its entries
  for (int j = tid; j < p.k; j += TH) {
    const uint32_t id = ids[j];
    if (id < e0 || id >= e1) continue;
    float mass = 0.f;
    bool first = true;
    for (int i = 0; i < p.k; ++i) {
      if (ids[i] == id) {
        first = first && i >= j;
        mass += ex2((tval[i] - tmax) * c);
      }
    }
    if (first) dz[id] = from_f32<T>(ex2((zval[j] - sub) * c) * scale - w * temp * (mass / tsum));
  }
}

template <typename T, int TH>
cudaError_t launch_rows(const DistillArgs& p, int cluster, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(p.M * cluster));
  cfg.blockDim = dim3(TH);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)cluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, distill_rows_kernel<T, TH>, p);
}

template <typename T>
cudaError_t launch_type(const DistillArgs& p, int sm_count, cudaStream_t stream) {
  const int64_t bytes = p.V * (int64_t)sizeof(T);
  if (bytes <= 128 * kVec * 16) return launch_rows<T, 128>(p, 1, stream);
  // as many CTAs as hold the row in registers; with few rows, more, down to 8 KB a CTA, while they fit the SMs
  int64_t cluster = (bytes + 512 * kVec * 16 - 1) / (512 * kVec * 16);
  while (cluster < kClusterMax && p.M * (cluster + 1) <= sm_count && bytes / (cluster + 1) >= 8192) ++cluster;
  if (cluster > kClusterMax) cluster = kClusterMax;
  return launch_rows<T, 512>(p, (int)cluster, stream);
}

}  // namespace

int distill_max_top() { return kTopMax; }

cudaError_t launch_distill(const DistillArgs& p, int sm_count, cudaStream_t stream) {
  if (p.M == 0) return cudaSuccess;
  if (p.dtype == QW_F16) return launch_type<__half>(p, sm_count, stream);
  if (p.dtype == QW_BF16) return launch_type<__nv_bfloat16>(p, sm_count, stream);
  return launch_type<float>(p, sm_count, stream);
}

}  // namespace qw
