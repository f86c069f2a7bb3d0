// qw_lora.cuh -- device helpers shared by the adapter kernels.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "qw_internal.h"
#include "qw_ptx.cuh"

namespace qw {

__device__ __forceinline__ int64_t adapter_of(const LoraArgs& p, int64_t m) {
  const uint32_t a = p.idx ? p.idx[m] : 0u;
  return (int64_t)a < p.L ? (int64_t)a : -1;
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  __syncwarp();  // .aligned takes a whole warp
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float ld_cluster_f32(const float* p, uint32_t rank) {
  uint32_t a;
  float v;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ float4 ld_cluster_f32x4(const float* p, uint32_t rank) {
  uint32_t a;
  float4 v;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(a)
               : "memory");
  return v;
}

// List of token tile t: its adapters in ascending order and, for each of its
// rows, the place of the row's adapter (none: 0xFFFFFFFF).  One CTA.
__device__ inline void token_list(const LoraArgs& p, const TokenLists& q, int t) {
  constexpr int kWords = (int)kLoraMaxAdapters / 32;
  __shared__ uint32_t bits[kWords], before[kWords];
  const int tid = threadIdx.x, threads = blockDim.x, lane = tid % 32;
  for (int i = tid; i < kWords; i += threads) bits[i] = 0u;
  __syncthreads();
  for (int i = tid; i < q.tile; i += threads) {
    const int64_t m = (int64_t)t * q.tile + i;
    if (m < p.M) {
      const int64_t a = adapter_of(p, m);
      if (a >= 0) atomicOr(&bits[a / 32], 1u << (a % 32));
    }
  }
  __syncthreads();
  if (tid < 32) {  // a lane the bits of 4 words
    uint32_t w[kWords / 32], n = 0;
#pragma unroll
    for (int i = 0; i < kWords / 32; ++i) {
      w[i] = bits[lane * (kWords / 32) + i];
      n += __popc(w[i]);
    }
    uint32_t at = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t v = __shfl_up_sync(0xffffffffu, at, o);
      if (lane >= o) at += v;
    }
    if (lane == 31) q.n[t] = at;
    at -= n;
#pragma unroll
    for (int i = 0; i < kWords / 32; ++i) {
      before[lane * (kWords / 32) + i] = at;
      for (uint32_t b = w[i]; b; b &= b - 1)
        q.ids[(size_t)t * q.tile + at++] = (uint32_t)((lane * (kWords / 32) + i) * 32 + __ffs(b) - 1);
    }
  }
  __syncthreads();
  for (int i = tid; i < q.tile; i += threads) {
    const int64_t m = (int64_t)t * q.tile + i;
    if (m >= p.M) break;
    const int64_t a = adapter_of(p, m);
    q.slots[m] = a < 0 ? 0xFFFFFFFFu : before[a / 32] + __popc(bits[a / 32] & ((1u << (a % 32)) - 1u));
  }
}

}  // namespace qw
