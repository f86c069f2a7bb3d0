// qw_lora.cu -- low-rank adapters beside a quantized projection, many at once:
// row m of x takes adapter idx[m] (none when idx[m] >= L),
//   y[m] += s (x[m] A^T) B^T,            A [R, K], B [N, R], s the adapter's scale
// and the gradient of that term:
//   h = s x A^T, g = s dy B, dA = g^T x, dB = dy^T h, dx = g A
// with the sums over the rows of each adapter.
//
// Forward, two launches chained by programmatic dependent launch:
//   rank_rows     h = s x A^T (below; many rows of a high rank: lora_products);
//   the projection's own kernel: the decode kernel (at most 16 rows) adds h B^T
//                 in its epilogue, the tcgen05 kernel takes h and B as further
//                 columns of its reduction.
#include <cuda_fp16.h>

#include "qw_internal.h"
#include "qw_lora.cuh"
#include "qw_ptx.cuh"

namespace qw {

namespace {

// h = s x A^T for the forward.  Memory- and latency-bound: x is read once and
// the A of every adapter present once per 16 rows; the products are few.
//
// A cluster takes a tile of 16 rows and every G-th of the adapters its rows
// name (a row belongs to one of them, so groups write disjoint rows); its CTAs
// and their warps split K.  A warp's operands come straight from memory in
// mma.sync m16n8k16 fragment order: one 16-byte load a lane brings a row's 8
// consecutive k for two products' slots, the order of k within a sum being
// free as long as x and A agree, so no shared memory, no barrier and no copy
// stands between the loads and the products, and a warp keeps U steps of 32 k
// in flight.  CTAs of 128 threads fit beside the decode kernel's, which starts
// while this one runs.  Each adapter has its own accumulators: what a row that is not its
// own, or A of another, holds never meets it.  Sums over warps and CTAs go
// through (distributed) shared memory in a fixed order.
//
// Blocks behind the tiles' list, for the tcgen05 kernel, the adapters of every
// token tile, and zero the decode kernel's counters.
struct RankRows {
  LoraArgs p;
  float* h32;         // [M][R] fp32 (at most 16 rows), or
  __half* h16;        // [M][R8] fp16, zero-padded rank, and
  float* full;        // [M][R8] fp32, where that is not finite
  int R8;
  int tiles, groups;  // row tiles, adapter groups per tile
  TokenLists lists;
  uint4* zero;        // cleared by the blocks behind the lists
  int zero_vecs;
  int prefetch;       // bring B of the adapters present to L2 (for the decode kernel's epilogue)
};

// The second bound keeps a CTA up to rank 16 within the registers that the decode
// kernel leaves of an SM (12 thousand at 9 to 16 rows).
template <int RT, int WARPS, int U>
__global__ void __launch_bounds__(WARPS * 32, RT <= 2 ? 5 : (RT <= 4 ? 4 : 2)) rank_rows_kernel(const RankRows q) {
  constexpr int RP = 8 * RT;
  extern __shared__ float red[];  // [WARPS][16][RP], then the CTA's sum [16][RP]
  __shared__ uint32_t row_id[16];
  __shared__ uint32_t list[16];
  __shared__ int list_n;
  const LoraArgs& p = q.p;
  pdl_wait();
  pdl_launch_dependents();
  const uint32_t rank = cluster_rank(), C = cluster_size();
  const int unit = (int)(blockIdx.x / C);
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;

  if (unit >= q.tiles * q.groups) {
    if (rank != 0) return;
    const int t = unit - q.tiles * q.groups;
    if (t < q.lists.tiles) {
      token_list(p, q.lists, t);
    } else {
      for (int i = tid; i < q.zero_vecs; i += WARPS * 32) q.zero[i] = make_uint4(0u, 0u, 0u, 0u);
    }
    return;
  }

  const int64_t m0 = (int64_t)(unit / q.groups) * 16;
  const int group = unit % q.groups;
  if (warp == 0) {
    const int64_t a = lane < 16 && m0 + lane < p.M ? adapter_of(p, m0 + lane) : -1;
    const uint32_t same = __match_any_sync(0xffffffffu, (int)a);
    const bool first = a >= 0 && __ffs(same) - 1 == lane;
    const uint32_t leaders = __ballot_sync(0xffffffffu, first);
    if (lane < 16) row_id[lane] = (uint32_t)a;
    if (first) list[__popc(leaders & ((1u << lane) - 1u))] = (uint32_t)a;
    if (lane == 0) list_n = __popc(leaders);
  }
  __syncthreads();
  const int n = list_n;
  const int steps = (int)(p.K / 32);
  const int s0 = (int)((int64_t)steps * rank / C), s1 = (int)((int64_t)steps * (rank + 1) / C);
  const int r = lane / 4, kq = (lane % 4) * 8;
  float* const mine = red + warp * 16 * RP;
  float* const cta = red + WARPS * 16 * RP;
  for (int j = group; j < n; j += q.groups) {
    const uint32_t a = list[j];
    const bool own0 = row_id[r] == a, own1 = row_id[r + 8] == a;
    const __half* x0 = reinterpret_cast<const __half*>(p.x) + (m0 + r) * p.x_ld + kq;
    const __half* x1 = x0 + 8 * p.x_ld;
    const __half* w0 = reinterpret_cast<const __half*>(p.a) + ((int64_t)a * p.R + r) * p.K + kq;
    float acc[RT][4];
#pragma unroll
    for (int t = 0; t < RT; ++t) acc[t][0] = acc[t][1] = acc[t][2] = acc[t][3] = 0.f;
    const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
    for (int s = s0 + warp; s < s1; s += WARPS * U) {
      uint4 xa[U], xb[U], w[U][RT];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t k = (int64_t)(s + u * WARPS) * 32;
        const bool in = s + u * WARPS < s1;
        xa[u] = in && own0 ? __ldg(reinterpret_cast<const uint4*>(x0 + k)) : zero;
        xb[u] = in && own1 ? __ldg(reinterpret_cast<const uint4*>(x1 + k)) : zero;
#pragma unroll
        for (int t = 0; t < RT; ++t)
          w[u][t] = in && r + 8 * t < p.R ? __ldg(reinterpret_cast<const uint4*>(w0 + (int64_t)t * 8 * p.K + k)) : zero;
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int t = 0; t < RT; ++t) {
          mma_16816(acc[t], xa[u].x, xb[u].x, xa[u].y, xb[u].y, w[u][t].x, w[u][t].y);
          mma_16816(acc[t], xa[u].z, xb[u].z, xa[u].w, xb[u].w, w[u][t].z, w[u][t].w);
        }
    }
    if (q.prefetch) {  // this adapter's B, split over the cluster
      const char* b = reinterpret_cast<const char*>(p.b) + (int64_t)a * p.N * p.R * 2;
      for (int64_t i = ((int64_t)rank * WARPS * 32 + tid) * 128; i < p.N * p.R * 2; i += (int64_t)C * WARPS * 32 * 128)
        asm volatile("prefetch.global.L2 [%0];" ::"l"(b + i));
    }
    __syncthreads();  // the sums of the adapter before are read
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      float2* d0 = reinterpret_cast<float2*>(mine + r * RP + t * 8 + (lane % 4) * 2);
      float2* d1 = reinterpret_cast<float2*>(mine + (r + 8) * RP + t * 8 + (lane % 4) * 2);
      *d0 = make_float2(acc[t][0], acc[t][1]);
      *d1 = make_float2(acc[t][2], acc[t][3]);
    }
    __syncthreads();
    const float scale = p.scales ? p.scales[a] : 1.f;
    for (int i = tid; i < 16 * RP; i += WARPS * 32) {
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) v += red[w * 16 * RP + i];
      cta[i] = v;
    }
    if (C > 1) cluster_sync();
    else __syncthreads();
    for (int i = (int)rank * WARPS * 32 + tid; i < 16 * RP; i += (int)C * WARPS * 32) {
      const int row = i / RP, c = i % RP;
      if (row_id[row] != a) continue;
      float v = 0.f;
      for (uint32_t k = 0; k < C; ++k) v += C > 1 ? ld_cluster_f32(&cta[i], k) : cta[i];
      v *= scale;
      if (q.h32) {
        if (c < p.R) q.h32[(m0 + row) * p.R + c] = v;
      } else if (c < q.R8) {
        // One rounding to fp16, relative to the adapter's term what y's own rounding is to
        // y: the tensor cores take the second product in fp16, and a second term of h
        // would double the adapters' k blocks.  Values beyond fp16 are kept in fp32.
        const int64_t at = (m0 + row) * q.R8 + c;
        const __half h = c < p.R ? __float2half_rn(v) : __half(0);
        q.h16[at] = h;
        if (!isfinite(__half2float(h))) q.full[at] = v;
      }
    }
    if (C > 1) cluster_sync();  // the peers' sums are read before they change or go
  }
}

constexpr size_t align256(size_t v) { return (v + 255) & ~(size_t)255; }
int round8(int r) { return (r + 7) / 8 * 8; }

// Forward workspace: at most 16 rows, h fp32; above, h fp16 (zero-padded rank),
// the token tiles' lists, and h fp32.
struct ForwardSpace {
  size_t second, third, fourth, full, end;
};
ForwardSpace forward_space(int64_t M, int R, int token_tile) {
  ForwardSpace f;
  if (token_tile == 0) {
    f.second = f.third = f.fourth = f.full = f.end = align256((size_t)M * R * sizeof(float));
  } else {
    const size_t tiles = (size_t)((M + token_tile - 1) / token_tile);
    f.second = align256((size_t)M * round8(R) * sizeof(__half));
    f.third = f.second + align256(tiles * sizeof(uint32_t));
    f.fourth = f.third + align256(tiles * token_tile * sizeof(uint32_t));
    f.full = f.fourth + align256((size_t)M * sizeof(uint32_t));
    f.end = f.full + align256((size_t)M * round8(R) * sizeof(float));
  }
  return f;
}

template <int RT, int WARPS, int U>
cudaError_t launch_rank_rows(RankRows& q, int sm_count, bool pdl, cudaStream_t stream) {
  // K over the warps, then over up to 8 CTAs while a warp has more than U
  // steps; the tile's adapters over groups while SMs are free.
  const int steps = (int)(q.p.K / 32);
  int C = (steps + WARPS * U - 1) / (WARPS * U);
  C = C > 8 ? 8 : C;
  while (C > 1 && (int64_t)q.tiles * C > 4 * sm_count) --C;
  int64_t groups = 4 * sm_count / ((int64_t)q.tiles * C);
  const int64_t most = q.p.L < 16 ? q.p.L : 16;
  groups = groups > most ? most : groups;
  groups = groups < 1 ? 1 : groups;
  q.groups = (int)groups;
  constexpr int smem = (WARPS + 1) * 16 * 8 * RT * (int)sizeof(float);
  static thread_local int configured_dev = -1;
  int dev = 0;
  cudaGetDevice(&dev);
  if (configured_dev != dev) {
    const cudaError_t e = cudaFuncSetAttribute(rank_rows_kernel<RT, WARPS, U>,
                                               cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    configured_dev = dev;
  }
  const int64_t units = (int64_t)q.tiles * q.groups + q.lists.tiles + (q.zero_vecs ? 1 : 0);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(units * C));
  cfg.blockDim = dim3(WARPS * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)C;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, rank_rows_kernel<RT, WARPS, U>, q);
}

}  // namespace

size_t lora_forward_bytes(int64_t M, int R, int token_tile) { return forward_space(M, R, token_tile).end; }

cudaError_t launch_lora_rank(const LoraArgs& p, int token_tile, void* ws, void* zero, size_t zero_bytes,
                             unsigned int* status, int sm_count, bool pdl, cudaStream_t stream, std::string* err) {
  const ForwardSpace f = forward_space(p.M, p.R, token_tile);
  uint8_t* base = static_cast<uint8_t*>(ws);
  RankRows q{};
  q.p = p;
  q.R8 = round8(p.R);
  if (token_tile == 0) {
    q.h32 = reinterpret_cast<float*>(base);
    q.prefetch = 1;
  } else {
    q.h16 = reinterpret_cast<__half*>(base);
    q.full = reinterpret_cast<float*>(base + f.full);
    q.lists.tile = token_tile;
    q.lists.tiles = (int)((p.M + token_tile - 1) / token_tile);
    q.lists.n = reinterpret_cast<uint32_t*>(base + f.second);
    q.lists.ids = reinterpret_cast<uint32_t*>(base + f.third);
    q.lists.slots = reinterpret_cast<uint32_t*>(base + f.fourth);
    // Many rows of a high rank are worth the tcgen05 products' tiles of 128 rows.  The
    // whole call in us with them and without, 8 adapters, 5120 -> 5120: 1024 rows of
    // rank 64 113 and 119, of rank 128 156 and 165; 512 rows 75 and 74, 98 and 93;
    // 300 rows 68 and 62, 82 and 73; rank 32 at 2048 rows 154 and 150.
    // (An empty stack has no tensor maps.)
    if (p.L > 0 && p.R > 32 && p.M > 512)
      return launch_lora_products(p, q.lists, q.h16, q.full, status, sm_count, pdl, stream, err);
  }
  q.tiles = (int)((p.M + 15) / 16);
  q.zero = static_cast<uint4*>(zero);
  q.zero_vecs = (int)((zero_bytes + 15) / 16);
  if (p.R <= 8) return launch_rank_rows<1, 4, 4>(q, sm_count, pdl, stream);
  if (p.R <= 16) return launch_rank_rows<2, 4, 3>(q, sm_count, pdl, stream);
  if (p.R <= 32) return launch_rank_rows<4, 4, 2>(q, sm_count, pdl, stream);
  if (p.R <= 64) return launch_rank_rows<8, 4, 1>(q, sm_count, pdl, stream);
  return launch_rank_rows<16, 4, 1>(q, sm_count, pdl, stream);
}

SkinnyLora lora_skinny_operands(const LoraArgs& p, void* ws, const void* bias) {
  return SkinnyLora{static_cast<const float*>(ws), p.b, p.idx, bias, p.R, (int)p.L};
}

PrefillLora lora_prefill_operands(const LoraArgs& p, int token_tile, void* ws, const void* bias) {
  const ForwardSpace f = forward_space(p.M, p.R, token_tile);
  uint8_t* base = static_cast<uint8_t*>(ws);
  PrefillLora l{};
  l.h = base;
  l.full = reinterpret_cast<const float*>(base + f.full);
  l.b = p.b;
  l.idx = p.idx;
  l.tile_n = reinterpret_cast<uint32_t*>(base + f.second);
  l.tile_ids = reinterpret_cast<uint32_t*>(base + f.third);
  l.slots = reinterpret_cast<uint32_t*>(base + f.fourth);
  l.bias = bias;
  l.R = p.R;
  l.L = (int)p.L;
  return l;
}

}  // namespace qw
