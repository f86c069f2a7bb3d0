// qw_lora_grad.cu -- gradient of the adapters beside a projection (and the
// rank-space product of a long forward):
//   h = s x A^T, g = s dy B                    per row, its adapter's A, B, s
//   dA = g^T x, dB = dy^T h                    sums over the adapter's rows
//   dx = g A (+ dx)
// Three launches, chained by programmatic dependent launch:
//   plan     sorts the rows by adapter and cuts each adapter's rows into chunks;
//   products h and g, fp32, and the largest magnitude of each per adapter
//            (runs beside the plan until its results);
//   sums     dA, dB and dx, a chunk of rows and 256 columns at a time.
// x and dy are read twice, once across their width and once along their rows;
// everything else is rank-sized.
#include <cuda_fp16.h>

#include <cstring>

#include "qw_internal.h"
#include "qw_lora.cuh"
#include "qw_ptx.cuh"

namespace qw {

namespace {

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid) {
  const int n = valid ? 16 : 0;  // 0 bytes read: 16 zeros written
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t addr, uint32_t& r0, uint32_t& r1, uint32_t& r2,
                                                  uint32_t& r3) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3)
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void sts16(uint32_t addr, uint4 v) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w)
               : "memory");
}
// Eight halves from any address, those at or past `n` zero.
__device__ __forceinline__ uint4 load_halves(const __half* p, int64_t n) {
  uint32_t h[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) h[i] = i < n ? __half_as_ushort(p[i]) : 0u;
  return make_uint4(h[0] | (h[1] << 16), h[2] | (h[3] << 16), h[4] | (h[5] << 16), h[6] | (h[7] << 16));
}

// ------------------------------------------------------- tensor-core operands
// Shared-memory operands of tcgen05.mma, all with the 128-byte swizzle: rows of
// 128 bytes (64 halves), 16-byte piece q of row i at place q ^ (i & 7), eight rows
// to an atom of 1024 bytes.
//   along K: the rows are the operand's M or N and hold 64 k; a step of 16 k is 32
//            bytes further on.
//   along MN: the rows are k and hold 64 of M or N, the next 64 are `next` bytes
//            away; a step of 16 k is 16 rows further on.
__device__ __forceinline__ uint32_t swizzled(int row, int piece) { return row * 128 + ((piece ^ (row & 7)) << 4); }
__device__ __forceinline__ uint64_t operand_k(uint32_t addr) {
  return (uint64_t)((addr >> 4) & 0x3FFF) | ((uint64_t)1 << 16) | ((uint64_t)(1024 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
__device__ __forceinline__ uint64_t operand_mn(uint32_t addr, uint32_t next) {
  return (uint64_t)((addr >> 4) & 0x3FFF) | ((uint64_t)(next >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// kind::f16, D fp32, A and B fp16 (each along K, or along MN), M x N.
constexpr uint32_t mma_desc(int m, int n, bool a_mn, bool b_mn) {
  return (1u << 4) | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(m >> 4) << 24);
}

// ---------------------------------------------------------------- products
// v W of each row's adapter, a tile of 128 rows at a time: out[m][r] = s sum_i
// v[m][i] W[i][r].  HBM-bound by v, which is read once.
//
// A cluster takes a tile and its CTAs split the reduction; a CTA walks 64 values
// of it at a time, four TMA loads deep, and within those the adapters that the
// tile's rows name, so v is staged once however mixed the rows are.  Rows or
// weights that TMA cannot take (dy of a width, or lora_b of a rank, that is no
// multiple of 8) are copied by the threads instead; that path pays a proxy fence
// a step, which waits for every copy in flight.
// Every adapter has columns of its own in TMEM (four adapters at a time, two
// above rank 64) and a row reads those of its own adapter: no row's sum ever
// meets another adapter's values.  Sums over the cluster go through distributed
// shared memory in rank order.
constexpr int kStages = 4;
constexpr int kProdThreads = 128;
constexpr int kChunk = 64;  // reduction values per step
constexpr int kTileRows = 128;

struct Product {
  const __half* v;  // [M][len], rows ld apart
  int64_t ld, len;
  const __half* w;  // [L][R][len], or for the second product [L][len][R]
  float* out32;     // [M][RP] fp32, RP the kernel's padded rank (null: out16)
  __half* out16;    // [M][R8] fp16
  uint32_t* amax;   // [L] largest magnitude of out32, as fp32 bits
};
struct Products {
  LoraArgs p;
  Product a, b;      // b.v null: one product
  __half* dx_zero;   // [M][K]: rows without an adapter are cleared (nullable)
  int R8;
  int tiles;         // row tiles
  int b_tma;         // TMA can take the second product's operands
  TokenLists lists;  // forward
  unsigned int* status;
};

template <int RP>
struct ProdCfg {
  static constexpr int BLOCK = RP > 64 ? 128 : 64;    // TMEM columns of an adapter
  static constexpr int COLUMNS = 256;                 // two CTAs an SM
  static constexpr int GROUP = COLUMNS / BLOCK;       // adapters at a time
  static constexpr int V_STAGE = kTileRows * 128;
  static constexpr int W_STAGE = 64 * BLOCK * 2;
  static constexpr int STAGE = V_STAGE + W_STAGE;
  static constexpr int PITCH = RP + 4;                // floats of a row of sums
  static constexpr int SUMS = kTileRows * PITCH * 4;
  static constexpr int SMEM = (kStages * STAGE > SUMS ? kStages * STAGE : SUMS) + 1024;
  static_assert(SMEM <= (RP > 64 ? 224 : 112) * 1024, "two CTAs an SM up to rank 64");
};

struct ProductMaps {
  CUtensorMap av, aw, bv, bw;  // operands of the two products: v [M][len], w 3-D
};
struct ProdShared {
  uint32_t row_id[kTileRows], row_slot[kTileRows], list[2 * kTileRows], slot_max[kTileRows];
  uint64_t full[kStages], done[kStages];
  int list_n;
  uint32_t tmem;
};

template <int RP, bool TRANS, bool TMA>
__device__ void product_tile(const Products& q, const Product& f, const CUtensorMap* map_v, const CUtensorMap* map_w,
                             int tile, uint32_t rank, uint32_t C, uint8_t* smem, ProdShared& sh) {
  using Cfg = ProdCfg<RP>;
  const LoraArgs& p = q.p;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const int64_t m0 = (int64_t)tile * kTileRows;

  // the tile's adapters in order of first appearance, and each row's place among them
  sh.row_id[tid] = m0 + tid < p.M ? (uint32_t)adapter_of(p, m0 + tid) : 0xFFFFFFFFu;
  sh.slot_max[tid] = 0u;
  __syncthreads();
  const uint32_t my_id = sh.row_id[tid];
  {
    const uint4* ids = reinterpret_cast<const uint4*>(sh.row_id);
    int first = tid;
    for (int k = tid / 4; k >= 0; --k) {  // four rows at a time, downwards
      const uint4 w = ids[k];
      first = w.w == my_id && 4 * k + 3 < first ? 4 * k + 3 : first;
      first = w.z == my_id && 4 * k + 2 < first ? 4 * k + 2 : first;
      first = w.y == my_id && 4 * k + 1 < first ? 4 * k + 1 : first;
      first = w.x == my_id && 4 * k < first ? 4 * k : first;
    }
    const bool lead = my_id != 0xFFFFFFFFu && first == tid;
    const uint32_t leaders = __ballot_sync(0xffffffffu, lead);
    if (lane == 0) sh.row_slot[warp] = __popc(leaders);
    __syncthreads();
    int at = __popc(leaders & ((1u << lane) - 1u));
    for (int w = 0; w < warp; ++w) at += (int)sh.row_slot[w];
    if (tid == kProdThreads - 1) sh.list_n = at + lead;
    if (lead) {
      sh.list[at] = my_id;
      sh.list[kTileRows + tid] = (uint32_t)at;
    }
    __syncthreads();
    sh.row_slot[tid] = my_id == 0xFFFFFFFFu ? my_id : sh.list[kTileRows + first];
  }
  const int n = sh.list_n;
  const int my_slot = (int)sh.row_slot[tid];  // -1: none
  if (!TRANS && q.dx_zero) {  // rows without an adapter
    for (int row = warp; row < kTileRows && m0 + row < p.M; row += kProdThreads / 32) {
      if (sh.row_id[row] != 0xFFFFFFFFu) continue;
      uint4* dst = reinterpret_cast<uint4*>(q.dx_zero + (m0 + row) * p.K);
      for (int64_t c = rank * 32 + lane; c < p.K / 8; c += C * 32) dst[c] = make_uint4(0u, 0u, 0u, 0u);
    }
  }
  if (n == 0) {  // the whole cluster: nobody's rows
    pdl_wait();  // a kernel behind this one counts on the plan, too
    return;
  }

  const int chunks = (int)((f.len + kChunk - 1) / kChunk);
  const int c0 = (int)((int64_t)chunks * rank / C), c1 = (int)((int64_t)chunks * (rank + 1) / C);
  const uint32_t base = smem_u32(smem);
  const bool v16 = f.ld % 8 == 0 && f.len % 8 == 0 && (reinterpret_cast<uintptr_t>(f.v) & 15) == 0;
  const bool w16 = !TRANS || p.R % 8 == 0;
  bool ok = true;        // a bounded wait that ran out: go on without waiting
  uint32_t it0 = 0, vit0 = 0;  // TMA: steps and chunks of earlier rounds
  constexpr uint32_t kDesc = mma_desc(kTileRows, TRANS ? Cfg::BLOCK : RP, false, TRANS);
  auto multiply = [&](int chunk, int j, uint32_t vs, uint32_t ws) {
    const uint64_t a = operand_k(vs), b = TRANS ? operand_mn(ws, 8192) : operand_k(ws);
#pragma unroll
    for (int kk = 0; kk < kChunk / 16; ++kk)
      tc_mma_ss(sh.tmem + j * Cfg::BLOCK, a + (uint64_t)(2 * kk), b + (uint64_t)((TRANS ? 128 : 2) * kk), kDesc,
                chunk > 0 || kk > 0);
  };
  uint32_t parities = 0; // copies: of done[i], a bit each: flips with every use waited for
  auto wait_step = [&](int step) {
    const int i = step % kStages;
    ok = ok && mbar_wait(&sh.done[i], (parities >> i) & 1u, q.status, kDevTimeoutAccum);
    parities ^= 1u << i;
  };

  for (int j0 = 0; j0 < n; j0 += Cfg::GROUP) {
    const int nj = n - j0 < Cfg::GROUP ? n - j0 : Cfg::GROUP;
    const int steps = (c1 - c0) * nj;
    if constexpr (TMA) {
      if (warp == 1 && lane == 0) {  // loads
        uint32_t it = it0, vit = vit0;
        for (int c = c0; c < c1; ++c, ++vit) {
          for (int j = 0; j < nj; ++j, ++it) {
            const uint32_t s = it % kStages;
            if (it >= kStages)
              ok = ok && mbar_wait(&sh.done[s], (it / kStages - 1) & 1, q.status, kDevTimeoutEmpty);
            mbar_arrive_expect_tx(&sh.full[s], (uint32_t)((j == 0 ? Cfg::V_STAGE : 0) + (TRANS ? Cfg::W_STAGE : RP * 128)));
            if (j == 0)
              tma_load_2d(smem + (vit % kStages) * Cfg::STAGE, map_v, &sh.full[s], c * kChunk, (int)m0);
            uint8_t* dst = smem + s * Cfg::STAGE + Cfg::V_STAGE;
            const int a = (int)sh.list[j0 + j];
            if (TRANS) {
              for (int b = 0; b < Cfg::BLOCK / 64; ++b)
                tma_load_3d(dst + b * 8192, map_w, &sh.full[s], b * 64, c * kChunk, a);
            } else {
              tma_load_3d(dst, map_w, &sh.full[s], c * kChunk, 0, a);
            }
          }
        }
      } else if (warp == 0 && lane == 0) {  // products
        uint32_t it = it0, vit = vit0;
        for (int c = c0; c < c1; ++c, ++vit) {
          for (int j = 0; j < nj; ++j, ++it) {
            const uint32_t s = it % kStages;
            ok = ok && mbar_wait(&sh.full[s], (it / kStages) & 1, q.status, kDevTimeoutFull);
            tc_fence_after();
            multiply(c - c0, j, base + (vit % kStages) * Cfg::STAGE, base + s * Cfg::STAGE + Cfg::V_STAGE);
            tc_commit(&sh.done[s]);
          }
        }
      }
      it0 += (uint32_t)steps;
      vit0 += (uint32_t)(c1 - c0);
      __syncwarp();
      // The last step's barrier has seen every earlier use waited for by the
      // thread that loads, but for those of the last turn of the ring, which
      // complete in order.
      if (steps > 0) {
        __syncthreads();
        ok = ok && mbar_wait(&sh.done[(it0 - 1) % kStages], ((it0 - 1) / kStages) & 1, q.status, kDevTimeoutAccum);
      }
    } else {
      auto load = [&](int step) {
        const int64_t i0 = (int64_t)(c0 + step / nj) * kChunk;
        const int j = step % nj;
        if (j == 0) {
          const uint32_t dst = base + (uint32_t)((step / nj) % kStages) * Cfg::STAGE;
#pragma unroll
          for (int k = 0; k < kTileRows * 8 / kProdThreads; ++k) {
            const int row = (k * kProdThreads + tid) / 8, piece = tid % 8;
            const int64_t i = i0 + piece * 8;
            const bool in = m0 + row < p.M && i < f.len;
            const __half* src = f.v + (in ? (m0 + row) * f.ld + i : 0);
            const uint32_t at = dst + swizzled(row, piece);
            if (v16) cp_async16(at, src, in);
            else sts16(at, load_halves(src, in ? f.len - i : 0));
          }
        }
        const uint32_t dst = base + (uint32_t)(step % kStages) * Cfg::STAGE + Cfg::V_STAGE;
        const __half* w = f.w + (int64_t)sh.list[j0 + j] * p.R * f.len;
        constexpr int kPieces = 8 * RP;
#pragma unroll
        for (int k = 0; k < kPieces / kProdThreads; ++k) {
          const int e = k * kProdThreads + tid;
          if (TRANS) {
            const int row = e / (RP / 8), r = e % (RP / 8) * 8;
            const bool in = i0 + row < f.len && r < p.R;
            const __half* src = w + (in ? (i0 + row) * p.R + r : 0);
            const uint32_t at = dst + (r / 64) * 8192 + swizzled(row, r % 64 / 8);
            if (w16) cp_async16(at, src, in);
            else sts16(at, load_halves(src, in ? p.R - r : 0));
          } else {
            const int r = e / 8, piece = e % 8;
            const bool in = r < p.R && i0 + piece * 8 < f.len;
            cp_async16(dst + swizzled(r, piece), w + (in ? (int64_t)r * f.len + i0 + piece * 8 : 0), in);
          }
        }
      };
#pragma unroll
      for (int s = 0; s < kStages - 1; ++s) {
        if (s < steps) load(s);
        cp_async_commit();
      }
      for (int step = 0; step < steps; ++step) {
        cp_async_wait<kStages - 2>();
        fence_proxy_async_smem();
        tc_fence_before();
        __syncthreads();
        if (tid == 0) {
          tc_fence_after();
          multiply(step / nj, step % nj, base + (uint32_t)((step / nj) % kStages) * Cfg::STAGE,
                   base + (uint32_t)(step % kStages) * Cfg::STAGE + Cfg::V_STAGE);
          tc_commit(&sh.done[step % kStages]);
        }
        // the products that read the stage loaded next are the previous step's
        if (step > 0) wait_step(step - 1);
        if (step + kStages - 1 < steps) load(step + kStages - 1);
        cp_async_commit();
      }
      if (steps > 0) wait_step(steps - 1);
    }
    tc_fence_after();
    cp_async_wait<0>();
    __syncthreads();

    // each row's own columns, to shared memory
    float* const sums = reinterpret_cast<float*>(smem);
    for (int b = 0; b < nj; ++b) {
      const bool own = my_slot == j0 + b;
      if (!__any_sync(0xffffffffu, own)) continue;
#pragma unroll
      for (int c = 0; c < RP; c += 16) {
        uint32_t v[16];
        if (steps > 0) {
          tmem_ld_32x32b_x16(sh.tmem + ((uint32_t)(warp * 32) << 16) + b * Cfg::BLOCK + c, v);
          tmem_wait_ld();
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i) v[i] = 0u;  // this CTA has no part of the reduction
        }
        if (own) {
#pragma unroll
          for (int i = 0; i < 16; i += 4)
            *reinterpret_cast<uint4*>(sums + tid * Cfg::PITCH + c + i) = make_uint4(v[i], v[i + 1], v[i + 2], v[i + 3]);
        }
      }
    }
    tc_fence_before();
    if (C > 1) cluster_sync();
    else __syncthreads();
    pdl_wait();  // the maxima's start values are the plan's (a forward has waited)
    for (int i = (int)rank * kProdThreads + tid; i < kTileRows * RP / 4; i += (int)C * kProdThreads) {
      const int row = i / (RP / 4), c = i % (RP / 4) * 4;
      const int slot = (int)sh.row_slot[row];
      if (slot < j0 || slot >= j0 + nj) continue;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      for (uint32_t k = 0; k < C; ++k) {
        const float4 t = ld_cluster_f32x4(sums + row * Cfg::PITCH + c, k);
        v.x += t.x;
        v.y += t.y;
        v.z += t.z;
        v.w += t.w;
      }
      const float s = p.scales ? p.scales[sh.row_id[row]] : 1.f;
      v.x *= s;
      v.y *= s;
      v.z *= s;
      v.w *= s;
      if (f.out32) {
        *reinterpret_cast<float4*>(f.out32 + (m0 + row) * RP + c) = v;
        const uint32_t b0 = __float_as_uint(fabsf(v.x)), b1 = __float_as_uint(fabsf(v.y));
        const uint32_t b2 = __float_as_uint(fabsf(v.z)), b3 = __float_as_uint(fabsf(v.w));
        const uint32_t lo = b0 > b1 ? b0 : b1, hi = b2 > b3 ? b2 : b3;
        atomicMax(&sh.slot_max[slot], lo > hi ? lo : hi);  // a NaN is above every number
      } else if (c < q.R8) {
        // one rounding to fp16: the tensor cores take y's second product in fp16
        const __half2 x = __floats2half2_rn(v.x, v.y), y = __floats2half2_rn(v.z, v.w);
        *reinterpret_cast<uint2*>(f.out16 + (m0 + row) * q.R8 + c) =
            make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
      }
    }
    fence_proxy_async_smem();   // TMA writes there next
    if (C > 1) cluster_sync();  // the peers' sums are read before they change or go
    else __syncthreads();
  }
  if (f.out32)
    for (int i = tid; i < n; i += kProdThreads)
      if (sh.slot_max[i]) atomicMax(f.amax + sh.list[i], sh.slot_max[i]);
}

template <int RP>
__global__ void __launch_bounds__(kProdThreads) lora_products_kernel(const __grid_constant__ Products q,
                                                                     const __grid_constant__ ProductMaps maps) {
  extern __shared__ uint8_t prod_smem[];
  __shared__ __align__(16) ProdShared sh;
  uint8_t* smem = prod_smem + ((1024u - (smem_u32(prod_smem) & 1023u)) & 1023u);
  const uint32_t rank = cluster_rank(), C = cluster_size();
  const int unit = (int)(blockIdx.x / C);
  // The operands were there before the kernel that this launch may overlap (the
  // plan started its dependents only once they were); a forward waits.
  if (q.lists.tile) pdl_wait();
  pdl_launch_dependents();
  const bool first = unit < q.tiles, second = !first && q.b.v && unit < 2 * q.tiles;
  if (!first && !second) {
    if (rank == 0) token_list(q.p, q.lists, unit - q.tiles);
    return;
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&sh.full[i], 1);
      mbar_init(&sh.done[i], 1);
    }
    fence_barrier_init();
  }
  if (threadIdx.x < 32) {
    tmem_alloc(&sh.tmem, ProdCfg<RP>::COLUMNS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (first) {
    product_tile<RP, false, true>(q, q.a, &maps.av, &maps.aw, unit, rank, C, smem, sh);
  } else if (q.b_tma) {
    product_tile<RP, true, true>(q, q.b, &maps.bv, &maps.bw, unit - q.tiles, rank, C, smem, sh);
  } else {
    product_tile<RP, true, false>(q, q.b, nullptr, nullptr, unit - q.tiles, rank, C, smem, sh);
  }
  tc_fence_before();
  __syncthreads();
  if (threadIdx.x < 32) {
    tc_fence_after();
    tmem_dealloc(sh.tmem, ProdCfg<RP>::COLUMNS);
  }
}

template <int RP>
cudaError_t launch_products(Products& q, int sm_count, bool pdl, cudaStream_t stream, std::string* err) {
  using Cfg = ProdCfg<RP>;
  static thread_local int configured_dev = -1;
  int dev = 0;
  cudaGetDevice(&dev);
  if (configured_dev != dev) {
    const cudaError_t e = cudaFuncSetAttribute(lora_products_kernel<RP>,
                                               cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::SMEM);
    if (e != cudaSuccess) return e;
    configured_dev = dev;
  }
  q.tiles = (int)((q.p.M + kTileRows - 1) / kTileRows);
  const LoraArgs& p = q.p;
  ProductMaps maps;
  std::memset(&maps, 0, sizeof(maps));
  {
    const uint64_t dims[3] = {(uint64_t)p.K, (uint64_t)p.R, (uint64_t)p.L};
    const uint64_t strides[2] = {(uint64_t)p.K * 2, (uint64_t)p.K * p.R * 2};
    const uint32_t box[3] = {kChunk, RP, 1};
    if (!encode_tmap_2d(&maps.av, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, q.a.v, (uint64_t)p.K, (uint64_t)p.M,
                        (uint64_t)q.a.ld * 2, kChunk, kTileRows, CU_TENSOR_MAP_SWIZZLE_128B, err) ||
        !encode_tmap_3d(&maps.aw, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, q.a.w, dims, strides, box,
                        CU_TENSOR_MAP_SWIZZLE_128B, err))
      return cudaErrorInvalidValue;
  }
  q.b_tma = q.b.v && q.b.ld % 8 == 0 && reinterpret_cast<uintptr_t>(q.b.v) % 16 == 0 && p.R % 8 == 0;
  if (q.b_tma) {
    const uint64_t dims[3] = {(uint64_t)p.R, (uint64_t)p.N, (uint64_t)p.L};
    const uint64_t strides[2] = {(uint64_t)p.R * 2, (uint64_t)p.R * p.N * 2};
    const uint32_t box[3] = {64, kChunk, 1};
    if (!encode_tmap_2d(&maps.bv, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, q.b.v, (uint64_t)p.N, (uint64_t)p.M,
                        (uint64_t)q.b.ld * 2, kChunk, kTileRows, CU_TENSOR_MAP_SWIZZLE_128B, err) ||
        !encode_tmap_3d(&maps.bw, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, q.b.w, dims, strides, box,
                        CU_TENSOR_MAP_SWIZZLE_128B, err))
      return cudaErrorInvalidValue;
  }
  const int products = q.b.v ? 2 : 1;
  int64_t most = (q.a.len + kChunk - 1) / kChunk;
  if (q.b.v && (q.b.len + kChunk - 1) / kChunk > most) most = (q.b.len + kChunk - 1) / kChunk;
  // two CTAs an SM from the clusters' splits
  int C = most < 8 ? (int)most : 8;
  while (C > 1 && (int64_t)products * q.tiles * C > 2 * sm_count) --C;
  const int64_t units = (int64_t)products * q.tiles + q.lists.tiles;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(units * C));
  cfg.blockDim = dim3(kProdThreads);
  cfg.dynamicSmemBytes = Cfg::SMEM;
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
  return cudaLaunchKernelEx(&cfg, lora_products_kernel<RP>, q, maps);
}

cudaError_t dispatch_products(Products& q, int sm_count, bool pdl, cudaStream_t stream, std::string* err) {
  if (q.p.R <= 16) return launch_products<16>(q, sm_count, pdl, stream, err);
  if (q.p.R <= 32) return launch_products<32>(q, sm_count, pdl, stream, err);
  if (q.p.R <= 64) return launch_products<64>(q, sm_count, pdl, stream, err);
  return launch_products<128>(q, sm_count, pdl, stream, err);
}
int padded_rank(int R) { return R <= 16 ? 16 : R <= 32 ? 32 : R <= 64 ? 64 : 128; }

// -------------------------------------------------------------------- plan
// Rows sorted by adapter (stable) and cut into chunks.  One CTA: each warp
// counts the adapters of its share of the rows, the counts become positions, and
// each warp places its rows; a warp owns its counters, so nothing is atomic.
struct Chunk {
  int adapter, start, count;  // rows order[start .. start + count)
  int index, of;              // which of the adapter's chunks
  int joint, slot0;           // of an adapter of several chunks: its place among those, and its first partial sum's
};
struct Plan {
  int* total;       // chunks
  Chunk* chunks;
  int* order;       // [M] rows by adapter
  uint32_t* amax;   // [2][L] largest magnitude of h and g, as fp32 bits
  uint32_t* count;  // [joint][tiles] chunks of a sum that are done
};

constexpr int kPlanThreads = 1024;

__device__ int block_scan(int v, int* warp_tot) {  // exclusive prefix over the CTA
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  int incl = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int t = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += t;
  }
  __syncthreads();
  if (lane == 31) warp_tot[warp] = incl;
  __syncthreads();
  int before = 0;
  for (int w = 0; w < warp; ++w) before += warp_tot[w];
  return before + incl - v;
}

__global__ void __launch_bounds__(kPlanThreads) lora_plan_kernel(const LoraArgs p, const Plan plan, int warps,
                                                                 int chunk_rows, int64_t counters) {
  extern __shared__ int hist[];  // [warps][L]
  __shared__ int warp_tot[32];
  pdl_wait();
  pdl_launch_dependents();
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  const int L = (int)p.L;
  for (int i = tid; i < 2 * L; i += kPlanThreads) plan.amax[i] = 0u;
  for (int64_t i = tid; i < counters; i += kPlanThreads) plan.count[i] = 0u;
  for (int i = tid; i < warps * L; i += kPlanThreads) hist[i] = 0;
  __syncthreads();
  const int64_t per = ((p.M + warps - 1) / warps + 31) / 32 * 32;
  const int64_t r0 = per * warp, r1 = r0 + per < p.M ? r0 + per : p.M;
  int* const mine = hist + warp * L;
  auto walk = [&](auto&& place) {
    if (warp >= warps) return;
    for (int64_t b = r0; b < r1; b += 32) {
      const int64_t m = b + lane;
      const int a = m < r1 ? (int)adapter_of(p, m) : -1;
      const uint32_t same = __match_any_sync(0xffffffffu, a);
      const int rank = __popc(same & ((1u << lane) - 1u));
      const int at = a >= 0 ? mine[a] : 0;
      __syncwarp();
      if (a >= 0 && rank == 0) mine[a] = at + __popc(same);
      __syncwarp();
      if (a >= 0) place(m, at + rank);
    }
  };
  walk([](int64_t, int) {});
  __syncthreads();
  constexpr int kPer = (int)kLoraMaxAdapters / kPlanThreads;
  int rows[kPer], sum = 0;
  for (int i = 0; i < kPer; ++i) {
    const int a = tid * kPer + i;
    rows[i] = 0;
    for (int w = 0; w < warps && a < L; ++w) rows[i] += hist[w * L + a];
    sum += rows[i];
  }
  int start = block_scan(sum, warp_tot);
  int cuts[kPer], n_cuts = 0, joints = 0, parts = 0;
  for (int i = 0; i < kPer; ++i) {
    cuts[i] = tid * kPer + i < L ? (rows[i] + chunk_rows - 1) / chunk_rows : 0;
    if (cuts[i] == 0 && tid * kPer + i < L) cuts[i] = 1;  // an adapter without rows has zeros to write
    n_cuts += cuts[i];
    joints += cuts[i] > 1;
    parts += cuts[i] > 1 ? cuts[i] : 0;
  }
  int chunk = block_scan(n_cuts, warp_tot);
  int joint = block_scan(joints, warp_tot);
  int slot = block_scan(parts, warp_tot);
  if (tid == kPlanThreads - 1) *plan.total = chunk + n_cuts;
  for (int i = 0; i < kPer; ++i) {
    const int a = tid * kPer + i;
    if (a >= L) break;
    for (int k = 0; k < cuts[i]; ++k) {
      const int left = rows[i] - k * chunk_rows;
      plan.chunks[chunk++] =
          Chunk{a, start + k * chunk_rows, left < chunk_rows ? left : chunk_rows, k, cuts[i], joint, slot};
    }
    joint += cuts[i] > 1;
    slot += cuts[i] > 1 ? cuts[i] : 0;
    for (int w = 0; w < warps; ++w) {  // counts to positions
      const int c = hist[w * L + a];
      hist[w * L + a] = start;
      start += c;
    }
  }
  __syncthreads();
  walk([&](int64_t m, int at) { plan.order[at] = (int)m; });
}

// -------------------------------------------------------------------- sums
// A chunk of an adapter's rows and 256 columns of x (dA, and dx of those rows)
// or of dy (dB) at a time, by a persistent grid.  Rows come 64 a step by
// cp.async, three steps deep, their h or g beside them.  Products run over rows,
// so both operands are read through transposing ldmatrix; D is [columns][ranks].
//
// The tensor cores take fp16, h and g are fp32: scaled by a power of two that
// puts the adapter's largest magnitude below 2^15, each is split into the nearest
// fp16 and the nearest fp16 of the rest (22 bits together) and both halves are
// multiplied, so dA and dB keep what an fp32 product would.
//
// A sum of several chunks is joined by the last CTA to finish one of them, from
// fp32 partial sums in chunk order, so that results do not depend on timing.
constexpr int kCols(int rp) { return rp > 64 ? 128 : 256; }  // columns of an item, 32 a warp
constexpr int kRows = 64;  // rows per step

struct Sums {
  LoraArgs p;
  const __half* dy;
  int64_t dy_ld;
  const float *h, *g;  // [M][RP]
  Plan plan;
  __half* dx;
  float *da, *db;
  float* part;         // [chunk of a joint sum][tiles][columns][RP]
  bool add_dx;
  int x_tiles, tiles;  // column tiles of x, and of x and dy together
};

template <int RT>
struct SumCfg {
  static constexpr int RP = 8 * RT;
  static constexpr int COLS = kCols(RP);
  static constexpr int THREADS = COLS;
  static constexpr int STAGES = 3;
  static constexpr int ROW = COLS * 2;              // bytes of a V or lora_a row, 16-byte pieces swizzled by row
  static constexpr int V_STAGE = kRows * ROW;
  static constexpr int G_STAGE = kRows * RP * 4;
  static constexpr int PITCH = RP * 2 + 16;          // of the split h or g, [64][RP] fp16
  static constexpr int OFF_G = STAGES * V_STAGE;
  static constexpr int OFF_HI = OFF_G + 2 * G_STAGE;  // a step's is free once it is split
  static constexpr int OFF_LO = OFF_HI + kRows * PITCH;
  static constexpr int OFF_A = OFF_LO + kRows * PITCH;  // lora_a [RP][columns]
  static constexpr int OFF_DX = OFF_A + RP * ROW;      // dx, [16 rows][32 columns] fp32 a warp
  static constexpr int SMEM = OFF_DX + THREADS / 32 * 16 * 32 * 4;
  static_assert(SMEM <= 227 * 1024, "shared memory budget");
};

template <int RT>
__global__ void __launch_bounds__(SumCfg<RT>::THREADS) lora_sums_kernel(const Sums q) {
  using Cfg = SumCfg<RT>;
  constexpr int RP = Cfg::RP, STAGES = Cfg::STAGES, COLS = Cfg::COLS, THREADS = Cfg::THREADS, PIECES = COLS / 8;
  extern __shared__ __align__(128) uint8_t sum_smem[];
  __shared__ int last;
  const LoraArgs& p = q.p;
  const uint32_t base = smem_u32(sum_smem);
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  pdl_wait();
  const int total = *q.plan.total;
  const int64_t items = (int64_t)total * q.tiles;
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const Chunk ck = q.plan.chunks[item / q.tiles];
    const int tile = (int)(item % q.tiles);
    const bool is_x = tile < q.x_tiles;
    const int64_t col0 = (int64_t)(is_x ? tile : tile - q.x_tiles) * COLS;
    const int64_t width = is_x ? p.K : p.N;
    const __half* v = is_x ? reinterpret_cast<const __half*>(p.x) : q.dy;
    const int64_t ld = is_x ? p.x_ld : q.dy_ld;
    const float* t = is_x ? q.g : q.h;
    float* out = is_x ? q.da : q.db;
    const bool want_dx = is_x && q.dx;
    if (!out && !want_dx) continue;
    const bool v16 = ld % 8 == 0 && width % 8 == 0 && (reinterpret_cast<uintptr_t>(v) & 15) == 0;
    // 2^e brings the largest magnitude into [2^14, 2^15); nothing to scale by where it is 0 or not finite
    const uint32_t top = q.plan.amax[(is_x ? p.L : 0) + ck.adapter];
    int e = top == 0u || top >= 0x7F800000u ? 0 : 14 - ((int)(top >> 23) - 127);
    e = e > 126 ? 126 : (e < -126 ? -126 : e);
    const float up = __uint_as_float((uint32_t)(127 + e) << 23), down = __uint_as_float((uint32_t)(127 - e) << 23);

    auto load = [&](int step) {
      const int s = step % STAGES;
#pragma unroll
      for (int k = 0; k < kRows * PIECES / THREADS; ++k) {
        const int row = (k * THREADS + tid) / PIECES, piece = tid % PIECES;
        const int64_t c = col0 + piece * 8;
        const bool in = step * kRows + row < ck.count && c < width;
        const __half* src = v + (in ? q.plan.order[ck.start + step * kRows + row] * ld + c : 0);
        const uint32_t at = base + s * Cfg::V_STAGE + row * Cfg::ROW + ((piece ^ (row & 7)) << 4);
        if (v16) cp_async16(at, src, in);
        else sts16(at, load_halves(src, in ? width - c : 0));
      }
#pragma unroll
      for (int k = 0; k < kRows * RP / 4 / THREADS; ++k) {
        const int i = k * THREADS + tid, row = i / (RP / 4), piece = i % (RP / 4);
        const bool in = step * kRows + row < ck.count;
        const float* src = t + (in ? (int64_t)q.plan.order[ck.start + step * kRows + row] * RP + piece * 4 : 0);
        cp_async16(base + Cfg::OFF_G + (step % 2) * Cfg::G_STAGE + i * 16, src, in);
      }
    };
    const int steps = (ck.count + kRows - 1) / kRows;
    __syncthreads();  // the item before has left shared memory
    if (want_dx) {    // with the first step's group
#pragma unroll
      for (int k = 0; k < RP * PIECES / THREADS; ++k) {
        const int i = k * THREADS + tid, r = i / PIECES, piece = i % PIECES;
        const bool in = r < p.R && col0 + piece * 8 < width;
        const __half* src = reinterpret_cast<const __half*>(p.a) +
                            (in ? ((int64_t)ck.adapter * p.R + r) * p.K + col0 + piece * 8 : 0);
        cp_async16(base + Cfg::OFF_A + r * Cfg::ROW + ((piece ^ (r & 7)) << 4), src, in);
      }
    }
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s) {
      if (s < steps) load(s);
      cp_async_commit();
    }
    float acc[2][RT][4];  // columns 32 warp + 16 i + .., ranks
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int r = 0; r < RT; ++r) acc[i][r][0] = acc[i][r][1] = acc[i][r][2] = acc[i][r][3] = 0.f;
    for (int step = 0; step < steps; ++step) {
      cp_async_wait<STAGES - 2>();
      __syncthreads();
      // split h or g
      const uint32_t gs = base + Cfg::OFF_G + (step % 2) * Cfg::G_STAGE;
#pragma unroll
      for (int k = 0; k < kRows * RP / 4 / THREADS; ++k) {
        const int i = k * THREADS + tid, row = i / (RP / 4), c = i % (RP / 4) * 4;
        float f[4];
        asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                     : "=f"(f[0]), "=f"(f[1]), "=f"(f[2]), "=f"(f[3])
                     : "r"(gs + i * 16)
                     : "memory");
        __half hi[4], lo[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          f[x] *= up;
          hi[x] = __float2half_rn(f[x]);
          lo[x] = __float2half_rn(f[x] - __half2float(hi[x]));
        }
        auto pack = [](const __half (&h)[4]) {
          return make_uint2((uint32_t)__half_as_ushort(h[0]) | ((uint32_t)__half_as_ushort(h[1]) << 16),
                            (uint32_t)__half_as_ushort(h[2]) | ((uint32_t)__half_as_ushort(h[3]) << 16));
        };
        const uint2 a = pack(hi), b = pack(lo);
        asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(base + Cfg::OFF_HI + row * Cfg::PITCH + c * 2), "r"(a.x),
                     "r"(a.y)
                     : "memory");
        asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(base + Cfg::OFF_LO + row * Cfg::PITCH + c * 2), "r"(b.x),
                     "r"(b.y)
                     : "memory");
      }
      __syncthreads();
      if (step + STAGES - 1 < steps) load(step + STAGES - 1);
      cp_async_commit();
      const uint32_t vs = base + (step % STAGES) * Cfg::V_STAGE;
      if (out) {
#pragma unroll
        for (int kk = 0; kk < kRows / 16; ++kk) {
          uint32_t a[2][4];
#pragma unroll
          for (int i = 0; i < 2; ++i) {  // V^T: [16 columns][16 rows]
            const int row = kk * 16 + (lane >> 4) * 8 + (lane & 7);
            const int piece = warp * 4 + i * 2 + ((lane >> 3) & 1);
            ldmatrix_x4_trans(vs + row * Cfg::ROW + ((piece ^ (row & 7)) << 4), a[i][0], a[i][1], a[i][2], a[i][3]);
          }
          const int row = kk * 16 + ((lane >> 3) & 1) * 8 + (lane & 7);
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const uint32_t ts = base + (half ? Cfg::OFF_LO : Cfg::OFF_HI) + row * Cfg::PITCH + (lane >> 4) * 16;
#pragma unroll
            for (int r = 0; r < RT; r += 2) {
              uint32_t b[4];
              ldmatrix_x4_trans(ts + r * 16, b[0], b[1], b[2], b[3]);
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                mma_16816(acc[i][r], a[i][0], a[i][1], a[i][2], a[i][3], b[0], b[1]);
                mma_16816(acc[i][r + 1], a[i][0], a[i][1], a[i][2], a[i][3], b[2], b[3]);
              }
            }
          }
        }
      }
      if (want_dx) {
        // dx of the step's rows: [64 rows][32 columns] a warp, ranks the reduction
#pragma unroll 1
        for (int mt = 0; mt < kRows / 16; ++mt) {
          if (step * kRows + mt * 16 >= ck.count) break;
          float d[4][4];
#pragma unroll
          for (int c = 0; c < 4; ++c) d[c][0] = d[c][1] = d[c][2] = d[c][3] = 0.f;
#pragma unroll
          for (int kk = 0; kk < RP / 16; ++kk) {
            uint32_t hi[4], lo[4];
            const uint32_t at = (uint32_t)((mt * 16 + (lane & 15)) * Cfg::PITCH + kk * 32 + (lane >> 4) * 16);
            ldmatrix_x4(base + Cfg::OFF_HI + at, hi[0], hi[1], hi[2], hi[3]);
            ldmatrix_x4(base + Cfg::OFF_LO + at, lo[0], lo[1], lo[2], lo[3]);
#pragma unroll
            for (int c = 0; c < 4; c += 2) {
              uint32_t b[4];
              const int r = kk * 16 + ((lane >> 3) & 1) * 8 + (lane & 7), piece = warp * 4 + c + (lane >> 4);
              ldmatrix_x4_trans(base + Cfg::OFF_A + r * Cfg::ROW + ((piece ^ (r & 7)) << 4), b[0], b[1], b[2], b[3]);
              mma_16816(d[c], hi[0], hi[1], hi[2], hi[3], b[0], b[1]);
              mma_16816(d[c + 1], hi[0], hi[1], hi[2], hi[3], b[2], b[3]);
              mma_16816(d[c], lo[0], lo[1], lo[2], lo[3], b[0], b[1]);
              mma_16816(d[c + 1], lo[0], lo[1], lo[2], lo[3], b[2], b[3]);
            }
          }
          // through shared memory (this warp's 64 bytes of each row) into rows of 16-byte stores
          float* stage = reinterpret_cast<float*>(sum_smem + Cfg::OFF_DX) + warp * 16 * 32;  // [16][32] fp32
          __syncwarp();
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int row = lane / 4 + 8 * h, col = c * 8 + (lane % 4) * 2;
              *reinterpret_cast<float2*>(stage + row * 32 + (col ^ ((row & 7) << 2))) =
                  make_float2(d[c][2 * h] * down, d[c][2 * h + 1] * down);
            }
          __syncwarp();
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const int i = k * 32 + lane, row = i / 4, col = i % 4 * 8;  // 8 columns a lane
            const int at = step * kRows + mt * 16 + row;
            const int64_t cg = col0 + warp * 32 + col;
            if (at < ck.count && cg < width) {
              uint4* dst = reinterpret_cast<uint4*>(q.dx + q.plan.order[ck.start + at] * p.K + cg);
              uint4 old = make_uint4(0u, 0u, 0u, 0u);
              if (q.add_dx) old = *dst;
              uint32_t* o = &old.x;
#pragma unroll
              for (int x = 0; x < 4; ++x) {
                const float2 f = *reinterpret_cast<const float2*>(stage + row * 32 + ((col + 2 * x) ^ ((row & 7) << 2)));
                float2 s = __half22float2(*reinterpret_cast<const __half2*>(&o[x]));
                s.x += f.x;
                s.y += f.y;
                const __half2 r = __floats2half2_rn(s.x, s.y);
                o[x] = *reinterpret_cast<const uint32_t*>(&r);
              }
              *dst = old;
            }
          }
        }
      }
    }
    cp_async_wait<0>();
    if (!out) continue;
    // D[column][rank] of this chunk, then the sum's
    auto put = [&](auto&& f) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
          for (int h = 0; h < 2; ++h) f(warp * 32 + i * 16 + lane / 4 + 8 * h, r * 8 + (lane % 4) * 2, acc[i][r] + 2 * h);
    };
    if (ck.of > 1) {
      const int64_t sum = (int64_t)ck.joint * q.tiles + tile;
      // slot of the adapter's first chunk; its next ones follow, q.tiles apart
      float* slots = q.part + ((int64_t)ck.slot0 * q.tiles + tile) * COLS * RP;
      const int64_t apart = (int64_t)q.tiles * COLS * RP;
      put([&](int c, int r, float* a) {
        __stcg(reinterpret_cast<float2*>(slots + ck.index * apart + c * RP + r), make_float2(a[0], a[1]));
      });
      __threadfence();
      __syncthreads();
      if (tid == 0) last = atomicAdd(q.plan.count + sum, 1u) == (uint32_t)ck.of - 1;
      __syncthreads();
      if (!last) continue;
      __threadfence();
      put([&](int c, int r, float* a) {
        float2 s = make_float2(0.f, 0.f);
        for (int k = 0; k < ck.of; ++k) {
          const float2 x = __ldcg(reinterpret_cast<const float2*>(slots + k * apart + c * RP + r));
          s.x += x.x;
          s.y += x.y;
        }
        a[0] = s.x;
        a[1] = s.y;
      });
    }
    const int64_t a0 = (int64_t)ck.adapter * p.R * width;
    put([&](int c, int r, float* a) {
      if (col0 + c >= width) return;
#pragma unroll
      for (int x = 0; x < 2; ++x)
        if (r + x < p.R)
          out[is_x ? a0 + (int64_t)(r + x) * width + col0 + c : a0 + (col0 + c) * p.R + r + x] = a[x] * down;
    });
  }
}

constexpr size_t align256(size_t v) { return (v + 255) & ~(size_t)255; }

// How a gradient call is cut: chunks long enough that the column tiles alone
// fill the GPU, shorter ones only where they would not.
struct GradSpace {
  int RP, x_tiles, tiles, chunk_rows;
  int64_t max_chunks, joints;
  size_t h, g, chunks, order, amax, count, part, end;
};
GradSpace grad_space(int64_t M, int64_t N, int64_t K, int R, int64_t L, int sm_count) {
  GradSpace s;
  s.RP = padded_rank(R);
  const int cols = kCols(s.RP);
  s.x_tiles = (int)((K + cols - 1) / cols);
  s.tiles = s.x_tiles + (int)((N + cols - 1) / cols);
  // about two items an SM
  int64_t cuts = (2 * (int64_t)sm_count + s.tiles - 1) / s.tiles;
  const int64_t most = (M + kRows - 1) / kRows;
  cuts = cuts > most ? most : cuts;
  cuts = cuts < 1 ? 1 : cuts;
  s.chunk_rows = (int)(((M + cuts - 1) / cuts + kRows - 1) / kRows * kRows);
  if (s.chunk_rows < kRows) s.chunk_rows = kRows;
  s.max_chunks = M / s.chunk_rows + L;
  s.joints = M / (s.chunk_rows + 1);  // adapters of more than chunk_rows rows
  if (s.joints > L) s.joints = L;
  const int64_t parts = s.joints ? M / s.chunk_rows + s.joints : 0;  // their chunks
  size_t at = 256;  // the chunks' total
  auto take = [&](size_t bytes) {
    const size_t was = at;
    at += align256(bytes);
    return was;
  };
  s.h = take((size_t)M * s.RP * sizeof(float));
  s.g = take((size_t)M * s.RP * sizeof(float));
  s.chunks = take((size_t)s.max_chunks * sizeof(Chunk));
  s.order = take((size_t)M * sizeof(int));
  s.amax = take((size_t)2 * L * sizeof(uint32_t));
  s.count = take((size_t)s.joints * s.tiles * sizeof(uint32_t));
  s.part = take((size_t)parts * s.tiles * cols * s.RP * sizeof(float));
  s.end = at;
  return s;
}

template <int RT>
cudaError_t launch_sums(const Sums& q, int64_t items, int sm_count, bool pdl, cudaStream_t stream) {
  using Cfg = SumCfg<RT>;
  static thread_local int configured_dev = -1, per_sm = 1;
  int dev = 0;
  cudaGetDevice(&dev);
  if (configured_dev != dev) {
    cudaError_t e = cudaFuncSetAttribute(lora_sums_kernel<RT>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::SMEM);
    if (e == cudaSuccess)
      e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, lora_sums_kernel<RT>, Cfg::THREADS, Cfg::SMEM);
    if (e != cudaSuccess) return e;
    if (per_sm < 1) return cudaErrorInvalidConfiguration;
    configured_dev = dev;
  }
  const int64_t grid = items < (int64_t)sm_count * per_sm ? items : (int64_t)sm_count * per_sm;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(Cfg::THREADS);
  cfg.dynamicSmemBytes = Cfg::SMEM;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, lora_sums_kernel<RT>, q);
}

}  // namespace

cudaError_t launch_lora_products(const LoraArgs& p, const TokenLists& lists, void* h16, unsigned int* status,
                                 int sm_count, bool pdl, cudaStream_t stream, std::string* err) {
  Products q{};
  q.p = p;
  q.R8 = (p.R + 7) / 8 * 8;
  q.a.v = static_cast<const __half*>(p.x);
  q.a.ld = p.x_ld;
  q.a.len = p.K;
  q.a.w = static_cast<const __half*>(p.a);
  q.a.out16 = static_cast<__half*>(h16);
  q.lists = lists;
  q.status = status;
  return dispatch_products(q, sm_count, pdl, stream, err);
}

size_t lora_backward_bytes(int64_t M, int64_t N, int64_t K, int64_t R, int64_t L, int sm_count) {
  return grad_space(M, N, K, (int)R, L, sm_count).end;
}

cudaError_t launch_lora_backward(const LoraArgs& p, const LoraGrads& g, void* ws, int sm_count, bool pdl,
                                 cudaStream_t stream, std::string* err) {
  cudaError_t e;
  const GradSpace s = grad_space(p.M, p.N, p.K, p.R, p.L, sm_count);
  uint8_t* base = static_cast<uint8_t*>(ws);
  if (p.L == 0) {  // nobody has an adapter
    return g.dx && !g.add_dx && p.M ? cudaMemsetAsync(g.dx, 0, (size_t)p.M * p.K * sizeof(__half), stream)
                                    : cudaSuccess;
  }
  Plan plan;
  plan.total = reinterpret_cast<int*>(base);
  plan.chunks = reinterpret_cast<Chunk*>(base + s.chunks);
  plan.order = reinterpret_cast<int*>(base + s.order);
  plan.amax = reinterpret_cast<uint32_t*>(base + s.amax);
  plan.count = reinterpret_cast<uint32_t*>(base + s.count);
  {
    // a warp's counters for every adapter; as many warps as fit 192 KB
    int warps = (int)(192 * 1024 / (p.L * 4));
    warps = warps > 32 ? 32 : warps;
    static thread_local int configured_dev = -1;
    int dev = 0;
    cudaGetDevice(&dev);
    if (configured_dev != dev) {
      e = cudaFuncSetAttribute(lora_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 192 * 1024);
      if (e != cudaSuccess) return e;
      configured_dev = dev;
    }
    lora_plan_kernel<<<1, kPlanThreads, (size_t)warps * p.L * 4, stream>>>(p, plan, warps, s.chunk_rows,
                                                                          s.joints * s.tiles);
    if ((e = cudaGetLastError()) != cudaSuccess) return e;
  }
  if (p.M) {
    Products q{};
    q.p = p;
    q.R8 = (p.R + 7) / 8 * 8;
    q.a.v = static_cast<const __half*>(p.x);
    q.a.ld = p.x_ld;
    q.a.len = p.K;
    q.a.w = static_cast<const __half*>(p.a);
    q.a.out32 = reinterpret_cast<float*>(base + s.h);
    q.a.amax = plan.amax;
    q.b.v = static_cast<const __half*>(g.dy);
    q.b.ld = g.dy_ld;
    q.b.len = p.N;
    q.b.w = static_cast<const __half*>(p.b);
    q.b.out32 = reinterpret_cast<float*>(base + s.g);
    q.b.amax = plan.amax + p.L;
    q.status = g.status;
    q.dx_zero = g.add_dx ? nullptr : static_cast<__half*>(g.dx);
    if ((e = dispatch_products(q, sm_count, pdl, stream, err)) != cudaSuccess) return e;
  }
  Sums q{};
  q.p = p;
  q.dy = static_cast<const __half*>(g.dy);
  q.dy_ld = g.dy_ld;
  q.h = reinterpret_cast<const float*>(base + s.h);
  q.g = reinterpret_cast<const float*>(base + s.g);
  q.plan = plan;
  q.dx = static_cast<__half*>(g.dx);
  q.da = g.da;
  q.db = g.db;
  q.part = reinterpret_cast<float*>(base + s.part);
  q.add_dx = g.add_dx;
  q.x_tiles = s.x_tiles;
  q.tiles = s.tiles;
  const int64_t items = s.max_chunks * s.tiles;
  if (p.R <= 16) return launch_sums<2>(q, items, sm_count, pdl, stream);
  if (p.R <= 32) return launch_sums<4>(q, items, sm_count, pdl, stream);
  if (p.R <= 64) return launch_sums<8>(q, items, sm_count, pdl, stream);
  return launch_sums<16>(q, items, sm_count, pdl, stream);
}

}  // namespace qw
