// qw_lora_grad.cu -- gradient of the adapters beside a projection (and the
// rank-space product of a forward with many rows of a high rank):
//   h = s x A^T, g = s dy B                    per row, its adapter's A, B, s
//   dA = g^T x, dB = dy^T h                    sums over the adapter's rows
//   dx = g A (+ dx)
// Three launches, chained by programmatic dependent launch:
//   products h and g, fp32, and the largest magnitude of each by tile and adapter;
//            one more CTA sorts the rows by adapter and cuts each adapter's rows
//            into chunks (the plan);
//   split    h and g of the sorted rows as two fp16 terms, laid out as the tensor
//            cores take them from shared memory;
//   sums     dA, dB and dx, a chunk of rows and 128 columns at a time.
// (dy of odd width and lora_b of odd rank are first laid out anew.)  x and dy are
// read twice, once across their width and once along their rows; everything else
// is rank-sized.
#include <cuda_fp16.h>

#include <cstring>

#include "qw_internal.h"
#include "qw_lora.cuh"
#include "qw_ptx.cuh"

namespace qw {

namespace {

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

// -------------------------------------------------------------------- plan
// Rows sorted by adapter (stable) and cut into chunks of whole steps (128 rows).
// One CTA: each warp counts the adapters of its share of the rows, the counts
// become positions, and each warp places its rows; a warp owns its counters, so
// nothing is atomic.
constexpr int kStepRows = 128;
struct Chunk {
  int adapter, start, count;  // rows order[start .. start + count)
  int step0;                  // first of its steps
  int index, of;              // which of the adapter's chunks
  int joint, slot0;           // of an adapter of several chunks: its place among those, and its first partial sum's
};
struct Step {
  int adapter, start, rows;  // rows order[start .. start + rows)
  int chunk;                 // whose first step it is, else -1
};
struct PlanArgs {
  int* total;         // chunks, and steps
  Chunk* chunks;
  Step* steps;
  int* order;         // [M] rows by adapter
  uint32_t* count;    // [joint][tiles] chunks of a sum that are done
  int64_t counters;
  int chunk_rows;
};
constexpr int kPlanWarps = 4;

// Exclusive prefix over the CTA's 128 threads, and their total.
__device__ __forceinline__ int block_scan(int v, int* warp_tot, int* total) {
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
  int before = 0, all = 0;
  for (int w = 0; w < kPlanWarps; ++w) {
    before += w < warp ? warp_tot[w] : 0;
    all += warp_tot[w];
  }
  *total = all;
  return before + incl - v;
}

__device__ void make_plan(const LoraArgs& p, const PlanArgs& plan, int* hist) {  // hist [kPlanWarps][L]
  __shared__ int warp_tot[kPlanWarps];
  constexpr int kThreads = kPlanWarps * 32;
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  const int L = (int)p.L;
  for (int64_t i = tid; i < plan.counters; i += kThreads) plan.count[i] = 0u;
  for (int i = tid; i < kPlanWarps * L; i += kThreads) hist[i] = 0;
  __syncthreads();
  const int64_t per = ((p.M + kPlanWarps - 1) / kPlanWarps + 31) / 32 * 32;
  const int64_t r0 = per * warp, r1 = r0 + per < p.M ? r0 + per : p.M;
  int* const mine = hist + warp * L;
  auto walk = [&](auto&& place) {
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
  int start0 = 0, chunk0 = 0, step0 = 0, joint0 = 0, slot0 = 0;  // of the adapters before
  for (int base = 0; base < L; base += kThreads) {
    const int a = base + tid;
    int rows = 0;
    for (int w = 0; w < kPlanWarps && a < L; ++w) rows += hist[w * L + a];
    // an adapter without rows has zeros to write
    const int cuts = a < L ? (rows > 0 ? (rows + plan.chunk_rows - 1) / plan.chunk_rows : 1) : 0;
    const int steps = (rows + kStepRows - 1) / kStepRows;  // chunks are whole steps
    int total;
    int start = start0 + block_scan(rows, warp_tot, &total);
    start0 += total;
    int chunk = chunk0 + block_scan(cuts, warp_tot, &total);
    chunk0 += total;
    int step = step0 + block_scan(steps, warp_tot, &total);
    step0 += total;
    const int joint = joint0 + block_scan(cuts > 1, warp_tot, &total);
    joint0 += total;
    const int slot = slot0 + block_scan(cuts > 1 ? cuts : 0, warp_tot, &total);
    slot0 += total;
    for (int k = 0; k < cuts; ++k) {
      const int left = rows - k * plan.chunk_rows;
      const int count = left < plan.chunk_rows ? left : plan.chunk_rows;
      plan.chunks[chunk] = Chunk{a, start + k * plan.chunk_rows, count, step, k, cuts, joint, slot};
      for (int i = 0; i < count; i += kStepRows)
        plan.steps[step++] = Step{a, start + k * plan.chunk_rows + i, count - i < kStepRows ? count - i : kStepRows,
                                  i == 0 ? chunk : -1};
      ++chunk;
    }
    for (int w = 0; w < kPlanWarps && a < L; ++w) {  // counts to positions
      const int c = hist[w * L + a];
      hist[w * L + a] = start;
      start += c;
    }
  }
  if (tid == 0) {
    plan.total[0] = chunk0;
    plan.total[1] = step0;
  }
  __syncthreads();
  walk([&](int64_t m, int at) { plan.order[at] = (int)m; });
}

// Rows of `width` halves, laid out anew `pitch` apart (a multiple of 8, zero
// behind the width): what TMA cannot take as it is.
struct Repack {
  const __half* src;
  __half* dst;  // null: nothing to do
  int64_t rows, width, ld, pitch;
};
__device__ __forceinline__ void repack(const Repack& r) {
  const int64_t pieces = r.pitch / 8;
  const int64_t step = (int64_t)gridDim.x * blockDim.x;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < r.rows * pieces; i += step) {
    const int64_t row = i / pieces, c = i % pieces * 8;
    *reinterpret_cast<uint4*>(r.dst + row * r.pitch + c) = load_halves(r.src + row * r.ld + c, r.width - c);
  }
}
__global__ void __launch_bounds__(256) lora_repack_kernel(const Repack dy, const Repack b) {
  if (dy.dst) repack(dy);
  if (b.dst) repack(b);
}

// ---------------------------------------------------------------- products
// v W of each row's adapter, a tile of 128 rows at a time: out[m][r] = s sum_i
// v[m][i] W[i][r].  HBM-bound by v, which is read once; short batches are bound by
// the chain of loads, products and the cluster's sum.
//
// A cluster takes a tile and its CTAs split the reduction; a CTA walks 64 values
// of it at a time, three steps of TMA loads deep, and within those the adapters
// that the tile's rows name, two a step (one above rank 64), so v is staged once
// however mixed the rows are.  Every adapter has columns of its own in TMEM (eight
// adapters at a time, four above rank 32, two above 64) and a row reads those of
// its own adapter: no row's sum ever meets another adapter's values.  Sums over
// the cluster go through distributed shared memory in rank order.
// x of 4096 x 17408 and dy of 4096 x 5120, rank 64: 53 us, 3.5 TB/s; one adapter a
// step took 63, as tiles of several adapters were last.
constexpr int kStages = 3;
constexpr int kProdThreads = 128;
constexpr int kChunk = 64;  // reduction values per step
constexpr int kTileRows = 128;
constexpr int kMaxSplit = 16;  // CTAs of a cluster

struct Product {
  const __half* v;  // [M][len], rows ld apart
  int64_t ld, len;
  const __half* w;  // [L][R][len], or for the second product [L][len][R8]
  float* out32;     // [M][RP] fp32, RP the kernel's padded rank (null: out16)
  __half* out16;    // [M][R8] fp16, zero-padded rank, and
  float* full;      // [M][R8] fp32, where that is not finite
  uint32_t* top;    // [tiles][kMaxSplit][kTileRows] largest magnitude of out32 by adapter, as fp32 bits
};
struct Products {
  LoraArgs p;
  Product a, b;      // b.v null: one product
  __half* dx_zero;   // [M][K]: rows without an adapter are cleared (nullable)
  int R8;
  int tiles, split;  // row tiles and CTAs of a tile's cluster, filled at the launch
  uint32_t* tile_ids;  // gradient: adapters of each row tile (0xFFFFFFFF: no more), [tiles][kTileRows]
  PlanArgs plan;     // gradient (plan.total null: none)
  TokenLists lists;  // forward
  unsigned int* status;
};

template <int RP>
struct ProdCfg {
  static constexpr int BLOCK = RP > 64 ? 128 : 64;    // ranks in a step's rows of w
  static constexpr int PITCH_T = RP < 32 ? 32 : RP;   // TMEM columns of an adapter
  static constexpr int COLUMNS = 256;                 // two CTAs an SM
  static constexpr int GROUP = COLUMNS / PITCH_T;     // adapters at a time
  static constexpr int V_STAGE = kTileRows * 128;
  static constexpr int W_STAGE = 64 * BLOCK * 2;
  static constexpr int PER = RP > 64 ? 1 : 2;         // adapters a step
  static constexpr int STAGE = V_STAGE + PER * W_STAGE;
  static constexpr int PITCH = RP + 4;                // floats of a row of sums
  static constexpr int SUMS = kTileRows * PITCH * 4;
  static constexpr int SMEM = (kStages * STAGE > SUMS ? kStages * STAGE : SUMS) + 1024;
  static_assert(SMEM <= 112 * 1024, "two CTAs an SM");
};

struct ProductMaps {
  CUtensorMap av, aw, bv, bw;  // operands of the two products: v [M][len], w 3-D
};
struct ProdShared {
  uint32_t row_id[kTileRows], row_slot[kTileRows], list[2 * kTileRows], slot_max[kTileRows];
  uint64_t full[kStages], done[kStages], drained;
  int list_n;
  uint32_t tmem;
};

template <int RP, bool TRANS>
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
  const bool none = my_id == 0xFFFFFFFFu;
  const bool some_none = __syncthreads_or(none && m0 + tid < p.M);
  {  // one adapter in the whole tile, mostly
    const uint32_t low = __reduce_min_sync(0xffffffffu, my_id);
    if (lane == 0) sh.list[warp] = low;
  }
  __syncthreads();
  const uint32_t low = min(min(sh.list[0], sh.list[1]), min(sh.list[2], sh.list[3]));
  if (__syncthreads_and(none || my_id == low)) {
    sh.row_slot[tid] = none ? my_id : 0u;
    if (tid == 0) {
      sh.list[0] = low;
      sh.list_n = low != 0xFFFFFFFFu;
    }
    __syncthreads();
  } else {
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
  if (!TRANS && q.dx_zero && some_none) {  // rows without an adapter
    for (int row = warp; row < kTileRows && m0 + row < p.M; row += kProdThreads / 32) {
      if (sh.row_id[row] != 0xFFFFFFFFu) continue;
      uint4* dst = reinterpret_cast<uint4*>(q.dx_zero + (m0 + row) * p.K);
      for (int64_t c = rank * 32 + lane; c < p.K / 8; c += C * 32) dst[c] = make_uint4(0u, 0u, 0u, 0u);
    }
  }
  if (!TRANS && f.out32 && rank == 0)  // for the split
    q.tile_ids[(int64_t)tile * kTileRows + tid] = tid < n ? sh.list[tid] : 0xFFFFFFFFu;
  if (n == 0) return;  // the whole cluster: nobody's rows

  const int chunks = (int)((f.len + kChunk - 1) / kChunk);
  const int c0 = (int)((int64_t)chunks * rank / C), c1 = (int)((int64_t)chunks * (rank + 1) / C);
  const uint32_t base = smem_u32(smem);
  bool ok = true;        // false: a bounded wait ran out, nothing more is loaded or multiplied
  uint32_t it0 = 0, vit0 = 0;  // steps and chunks of earlier rounds
  uint32_t issued = 0;         // steps loaded, by the thread that loads
  constexpr uint32_t kDesc = mma_desc(kTileRows, RP, false, TRANS);
  // Few adapters: two sums of every other chunk, as the tensor cores' additions
  // truncate and an error grows with the number that follow one another.
  constexpr int kHalf = Cfg::GROUP / 2;
  bool two = false;
  auto multiply = [&](int chunk, int j, uint32_t vs, uint32_t ws) {
    const uint64_t a = operand_k(vs), b = TRANS ? operand_mn(ws, 8192) : operand_k(ws);
    const int col = (j + (two && (chunk & 1) ? kHalf : 0)) * Cfg::PITCH_T;
#pragma unroll
    for (int kk = 0; kk < kChunk / 16; ++kk)
      tc_mma_ss(sh.tmem + col, a + (uint64_t)(2 * kk), b + (uint64_t)((TRANS ? 128 : 2) * kk), kDesc,
                chunk > (two ? 1 : 0) || kk > 0);
  };

  for (int j0 = 0; j0 < n; j0 += Cfg::GROUP) {
    const int nj = n - j0 < Cfg::GROUP ? n - j0 : Cfg::GROUP;
    const int steps = (c1 - c0) * ((nj + Cfg::PER - 1) / Cfg::PER);
    two = nj <= kHalf && c1 - c0 > 1;
    const bool working = ok;
    if (warp == 1 && lane == 0 && working) {  // loads
      uint32_t it = it0, vit = vit0;
      for (int c = c0; c < c1 && ok; ++c, ++vit) {
        for (int j = 0; j < nj; j += Cfg::PER, ++it) {
          const uint32_t s = it % kStages;
          const int here = nj - j < Cfg::PER ? nj - j : Cfg::PER;
          if (it >= kStages) {
            ok = mbar_wait(&sh.done[s], (it / kStages - 1) & 1, q.status, kDevTimeoutEmpty);
            if (!ok) break;
          }
          mbar_arrive_expect_tx(&sh.full[s], (uint32_t)((j == 0 ? Cfg::V_STAGE : 0) +
                                                        here * (TRANS ? Cfg::W_STAGE : RP * 128)));
          if (j == 0)
            tma_load_2d(smem + (vit % kStages) * Cfg::STAGE, map_v, &sh.full[s], c * kChunk, (int)m0);
          for (int i = 0; i < here; ++i) {
            uint8_t* dst = smem + s * Cfg::STAGE + Cfg::V_STAGE + i * Cfg::W_STAGE;
            const int a = (int)sh.list[j0 + j + i];
            if (TRANS) {
              for (int b = 0; b < Cfg::BLOCK / 64; ++b)
                tma_load_3d(dst + b * 8192, map_w, &sh.full[s], b * 64, c * kChunk, a);
            } else {
              tma_load_3d(dst, map_w, &sh.full[s], c * kChunk, 0, a);
            }
          }
          issued = it + 1;
        }
      }
    } else if (warp == 0 && lane == 0 && working) {  // products
      uint32_t it = it0, vit = vit0;
      for (int c = c0; c < c1 && ok; ++c, ++vit) {
        for (int j = 0; j < nj; j += Cfg::PER, ++it) {
          const uint32_t s = it % kStages;
          ok = mbar_wait(&sh.full[s], (it / kStages) & 1, q.status, kDevTimeoutFull);
          if (!ok) break;
          tc_fence_after();
          for (int i = 0; i < Cfg::PER && j + i < nj; ++i)
            multiply(c - c0, j + i, base + (vit % kStages) * Cfg::STAGE,
                     base + s * Cfg::STAGE + Cfg::V_STAGE + i * Cfg::W_STAGE);
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
    ok = !__syncthreads_or(!ok);
    if (working && !ok) {  // loads and products under way end before their memory goes
      if (tid == 0) {
        tc_commit(&sh.drained);
        mbar_wait(&sh.drained, 0, q.status, kDevTimeoutAccum);
      }
      for (uint32_t u = issued < kStages ? 0 : issued - kStages; u < issued; ++u)
        mbar_wait(&sh.full[u % kStages], (u / kStages) & 1, q.status, kDevTimeoutFull);
      __syncthreads();
    }
    tc_fence_after();

    // each row's own columns, to shared memory
    float* const sums = reinterpret_cast<float*>(smem);
    for (int b = 0; b < nj; ++b) {
      const bool own = my_slot == j0 + b;
      if (!__any_sync(0xffffffffu, own)) continue;
#pragma unroll
      for (int c = 0; c < RP; c += 16) {
        uint32_t v[16];
        __syncwarp();  // tcgen05.ld takes a whole warp, stores below are some lanes'
        if (steps > 0) {
          const uint32_t at = sh.tmem + ((uint32_t)(warp * 32) << 16) + b * Cfg::PITCH_T + c;
          tmem_ld_32x32b_x16(at, v);
          tmem_wait_ld();
          if (two) {
            uint32_t w[16];
            tmem_ld_32x32b_x16(at + kHalf * Cfg::PITCH_T, w);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) + __uint_as_float(w[i]));
          }
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
    for (int i = (int)rank * kProdThreads + tid; i < kTileRows * RP / 4; i += (int)C * kProdThreads) {
      const int row = i / (RP / 4), c = i % (RP / 4) * 4;
      const int slot = (int)sh.row_slot[row];
      if (slot < j0 || slot >= j0 + nj) continue;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      for (uint32_t k0 = 0; k0 < C; k0 += 8) {  // in rank order, eight reads in flight
        float4 t[8];
#pragma unroll
        for (uint32_t k = 0; k < 8; ++k)
          t[k] = k0 + k < C ? ld_cluster_f32x4(sums + row * Cfg::PITCH + c, k0 + k) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (uint32_t k = 0; k < 8; ++k) {
          v.x += t[k].x;
          v.y += t[k].y;
          v.z += t[k].z;
          v.w += t[k].w;
        }
      }
      const float s = p.scales ? p.scales[sh.row_id[row]] : 1.f;
      v.x *= s;
      v.y *= s;
      v.z *= s;
      v.w *= s;
      if (f.out32) {
        *reinterpret_cast<float4*>(f.out32 + (m0 + row) * RP + c) = v;
        const float each[4] = {v.x, v.y, v.z, v.w};
        uint32_t most = 0u;  // finite values alone: the others need no scale
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const uint32_t b = __float_as_uint(fabsf(each[x]));
          most = b < 0x7F800000u && b > most ? b : most;
        }
        atomicMax(&sh.slot_max[slot], most);
      } else if (c < q.R8) {
        // one rounding to fp16, as rank_rows has it
        const int left = p.R - c;
        const __half2 x = __floats2half2_rn(left > 0 ? v.x : 0.f, left > 1 ? v.y : 0.f);
        const __half2 y = __floats2half2_rn(left > 2 ? v.z : 0.f, left > 3 ? v.w : 0.f);
        *reinterpret_cast<uint2*>(f.out16 + (m0 + row) * q.R8 + c) =
            make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
        const float2 bx = __half22float2(x), by = __half22float2(y);
        if (!isfinite(bx.x) || !isfinite(bx.y) || !isfinite(by.x) || !isfinite(by.y))
          *reinterpret_cast<float4*>(f.full + (m0 + row) * q.R8 + c) = v;
      }
    }
    fence_proxy_async_smem();   // TMA writes there next
    if (C > 1) cluster_sync();  // the peers' sums are read before they change or go
    else __syncthreads();
  }
  if (f.out32)
    for (int i = tid; i < n; i += kProdThreads)
      f.top[((int64_t)tile * kMaxSplit + rank) * kTileRows + i] = sh.slot_max[i];
}

template <int RP>
__global__ void __launch_bounds__(kProdThreads) lora_products_kernel(const __grid_constant__ Products q,
                                                                     const __grid_constant__ ProductMaps maps) {
  extern __shared__ uint8_t prod_smem[];
  __shared__ __align__(16) ProdShared sh;
  uint8_t* smem = prod_smem + ((1024u - (smem_u32(prod_smem) & 1023u)) & 1023u);
  const uint32_t rank = cluster_rank(), C = cluster_size();
  const int unit = (int)(blockIdx.x / C) - (q.plan.total ? 1 : 0);
  pdl_wait();
  pdl_launch_dependents();
  if (unit < 0) {
    if (rank == 0) make_plan(q.p, q.plan, reinterpret_cast<int*>(smem));
    return;
  }
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
    mbar_init(&sh.drained, 1);
    fence_barrier_init();
  }
  if (threadIdx.x < 32) {
    tmem_alloc(&sh.tmem, ProdCfg<RP>::COLUMNS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (first) product_tile<RP, false>(q, q.a, &maps.av, &maps.aw, unit, rank, C, smem, sh);
  else product_tile<RP, true>(q, q.b, &maps.bv, &maps.bw, unit - q.tiles, rank, C, smem, sh);
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
    cudaError_t e = cudaFuncSetAttribute(lora_products_kernel<RP>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         Cfg::SMEM);
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(lora_products_kernel<RP>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
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
  if (q.b.v) {
    const uint64_t dims[3] = {(uint64_t)q.R8, (uint64_t)p.N, (uint64_t)p.L};
    const uint64_t strides[2] = {(uint64_t)q.R8 * 2, (uint64_t)q.R8 * p.N * 2};
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
  // Splits for about four CTAs an SM, each two SM's worth in flight: an SM's TMA
  // loads run at 46 GB/s (a 128-byte row in 5 cycles), so all SMs are needed.  16
  // CTAs to a cluster, twice the portable size, where the tiles are few.  (Fewer
  // CTAs of six stages, one an SM: 1024 rows, 17408 and 5120 columns, rank 64, 71 us
  // a call; so 63.)
  int C = most < kMaxSplit ? (int)most : kMaxSplit;
  while (C > 1 && (int64_t)products * q.tiles * C > (C > 8 ? 1 : 4) * sm_count) --C;
  q.split = C;
  const int64_t units = (int64_t)products * q.tiles + q.lists.tiles + (q.plan.total ? 1 : 0);
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

// ------------------------------------------------------------------- split
// The tensor cores take fp16, h and g are fp32: scaled by a power of two that
// puts the adapter's largest finite magnitude below 2^15, each is split into the nearest
// fp16 and the nearest fp16 of the rest (22 bits together), so dA and dB keep what
// an fp32 product would.  A CTA lays out one step, 128 sorted rows of both, as the
// sums' shared memory holds them: high halves then low halves, blocks of 64 ranks,
// 128 rows of 128 swizzled bytes, so that a step is one bulk copy there however
// many column tiles read it (made anew by each column tile's CTA instead: 4096
// rows to 5120 x 17408 columns, rank 64, 174 us, not 142).  Latency-bound, 4 us of
// 256 rows' 19: three reads, each of what the one before names.
template <int RP>
struct SplitCfg {
  static constexpr int NRANK = RP > 64 ? 128 : 64;          // ranks in whole 128-byte rows
  static constexpr int HALF = kStepRows * NRANK * 2;        // high or low halves
  static constexpr int IMAGE = 2 * HALF;                    // h or g of a step
};
struct Split {
  LoraArgs p;
  PlanArgs plan;
  const float *h, *g;                 // [M][RP]
  const uint32_t *top_h, *top_g;      // [tiles][kMaxSplit][kTileRows]
  const uint32_t* tile_ids;
  int tiles, split;                   // row tiles and cluster size of the products
  uint8_t* images;                    // [steps][h, g][IMAGE]
  float* down;                        // [chunks][h, g] 2^-e, the scale back
  int2* runs;                         // [steps] first row of a whole step of consecutive rows, else -1, and bits of
                                      // the groups of 8 rows that are consecutive
};
constexpr int kSplitThreads = 128, kSplitRows = 32;

// blockIdx.y: h or g, and which 32 of the step's rows.
template <int RP>
__global__ void __launch_bounds__(kSplitThreads) lora_split_kernel(const Split q) {
  using Cfg = SplitCfg<RP>;
  __shared__ uint32_t top, runs[kStepRows / 32];
  pdl_wait();
  pdl_launch_dependents();
  const int step = blockIdx.x, tid = threadIdx.x;
  const int which = blockIdx.y % 2, row0 = blockIdx.y / 2 * kSplitRows;
  const int steps = __ldcg(q.plan.total + 1);
  const int4 info = __ldcg(reinterpret_cast<const int4*>(q.plan.steps) + step);  // there whatever the plan wrote
  if (step >= steps) return;
  const int adapter = info.x, rows = info.z, chunk = info.w;
  const int* order = q.plan.order + info.y;
  const uint32_t* tops = which ? q.top_g : q.top_h;
  constexpr int kPieces = RP / 4, kRowStep = kSplitThreads / kPieces, kPasses = kSplitRows / kRowStep;
  const int c = tid % kPieces * 4;
  const float* src = which ? q.g : q.h;
  // All that is read is asked for as early as its place is known: the time is the
  // chain of reads (the plan, rows and tiles' adapters, values and maxima).
  int m[kPasses];
#pragma unroll
  for (int k = 0; k < kPasses; ++k) {
    const int row = row0 + k * kRowStep + tid / kPieces;
    m[k] = row < rows ? __ldcg(order + row) : -1;
  }
  const int mine = tid < rows ? __ldcg(order + tid) : -1, next = tid + 1 < rows ? __ldcg(order + tid + 1) : -1;
  float4 v[kPasses];
#pragma unroll
  for (int k = 0; k < kPasses; ++k) {
    v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (m[k] >= 0) v[k] = __ldcg(reinterpret_cast<const float4*>(src + (int64_t)m[k] * RP + c));
  }
  if (tid == 0) top = 0u;
  // the adapter's largest magnitude over the products' tiles, 16 of a tile's adapters a thread
  uint32_t bits = 0u;
  for (int t = tid / 8; t < q.tiles; t += kSplitThreads / 8) {
    const int first = tid % 8 * 16;
    uint4 id[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      id[j] = __ldcg(reinterpret_cast<const uint4*>(q.tile_ids + (int64_t)t * kTileRows + first) + j);
    int at = -1;  // a tile names an adapter once
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t a = (uint32_t)adapter;
      at = id[j].x == a ? 4 * j : id[j].y == a ? 4 * j + 1 : id[j].z == a ? 4 * j + 2 : id[j].w == a ? 4 * j + 3 : at;
    }
    if (at >= 0) {
      const uint32_t* of = tops + (int64_t)t * kMaxSplit * kTileRows + first + at;
      uint32_t b[kMaxSplit];
#pragma unroll
      for (int k = 0; k < kMaxSplit; ++k) b[k] = k < q.split ? __ldcg(of + k * kTileRows) : 0u;
#pragma unroll
      for (int k = 0; k < kMaxSplit; ++k) bits = b[k] > bits ? b[k] : bits;
    }
  }
  if (blockIdx.y == 0) {  // a row a thread
    const uint32_t here = __ballot_sync(0xffffffffu, mine >= 0 && next == mine + 1);
    if (tid % 32 == 0) runs[tid / 32] = here;
  }
  __syncthreads();
  if (blockIdx.y == 0 && tid == 0) {
    uint32_t mask = 0u;
    for (int g = 0; g < kStepRows / 8; ++g) mask |= ((runs[g / 4] >> g % 4 * 8 & 0x7Fu) == 0x7Fu ? 1u : 0u) << g;
    const bool all = (runs[0] & runs[1] & runs[2]) == 0xFFFFFFFFu && runs[3] == 0x7FFFFFFFu;
    q.runs[step] = make_int2(all ? mine : -1, (int)mask);
  }
  if (bits) atomicMax(&top, bits);
  __syncthreads();
  // 2^e brings the largest magnitude into [2^14, 2^15)
  bits = top;
  int e = bits == 0u ? 0 : 14 - ((int)(bits >> 23) - 127);
  e = e > 126 ? 126 : (e < -126 ? -126 : e);
  const float up = __uint_as_float((uint32_t)(127 + e) << 23);
  if (row0 == 0 && tid == 0 && chunk >= 0) q.down[2 * chunk + which] = __uint_as_float((uint32_t)(127 - e) << 23);
  uint8_t* image = q.images + ((int64_t)step * 2 + which) * Cfg::IMAGE + c / 64 * (kStepRows * 128);
#pragma unroll
  for (int k = 0; k < kPasses; ++k) {
    const float f[4] = {v[k].x * up, v[k].y * up, v[k].z * up, v[k].w * up};
    uint32_t hi[2], lo[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const __half2 h = __floats2half2_rn(f[2 * x], f[2 * x + 1]);
      const float2 back = __half22float2(h);
      // nothing is left of an infinity
      const __half2 l = __floats2half2_rn(isinf(back.x) ? 0.f : f[2 * x] - back.x,
                                          isinf(back.y) ? 0.f : f[2 * x + 1] - back.y);
      hi[x] = *reinterpret_cast<const uint32_t*>(&h);
      lo[x] = *reinterpret_cast<const uint32_t*>(&l);
    }
    uint8_t* at = image + swizzled(row0 + k * kRowStep + tid / kPieces, c % 64 / 8) + c % 8 * 2;
    *reinterpret_cast<uint2*>(at) = make_uint2(hi[0], hi[1]);
    *reinterpret_cast<uint2*>(at + Cfg::HALF) = make_uint2(lo[0], lo[1]);
  }
}

// -------------------------------------------------------------------- sums
// A chunk of an adapter's rows and 128 columns of x (dA, and dx of those rows)
// or of dy (dB) at a time, by a persistent grid of one CTA an SM, 128 rows a step.
// The CTAs take the column tiles in turns, so that at a time they read a stretch
// of the same rows (equal shares of all the work, a range of columns each, took
// 110 us where this took 77):
//   warps 8-13  load, two to a step in turn: its image of h or g (one bulk copy)
//               and its rows of x or dy, all 128 or 8 at a time by TMA where they
//               are consecutive, else copied (cp.async; a warp's proxy fence waits
//               for its own step's copies alone, and three steps are in flight.
//               One warp a step: 4096 rows in any order 187 us a call, not 173.
//               TMA's four-row gathers were issued at one in 80 cycles: 12 GB/s an
//               SM); warp 8 also an item's lora_a;
//   warp 14     issues tcgen05.mma: D[ranks][columns] += (h or g)^T v, both
//               operands along MN since the rows are the reduction, and
//               dx[rows][columns] = g A into one of two TMEM buffers;
//   warps 0-7   take a step's dx from TMEM to memory, and an item's D.
// Odd steps of a chunk have a D of their own: the tensor cores' additions truncate,
// and an error grows with the number that follow one another (dA of 4096 rows to
// 1.2e-6 of its size, 2.0e-6 in one sum; of 256 rows 4.0e-7 and 5.4e-7; the plain
// fp32 form 1.4e-6 and 4.8e-7; the times are the same, 135.1 and 19.8 us).
// HBM-bound by x, dy and dx (4.1 TB/s of them over 4096 rows, 17408 and 5120 columns,
// rank 64: 80 us).  Up to rank 64 the two halves of h or g are rows of one D (64 of
// each) and are added when it is read; dx takes both into one sum.
//
// A sum of several chunks is joined by the last CTA to finish one of them, from
// fp32 partial sums in chunk order, so that results do not depend on timing.
constexpr int kCols = 128;
constexpr int kWorkers = 256;
constexpr int kWarpCols = kCols / (kWorkers / 128);  // columns of D or dx a worker warp reads, of 32 rows
constexpr int kVStages = 3;                          // and two warps for each that load
constexpr int kLoaders = 2;
constexpr int kMmaWarp = kWorkers / 32 + kLoaders * kVStages;
constexpr int kSumThreads = (kMmaWarp + 1) * 32;

struct Sums {
  LoraArgs p;
  const __half* dy;
  int64_t dy_ld;
  PlanArgs plan;
  const uint8_t* images;
  const float* down;
  const int2* runs;
  __half* dx;
  float *da, *db;
  float* part;         // [chunk of a joint sum][tiles][kCols][RP]
  bool add_dx;
  int x_tiles, tiles;  // column tiles of x, and of x and dy together
  unsigned int* status;
};
struct SumMaps {
  CUtensorMap x, dy;    // 128 rows of 64 columns
  CUtensorMap x8, dy8;  // 8 rows of them
  CUtensorMap a;        // 3-D
};

template <int RP>
struct SumCfg {
  static constexpr bool STACK = RP <= 64;                        // a D's rows are 64 high and 64 low halves
  static constexpr int V_STAGE = kStepRows * kCols * 2;          // two blocks of 64 columns
  static constexpr int BLOCK = kStepRows * 128;                  // 64 ranks or columns of a step's rows
  static constexpr int G_HALF = SplitCfg<RP>::HALF, G_STAGE = SplitCfg<RP>::IMAGE;
  static constexpr int G_BUFS = RP > 64 ? 1 : kVStages;
  static constexpr int OFF_G = kVStages * V_STAGE;
  static constexpr int OFF_A = OFF_G + G_BUFS * G_STAGE;         // lora_a: two blocks of [RP][64 columns]
  static constexpr int OFF_X = OFF_A + RP * kCols * 2;           // 2 KB a worker warp, for transposing
  static constexpr int SMEM = OFF_X + kWorkers / 32 * 2048 + 1024;
  static_assert(SMEM <= 226 * 1024, "shared memory budget");
};

struct SumShared {
  uint64_t vfull[kVStages], vempty[kVStages], gfull[kVStages], dxfull[2], dxempty[2];
  uint64_t accfull, accempty, afull, aempty, drained;
  uint32_t tmem;
  int last;
  int late;  // a bounded wait ran out
};

// 16 bytes from src (zeros where !valid)
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid) {
  const int n = valid ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void bulk_copy(uint32_t dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ uint4 lds16(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}
__device__ __forceinline__ void pair_sync(int pair) {  // two warps
  asm volatile("bar.sync %0, 64;" ::"r"(2 + pair) : "memory");
}
__device__ __forceinline__ void worker_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kWorkers) : "memory"); }

// One item of the persistent loop.
struct Item {
  Chunk ck;
  int chunk, tile, steps;
  bool is_x, sum, dx;  // columns of x; dA or dB wanted; dx wanted
  int64_t col0, width;
};
__device__ __forceinline__ Item item_at(const Sums& q, int64_t i) {
  Item t;
  t.chunk = (int)(i / q.tiles);
  t.ck = q.plan.chunks[t.chunk];
  t.tile = (int)(i % q.tiles);
  t.is_x = t.tile < q.x_tiles;
  t.col0 = (int64_t)(t.is_x ? t.tile : t.tile - q.x_tiles) * kCols;
  t.width = t.is_x ? q.p.K : q.p.N;
  t.sum = t.is_x ? q.da != nullptr : q.db != nullptr;
  t.dx = t.is_x && q.dx != nullptr;
  t.steps = t.sum || t.dx ? (t.ck.count + kStepRows - 1) / kStepRows : 0;
  return t;
}

template <int RP>
__global__ void __launch_bounds__(kSumThreads, 1)
    lora_sums_kernel(const __grid_constant__ Sums q, const __grid_constant__ SumMaps maps) {
  using Cfg = SumCfg<RP>;
  extern __shared__ uint8_t sum_smem[];
  __shared__ SumShared sh;
  uint8_t* smem = sum_smem + ((1024u - (smem_u32(sum_smem) & 1023u)) & 1023u);
  const uint32_t base = smem_u32(smem);
  const LoraArgs& p = q.p;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;

  if (tid == 0) {
    for (int i = 0; i < kVStages; ++i) {
      mbar_init(&sh.vfull[i], kLoaders);
      mbar_init(&sh.vempty[i], 1);
      mbar_init(&sh.gfull[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sh.dxfull[i], 1);
      mbar_init(&sh.dxempty[i], kWorkers / 32);
    }
    mbar_init(&sh.accfull, 1);
    mbar_init(&sh.accempty, kWorkers / 32);
    mbar_init(&sh.afull, 1);
    mbar_init(&sh.aempty, 1);
    mbar_init(&sh.drained, 1);
    sh.late = 0;
    fence_barrier_init();
  }
  if (warp == kMmaWarp) {
    tmem_alloc(&sh.tmem, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh.tmem;
  constexpr uint32_t kDx = 128, kOdd = 384;  // TMEM columns of the two dx buffers, and of D's odd steps
  pdl_wait();
  const int64_t items = (int64_t)q.plan.total[0] * q.tiles;
  // After a bounded wait that ran out the workers go on without waiting (they meet at
  // barriers of their own); the others stop, one after the other, and see to what they
  // have under way.
  bool ok = true;
  int last_image = -1;  // the last step whose image this thread loaded
  auto wait = [&](uint64_t* bar, uint32_t parity, unsigned int code) {
    if (ok && !mbar_wait(bar, parity, q.status, code)) {
      ok = false;
      sh.late = 1;
    }
  };

  if (warp >= kWorkers / 32 && warp < kMmaWarp) {
    // -------------------------------------------------------------- loads
    const int slot = (warp - kWorkers / 32) / kLoaders, part = (warp - kWorkers / 32) % kLoaders;
    constexpr int kQuarters = 4 / kLoaders;  // of the step's rows
    uint32_t it = 0, ai = 0;
    int last = -1;  // the last step that this warp loaded
    for (int64_t i = blockIdx.x; i < items && ok; i += gridDim.x) {
      const Item t = item_at(q, i);
      if (t.steps == 0) continue;
      if (t.dx && slot == 0 && part == 0) {
        if (lane == 0 && ai > 0) wait(&sh.aempty, (ai - 1) & 1, kDevTimeoutEmpty);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        if (lane == 0) {
          mbar_arrive_expect_tx(&sh.afull, RP * kCols * 2);
          for (int b = 0; b < 2; ++b)
            tma_load_3d(smem + Cfg::OFF_A + b * RP * 128, &maps.a, &sh.afull, (int)t.col0 + b * 64, 0, t.ck.adapter);
        }
        __syncwarp();
        ++ai;
      }
      const __half* v = t.is_x ? reinterpret_cast<const __half*>(p.x) : q.dy;
      const int64_t ld = t.is_x ? p.x_ld : q.dy_ld;
      const int64_t c = t.col0 + lane % 16 * 8;
      const bool in_c = c < t.width;
      const int* order = q.plan.order + t.ck.start;
      for (int step = 0; step < t.steps; ++step, ++it) {
        if (it % kVStages != (uint32_t)slot) continue;
        const uint32_t gb = it % Cfg::G_BUFS;
        const int2 runs = __ldcg(q.runs + t.ck.step0 + step);
        const int rows = t.ck.count - step * kStepRows;
        int at[kQuarters];  // this warp's rows of the step
#pragma unroll
        for (int k = 0; k < kQuarters; ++k) {
          const int r = 32 * (part * kQuarters + k) + lane;
          at[k] = r < rows ? __ldcg(order + step * kStepRows + r) : -1;
        }
        const int head = lane % 16 * 8 < rows ? __ldcg(order + step * kStepRows + lane % 16 * 8) : -1;
        // The products that read this stage are done; then those that read the
        // image's buffer, which are at most two steps later (so that a barrier
        // is never a whole turn ahead of its waiter).
        if (it >= kVStages) wait(&sh.vempty[slot], (it / kVStages - 1) & 1, kDevTimeoutEmpty);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        last = (int)it;
        uint8_t* const stage = smem + slot * Cfg::V_STAGE;
        if (lane == 0 && part == 0 && runs.y) mbar_expect_tx(&sh.vfull[slot], (uint32_t)__popc(runs.y) * 2048u);
        __syncwarp();
        if (runs.x >= 0) {
          if (lane == 0 && part == 0)
            for (int b = 0; b < 2; ++b)
              tma_load_2d(stage + b * Cfg::BLOCK, t.is_x ? &maps.x : &maps.dy, &sh.vfull[slot], (int)t.col0 + b * 64,
                          runs.x);
        } else {
          // groups of 8 consecutive rows by TMA, a group and a block of columns a lane
          if (part == 0 && (runs.y >> lane % 16 & 1))
            tma_load_2d(stage + lane / 16 * Cfg::BLOCK + lane % 16 * 1024, t.is_x ? &maps.x8 : &maps.dy8,
                        &sh.vfull[slot], (int)t.col0 + lane / 16 * 64, head);
          const uint32_t dst = smem_u32(stage) + lane % 16 / 8 * Cfg::BLOCK;
#pragma unroll
          for (int k = 0; k < kQuarters; ++k)
#pragma unroll 1
            for (int g = 0; g < 4; ++g) {
              const int group = 4 * (part * kQuarters + k) + g;
              // the products take no rows behind the last 16 that hold one
              if ((runs.y >> group & 1) || group / 2 * 16 >= rows) continue;
#pragma unroll
              for (int j = 0; j < 4; ++j) {  // two rows of 256 bytes
                const int in_k = g * 8 + 2 * j + lane / 16;
                const int m = __shfl_sync(0xffffffffu, at[k], in_k);
                const bool in = in_c && m >= 0;
                cp_async16(dst + swizzled(group * 8 + 2 * j + lane / 16, lane % 8), v + (in ? m * ld + c : 0), in);
              }
            }
        }
        if (lane == 0 && part == 0) {
          if (it >= Cfg::G_BUFS) {
            const uint32_t was = it - Cfg::G_BUFS;
            wait(&sh.vempty[was % kVStages], (was / kVStages) & 1, kDevTimeoutEmpty);
          }
          if (ok) {
            last_image = (int)it;
            mbar_arrive_expect_tx(&sh.gfull[gb], Cfg::G_STAGE);
            bulk_copy(base + Cfg::OFF_G + gb * Cfg::G_STAGE,
                      q.images + ((int64_t)(t.ck.step0 + step) * 2 + (t.is_x ? 1 : 0)) * Cfg::G_STAGE, Cfg::G_STAGE,
                      &sh.gfull[gb]);
          }
        }
        __syncwarp();
        if (runs.x < 0) {
          asm volatile("cp.async.wait_all;" ::: "memory");
          fence_proxy_async_smem();
          __syncwarp();
        }
        if (lane == 0) mbar_arrive(&sh.vfull[slot]);
      }
    }
    // What is under way lands before the CTA goes (a step counts as landed when both
    // its warps have arrived, so the one that gives up does).
    if (lane == 0 && part == 1 && !ok) mbar_arrive(&sh.vfull[slot]);
    if (lane == 0 && part == 0) {
      if (last >= 0) mbar_wait(&sh.vfull[slot], (last / kVStages) & 1, q.status, kDevTimeoutFull);
      if (ai > 0) mbar_wait(&sh.afull, (ai - 1) & 1, q.status, kDevTimeoutFull);
    }
    __syncwarp();
  } else if (warp == kMmaWarp) {
    // ----------------------------------------------------------- products
    uint32_t it = 0, dxs = 0, sums = 0, ai = 0;
    if (lane == 0) {
      constexpr uint32_t kSumDesc = mma_desc(128, kCols, true, true);
      constexpr uint32_t kDxDesc = mma_desc(kStepRows, kCols, false, true);
      for (int64_t i = blockIdx.x; i < items && ok; i += gridDim.x) {
        const Item t = item_at(q, i);
        if (t.steps == 0) continue;
        if (t.sum && sums > 0) wait(&sh.accempty, (sums - 1) & 1, kDevTimeoutAccum);
        for (int step = 0; step < t.steps; ++step, ++it) {
          const uint32_t s = it % kVStages, gb = it % Cfg::G_BUFS;
          wait(&sh.vfull[s], (it / kVStages) & 1, kDevTimeoutFull);
          wait(&sh.gfull[gb], (it / Cfg::G_BUFS) & 1, kDevTimeoutFull);
          if (t.dx && dxs >= 2) wait(&sh.dxempty[dxs & 1], (dxs / 2 - 1) & 1, kDevTimeoutAccum);
          if (!ok) break;
          tc_fence_after();
          const uint32_t vs = base + s * Cfg::V_STAGE, gs = base + Cfg::OFF_G + gb * Cfg::G_STAGE;
          auto dx = [&]() {
            const uint64_t b = operand_mn(base + Cfg::OFF_A, RP * 128);
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
              for (int kk = 0; kk < RP / 16; ++kk) {
                const uint64_t a =
                    operand_k(gs + half * Cfg::G_HALF + kk / 4 * Cfg::BLOCK) + (uint64_t)(2 * (kk % 4));
                tc_mma_ss(tmem + kDx + (dxs & 1) * kCols, a, b + (uint64_t)(128 * kk), kDxDesc, half > 0 || kk > 0);
              }
            tc_commit(&sh.dxfull[dxs & 1]);
            ++dxs;
          };
          if (t.dx && step > 0) dx();  // before the sums: the workers wait for it
          if (t.sum) {
            const int blocks = (t.ck.count - step * kStepRows + 15) / 16;
            const bool two = t.steps > 1;
            const uint64_t b = operand_mn(vs, Cfg::BLOCK);
#pragma unroll
            for (int half = 0; half < (Cfg::STACK ? 1 : 2); ++half) {
              // both halves, 64 ranks of each, or one half's 128
              const uint64_t a = operand_mn(gs + half * Cfg::G_HALF, Cfg::BLOCK);
#pragma unroll
              for (int kk = 0; kk < kStepRows / 16; ++kk)
                if (kk < blocks)
                  tc_mma_ss(tmem + (two && (step & 1) ? kOdd : 0u), a + (uint64_t)(128 * kk),
                            b + (uint64_t)(128 * kk), kSumDesc, step > (two ? 1 : 0) || half > 0 || kk > 0);
            }
          }
          if (t.dx && step == 0) {  // lora_a comes when the item before is done
            wait(&sh.afull, ai & 1, kDevTimeoutFull);
            if (ok) dx();
          }
          tc_commit(&sh.vempty[s]);
        }
        if (t.sum) {
          tc_commit(&sh.accfull);
          ++sums;
        }
        if (t.dx) {
          tc_commit(&sh.aempty);
          ++ai;
        }
      }
      // every product and every arrival has ended before the CTA's memory goes
      tc_commit(&sh.drained);
      mbar_wait(&sh.drained, 0, q.status, kDevTimeoutAccum);
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ workers
    const int quarter = warp % 4, upper = warp / 4;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    uint32_t dxs = 0, sums = 0;
    for (int64_t i = blockIdx.x; i < items; i += gridDim.x) {
      const Item t = item_at(q, i);
      const Chunk& ck = t.ck;
      const int* order = q.plan.order + ck.start;
      float* out = t.is_x ? q.da : q.db;
      const float down = ck.count > 0 ? __ldcg(q.down + 2 * t.chunk + (t.is_x ? 1 : 0)) : 1.f;
      // dx of a step: a row a lane and 64 columns a warp out of TMEM, through
      // shared memory into pieces of 64 bytes of a row.  Added to what dx holds,
      // it goes there directly, in fp32 up to its one rounding.
      int next_row = -1;
      auto fetch_row = [&](int step) {
        const int r = step * kStepRows + quarter * 32 + lane;
        next_row = r < ck.count ? __ldcg(order + r) : -1;
      };
      if (t.dx) fetch_row(0);
      for (int step = 0; t.dx && step < t.steps; ++step, ++dxs) {
        const uint32_t b = dxs & 1;
        const int mine = next_row;
        if (step + 1 < t.steps) fetch_row(step + 1);
        wait(&sh.dxfull[b], (dxs / 2) & 1, kDevTimeoutAccum);
        __syncwarp();  // lanes without a row came early
        tc_fence_after();
        uint32_t d[kWarpCols / 16][16];
#pragma unroll
        for (int c = 0; c < kWarpCols / 16; ++c)
          tmem_ld_32x32b_x16(tmem + lanes + kDx + b * kCols + upper * kWarpCols + c * 16, d[c]);
        tmem_wait_ld();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.dxempty[b]);
        if (q.add_dx) {
          if (mine < 0) continue;
          __half* row = q.dx + (int64_t)mine * p.K + t.col0 + upper * kWarpCols;
#pragma unroll
          for (int c = 0; c < kWarpCols / 16; ++c) {
            if (t.col0 + upper * kWarpCols + c * 16 >= t.width) continue;
            uint32_t o[8];
#pragma unroll
            for (int x = 0; x < 2; ++x)
              *reinterpret_cast<uint4*>(o + 4 * x) = *reinterpret_cast<const uint4*>(row + c * 16 + 8 * x);
#pragma unroll
            for (int x = 0; x < 8; ++x) {
              const float2 w = __half22float2(*reinterpret_cast<const __half2*>(&o[x]));
              const __half2 r = __floats2half2_rn(fmaf(__uint_as_float(d[c][2 * x]), down, w.x),
                                                  fmaf(__uint_as_float(d[c][2 * x + 1]), down, w.y));
              o[x] = *reinterpret_cast<const uint32_t*>(&r);
            }
#pragma unroll
            for (int x = 0; x < 2; ++x)
              *reinterpret_cast<uint4*>(row + c * 16 + 8 * x) =
                  make_uint4(o[4 * x], o[4 * x + 1], o[4 * x + 2], o[4 * x + 3]);
          }
          continue;
        }
        const uint32_t area = base + Cfg::OFF_X + warp * 2048;  // 32 rows of 64 bytes, swizzled
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            uint32_t o[4];
#pragma unroll
            for (int y = 0; y < 4; ++y) {
              const uint32_t* v = &d[2 * h + x / 2][8 * (x % 2) + 2 * y];
              const __half2 r = __floats2half2_rn(__uint_as_float(v[0]) * down, __uint_as_float(v[1]) * down);
              o[y] = *reinterpret_cast<const uint32_t*>(&r);
            }
            sts16(area + lane * 64 + ((x ^ (lane / 2 & 3)) << 4), make_uint4(o[0], o[1], o[2], o[3]));
          }
          __syncwarp();
          const int64_t col = t.col0 + upper * kWarpCols + h * 32 + lane % 4 * 8;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int r = 8 * k + lane / 4;
            const int m = __shfl_sync(0xffffffffu, mine, r);
            const uint4 w = lds16(area + r * 64 + ((lane % 4 ^ (r / 2 & 3)) << 4));
            if (m >= 0 && col < t.width) *reinterpret_cast<uint4*>(q.dx + (int64_t)m * p.K + col) = w;
          }
          __syncwarp();
        }
      }
      if (!t.sum) continue;

      // D[rank][column] of this chunk: a rank a lane, 64 columns a warp, all read
      // at once so that the next item's products may start.  The high and the low
      // halves of a sum are in two warps: each gives the other 32 of its columns,
      // 16 at a time through shared memory (2 KB, as 128 pieces of 16 bytes).
      uint32_t d[4][16];
      if (t.steps > 0) {
        wait(&sh.accfull, sums & 1, kDevTimeoutAccum);
        ++sums;
        __syncwarp();
        tc_fence_after();
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld_32x32b_x16(tmem + lanes + upper * kWarpCols + c * 16, d[c]);
        tmem_wait_ld();
        if (t.steps > 1) {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t w[16];
            tmem_ld_32x32b_x16(tmem + lanes + kOdd + upper * kWarpCols + c * 16, w);
            tmem_wait_ld();
#pragma unroll
            for (int x = 0; x < 16; ++x)
              d[c][x] = __float_as_uint(__uint_as_float(d[c][x]) + __uint_as_float(w[x]));
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.accempty);
      } else {
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int x = 0; x < 16; ++x) d[c][x] = 0u;
      }
      constexpr int kOwn = Cfg::STACK ? 2 : 4;  // 16s of columns that this warp finishes
      const bool low = Cfg::STACK && quarter >= 2;
      const int r = (Cfg::STACK ? quarter & 1 : quarter) * 32 + lane;
      const int c0 = upper * kWarpCols + (low ? 32 : 0);
      float f[kOwn][16];
      if (Cfg::STACK) {
        const uint32_t area = base + Cfg::OFF_X + warp * 2048, peer = base + Cfg::OFF_X + (warp ^ 2) * 2048;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            uint4 w;
            w.x = low ? d[c][4 * x] : d[2 + c][4 * x];
            w.y = low ? d[c][4 * x + 1] : d[2 + c][4 * x + 1];
            w.z = low ? d[c][4 * x + 2] : d[2 + c][4 * x + 2];
            w.w = low ? d[c][4 * x + 3] : d[2 + c][4 * x + 3];
            sts16(area + lane * 64 + ((x ^ (lane / 2 & 3)) << 4), w);
          }
          pair_sync(quarter % 2 * 2 + upper);
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const uint4 w = lds16(peer + lane * 64 + ((x ^ (lane / 2 & 3)) << 4));
            f[c][4 * x] = __uint_as_float(low ? d[2 + c][4 * x] : d[c][4 * x]) + __uint_as_float(w.x);
            f[c][4 * x + 1] = __uint_as_float(low ? d[2 + c][4 * x + 1] : d[c][4 * x + 1]) + __uint_as_float(w.y);
            f[c][4 * x + 2] = __uint_as_float(low ? d[2 + c][4 * x + 2] : d[c][4 * x + 2]) + __uint_as_float(w.z);
            f[c][4 * x + 3] = __uint_as_float(low ? d[2 + c][4 * x + 3] : d[c][4 * x + 3]) + __uint_as_float(w.w);
          }
          pair_sync(quarter % 2 * 2 + upper);
        }
      } else {
#pragma unroll
        for (int c = 0; c < kOwn; ++c)
#pragma unroll
          for (int x = 0; x < 16; ++x) f[c][x] = __uint_as_float(d[c % 4][x]);
      }
      auto write = [&](int c, const float (&v)[16]) {
        const int64_t col = t.col0 + c0 + c;
        if (r >= p.R) return;
        if (t.is_x) {
          float* o = out + ((int64_t)ck.adapter * p.R + r) * t.width + col;
          if (col < t.width) {  // the width is a multiple of 64
#pragma unroll
            for (int x = 0; x < 16; x += 4)
              *reinterpret_cast<float4*>(o + x) =
                  make_float4(v[x] * down, v[x + 1] * down, v[x + 2] * down, v[x + 3] * down);
          }
        } else {
          float* o = out + ((int64_t)ck.adapter * t.width + col) * p.R + r;
#pragma unroll
          for (int x = 0; x < 16; ++x)
            if (col + x < t.width) o[x * p.R] = v[x] * down;
        }
      };
      if (ck.of == 1) {
#pragma unroll
        for (int c = 0; c < kOwn; ++c) write(c * 16, f[c]);
        continue;
      }
      // a chunk's sums lie [column][rank], those of the adapter's next chunk q.tiles further on
      float* slots = q.part + (((int64_t)ck.slot0 * q.tiles + t.tile) * kCols + c0) * RP + r;
      const int64_t apart = (int64_t)q.tiles * kCols * RP;
      if (r < RP) {
#pragma unroll
        for (int c = 0; c < kOwn; ++c)
#pragma unroll
          for (int x = 0; x < 16; ++x) __stcg(slots + ck.index * apart + (c * 16 + x) * RP, f[c][x]);
      }
      __threadfence();
      worker_sync();
      if (tid == 0) sh.last = atomicAdd(q.plan.count + (int64_t)ck.joint * q.tiles + t.tile, 1u) == (uint32_t)ck.of - 1;
      worker_sync();
      if (sh.last && r < RP) {
        __threadfence();
#pragma unroll
        for (int c = 0; c < kOwn; ++c) {
#pragma unroll
          for (int x = 0; x < 16; ++x) f[c][x] = 0.f;
          for (int k = 0; k < ck.of; ++k)
#pragma unroll
            for (int x = 0; x < 16; ++x) f[c][x] += __ldcg(slots + k * apart + (c * 16 + x) * RP);
          write(c * 16, f[c]);
        }
      }
      worker_sync();  // all have read sh.last
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
  if (sh.late && last_image >= 0)  // images too, where products did not wait for them
    mbar_wait(&sh.gfull[last_image % Cfg::G_BUFS], (last_image / Cfg::G_BUFS) & 1, q.status, kDevTimeoutFull);
}

constexpr size_t align256(size_t v) { return (v + 255) & ~(size_t)255; }

// How a gradient call is cut: chunks long enough that the column tiles alone
// fill the GPU, shorter ones only where they would not.
struct GradSpace {
  int RP, x_tiles, tiles, chunk_rows;
  int64_t max_chunks, joints;
  int64_t dy_pitch, b_pitch;  // of dy and lora_b laid out anew (0: as they are)
  int64_t max_steps;
  size_t h, g, chunks, steps, order, count, part, dy, b, top, ids, images, down, runs, end;
};
GradSpace grad_space(int64_t M, int64_t N, int64_t K, int R, int64_t L, int sm_count) {
  GradSpace s;
  s.RP = padded_rank(R);
  s.x_tiles = (int)((K + kCols - 1) / kCols);
  s.tiles = s.x_tiles + (int)((N + kCols - 1) / kCols);
  // The cuts of an adapter with all rows whose rounds of items take least, in
  // steps: an item's beginning and end cost about two, joining its sum two more
  // (256 rows, 6144 x 5120: two cuts of one step took 4 us more than one of two).
  int64_t cuts = 1, best = 0;
  for (int64_t c = 1; c <= 8 && (c - 1) * kStepRows < M; ++c) {
    const int64_t rounds = (c * s.tiles + sm_count - 1) / sm_count;
    const int64_t steps = ((M + c - 1) / c + kStepRows - 1) / kStepRows;
    const int64_t cost = rounds * (steps + (c > 1 ? 4 : 2));
    if (c == 1 || cost < best) {
      cuts = c;
      best = cost;
    }
  }
  s.chunk_rows = (int)(((M + cuts - 1) / cuts + kStepRows - 1) / kStepRows * kStepRows);
  if (s.chunk_rows < kStepRows) s.chunk_rows = kStepRows;
  s.max_chunks = M / s.chunk_rows + L;
  s.joints = M / (s.chunk_rows + 1);  // adapters of more than chunk_rows rows
  if (s.joints > L) s.joints = L;
  const int64_t parts = s.joints ? M / s.chunk_rows + s.joints : 0;  // their chunks
  s.max_steps = M / kStepRows + L;  // a whole step holds 128 rows, and an adapter has one that is not
  if (s.max_steps > M) s.max_steps = M;
  const size_t row_tiles = (size_t)((M + kTileRows - 1) / kTileRows);
  const size_t image = (size_t)kStepRows * (s.RP > 64 ? 128 : 64) * 2 * 2;
  size_t at = 256;  // the plan's totals
  auto take = [&](size_t bytes) {
    const size_t was = at;
    at += align256(bytes);
    return was;
  };
  s.h = take((size_t)M * s.RP * sizeof(float));
  s.g = take((size_t)M * s.RP * sizeof(float));
  s.chunks = take((size_t)s.max_chunks * sizeof(Chunk));
  s.steps = take((size_t)s.max_steps * sizeof(Step));
  s.order = take((size_t)M * sizeof(int));
  s.top = take(2 * row_tiles * kMaxSplit * kTileRows * sizeof(uint32_t));
  s.ids = take(row_tiles * kTileRows * sizeof(uint32_t));
  s.images = take((size_t)s.max_steps * 2 * image);
  s.down = take((size_t)s.max_chunks * 2 * sizeof(float));
  s.runs = take((size_t)s.max_steps * sizeof(int2));
  s.count = take((size_t)s.joints * s.tiles * sizeof(uint32_t));
  s.part = take((size_t)parts * s.tiles * kCols * s.RP * sizeof(float));
  s.dy_pitch = N % 8 ? (N + 7) / 8 * 8 : 0;
  s.b_pitch = R % 8 ? (R + 7) / 8 * 8 : 0;
  s.dy = take((size_t)M * s.dy_pitch * sizeof(__half));
  s.b = take((size_t)L * N * s.b_pitch * sizeof(__half));
  s.end = at;
  return s;
}

template <int RP>
cudaError_t launch_sums(const Split& sp, const Sums& q, const SumMaps& maps, int64_t steps, int64_t items, int sm_count,
                        bool pdl, cudaStream_t stream) {
  using Cfg = SumCfg<RP>;
  static thread_local int configured_dev = -1;
  int dev = 0;
  cudaGetDevice(&dev);
  if (configured_dev != dev) {
    const cudaError_t e =
        cudaFuncSetAttribute(lora_sums_kernel<RP>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::SMEM);
    if (e != cudaSuccess) return e;
    configured_dev = dev;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl ? 1 : 0;
  {
    cfg.gridDim = dim3((unsigned)steps, 2 * kStepRows / kSplitRows);
    cfg.blockDim = dim3(kSplitThreads);
    const cudaError_t e = cudaLaunchKernelEx(&cfg, lora_split_kernel<RP>, sp);
    if (e != cudaSuccess) return e;
  }
  cfg.gridDim = dim3((unsigned)(items < sm_count ? items : sm_count));
  cfg.blockDim = dim3(kSumThreads);
  cfg.dynamicSmemBytes = Cfg::SMEM;
  return cudaLaunchKernelEx(&cfg, lora_sums_kernel<RP>, q, maps);
}

}  // namespace

cudaError_t launch_lora_products(const LoraArgs& p, const TokenLists& lists, void* h16, float* full,
                                 unsigned int* status, int sm_count, bool pdl, cudaStream_t stream, std::string* err) {
  Products q{};
  q.p = p;
  q.R8 = (p.R + 7) / 8 * 8;
  q.a.v = static_cast<const __half*>(p.x);
  q.a.ld = p.x_ld;
  q.a.len = p.K;
  q.a.w = static_cast<const __half*>(p.a);
  q.a.out16 = static_cast<__half*>(h16);
  q.a.full = full;
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
  if (p.L == 0) {  // nobody has an adapter
    return g.dx && !g.add_dx && p.M ? cudaMemsetAsync(g.dx, 0, (size_t)p.M * p.K * sizeof(__half), stream)
                                    : cudaSuccess;
  }
  if (p.M == 0) {  // no rows: the adapters' gradients are zero
    e = g.da ? cudaMemsetAsync(g.da, 0, (size_t)p.L * p.R * p.K * sizeof(float), stream) : cudaSuccess;
    if (e == cudaSuccess && g.db) e = cudaMemsetAsync(g.db, 0, (size_t)p.L * p.N * p.R * sizeof(float), stream);
    return e;
  }
  const GradSpace s = grad_space(p.M, p.N, p.K, p.R, p.L, sm_count);
  uint8_t* base = static_cast<uint8_t*>(ws);
  const __half *dy = static_cast<const __half*>(g.dy), *lora_b = static_cast<const __half*>(p.b);
  int64_t dy_ld = g.dy_ld;
  if (s.dy_pitch || s.b_pitch) {
    Repack rdy{}, rb{};
    if (s.dy_pitch) rdy = Repack{dy, reinterpret_cast<__half*>(base + s.dy), p.M, p.N, p.N, s.dy_pitch};
    if (s.b_pitch) rb = Repack{lora_b, reinterpret_cast<__half*>(base + s.b), p.L * p.N, p.R, p.R, s.b_pitch};
    const int64_t pieces = (rdy.dst ? p.M * (s.dy_pitch / 8) : 0) + (rb.dst ? p.L * p.N * (s.b_pitch / 8) : 0);
    const int64_t blocks = (pieces + 255) / 256, most = 8 * (int64_t)sm_count;
    lora_repack_kernel<<<(unsigned)(blocks < most ? blocks : most), 256, 0, stream>>>(rdy, rb);
    if ((e = cudaGetLastError()) != cudaSuccess) return e;
    if (rdy.dst) {
      dy = rdy.dst;
      dy_ld = s.dy_pitch;
    }
    if (rb.dst) lora_b = rb.dst;
  }
  const int row_tiles = (int)((p.M + kTileRows - 1) / kTileRows);
  uint32_t* top = reinterpret_cast<uint32_t*>(base + s.top);
  Products q{};
  q.p = p;
  q.R8 = (p.R + 7) / 8 * 8;
  q.a.v = static_cast<const __half*>(p.x);
  q.a.ld = p.x_ld;
  q.a.len = p.K;
  q.a.w = static_cast<const __half*>(p.a);
  q.a.out32 = reinterpret_cast<float*>(base + s.h);
  q.a.top = top;
  q.b.v = dy;
  q.b.ld = dy_ld;
  q.b.len = p.N;
  q.b.w = lora_b;
  q.b.out32 = reinterpret_cast<float*>(base + s.g);
  q.b.top = top + (size_t)row_tiles * kMaxSplit * kTileRows;
  q.tile_ids = reinterpret_cast<uint32_t*>(base + s.ids);
  q.status = g.status;
  q.dx_zero = g.add_dx ? nullptr : static_cast<__half*>(g.dx);
  q.plan.total = reinterpret_cast<int*>(base);
  q.plan.chunks = reinterpret_cast<Chunk*>(base + s.chunks);
  q.plan.steps = reinterpret_cast<Step*>(base + s.steps);
  q.plan.order = reinterpret_cast<int*>(base + s.order);
  q.plan.count = reinterpret_cast<uint32_t*>(base + s.count);
  q.plan.counters = s.joints * s.tiles;
  q.plan.chunk_rows = s.chunk_rows;
  if ((e = dispatch_products(q, sm_count, pdl, stream, err)) != cudaSuccess) return e;
  Split sp{};
  sp.p = p;
  sp.plan = q.plan;
  sp.h = q.a.out32;
  sp.g = q.b.out32;
  sp.top_h = q.a.top;
  sp.top_g = q.b.top;
  sp.tile_ids = q.tile_ids;
  sp.tiles = q.tiles;
  sp.split = q.split;
  sp.images = base + s.images;
  sp.down = reinterpret_cast<float*>(base + s.down);
  sp.runs = reinterpret_cast<int2*>(base + s.runs);
  Sums u{};
  u.p = p;
  u.dy = dy;
  u.dy_ld = dy_ld;
  u.plan = q.plan;
  u.images = sp.images;
  u.down = sp.down;
  u.runs = sp.runs;
  u.dx = static_cast<__half*>(g.dx);
  u.da = g.da;
  u.db = g.db;
  u.part = reinterpret_cast<float*>(base + s.part);
  u.add_dx = g.add_dx;
  u.x_tiles = s.x_tiles;
  u.tiles = s.tiles;
  u.status = g.status;
  SumMaps maps;
  std::memset(&maps, 0, sizeof(maps));
  const uint64_t dims[3] = {(uint64_t)p.K, (uint64_t)p.R, (uint64_t)p.L};
  const uint64_t strides[2] = {(uint64_t)p.K * 2, (uint64_t)p.K * p.R * 2};
  const uint32_t box[3] = {64, (uint32_t)s.RP, 1};
  if (!encode_tmap_3d(&maps.a, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, p.a, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B,
                      err) ||
      !encode_tmap_2d(&maps.x, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, p.x, (uint64_t)p.K, (uint64_t)p.M,
                      (uint64_t)p.x_ld * 2, 64, kStepRows, CU_TENSOR_MAP_SWIZZLE_128B, err) ||
      !encode_tmap_2d(&maps.x8, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, p.x, (uint64_t)p.K, (uint64_t)p.M,
                      (uint64_t)p.x_ld * 2, 64, 8, CU_TENSOR_MAP_SWIZZLE_128B, err) ||
      !encode_tmap_2d(&maps.dy, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, dy, (uint64_t)p.N, (uint64_t)p.M,
                      (uint64_t)dy_ld * 2, 64, kStepRows, CU_TENSOR_MAP_SWIZZLE_128B, err) ||
      !encode_tmap_2d(&maps.dy8, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, dy, (uint64_t)p.N, (uint64_t)p.M,
                      (uint64_t)dy_ld * 2, 64, 8, CU_TENSOR_MAP_SWIZZLE_128B, err))
    return cudaErrorInvalidValue;
  const int64_t items = s.max_chunks * s.tiles;
  if (p.R <= 16) return launch_sums<16>(sp, u, maps, s.max_steps, items, sm_count, pdl, stream);
  if (p.R <= 32) return launch_sums<32>(sp, u, maps, s.max_steps, items, sm_count, pdl, stream);
  if (p.R <= 64) return launch_sums<64>(sp, u, maps, s.max_steps, items, sm_count, pdl, stream);
  return launch_sums<128>(sp, u, maps, s.max_steps, items, sm_count, pdl, stream);
}

}  // namespace qw
