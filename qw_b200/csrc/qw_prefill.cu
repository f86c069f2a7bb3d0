// qw_prefill.cu -- affine 4-bit group-64 quantized matmul for prefill-sized
// M (>= 17 rows of x) on the 5th-generation tensor cores.  Compute-bound.
//
// One CTA per SM walks output tiles of 128 weight rows x 256 tokens
// (persistent, token tiles fastest so a weight tile is reused from L2):
//
//   warp 0      TMA producer, per 64-wide k group: the x box (256 tokens x
//               64 halves, 128-byte swizzle, K-major: the UMMA B operand) and
//               the packed weights of the group (128 rows x 32 bytes).
//   warp 1      allocates TMEM and issues tcgen05.mma (one thread):
//               D[128 x 256, fp32, TMEM] += A[128 x 64, TMEM] * x^T, four
//               K=16 instructions per group, tcgen05.commit releasing stages.
//   warps 2-9   dequantize: the two warps of a TMEM lane quarter own its 32
//               weight rows (one row per lane) and take alternate groups, all
//               64 codes of each; they write fp16 weights to a TMEM A stage
//               with tcgen05.st.  After the last group of a tile they read D
//               back (tcgen05.ld, half of the tokens each) and store y.
//
// SwiGLU (gate and up projections with the activation fused): a tile is 64
// gate rows and the same 64 up rows, staged so that TMEM lanes l and l + 16
// of each lane quarter hold one output's gate and up sums; the epilogue pairs
// them with one shuffle per token and writes silu(gate) * up (64 outputs per
// tile, each op rounded to fp16).
//
// LORA (a separate instantiation): adapters beside the projection, as further
// columns of the reduction.  A token tile that names n adapters of rank R gets
// ceil(n R8 / 64) more k blocks (R8 the rank rounded up to 8): block columns
// (adapter, r) hold lora_b of the tile's weight rows as A and h = s x A^T, fp16,
// of the tokens that take that adapter as B, zero for the others.  Four more
// warps write both (TMEM and the swizzled x slot) while the dequant warps are at
// the weights; the producer only passes the stage on.  2048 x 17408 x 5120 with 8
// adapters of rank 32: 380 us, where the projection alone takes 369 (421 and 418 once
// the power cap lowers the clocks); a pass of its own over y would read and write 214 MB.
// A zero times another adapter's infinity would be NaN: lora_b and h values that
// are not finite fp16 enter as zero, and their terms, with h in fp32, are added in
// the epilogue for the tokens that own them (so h may pass 65504).
// The weights are fp16(s q + b), rounded once: the result's error is half of that
// with the two roundings below (2.8e-4 and 5.7e-4 of y in the mean, 2048 x 17408 x 5120;
// y's own rounding alone is 2.1e-4).  The rest would take a second fp16 term, twice the
// products and the tensor memory.
//
// Otherwise the weights the MMA consumes are exactly qw_dequantize's (fp16(fp16(s*q)
// + b)): pairs (1024 + q_even, 1024 + 16 q_odd) come from one prmt and one
// and, fma.rn.f16x2 with (s, s/16) and (-1024 s, -64 s) gives fp16(s*q)
// rounded once from the exact product, and add.rn.f16x2 adds b.  Scales too
// small for s/16 to be exact, or too large for 1024 s, take an exact
// per-element path.  Accumulation is fp32 in the tensor cores.
#include <cuda_fp16.h>

#include <type_traits>

#include "qw_internal.h"
#include "qw_ptx.cuh"

namespace qw {

namespace {

constexpr int kGroup = 64;
constexpr int BM = 128;       // weight rows per tile (UMMA M, TMEM lanes)
// Packed codes of one 64-wide k block: BITS/2 words (4-bit: 8, 8-bit: 16) per
// row.  BT tokens per tile (UMMA N): 256 for prefill; 32 for calls of at most
// 32 rows of x (the configurations without the decode kernel: 8-bit codes,
// groups of 128, and 17..32 rows), whose narrow x tiles leave room for a
// deeper pipeline of weight blocks.
template <int BITS, int BT_>
struct PfCfg {
  static constexpr int BT = BT_;
  static constexpr int STAGES = BT >= 128 ? 4 : 8;  // pipeline depth (x box, packed W, TMEM A)
  static constexpr int X_STAGE = BT * 128;          // 64 halves of k per token row
  static constexpr int WP_ROW = kGroup * BITS / 8;   // bytes per row per k block
  static constexpr int WORDS = kGroup * BITS / 32;   // packed words per row per k block
  static constexpr int WP_STAGE = BM * WP_ROW;
  static constexpr int OFF_X = 0;
  static constexpr int OFF_WP = STAGES * X_STAGE;
  // barriers: xfull, wpfull, wpempty, afull, aempty (per stage), dfull, dempty
  static constexpr int NBAR = 5 * STAGES + 2;
  static constexpr int OFF_BAR = OFF_WP + STAGES * WP_STAGE;
  // LORA: whether a weight row has non-finite lora_b values, a slot for each of the
  // last STAGES tiles.  The slot of a tile STAGES further on is written with its last
  // block, when the block STAGES before that one has been multiplied.  The tiles from
  // the next on have at least STAGES + 1 blocks together (one each, two where adapters
  // are), so that block belongs to them, and their products wait for this tile's epilogue.
  static constexpr int OFF_BAD = OFF_BAR + NBAR * 8 + 64;
  // LORA: barriers, the producer has freed the stage for an adapters' block
  static constexpr int OFF_XGO = OFF_BAD + STAGES * BM;
  // LORA: of the same tiles as OFF_BAD's, whether a warp met such values in h
  static constexpr int OFF_WIDE = OFF_XGO + 8 * STAGES;
  static constexpr int SMEM = OFF_BAD + 1024;
  static constexpr int SMEM_LORA = SMEM + STAGES * BM + 12 * STAGES;
  // TMEM: D (BT fp32 columns) at 0, then the A stages (32 columns each)
  static constexpr uint32_t D_COL = 0;
  static constexpr uint32_t A_COL = BT >= 128 ? BT : 128;
  static constexpr uint32_t TMEM_COLS = A_COL + 32 * STAGES <= 256 ? 256 : 512;
  static_assert(A_COL + 32 * STAGES <= 512, "TMEM columns");
  static_assert(SMEM_LORA <= 232448, "shared memory budget");
};
constexpr int DQW = 8;             // dequant / epilogue warps: 2 per TMEM lane quarter
constexpr int THREADS = (2 + DQW) * 32;
constexpr int THREADS_LORA = THREADS + 128;  // and four warps that stage the adapters' blocks

struct PrefillParams {
  int M, N, K;
  int n_tiles, m_tiles, groups;  // groups: 64-wide k blocks
  int gsh;                       // k blocks per quantization group (group_size / 64)
  int sb_groups;                 // quantization groups per row (K / group_size)
  int y_f32;
  int swiglu;      // gate (tm_w, scales, biases) and up (tm_w2, scales2, biases2), 64 rows of each per tile
  int tile_rows;   // output rows per tile: 128, or 64 with swiglu
  void* y;
  const __half* scales;
  const __half* biases;
  const __half* scales2;
  const __half* biases2;
  unsigned int* status;
  PrefillLora lora;  // LORA
  int lora_r8;       // rank rounded up to 8, in 8-wide chunks
};

// 8 consecutive ranks of one lora_b row from rank r0 on, zero past the rank.
__device__ __forceinline__ uint4 lora_chunk(const __half* row, int r0, int R) {
  if (R % 8 == 0) return __ldg(reinterpret_cast<const uint4*>(row + r0));
  uint32_t w[4] = {0u, 0u, 0u, 0u};
  if (R % 4 == 0) {  // rows of 8-byte alignment
#pragma unroll
    for (int i = 0; i < 4; i += 2)
      if (r0 + 2 * i < R) {
        const uint2 v = __ldg(reinterpret_cast<const uint2*>(row + r0 + 2 * i));
        w[i] = v.x;
        w[i + 1] = v.y;
      }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t lo = r0 + 2 * i < R ? __half_as_ushort(row[r0 + 2 * i]) : 0;
      const uint32_t hi = r0 + 2 * i + 1 < R ? __half_as_ushort(row[r0 + 2 * i + 1]) : 0;
      w[i] = lo | (hi << 16);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
// Replaces non-finite fp16 values (exponent all ones) by zero; whether there were
// any.  One more in the exponent's place carries into the sign's where it is all
// ones, so that the usual case takes two operations a pair.
__device__ __forceinline__ bool make_finite(uint4 (&v)[8]) {
  uint32_t met = 0u;
#pragma unroll
  for (int c = 0; c < 8; ++c)
    met |= ((v[c].x & 0x7C007C00u) + 0x04000400u) | ((v[c].y & 0x7C007C00u) + 0x04000400u) |
           ((v[c].z & 0x7C007C00u) + 0x04000400u) | ((v[c].w & 0x7C007C00u) + 0x04000400u);
  if ((met & 0x80008000u) == 0u) return false;
  auto finite = [](uint32_t w) {
    return ((w & 0x7C00u) == 0x7C00u ? 0u : w & 0xFFFFu) | ((w & 0x7C000000u) == 0x7C000000u ? 0u : w & 0xFFFF0000u);
  };
#pragma unroll
  for (int c = 0; c < 8; ++c) v[c] = make_uint4(finite(v[c].x), finite(v[c].y), finite(v[c].z), finite(v[c].w));
  return true;
}
__device__ __forceinline__ uint32_t lora_adapter_of(const PrefillLora& l, int tok, int M) {
  if (tok >= M) return 0xFFFFFFFFu;
  return l.idx ? l.idx[tok] : 0u;
}

__device__ __forceinline__ uint64_t smem_desc_sw128(uint32_t addr) {
  // K-major, 128-byte swizzle: rows of 128 bytes, 8-row atoms 1024 bytes apart.
  return (uint64_t)((addr >> 4) & 0x3FFF) | ((uint64_t)1 << 16) | ((uint64_t)(1024 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}

// kind::f16 instruction descriptor: D fp32, A/B fp16, both K-major, M x N.
constexpr uint32_t idesc_f16(int m, int n) {
  return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

__device__ __forceinline__ void tmem_st_x16(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}

__device__ __forceinline__ uint32_t h2_bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }

// Exact per-element dequantization, for scales outside the fast path's range.
// Inlined and fully unrolled so that `out` stays in registers on both paths.
__device__ __forceinline__ void dequant_group_slow(const uint32_t (&wd)[4], __half s, __half b, uint32_t (&out)[16]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#pragma unroll
    for (int pp = 0; pp < 4; ++pp) {
      const uint32_t q0 = (wd[i] >> (8 * pp)) & 0xFu, q1 = (wd[i] >> (8 * pp + 4)) & 0xFu;
      const __half t0 = __hmul_rn(s, __uint2half_rn(q0));
      const __half t1 = __hmul_rn(s, __uint2half_rn(q1));
      out[4 * i + pp] = h2_bits(__halves2half2(__hadd_rn(t0, b), __hadd_rn(t1, b)));
    }
  }
}

// fp16(s q + b) of a block's 64 codes, rounded once.  A code's bits in the low
// byte of a half are the subnormal 16 q 2^-24 (4 bits) or q 2^-24 (8 bits), exact:
// one fma with s 2^20 or s 2^24, as long as that is finite; larger scales take
// 1024 + 16 q (or q) less 1024, with s/16 (or s) and for the even 4-bit codes s.
template <int BITS>
__device__ __forceinline__ void weights_once(const uint32_t (&wd)[BITS * 2], __half s, uint32_t b2,
                                             uint32_t (&out)[2][16]) {
  const float sf = __half2float(s);
  if (fabsf(sf) < (BITS == 4 ? 0.0624f : 0.0039f)) {
    const __half up = __float2half_rn(sf * (BITS == 4 ? 1048576.f : 16777216.f));
    const uint32_t up2 = h2_bits(__halves2half2(up, up));
#pragma unroll
    for (int i = 0; i < BITS * 2; ++i) {
      if (BITS == 4) {
        const uint32_t even = wd[i] << 4;
#pragma unroll
        for (int pp = 0; pp < 4; ++pp)
          out[i / 4][4 * (i % 4) + pp] = hfma2_rn(prmt(even, wd[i], 0x0400u + 0x0101u * pp) & 0x00F000F0u, up2, b2);
      } else {
        out[i / 8][2 * (i % 8)] = hfma2_rn(prmt(wd[i], 0u, 0x5140u), up2, b2);
        out[i / 8][2 * (i % 8) + 1] = hfma2_rn(prmt(wd[i], 0u, 0x5342u), up2, b2);
      }
    }
  } else {
    const uint32_t s2 = h2_bits(__halves2half2(s, BITS == 4 ? __float2half_rn(sf * 0.0625f) : s));
#pragma unroll
    for (int i = 0; i < BITS * 2; ++i) {
      if (BITS == 4) {
#pragma unroll
        for (int pp = 0; pp < 4; ++pp) {
          const uint32_t t = prmt(wd[i], 0x64646464u, 0x4040u + 0x0101u * pp) & 0xFFF0FF0Fu;
          out[i / 4][4 * (i % 4) + pp] = hfma2_rn(hsub2_rn(t, 0x64006400u), s2, b2);
        }
      } else {
        out[i / 8][2 * (i % 8)] = hfma2_rn(hsub2_rn(prmt(wd[i], 0x64646464u, 0x5140u), 0x64006400u), s2, b2);
        out[i / 8][2 * (i % 8) + 1] = hfma2_rn(hsub2_rn(prmt(wd[i], 0x64646464u, 0x5342u), 0x64006400u), s2, b2);
      }
    }
  }
}

// Terms of a token's own adapter in which lora_b or h is not finite fp16.  No part of
// the epilogue's code: inlined, it made the usual case slower too (37 x 4099 x 2560
// 33.4 us, not 31.6; 2048 x 17408 x 5120 390, not 377).
__device__ __noinline__ float own_terms(const PrefillParams& p, int tok, int row) {
  const PrefillLora& l = p.lora;
  const uint32_t a = lora_adapter_of(l, tok, p.M);
  if (a >= (uint32_t)l.L) return 0.f;
  const __half* h = reinterpret_cast<const __half*>(l.h) + (size_t)tok * 8 * p.lora_r8;
  const float* full = l.full + (size_t)tok * 8 * p.lora_r8;
  const __half* b = reinterpret_cast<const __half*>(l.b) + ((size_t)a * p.N + row) * l.R;
  float f = 0.f;
  for (int r = 0; r < l.R; ++r) {
    const float bv = __half2float(b[r]), hr = __half2float(h[r]);
    if (!isfinite(hr)) f += __ldcg(full + r) * bv;
    else if (!isfinite(bv)) f += hr * bv;
  }
  return f;
}

template <int BITS, int BT_, bool LORA>
__global__ void __launch_bounds__(LORA ? THREADS_LORA : THREADS, 1)
    qmm_prefill_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w,
                       const __grid_constant__ CUtensorMap tm_w2, const PrefillParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  using Cfg = PfCfg<BITS, BT_>;
  constexpr int BT = Cfg::BT;
  constexpr int STAGES = Cfg::STAGES;
  constexpr int X_STAGE = Cfg::X_STAGE;
  constexpr int OFF_X = Cfg::OFF_X;
  constexpr uint32_t D_COL = Cfg::D_COL, A_COL = Cfg::A_COL, TMEM_COLS = Cfg::TMEM_COLS;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Cfg::OFF_BAR);
  uint64_t* xfull = bars;
  uint64_t* wpfull = bars + STAGES;
  uint64_t* wpempty = bars + 2 * STAGES;
  uint64_t* afull = bars + 3 * STAGES;
  uint64_t* aempty = bars + 4 * STAGES;  // arrived by tcgen05.commit: x slot and A stage are free
  uint64_t* dfull = bars + 5 * STAGES;
  uint64_t* dempty = dfull + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(dempty + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x / 32;
  const int lane = threadIdx.x % 32;
  const int total_tiles = p.n_tiles * p.m_tiles;
  uint8_t* const bad_rows = smem + Cfg::OFF_BAD;  // LORA: [tile % STAGES][BM]
  uint32_t* const wide_tiles = reinterpret_cast<uint32_t*>(smem + Cfg::OFF_WIDE);  // LORA: [tile % STAGES], a byte a warp
  uint64_t* const xgo = reinterpret_cast<uint64_t*>(smem + Cfg::OFF_XGO);  // LORA
  // k blocks of a token tile: the weights' groups, then its adapters'
  auto blocks_of = [&](int mt) {
    if constexpr (LORA) return p.groups + ((int)__ldcg(p.lora.tile_n + mt) * p.lora_r8 + 7) / 8;
    else return p.groups;
  };

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&xfull[s], 1);
      mbar_init(&wpfull[s], 1);
      mbar_init(&wpempty[s], DQW / 2);  // the four warps (lane quarters) that own the group
      mbar_init(&afull[s], DQW / 2);
      mbar_init(&aempty[s], 1);
      if (LORA) mbar_init(&xgo[s], 1);
    }
    mbar_init(dfull, 1);
    mbar_init(dempty, DQW);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_launch_dependents();

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    if (lane == 0) {
      prefetch_tensormap(&tm_x);
      prefetch_tensormap(&tm_w);
      if (p.swiglu) prefetch_tensormap(&tm_w2);
      pdl_wait();
      const uint64_t pol_w = l2_policy_evict_last();
      uint32_t it = 0;
      for (int tile = blockIdx.x; tile < total_tiles && !*abort_flag; tile += gridDim.x) {
        const int nt = tile / p.m_tiles, mt = tile % p.m_tiles;
        const int blocks = blocks_of(mt);
        for (int g = 0; g < blocks; ++g, ++it) {
          const int s = it % STAGES;
          const uint32_t ph = (it / STAGES) & 1;
          if (it >= STAGES) {
            // x slot s is free once the MMAs that read it completed; the
            // packed-weight slot once the dequant warps read it.
            if (!mbar_wait(&aempty[s], ph ^ 1, p.status, kDevTimeoutEmpty) ||
                !mbar_wait(&wpempty[s], ph ^ 1, p.status, kDevTimeoutEmpty)) {
              *abort_flag = 1;
              break;
            }
          }
          if (LORA && g >= p.groups) {  // the stage is free: the adapters' warps fill it
            mbar_arrive(&xfull[s]);
            mbar_arrive(&wpfull[s]);
            mbar_arrive(&xgo[s]);
            continue;
          }
          mbar_arrive_expect_tx(&xfull[s], X_STAGE);
          tma_load_2d(smem + OFF_X + s * X_STAGE, &tm_x, &xfull[s], g * kGroup, mt * BT);
          mbar_arrive_expect_tx(&wpfull[s], Cfg::WP_STAGE);
          uint8_t* wp = smem + Cfg::OFF_WP + s * Cfg::WP_STAGE;
          if (!p.swiglu) {
            tma_load_2d_hint(wp, &tm_w, &wpfull[s], g * Cfg::WP_ROW, nt * BM, pol_w);
          } else {  // 64 gate rows, then the same 64 up rows
            tma_load_2d_hint(wp, &tm_w, &wpfull[s], g * Cfg::WP_ROW, nt * (BM / 2), pol_w);
            tma_load_2d_hint(wp + (BM / 2) * Cfg::WP_ROW, &tm_w2, &wpfull[s], g * Cfg::WP_ROW, nt * (BM / 2), pol_w);
          }
        }
      }
      // what is under way lands before the CTA goes, whoever gave up waiting for it
      for (uint32_t u = it < (uint32_t)STAGES ? 0u : it - STAGES; u < it; ++u) {
        mbar_wait(&xfull[u % STAGES], (u / STAGES) & 1, p.status, kDevTimeoutFull);
        mbar_wait(&wpfull[u % STAGES], (u / STAGES) & 1, p.status, kDevTimeoutFull);
      }
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------- MMA issuer
    constexpr uint32_t idesc = idesc_f16(BM, BT);
    uint32_t it = 0, tile_count = 0;
    if (LORA) pdl_wait();  // the lists are the previous kernel's
    for (int tile = blockIdx.x; tile < total_tiles; tile += gridDim.x, ++tile_count) {
      // the epilogue has drained D from the previous tile
      if (tile_count > 0 && !*abort_flag &&
          !mbar_wait(dempty, (tile_count - 1) & 1, p.status, kDevTimeoutAccum))
        *abort_flag = 1;
      tc_fence_after();
      const int blocks = blocks_of(tile % p.m_tiles);
      for (int g = 0; g < blocks; ++g, ++it) {
        const int s = it % STAGES;
        const uint32_t ph = (it / STAGES) & 1;
        if (!*abort_flag) {
          if (!mbar_wait(&xfull[s], ph, p.status, kDevTimeoutFull) ||
              !mbar_wait(&afull[s], ph, p.status, kDevTimeoutFull))
            *abort_flag = 1;
        }
        tc_fence_after();
        if (lane == 0 && !*abort_flag) {
          const uint64_t bdesc = smem_desc_sw128(smem_u32(smem + OFF_X + s * X_STAGE));
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) {
            tc_mma_ts(tmem + D_COL, tmem + A_COL + s * 32 + kk * 8, bdesc + (uint64_t)(2 * kk), idesc,
                      (g > 0 || kk > 0) ? 1u : 0u);
          }
        }
        __syncwarp();
        if (lane == 0) tc_commit(&aempty[s]);  // frees x slot s and A stage s when these MMAs finish
        __syncwarp();
      }
      if (lane == 0) tc_commit(dfull);
      __syncwarp();
    }
  } else if (LORA && warp >= 2 + DQW) {
    // ------------------------------- the adapters' k blocks (A in TMEM, x slot)
    const int quarter = warp & 3;
    const int lane_row = quarter * 32 + lane;
    const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
    const __half* lb = reinterpret_cast<const __half*>(p.lora.b);
    const uint4* hb = reinterpret_cast<const uint4*>(p.lora.h);
    const int r8 = p.lora_r8;
    pdl_wait();
    // xgo[s] completes a phase per adapters' block in stage s, and its next one only after these warps have
    // passed the stage on (wpempty), so its parity is that of the blocks counted here
    uint32_t it0 = 0, tile_count = 0, parities = 0;
    for (int tile = blockIdx.x; tile < total_tiles; tile += gridDim.x, ++tile_count) {
      const int nt = tile / p.m_tiles, mt = tile % p.m_tiles;
      const int blocks = blocks_of(mt);
      const int n = (int)__ldcg(p.lora.tile_n + mt);
      const uint32_t* list = p.lora.tile_ids + (size_t)mt * BT;
      const int row = nt * BM + lane_row;
      const bool row_ok = row < p.N;
      bool bad = false, wide = false;
      for (int g = p.groups; g < blocks; ++g) {
        const int s = (int)((it0 + (uint32_t)g) % STAGES);
        // chunk c (8 wide) of the block is ranks 8 rc .. of entry j of the tile's list
        const int j0 = (g - p.groups) * 8 / r8, rc0 = (g - p.groups) * 8 % r8;
        uint4 v[8];
        {
          int j = j0, rc = rc0;
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            v[c] = make_uint4(0u, 0u, 0u, 0u);
            if (j < n && row_ok)
              v[c] = lora_chunk(lb + ((size_t)__ldcg(list + j) * p.N + row) * p.lora.R, rc * 8, p.lora.R);
            if (++rc == r8) rc = 0, ++j;
          }
        }
        uint32_t slot[BT > BM ? BT / BM : 1];
#pragma unroll
        for (int i = 0; i < (BT > BM ? BT / BM : 1); ++i) {
          const int tok = mt * BT + lane_row + i * BM;
          slot[i] = lane_row + i * BM < BT && tok < p.M ? __ldcg(p.lora.slots + tok) : 0xFFFFFFFFu;
        }
        if (!*abort_flag && !mbar_wait(&xgo[s], (parities >> s) & 1u, p.status, kDevTimeoutFull)) *abort_flag = 1;
        parities ^= 1u << s;
        // h of the tokens that take each column's adapter, at the places TMA's 128-byte swizzle gives them
#pragma unroll 1
        for (int i = 0; i < (BT > BM ? BT / BM : 1); ++i) {
          const int t = lane_row + i * BM;
          if (t >= BT) continue;
          const uint4* h = hb + (size_t)(mt * BT + t) * r8;
          uint4 hv[8];
          int j = j0, rc = rc0;
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            hv[c] = make_uint4(0u, 0u, 0u, 0u);
            if ((uint32_t)j == slot[i]) hv[c] = __ldcg(h + rc);
            if (++rc == r8) rc = 0, ++j;
          }
          wide |= make_finite(hv);
          uint8_t* dst = smem + OFF_X + s * X_STAGE + t * 128;
#pragma unroll
          for (int c = 0; c < 8; ++c) *reinterpret_cast<uint4*>(dst + ((c ^ (t & 7)) << 4)) = hv[c];
        }
        fence_proxy_async_smem();
        bad |= make_finite(v);
        uint32_t out[2][16];
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          out[c / 4][4 * (c % 4)] = v[c].x;
          out[c / 4][4 * (c % 4) + 1] = v[c].y;
          out[c / 4][4 * (c % 4) + 2] = v[c].z;
          out[c / 4][4 * (c % 4) + 3] = v[c].w;
        }
        if (g + 1 == blocks) {
          bad_rows[tile_count % STAGES * BM + lane_row] = bad;
          const bool met = __any_sync(0xffffffffu, wide);
          if (lane == 0) reinterpret_cast<uint8_t*>(wide_tiles + tile_count % STAGES)[quarter] = met;
        }
        __syncwarp();
        tc_fence_after();
        tmem_st_x16(tmem + lane_base + A_COL + s * 32, out[0]);
        tmem_st_x16(tmem + lane_base + A_COL + s * 32 + 16, out[1]);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&wpempty[s]);
          mbar_arrive(&afull[s]);
        }
      }
      it0 += (uint32_t)blocks;
    }
  } else {
    // ---------------------------------------------- dequant + epilogue
    const int dw = warp - 2;                 // 0..7
    const int quarter = warp & 3;            // TMEM lane quarter this warp may access
    const int khalf = dw >> 2;               // which groups (even / odd) / which 128 tokens
    // The weight row this lane dequantizes into its TMEM lane (quarter * 32 +
    // lane): the tile's row quarter * 32 + lane, or with SwiGLU, lanes 0-15
    // of a quarter take gate rows 16 quarter + lane and lanes 16-31 the same
    // rows' up projection (staged 64 rows further on), so lanes l and l + 16
    // hold the two halves of one output.
    const bool up_lane = p.swiglu && lane >= 16;
    const int row_in_tile = p.swiglu ? quarter * 16 + (lane & 15) : quarter * 32 + lane;  // output row
    const int smem_row = p.swiglu ? row_in_tile + (up_lane ? BM / 2 : 0) : row_in_tile;
    const __half* scales = up_lane ? p.scales2 : p.scales;
    const __half* biases = up_lane ? p.biases2 : p.biases;
    const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
    pdl_wait();
    uint32_t tile_count = 0, it0 = 0;  // it0: k blocks of the tiles before
    for (int tile = blockIdx.x; tile < total_tiles; tile += gridDim.x, ++tile_count) {
      const int nt = tile / p.m_tiles, mt = tile % p.m_tiles;
      const int blocks = blocks_of(mt);
      const int row = nt * p.tile_rows + row_in_tile;
      const bool row_ok = row < p.N;
      const __half* srow = scales + (size_t)(row_ok ? row : 0) * p.sb_groups;
      const __half* brow = biases + (size_t)(row_ok ? row : 0) * p.sb_groups;
      // This warp dequantizes every other k block of the tile in full (the
      // other warp of its lane quarter takes the rest), so each warp has two
      // MMA block-times per block of its own.
      __half s_next = (row_ok && khalf < p.groups) ? srow[khalf / p.gsh] : __float2half(0.f);
      __half b_next = (row_ok && khalf < p.groups) ? brow[khalf / p.gsh] : __float2half(0.f);
      for (int g = khalf; g < p.groups; g += 2) {
        const uint32_t it = it0 + (uint32_t)g;
        const int s = it % STAGES;
        const uint32_t ph = (it / STAGES) & 1;
        const __half sc = s_next, bi = b_next;
        if (g + 2 < p.groups && row_ok) {  // prefetch this warp's next block's scale/bias
          s_next = srow[(g + 2) / p.gsh];
          b_next = brow[(g + 2) / p.gsh];
        }
        if (!*abort_flag && !mbar_wait(&wpfull[s], ph, p.status, kDevTimeoutFull)) *abort_flag = 1;
        uint32_t wd[Cfg::WORDS];
        {
          const uint4* src =
              reinterpret_cast<const uint4*>(smem + Cfg::OFF_WP + s * Cfg::WP_STAGE + smem_row * Cfg::WP_ROW);
#pragma unroll
          for (int i = 0; i < Cfg::WORDS / 4; ++i) {
            const uint4 a = src[i];
            wd[4 * i] = a.x; wd[4 * i + 1] = a.y; wd[4 * i + 2] = a.z; wd[4 * i + 3] = a.w;
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&wpempty[s]);
        // dequantize the block's 64 codes into 32 fp16 pairs (k ascending)
        uint32_t out[2][16];
        const float sf = __half2float(sc);
        const uint32_t b2 = h2_bits(__halves2half2(bi, bi));
        if (LORA) {
          weights_once<BITS>(wd, sc, b2, out);
        } else if (BITS == 4) {
          const bool fast = fabsf(sf) >= 0.0009765625f && fabsf(sf) < 63.0f;  // s/16 exact, 1024 s finite
          if (fast) {
            const __half s16 = __float2half_rn(sf * 0.0625f);  // exact: s >= 2^-10
            const uint32_t s2 = h2_bits(__halves2half2(sc, s16));
            const uint32_t c2 =
                h2_bits(__halves2half2(__float2half_rn(-1024.f * sf), __float2half_rn(-64.f * sf)));
#pragma unroll
            for (int hh = 0; hh < 2; ++hh)
#pragma unroll
              for (int i = 0; i < 4; ++i) {
#pragma unroll
                for (int pp = 0; pp < 4; ++pp) {
                  const uint32_t t = prmt(wd[4 * hh + i], 0x64646464u, 0x4040u + 0x0101u * pp) & 0xFFF0FF0Fu;
                  out[hh][4 * i + pp] = hadd2_rn(hfma2_rn(t, s2, c2), b2);
                }
              }
          } else {
            uint32_t w0[4] = {wd[0], wd[1], wd[2], wd[3]}, w1[4] = {wd[4], wd[5], wd[6], wd[7]};
            dequant_group_slow(w0, sc, bi, out[0]);
            dequant_group_slow(w1, sc, bi, out[1]);
          }
        } else {
          // 8-bit: a word holds 4 codes; prmt pairs them with 0x64 into
          // (1024 + q_even, 1024 + q_odd), and fma with (s, s), (-1024 s,
          // -1024 s) rounds s*q once from the exact product.
          const bool fast = fabsf(sf) < 63.0f;  // 1024 s finite
          if (fast) {
            const uint32_t s2 = h2_bits(__halves2half2(sc, sc));
            const __half c = __float2half_rn(-1024.f * sf);
            const uint32_t c2 = h2_bits(__halves2half2(c, c));
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const uint32_t t0 = prmt(wd[i], 0x64646464u, 0x5140u);
              const uint32_t t1 = prmt(wd[i], 0x64646464u, 0x5342u);
              out[i / 8][2 * (i % 8)] = hadd2_rn(hfma2_rn(t0, s2, c2), b2);
              out[i / 8][2 * (i % 8) + 1] = hadd2_rn(hfma2_rn(t1, s2, c2), b2);
            }
          } else {
#pragma unroll
            for (int i = 0; i < 16; ++i)
#pragma unroll
              for (int pp = 0; pp < 2; ++pp) {
                const uint32_t q0 = (wd[i] >> (16 * pp)) & 0xFFu, q1 = (wd[i] >> (16 * pp + 8)) & 0xFFu;
                const __half t0 = __hmul_rn(sc, __uint2half_rn(q0));
                const __half t1 = __hmul_rn(sc, __uint2half_rn(q1));
                out[i / 8][2 * (i % 8) + pp] = h2_bits(__halves2half2(__hadd_rn(t0, bi), __hadd_rn(t1, bi)));
              }
          }
        }
        // write A stage s once the MMAs that read it last have completed
        if (it >= STAGES && !*abort_flag && !mbar_wait(&aempty[s], ph ^ 1, p.status, kDevTimeoutEmpty))
          *abort_flag = 1;
        __syncwarp();  // scales of two kinds took two ways
        tc_fence_after();
        tmem_st_x16(tmem + lane_base + A_COL + s * 32, out[0]);
        tmem_st_x16(tmem + lane_base + A_COL + s * 32 + 16, out[1]);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&afull[s]);
      }
      // ---------------------------------------------------------- epilogue
      it0 += (uint32_t)blocks;
      if (!*abort_flag && !mbar_wait(dfull, tile_count & 1, p.status, kDevTimeoutAccum)) *abort_flag = 1;
      tc_fence_after();
      float bias = 0.f;
      bool bad = false, wide = false;  // non-finite lora_b values in this row, h values in this tile
      if (LORA) {
        if (p.lora.bias && row_ok) bias = __half2float(reinterpret_cast<const __half*>(p.lora.bias)[row]);
        bad = blocks > p.groups && bad_rows[tile_count % STAGES * BM + quarter * 32 + lane];
        wide = blocks > p.groups && wide_tiles[tile_count % STAGES] != 0u;
      }
      auto store_tile = [&](auto with_bad) {
#pragma unroll 1
        for (int cb = khalf * (BT / 32); cb < (khalf + 1) * (BT / 32); ++cb) {
          uint32_t v[16];
          __syncwarp();  // lanes past the last row came early
          tmem_ld_32x32b_x16(tmem + lane_base + D_COL + cb * 16, v);
          tmem_wait_ld();
          if (p.swiglu) {
            // lane l < 16 finishes tokens 0-7 of the block and lane l + 16
            // tokens 8-15: each sends its partner the half the partner needs
            float g[8], u[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) {
              const float mine_lo = __uint_as_float(v[q]), mine_hi = __uint_as_float(v[q + 8]);
              const float other = __shfl_xor_sync(0xffffffffu, up_lane ? mine_lo : mine_hi, 16);
              g[q] = up_lane ? other : mine_lo;
              u[q] = up_lane ? mine_hi : other;
            }
            if (!row_ok || *abort_flag) continue;
#pragma unroll
            for (int q = 0; q < 8; ++q) {
              const int tok = mt * BT + cb * 16 + (up_lane ? 8 : 0) + q;
              if (tok < p.M) {
                const size_t idx = (size_t)tok * p.N + row;
                const float h = swiglu_f16(g[q], u[q]);
                if (p.y_f32) reinterpret_cast<float*>(p.y)[idx] = h;
                else reinterpret_cast<__half*>(p.y)[idx] = __float2half_rn(h);
              }
            }
            continue;
          }
          if (!row_ok || *abort_flag) continue;
#pragma unroll
          for (int q = 0; q < 16; ++q) {
            const int tok = mt * BT + cb * 16 + q;
            if (tok < p.M) {
              const size_t idx = (size_t)tok * p.N + row;
              float f = __uint_as_float(v[q]);
              if constexpr (LORA) {
                f += bias;
                if (decltype(with_bad)::value && (bad || wide)) f += own_terms(p, tok, row);
                reinterpret_cast<__half*>(p.y)[idx] = __float2half_rn(f);
                continue;
              }
              if (p.y_f32) reinterpret_cast<float*>(p.y)[idx] = f;
              else reinterpret_cast<__half*>(p.y)[idx] = __float2half_rn(f);
            }
          }
        }
      };
      // a branch an element for the rare case would cost the whole epilogue (2048 x 17408 x 5120: 45 us of 499)
      if (LORA && __any_sync(0xffffffffu, bad || wide)) store_tile(std::true_type{});
      else store_tile(std::false_type{});
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(dempty);
    }
  }

  // everyone: make sure all tcgen05 work is finished before freeing TMEM
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, TMEM_COLS);
  }
}

}  // namespace

bool prefill_available() { return true; }

namespace {
template <int BITS, int BT, bool LORA>
cudaError_t launch_cfg(const PrefillArgs& a, cudaStream_t stream, bool pdl, std::string* err) {
  constexpr int smem = LORA ? PfCfg<BITS, BT>::SMEM_LORA : PfCfg<BITS, BT>::SMEM;
  using Cfg = PfCfg<BITS, BT>;
  int dev = 0;
  cudaGetDevice(&dev);
  const DeviceInfo& di = device_info(dev);
  static thread_local int configured_dev = -1;
  if (configured_dev != dev) {
    cudaError_t e =
        cudaFuncSetAttribute(qmm_prefill_kernel<BITS, BT, LORA>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    configured_dev = dev;
  }
  PrefillParams p{};
  p.M = (int)a.M;
  p.N = (int)a.N;
  p.K = (int)a.K;
  p.groups = (int)(a.K / kGroup);
  p.gsh = a.group_size / kGroup;
  p.sb_groups = (int)(a.K / a.group_size);
  p.swiglu = a.swiglu ? 1 : 0;
  p.tile_rows = a.swiglu ? BM / 2 : BM;
  p.n_tiles = (int)((a.N + p.tile_rows - 1) / p.tile_rows);
  p.m_tiles = (int)((a.M + BT - 1) / BT);
  p.y_f32 = a.y_f32 ? 1 : 0;
  p.y = a.y;
  p.scales = reinterpret_cast<const __half*>(a.scales);
  p.biases = reinterpret_cast<const __half*>(a.biases);
  p.scales2 = reinterpret_cast<const __half*>(a.swiglu ? a.scales2 : a.scales);
  p.biases2 = reinterpret_cast<const __half*>(a.swiglu ? a.biases2 : a.biases);
  p.status = a.status;
  if (LORA) {
    p.lora = *a.lora;
    p.lora_r8 = (a.lora->R + 7) / 8;
  }
  CUtensorMap tx, tw, tw2;
  if (!encode_tmap_2d(&tx, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, a.x, (uint64_t)a.K, (uint64_t)a.M,
                      (uint64_t)(a.x_ld ? a.x_ld : a.K) * 2, kGroup, BT, CU_TENSOR_MAP_SWIZZLE_128B, err))
    return cudaErrorInvalidValue;
  const uint64_t row_bytes = (uint64_t)a.K * BITS / 8;
  if (!encode_tmap_2d(&tw, CU_TENSOR_MAP_DATA_TYPE_UINT8, a.w, row_bytes, (uint64_t)a.N, row_bytes, Cfg::WP_ROW,
                      p.tile_rows, CU_TENSOR_MAP_SWIZZLE_NONE, err))
    return cudaErrorInvalidValue;
  tw2 = tw;  // unused unless SwiGLU
  if (a.swiglu && !encode_tmap_2d(&tw2, CU_TENSOR_MAP_DATA_TYPE_UINT8, a.w2, row_bytes, (uint64_t)a.N, row_bytes,
                                  Cfg::WP_ROW, p.tile_rows, CU_TENSOR_MAP_SWIZZLE_NONE, err))
    return cudaErrorInvalidValue;
  const int tiles = p.n_tiles * p.m_tiles;
  int grid = di.sm_count < tiles ? di.sm_count : tiles;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(LORA ? THREADS_LORA : THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, qmm_prefill_kernel<BITS, BT, LORA>, tx, tw, tw2, p);
}
}  // namespace

cudaError_t launch_prefill(const PrefillArgs& a, cudaStream_t stream, bool pdl, std::string* err) {
  if ((a.bits != 4 && a.bits != 8) || (a.group_size != 64 && a.group_size != 128) || a.K % a.group_size) {
    *err = "the prefill kernel takes 4- or 8-bit codes in groups of 64 or 128";
    return cudaErrorInvalidValue;
  }
  // narrow token tiles for at most 32 rows of x
  if (a.lora) {
    if (a.M <= 32)
      return a.bits == 4 ? launch_cfg<4, 32, true>(a, stream, pdl, err) : launch_cfg<8, 32, true>(a, stream, pdl, err);
    return a.bits == 4 ? launch_cfg<4, 256, true>(a, stream, pdl, err) : launch_cfg<8, 256, true>(a, stream, pdl, err);
  }
  if (a.M <= 32)
    return a.bits == 4 ? launch_cfg<4, 32, false>(a, stream, pdl, err) : launch_cfg<8, 32, false>(a, stream, pdl, err);
  return a.bits == 4 ? launch_cfg<4, 256, false>(a, stream, pdl, err) : launch_cfg<8, 256, false>(a, stream, pdl, err);
}

int prefill_token_tile(int64_t M) { return M <= 32 ? 32 : 256; }

}  // namespace qw
