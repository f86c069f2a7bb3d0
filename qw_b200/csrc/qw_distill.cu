// qw_distill.cu -- distillation from a teacher's top logits, loss and gradient:
// with p = softmax(t / T) over a row's valid teacher entries (ids below V) and
// q = softmax(z / T) over its V logits,
//   loss = w T^2 sum_j p_j (log p_j - log q_{i_j}),   dz = w T (q - sum_j p_j e_{i_j}).
//
// HBM-bound: z has to be read once and dz written once.  q needs the whole
// row's maximum and sum before the first dz can leave, so a row is held on chip
// in between: a thread-block cluster of up to 8 CTAs per row, each CTA a
// contiguous share of it in shared memory (up to 40 KB, five CTAs of 128 threads
// an SM, or 72 KB, three of 256; longer rows up to 200 KB a CTA).  What a share has beyond that
// (rows of more than 1.6 MB) is read a second time, from L2.  Clusters are
// persistent: behind each vector of dz that a thread writes, it starts the
// asynchronous copy of the next row's vector into the same place, which only
// this thread reads, so loads run under the stores and the reductions and need
// no barrier of their own.
//   1. the teacher's k entries go to shared memory, every warp takes their
//      softmax's normaliser alone, and the z they point at are fetched;
//   2. maximum and sum of exponentials by thread and warp; each warp stores
//      (maximum, sum, its part of sum_j p_j (t_j - z_j)) into every CTA of the
//      cluster, and one cluster barrier later every warp joins them;
//   3. dz = w T q, then the columns the teacher names are written again by the
//      CTA that owns them, behind a barrier.
// Sums and exponentials are fp32 (ex2.approx, 2^-22 of a term; fp32 gradients are off
// by 6.5e-8 in the mean, those of the plain fp32 form by 1.1e-7); the loss, a
// difference of two log-normalisers, is put together in fp64 from them.
// Rows start at any element: up to 15 bytes before the first 16-byte boundary
// and after the last are single elements of rank 0's and the last rank's
// threads.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "../../include/qw_qmm.h"
#include "qw_internal.h"
#include "qw_ptx.cuh"

namespace qw {

namespace {

constexpr int kTopMax = 1024;    // teacher entries per row
constexpr int kClusterMax = 8;   // CTAs per row
constexpr int kWarpsMax = 8;     // warps per CTA
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
  static __device__ __forceinline__ uint4 max(const uint4& a, const uint4& b);  // elementwise, numbers over NaN
  static __device__ __forceinline__ uint4 fill(float v) {
    float f[N];
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = v;
    return pack(f);
  }
};
template <typename H2>
__device__ __forceinline__ uint4 max_pairs(const uint4& a, const uint4& b) {
  uint4 r;
  const uint32_t *pa = &a.x, *pb = &b.x;
  uint32_t* pr = &r.x;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const H2 h = __hmax2(*reinterpret_cast<const H2*>(pa + i), *reinterpret_cast<const H2*>(pb + i));
    pr[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  return r;
}
template <>
__device__ __forceinline__ uint4 Vec<__half>::max(const uint4& a, const uint4& b) {
  return max_pairs<__half2>(a, b);
}
template <>
__device__ __forceinline__ uint4 Vec<__nv_bfloat16>::max(const uint4& a, const uint4& b) {
  return max_pairs<__nv_bfloat162>(a, b);
}
template <>
__device__ __forceinline__ uint4 Vec<float>::max(const uint4& a, const uint4& b) {
  auto mx = [](uint32_t x, uint32_t y) {
    return __float_as_uint(fmaxf(__uint_as_float(x), __uint_as_float(y)));
  };
  return make_uint4(mx(a.x, b.x), mx(a.y, b.y), mx(a.z, b.z), mx(a.w, b.w));
}
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
// Exponentials of a share are taken relative to a reference: the largest
// exponent z c (c = log2(e) / T) rounded up to a whole number, so that one fused
// multiply-add makes an argument, z c - ref, and every term is at most 1.  Where
// the largest exponent is beyond +-kFar the product's own rounding (and that of
// c) would show, so z - max is taken first, the reference being max c; that
// costs an addition an element.  References follow from the maximum, and shares
// are joined by 2^(their difference), taken in fp64.
constexpr float kFar = 64.f;
struct Ref {
  float sub, off;  // argument of z: (z - sub) c - off
  bool far;
  double ref;
};
__device__ __forceinline__ Ref make_ref(float zmax, float c) {
  Ref r{0.f, 0.f, false, -INFINITY};
  if (zmax == -INFINITY) return r;  // nothing here: every exponential is 0
  const float top = zmax * c;
  r.far = !(fabsf(top) <= kFar);
  if (r.far) {
    r.sub = zmax;
    r.ref = (double)zmax * (double)c;
  } else {
    r.off = ceilf(top);
    r.ref = r.off;
  }
  return r;
}

// What a warp tells its cluster: the largest of its logits, the sum of their
// exponentials relative to that maximum's reference, and sum_j p_j (t_j - z_j)
// over its teacher entries.
struct __align__(16) Share {
  double gap;
  float max, sum;
};

// One row's layout: `head` single elements up to the first 16-byte boundary,
// then vectors, of which this thread has those at `first` + e TH N for e TH <
// `count`, then `tail` single elements.
struct RowLayout {
  int first;   // element index of this thread's first vector
  int count;   // vectors from it to the end of the CTA's share
  int edge;    // the single element of this thread, -1: none
  int lo, hi;  // the CTA's columns
};
template <typename T>
__device__ __forceinline__ RowLayout row_layout(const T* z, int V, uint32_t rank, uint32_t C) {
  constexpr int N = Vec<T>::N;
  const int off = (int)((16 - (reinterpret_cast<uintptr_t>(z) & 15)) & 15) / (int)sizeof(T);
  const int head = off < V ? off : V;
  const uint32_t nv = (uint32_t)(V - head) / N;
  const int tail = V - head - (int)nv * N;
  const int v0 = (int)(nv * rank / C), v1 = (int)(nv * (rank + 1) / C);
  const int tid = threadIdx.x;
  RowLayout r;
  r.first = head + (v0 + tid) * N;
  r.count = v1 - v0 - tid;
  r.edge = -1;
  if (rank == 0 && tid < head) r.edge = tid;
  if (rank == C - 1 && tid >= 32 && tid < 32 + tail) r.edge = V - tail + (tid - 32);
  r.lo = rank == 0 ? 0 : head + v0 * N;
  r.hi = rank == C - 1 ? V : head + v1 * N;
  return r;
}

__device__ __forceinline__ void copy_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ uint4 lds16(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

// EVEN: every row of logits and of dlogits starts on a 16-byte boundary and has
// whole vectors, so that one layout serves all.
// Shared memory: `held` vectors per thread, then ids [2][k], tval [2][k], zval [k].
template <typename T, int TH, int PER_SM, bool EVEN>
__global__ void __launch_bounds__(TH, PER_SM) distill_rows_kernel(const DistillArgs p, const int held) {
  using VT = Vec<T>;
  constexpr int kWarps = TH / 32;
  static_assert(kWarps <= kWarpsMax && kWarps * kClusterMax <= 64, "two shares a lane");
  extern __shared__ uint4 smem[];
  __shared__ Share shares_buf[2][kClusterMax * kWarps];
  uint32_t rank, C;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(C));
  // A CTA's shared memory may be written by its cluster only once it runs: waited
  // for before the first share, which the first row's loads come before.
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  const int V = (int)p.V, M = (int)p.M;
  const T* const z0 = reinterpret_cast<const T*>(p.logits);
  uint32_t* const teacher = reinterpret_cast<uint32_t*>(smem + (size_t)held * TH);
  float* const zval = reinterpret_cast<float*>(teacher) + 4 * p.k;
  const uint32_t mine = smem_u32(smem + tid);  // this thread's vectors, TH apart
  const int inside = held * TH;                // e below it is held
  const int stride = (int)(gridDim.x / C);
  int m = (int)(blockIdx.x / C);

  // What of a row is loaded while the row before it is written: this thread's
  // teacher entry, the weight, the vectors and the single element.
  uint32_t id_next = 0xFFFFFFFFu;
  float val_next = 0.f, w_next = 1.f, ze = -INFINITY;
  auto fetch_teacher = [&](int row) {
    if (tid < p.k) {
      id_next = p.idx[(int64_t)row * p.k + tid];
      val_next = load_value(p, (int64_t)row * p.k + tid);
    }
    if (p.weights) w_next = p.weights[row];
  };
  fetch_teacher(m);
  RowLayout lay = row_layout(z0 + (int64_t)m * V, V, rank, C);
  {
    const T* z = z0 + (int64_t)m * V;
    const int n = lay.count < inside ? lay.count : inside;
#pragma unroll 4
    for (int e = 0; e < n; e += TH) copy_async16(mine + e * 16, z + lay.first + e * VT::N);
    if (lay.edge >= 0) ze = to_f32(z[lay.edge]);
  }
  const float temp = p.temperature ? *p.temperature : 1.f;
  const float inv = 1.f / temp;
  const float c = inv * kLog2e;

  // Buffers alternate so that a barrier of their own guards none of them: the
  // teacher's by row, the shares by row that reached the cluster barrier (a CTA
  // may be ahead of its cluster by rows that skip it, but by one barrier only).
  int met = 0;
  bool begun = false;
  for (int parity = 0; m < M; parity ^= 1) {
    uint32_t* const ids = teacher + parity * p.k;
    float* const tval = reinterpret_cast<float*>(teacher) + (2 + parity) * p.k;
    Share* const shares = shares_buf[met];
    const T* const z = z0 + (int64_t)m * V;
    T* const dz = p.dlogits ? reinterpret_cast<T*>(p.dlogits) + (int64_t)m * V : nullptr;
    const float w = w_next;
    const RowLayout cur = lay;
    const int n = cur.count < inside ? cur.count : inside;
    const int next = m + stride;

    // the teacher's entries of the row
    const uint32_t my_id = id_next < (uint32_t)V && tid < p.k ? id_next : 0xFFFFFFFFu;
    const float my_val = my_id != 0xFFFFFFFFu ? val_next : -INFINITY;
    if (tid < p.k) {
      ids[tid] = my_id;
      tval[tid] = my_val;
    }
    for (int j = tid + TH; j < p.k; j += TH) {
      const uint32_t id = p.idx[(int64_t)m * p.k + j];
      const float v = load_value(p, (int64_t)m * p.k + j);
      ids[j] = id < (uint32_t)V ? id : 0xFFFFFFFFu;
      tval[j] = id < (uint32_t)V ? v : -INFINITY;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
    float tmax = -INFINITY, tsum = 0.f;
    bool unknown = false;
    for (int j = lane; j < p.k; j += 32) {
      tmax = fmaxf(tmax, tval[j]);
      unknown = unknown || tval[j] != tval[j];
    }
    tmax = warp_max(tmax);
    if (__any_sync(0xffffffffu, unknown)) tmax = NAN;  // a teacher of NaN alone is no row without entries
    // Writes the row from `value` of each element and, behind each vector's
    // store, starts the next row's copy into its place.
    auto write_row = [&](auto&& value) {
      const bool aligned = EVEN || ((reinterpret_cast<uintptr_t>(z) ^ reinterpret_cast<uintptr_t>(dz)) & 15) == 0;
      auto store = [&](int at, const uint4& v) {
        float f[VT::N];
        VT::load(v, f);
#pragma unroll
        for (int q = 0; q < VT::N; ++q) f[q] = value(f[q]);
        if (aligned) {
          *reinterpret_cast<uint4*>(dz + at) = VT::pack(f);
        } else {  // dlogits start at another offset from a 16-byte boundary than logits
#pragma unroll
          for (int q = 0; q < VT::N; ++q) dz[at + q] = from_f32<T>(f[q]);
        }
      };
      const T* const zn = z0 + (int64_t)next * V;
      int nn = -1;
      if (next < M) {
        fetch_teacher(next);
        if (!EVEN) lay = row_layout(zn, V, rank, C);
        nn = lay.count < inside ? lay.count : inside;
      }
      if (dz) {
        if (EVEN && next < M) {
#pragma unroll 2
          for (int e = 0; e < n; e += TH) {
            store(cur.first + e * VT::N, lds16(mine + e * 16));
            copy_async16(mine + e * 16, zn + cur.first + e * VT::N);
          }
        } else {
#pragma unroll 1
          for (int e = 0; e < n || e < nn; e += TH) {
            if (e < n) store(cur.first + e * VT::N, lds16(mine + e * 16));
            if (e < nn) copy_async16(mine + e * 16, zn + lay.first + e * VT::N);
          }
        }
#pragma unroll 1
        for (int e = inside; e < cur.count; e += TH) {
          const int at = cur.first + e * VT::N;
          store(at, __ldcg(reinterpret_cast<const uint4*>(z + at)));
        }
        if (!EVEN && cur.edge >= 0) dz[cur.edge] = from_f32<T>(value(ze));
      } else {
#pragma unroll 1
        for (int e = 0; e < nn; e += TH) copy_async16(mine + e * 16, zn + lay.first + e * VT::N);
      }
      if (!EVEN) ze = next < M && lay.edge >= 0 ? to_f32(zn[lay.edge]) : -INFINITY;
    };
    if (w == 0.f || tmax == -INFINITY) {  // no weight, or nothing to learn from: the whole cluster takes this branch
      if (rank == 0 && tid == 0) p.loss[m] = 0.f;
      write_row([](float) { return 0.f; });
      m = next;
      continue;
    }
    const bool mine_in = my_id >= (uint32_t)cur.lo && my_id < (uint32_t)cur.hi;
    float my_z = 0.f;
    if (mine_in) my_z = to_f32(z[my_id]);
    for (int j = lane; j < p.k; j += 32) tsum += ex2((tval[j] - tmax) * c);
    tsum = warp_sum(tsum);

    // maximum and sum of this thread's, warp's and cluster's logits
    uint4 mv = VT::fill(-INFINITY);
    auto over_rest = [&](auto&& f) {  // what is not held
#pragma unroll 1
      for (int e = inside; e < cur.count; e += TH)
        f(__ldcg(reinterpret_cast<const uint4*>(z + cur.first + e * VT::N)));
    };
#pragma unroll 4
    for (int e = 0; e < n; e += TH) mv = VT::max(mv, lds16(mine + e * 16));
    over_rest([&](const uint4& v) { mv = VT::max(mv, v); });
    float mx = ze;
    {
      float f[VT::N];
      VT::load(mv, f);
#pragma unroll
      for (int q = 0; q < VT::N; ++q) mx = fmaxf(mx, f[q]);
    }
    mx = warp_max(mx);
    const Ref wr = make_ref(mx, c);
    float sum = cur.edge >= 0 ? ex2((ze - wr.sub) * c - wr.off) : 0.f;
    auto add_all = [&](auto far) {
      auto add = [&](const uint4& v) {
        float f[VT::N];
        VT::load(v, f);
        float part[2] = {0.f, 0.f};
#pragma unroll
        for (int q = 0; q < VT::N; ++q)
          part[q & 1] += ex2(decltype(far)::value ? (f[q] - wr.sub) * c : fmaf(f[q], c, -wr.off));
        sum += part[0] + part[1];
      };
#pragma unroll 4
      for (int e = 0; e < n; e += TH) add(lds16(mine + e * 16));
      over_rest(add);
    };
    if (wr.far) add_all(std::true_type{});
    else add_all(std::false_type{});
    sum = warp_sum(sum);
    double gap = 0.0;
    auto entry = [&](int j, float t, float zj) {
      zval[j] = zj;
      const float pj = ex2((t - tmax) * c) / tsum;
      if (pj > 0.f) gap += zj == -INFINITY ? (double)INFINITY : (double)pj * ((double)t - (double)zj);
    };
    if (mine_in) entry(tid, my_val, my_z);
    for (int j = tid + TH; j < p.k; j += TH)
      if (ids[j] >= (uint32_t)cur.lo && ids[j] < (uint32_t)cur.hi) entry(j, tval[j], to_f32(z[ids[j]]));
    if (__any_sync(0xffffffffu, gap != 0.0)) gap = warp_sum(gap);
    if (!begun) {
      __syncwarp();
      asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
      begun = true;
    }
    if (lane < C) {  // this warp's share into CTA `lane` of the cluster
      uint32_t to;
      asm("mapa.shared::cluster.u32 %0, %1, %2;"
          : "=r"(to)
          : "r"(smem_u32(&shares[rank * kWarps + warp])), "r"((uint32_t)lane));
      asm volatile("st.shared::cluster.f64 [%0], %1;\nst.shared::cluster.v2.f32 [%0+8], {%2, %3};" ::"r"(to), "d"(gap),
                   "f"(mx), "f"(sum)
                   : "memory");
    }
    __syncwarp();  // .aligned takes a whole warp
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    met ^= 1;
    // two shares a lane, joined by every warp
    const int n_shares = (int)C * kWarps;
    Share sa{0.0, -INFINITY, 0.f}, sb = sa;
    if (lane < n_shares) sa = shares[lane];
    if (lane + 32 < n_shares) sb = shares[lane + 32];
    const float zmax = warp_max(fmaxf(sa.max, sb.max));
    const Ref row = make_ref(zmax, c);
    auto joined = [&](const Share& s) {
      return s.max == -INFINITY ? s.sum : s.sum * ex2((float)(make_ref(s.max, c).ref - row.ref));
    };
    const float zsum = warp_sum(joined(sa) + joined(sb));
    const float scale = zsum == 0.f ? 0.f : w * temp / zsum;
    if (row.far) write_row([&](float x) { return ex2((x - row.sub) * c) * scale; });
    else write_row([&](float x) { return ex2(fmaf(x, c, -row.off)) * scale; });
    if (rank == 0 && warp == kWarps - 1) {
      const double g = warp_sum(sa.gap + sb.gap);
      if (lane == 0) {
        // log of p's normaliser over q's; a student row of -inf alone has an infinite gap
        const double norm = (double)tmax * inv + log((double)tsum) -
                            (row.ref * 0.69314718055994531 + log((double)zsum));
        p.loss[m] = (float)((double)w * temp * temp * (isinf(g) ? g : g * inv - norm));
      }
    }
    if (dz) {
      __syncthreads();
      // the teacher's columns of this CTA, a warp an entry: the first entry of
      // an id writes it, with the mass of all its entries
      for (int j0 = warp; j0 < p.k; j0 += 32 * kWarps) {
        const int jl = j0 + lane * kWarps;
        const uint32_t idl = jl < p.k ? ids[jl] : 0xFFFFFFFFu;
        for (uint32_t in = __ballot_sync(0xffffffffu, idl >= (uint32_t)cur.lo && idl < (uint32_t)cur.hi); in;
             in &= in - 1) {
          const int j = j0 + (__ffs(in) - 1) * kWarps;
          const uint32_t id = __shfl_sync(0xffffffffu, idl, __ffs(in) - 1);
          float mass = 0.f;
          bool first = true;
          for (int i = lane; i < p.k; i += 32) {
            if (ids[i] == id) {
              first = first && i >= j;
              mass += ex2((tval[i] - tmax) * c);
            }
          }
          if (!__all_sync(0xffffffffu, first)) continue;
          mass = warp_sum(mass);
          if (lane == 0)
            dz[id] = from_f32<T>(ex2((zval[j] - row.sub) * c - row.off) * scale - w * temp * (mass / tsum));
        }
      }
    }
    m = next;
  }
  if (!begun) {  // no row had a share
    __syncwarp();
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
  }
}

constexpr int64_t kMaxSmem = 227 * 1024 - 2048;  // dynamic shared memory a CTA may take
constexpr int64_t kShortShare = 40 * 1024, kLongShare = 72 * 1024;  // shares of a row

template <typename T, int TH, int PER_SM, bool EVEN>
cudaError_t launch_even(const DistillArgs& p, int cluster, cudaStream_t stream) {
  auto* kernel = distill_rows_kernel<T, TH, PER_SM, EVEN>;
  // vectors per thread that cover a CTA's share of any row, as far as shared memory goes
  const int64_t nv = (p.V * (int64_t)sizeof(T) / 16 + cluster - 1) / cluster + 1;
  int64_t held = (nv + TH - 1) / TH;
  const int64_t top_bytes = (int64_t)p.k * 20;
  if (held * TH * 16 + top_bytes > kMaxSmem) held = (kMaxSmem - top_bytes) / (TH * 16);
  const size_t smem = (size_t)(held * TH * 16 + top_bytes);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)cluster);
  cfg.blockDim = dim3(TH);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)cluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  // as many clusters as the GPU holds at once (asked once per size), each walking rows a grid apart
  static thread_local int configured_dev = -1, asked_cluster = 0, resident = 0;
  static thread_local size_t asked_smem = 0;
  int dev = 0;
  cudaGetDevice(&dev);
  cudaError_t e;
  if (configured_dev != dev) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMaxSmem);
    if (e != cudaSuccess) return e;
    configured_dev = dev;
    asked_cluster = 0;
  }
  if (asked_cluster != cluster || asked_smem != smem) {
    if ((e = cudaOccupancyMaxActiveClusters(&resident, kernel, &cfg)) != cudaSuccess) return e;
    if (resident < 1) return cudaErrorInvalidConfiguration;
    asked_cluster = cluster;
    asked_smem = smem;
  }
  const int64_t clusters = p.M < resident ? p.M : resident;
  cfg.gridDim = dim3((unsigned)(clusters * cluster));
  return cudaLaunchKernelEx(&cfg, kernel, p, (int)held);
}

template <typename T, int TH, int PER_SM>
cudaError_t launch_rows(const DistillArgs& p, int cluster, cudaStream_t stream) {
  const bool even = ((reinterpret_cast<uintptr_t>(p.logits) | reinterpret_cast<uintptr_t>(p.dlogits) |
                      (uintptr_t)(p.V * (int64_t)sizeof(T))) & 15) == 0;
  return even ? launch_even<T, TH, PER_SM, true>(p, cluster, stream)
              : launch_even<T, TH, PER_SM, false>(p, cluster, stream);
}

template <typename T>
cudaError_t launch_type(const DistillArgs& p, int sm_count, cudaStream_t stream) {
  const int64_t bytes = p.V * (int64_t)sizeof(T);
  if (bytes <= 16384) return launch_rows<T, 128, 8>(p, 1, stream);
  // Many rows that a cluster holds in shares of 40 KB: five CTAs of 128 threads an
  // SM, whose rows' reductions cover one another's (2048 rows of 151936 fp16 in 290
  // us; 315 in shares of 72 KB, three CTAs of 256 threads; 333 rows of 32003 in 18.0
  // and 19.3).  Few rows, where a row's own time counts: 256 threads, and more CTAs
  // down to 8 KB a CTA while they fit the SMs (4 rows of 151936 in 7.7 us, 9.1 with
  // 128).  Longer rows: shares of 72 KB.
  const bool short_share = bytes <= kClusterMax * kShortShare;
  const int64_t share = short_share ? kShortShare : kLongShare;
  int64_t cluster = (bytes + share - 1) / share;
  while (cluster < kClusterMax && p.M * (cluster + 1) <= sm_count && bytes / (cluster + 1) >= 8192) ++cluster;
  if (cluster > kClusterMax) cluster = kClusterMax;
  if (short_share && p.M * cluster > sm_count) return launch_rows<T, 128, 5>(p, (int)cluster, stream);
  return launch_rows<T, 256, 3>(p, (int)cluster, stream);
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
