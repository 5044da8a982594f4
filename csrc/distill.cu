// Distillation from a teacher's top logits: per row t, with teacher entries
// (value, id), q = softmax(values / tau) over the entries with id >= 0 and
// p = softmax(logits / tau),
//   loss_t = tau^2 sum_k q_k (log q_k - log p_{id_k}),  mean over the N rows that count
//   d logits_v = tau (p_v - sum_k q_k [id_k = v]) / N.
//
//   distill_prep  a warp per row: q, the ids as int32, and N.
//   distill_rows  a CTA per row (a cluster per row when there are few rows),
//                 two passes: running maximum and sum, then the gradient.
//   distill_loss  the row losses, added in a fixed order.
//
// The gradient is written in the forward pass, for a loss that counts once.
// Where the backward brings another weight, distill_rows runs again with it: a
// bf16 gradient multiplied afterwards would be rounded twice, and reading it takes
// as long as reading the logits (8192 x 151936 bf16: 935 us in the forward, 2 more
// for a weight of 1, 1100 for another).
//
// What bounds it: one read and one write of each logit in HBM.  A row of
// 151,936 bf16 logits is 304 KB, more than an SM's shared memory, so the second
// pass reads it again, from L2 for two thirds and more: 2 CTAs on each of 148 SMs
// hold at most 90 MB of rows there, of which a CTA in its first pass has not read
// all and one in its second does not need all (it reads and writes with
// evict-first).
// Sharing a row between the 8 CTAs of a cluster, which keeps it in registers
// and needs no second read, was slower in every form that was tried (8192 x
// 151936 bf16: 1211 us as short-lived CTAs, 1229 us persistent with bulk-copy
// prefetch and the exponentials kept): each row then waits for an exchange
// between 8 SMs, with too few warps beside it to fill the time.  Measured: 8192
// x 151936 bf16, 64 entries: 877 us, 0.88 of the measured copy rate (of one
// read and one write; 935 on GPUs with less clock); 1021 x 32003 fp32: 58 us.
#include <cuda_bf16.h>
#include <math.h>

#include <algorithm>

#include "host_util.h"
#include "objectives.cuh"
#include "ptx.cuh"

namespace pb {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kMaxCluster = kDistillMaxCluster;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float load1(const float* p) { return *p; }
__device__ __forceinline__ float load1(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void store1(float* p, float v) { *p = v; }
__device__ __forceinline__ void store1(__nv_bfloat16* p, float v) { *p = __float2bfloat16(v); }

// ---------------------------------------------------------------- teacher side
constexpr int kPrepWarps = 8;

__device__ __forceinline__ float teacher_value(const DistillParams& p, int64_t t, int k, int64_t id) {
  // an id past the vocabulary has no probability: NaN, and so is the loss
  if (id >= p.V) return NAN;
  return p.top_bf16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p.top)[t * p.ld_top + k])
                    : reinterpret_cast<const float*>(p.top)[t * p.ld_top + k];
}

__device__ __forceinline__ int64_t teacher_id(const DistillParams& p, int64_t t, int k) {
  return p.ids32 ? (int64_t) reinterpret_cast<const int*>(p.ids)[t * p.ld_ids + k]
                 : reinterpret_cast<const int64_t*>(p.ids)[t * p.ld_ids + k];
}

// counters[0]: rows that count (an integer sum, the same in any order)
__global__ void __launch_bounds__(32 * kPrepWarps) distill_prep_kernel(const DistillParams p) {
  pdl_prologue();
  const int64_t t = (int64_t)blockIdx.x * kPrepWarps + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (t >= p.T) return;
  float m = -INFINITY;
  bool any = false, bad = false;
  if (!p.mask || p.mask[t * p.ld_mask]) {
    for (int k = lane; k < p.K; k += 32) {
      const int64_t id = teacher_id(p, t, k);
      if (id < 0) continue;
      const float v = teacher_value(p, t, k, id);
      any = any || v != -INFINITY;
      bad = bad || isnan(v);
      m = fmaxf(m, v);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  any = __any_sync(0xffffffffu, any);
  bad = __any_sync(0xffffffffu, bad);
  if (lane == 0) {
    p.live[t] = any ? 1 : 0;
    if (p.key) p.key[t] = any ? 0 : -1;
    if (any) atomicAdd(p.counters, 1);
  }
  if (!any) return;
  float s = 0.f;
  for (int k = lane; k < p.K; k += 32) {
    const int64_t id = teacher_id(p, t, k);
    if (id >= 0) s += expf((teacher_value(p, t, k, id) - m) * p.inv_tau);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (bad) s = NAN;
  const float inv = 1.f / s;
  for (int k = lane; k < p.K; k += 32) {
    const int64_t id = teacher_id(p, t, k);
    p.q[t * p.Kp + k] = id >= 0 ? expf((teacher_value(p, t, k, id) - m) * p.inv_tau) * inv : 0.f;
    p.id[t * p.Kp + k] = id >= 0 && id < p.V ? (int)id : -1;
  }
  for (int k = p.K + lane; k < p.Kp; k += 32) {
    p.q[t * p.Kp + k] = 0.f;
    p.id[t * p.Kp + k] = -1;
  }
}

// ---------------------------------------------------------------- student side
__device__ __forceinline__ float warp_max(float v) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Store v at this shared-memory location of CTA `rank` of the cluster.
__device__ __forceinline__ void st_cluster_f2(float2* p, uint32_t rank, float2 v) {
  const uint32_t a = mapa_shared(smem_u32(p), rank);
  asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(a), "f"(v.x), "f"(v.y) : "memory");
}

// A 16-byte vector of a row: its maximum, its sum of exponentials, its
// gradient.  ref: the reference maximum; k2 = log2(e) / tau.  Exponents are
// (l - ref) k2, the difference exact near the reference; for bf16 a single
// multiply-add l k2 - ref k2 where its addend is small enough (near): below 1024
// the addend is rounded by at most 2^-15, and for the type's lowest value, with
// which columns are masked, it would overflow.
template <typename E>
struct Vec;
constexpr float kNear = 1024.f;
template <>
struct Vec<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ uint4 lowest() {
    return make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u);
  }
  static __device__ __forceinline__ bool near(float ref, float k2) { return fabsf(ref) * k2 < kNear; }
  static __device__ __forceinline__ float max(const uint4& u) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&u);
    const float2 t = __bfloat1622float2(__hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3])));
    return fmaxf(t.x, t.y);
  }
  template <bool NEAR>
  static __device__ __forceinline__ float exponent(float l, float ref, float k2, float c) {
    return NEAR ? fmaf(l, k2, c) : fmaf(l - ref, k2, c);
  }
  template <bool NEAR>
  static __device__ __forceinline__ void sum(const uint4& u, float ref, float k2, float* s) {
    const uint32_t* w = &u.x;
    const float c = NEAR ? -ref * k2 : 0.f;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      s[q] += ex2(exponent<NEAR>(__uint_as_float(w[q] << 16), ref, k2, c));
      s[q] += ex2(exponent<NEAR>(__uint_as_float(w[q] & 0xffff0000u), ref, k2, c));
    }
  }
  // f exp((l - ref) / tau), lf = log2(|f|) inside the exponent, flip the signs of a pair where f < 0
  template <bool NEAR>
  static __device__ __forceinline__ uint4 grad(const uint4& u, float ref, float k2, float, float lf, uint32_t flip) {
    const float c = NEAR ? fmaf(-ref, k2, lf) : lf;
    const uint32_t* w = &u.x;
    uint4 g;
    uint32_t* o = &g.x;
#pragma unroll
    for (int q = 0; q < 4; ++q)
      o[q] = pack_bf16x2(ex2(exponent<NEAR>(__uint_as_float(w[q] << 16), ref, k2, c)),
                         ex2(exponent<NEAR>(__uint_as_float(w[q] & 0xffff0000u), ref, k2, c))) ^ flip;
    return g;
  }
};
template <>
struct Vec<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ uint4 lowest() {
    return make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u);
  }
  static __device__ __forceinline__ float max(const uint4& u) {
    return fmaxf(fmaxf(__uint_as_float(u.x), __uint_as_float(u.y)),
                 fmaxf(__uint_as_float(u.z), __uint_as_float(u.w)));
  }
  static __device__ __forceinline__ bool near(float, float) { return false; }
  template <bool>
  static __device__ __forceinline__ void sum(const uint4& u, float ref, float k2, float* s) {
    const uint32_t* w = &u.x;
#pragma unroll
    for (int q = 0; q < 4; ++q) s[q] += ex2((__uint_as_float(w[q]) - ref) * k2);
  }
  template <bool>
  static __device__ __forceinline__ uint4 grad(const uint4& u, float ref, float k2, float f, float, uint32_t) {
    const uint32_t* w = &u.x;
    uint4 g;
    uint32_t* o = &g.x;
#pragma unroll
    for (int q = 0; q < 4; ++q) o[q] = __float_as_uint(f * ex2((__uint_as_float(w[q]) - ref) * k2));
    return g;
  }
};

constexpr int kRowThreads = 512;
constexpr int kUnroll = 4;  // vectors a thread has in flight

// A cluster of p.cluster CTAs takes a row, t of this block of logits.  A row may
// start at any element: up to 16 bytes in front of and behind its aligned vectors
// are taken one by one by the first CTA.
template <typename E, bool WEIGHTED>
__device__ __forceinline__ void distill_row(const DistillParams& p, int64_t t, float weight) {
  using VE = Vec<E>;
  constexpr int WARPS = kRowThreads / 32;
  extern __shared__ __align__(16) uint8_t smem[];
  int* sid = reinterpret_cast<int*>(smem);             // [Kp] the row's teacher entries
  float* sq = reinterpret_cast<float*>(sid + p.Kp);    // [Kp]
  float* sl = sq + p.Kp;                               // [Kp] student logits at the ids in this CTA's columns
  __shared__ float2 stat[kMaxCluster * WARPS];
  __shared__ float red[WARPS], single[32];
  __shared__ int single_col[32];

  const int C = p.cluster;
  const int rank = C == 1 ? 0 : (int)cluster_ctarank();
  // Packed rows: those behind the last 64-deep step of a sum over the rows that
  // count are neither read nor written.
  if (p.perm && p.row0 + t >= (max(p.counters[0], (int)p.row0 + 1) + 63) / 64 * 64) {
    if (threadIdx.x == 0) p.row_loss[(int64_t)p.perm[p.row0 + t] * C + rank] = 0.f;
    return;
  }
  // row of the teacher's entries and of the loss
  const int64_t tg = p.perm ? p.perm[p.row0 + t] : p.row0 + t;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const E* row = reinterpret_cast<const E*>(p.logits) + t * p.ld;
  E* out = p.grad ? reinterpret_cast<E*>(p.grad) + t * p.ld_grad : nullptr;
  const int mis = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(E));
  const int head = min(p.V, mis ? VE::N - mis : 0);
  const int nvec = (p.V - head) / VE::N, per = (nvec + C - 1) / C;
  const int tail0 = head + nvec * VE::N;  // columns [0, head) and [tail0, V) stand outside the vectors
  const int v0 = min(nvec, rank * per), nv = min(nvec, v0 + per) - v0;
  const uint4* vin = reinterpret_cast<const uint4*>(row + head) + v0;
  uint4* vout = reinterpret_cast<uint4*>(out + head) + v0;
  int xcol = -1;  // a single column: one a thread of the first CTA's first warp
  if (rank == 0) {
    if (tid < head) xcol = tid;
    else if (tid >= 16 && tid < 16 + p.V - tail0) xcol = tail0 + tid - 16;
  }

  if (!p.live[tg]) {  // a row that does not count: its logits are not read, its gradient is 0
    if (out) {
      for (int i = tid; i < nv; i += kRowThreads) __stcs(vout + i, make_uint4(0u, 0u, 0u, 0u));
      if (xcol >= 0) store1(out + xcol, 0.f);
    }
    if (tid == 0) p.row_loss[tg * C + rank] = 0.f;
    return;
  }
  // A CTA's shared memory may be written by its peers once it has started: this
  // barrier says that all have.  Its wait stands before the first such write,
  // behind the first pass; the returns above are taken by whole clusters.
  if (C > 1) cluster_arrive();

  // The teacher's entries in this CTA's columns (the others' ids become -1) and
  // the student's logits there, before a gradient may take their place.
  for (int k = tid; k < p.Kp; k += kRowThreads) {
    int id = p.id[tg * p.Kp + k];
    const int c0 = head + v0 * VE::N, c1 = c0 + nv * VE::N;
    if (id < head || id >= tail0 ? rank != 0 : (id < c0 || id >= c1)) id = -1;
    sid[k] = id;
    sq[k] = p.q[tg * p.Kp + k];
    if (id >= 0) sl[k] = load1(row + id);
  }
  const float x = xcol >= 0 ? load1(row + xcol) : -INFINITY;
  if (tid < 32) {
    single_col[tid] = xcol;
    single[tid] = x;
  }

  // first pass: this thread's maximum and sum, rescaled once per kUnroll vectors
  const float k2 = kLog2e * p.inv_tau;
  float m = x, s[4] = {x == -INFINITY ? 0.f : 1.f + (x - x), 0.f, 0.f, 0.f};  // x - x: 0, or NaN if x is not finite
  // two groups of vectors in turn: one on its way while the other is summed
  uint4 ua[kUnroll], ub[kUnroll];
  auto load = [&](uint4* u, int i0) {
#pragma unroll
    for (int j = 0; j < kUnroll; ++j) {
      u[j] = VE::lowest();
      if (i0 + j * kRowThreads < nv) u[j] = __ldcg(vin + i0 + j * kRowThreads);
    }
  };
  auto add = [&](const uint4* u) {
    float mn = m;
#pragma unroll
    for (int j = 0; j < kUnroll; ++j) mn = fmaxf(mn, VE::max(u[j]));
    const float ref = mn == -INFINITY ? 0.f : mn;
    const float r = ex2((m - ref) * k2);
#pragma unroll
    for (int q = 0; q < 4; ++q) s[q] *= r;
    m = mn;
    if (VE::near(ref, k2)) {
#pragma unroll
      for (int j = 0; j < kUnroll; ++j) VE::template sum<true>(u[j], ref, k2, s);
    } else {
#pragma unroll
      for (int j = 0; j < kUnroll; ++j) VE::template sum<false>(u[j], ref, k2, s);
    }
  };
  constexpr int kStep = kUnroll * kRowThreads;
  load(ua, tid);
  for (int i0 = tid; i0 < nv; i0 += 2 * kStep) {
    load(ub, i0 + kStep);
    add(ua);
    load(ua, i0 + 2 * kStep);
    if (i0 + kStep < nv) add(ub);
  }
  auto again = [&](uint4* u, int i0) {
#pragma unroll
    for (int j = 0; j < kUnroll; ++j)
      if (i0 + j * kRowThreads < nv) u[j] = __ldcs(vin + i0 + j * kRowThreads);
  };
  if (out) again(ua, tid);  // the second pass's first vectors come while the statistics are exchanged
  {
    const float mw = warp_max(m);
    const float ref = mw == -INFINITY ? 0.f : mw;
    const float sw = warp_sum(((s[0] + s[1]) + (s[2] + s[3])) * ex2((m - ref) * k2));
    // every CTA of the cluster gets every warp's pair
    if (C == 1) {
      if (lane == 0) stat[warp] = make_float2(mw, sw);
      __syncthreads();
    } else {
      cluster_wait();
      if (lane < C) st_cluster_f2(&stat[rank * WARPS + warp], lane, make_float2(mw, sw));
      cluster_sync();
    }
  }
  // all warps of all CTAs add the pairs in the same order: the same bits everywhere
  float total;
  {
    m = -INFINITY;
    for (int i = lane; i < C * WARPS; i += 32) m = fmaxf(m, stat[i].x);
    m = warp_max(m);
    const float ref = m == -INFINITY ? 0.f : m;
    float a = 0.f;
    for (int i = lane; i < C * WARPS; i += 32) a += stat[i].y * ex2((stat[i].x - ref) * k2);
    total = warp_sum(a);
    if (m == -INFINITY) total = NAN;  // no finite logit
  }
  const float sc = weight * p.tau / (float)max(1, p.counters[0]);
  const float f = sc / total;

  if (out) {  // second pass: the gradient of the softmax
    const float lf = log2f(WEIGHTED ? fabsf(f) : f);
    const uint32_t flip = WEIGHTED && f < 0.f ? 0x80008000u : 0u;
    const bool near = VE::near(m, k2);
    auto store = [&](const uint4* u, int i0) {
#pragma unroll
      for (int j = 0; j < kUnroll; ++j)
        if (i0 + j * kRowThreads < nv)
          __stcs(vout + i0 + j * kRowThreads,
                 near ? VE::template grad<true>(u[j], m, k2, f, lf, flip)
                      : VE::template grad<false>(u[j], m, k2, f, lf, flip));
    };
    for (int i0 = tid; i0 < nv; i0 += 2 * kStep) {
      again(ub, i0 + kStep);
      store(ua, i0);
      again(ua, i0 + 2 * kStep);
      store(ub, i0 + kStep);
    }
    if (tid < 32 && single_col[tid] >= 0) store1(out + single_col[tid], f * ex2((single[tid] - m) * k2));
    __syncthreads();  // the plain gradients stand before the teacher's columns are corrected
  }
  // the teacher's entries in this CTA's columns: their share of the loss, and their gradient
  const float ls = logf(total);
  float acc = 0.f;
  for (int k = tid; k < p.K; k += kRowThreads) {
    const int id = sid[k];
    const float q = sq[k];
    if (id < 0) {
      if (isnan(q)) acc = q;
      continue;
    }
    const float l = sl[k];
    // log p = (l - m) / tau - log s
    if (q != 0.f) acc += q * (logf(q) - ((l - m) * p.inv_tau - ls));
    if (out) {
      // entries of one id: each writes the gradient with the sum of their q
      float together = 0.f;
      for (int i = 0; i < p.Kp; i += 4) {
        const int4 ids = *reinterpret_cast<const int4*>(sid + i);
        const float4 qs = *reinterpret_cast<const float4*>(sq + i);
        together += (ids.x == id ? qs.x : 0.f) + (ids.y == id ? qs.y : 0.f) + (ids.z == id ? qs.z : 0.f) +
                    (ids.w == id ? qs.w : 0.f);
      }
      store1(out + id, f * ex2((l - m) * k2) - sc * together);
    }
  }
  acc = warp_sum(acc);
  if (lane == 0) red[warp] = acc;
  __syncthreads();
  if (tid == 0) {
    for (int i = 1; i < WARPS; ++i) acc += red[i];
    p.row_loss[tg * C + rank] = p.tau * p.tau * acc;
  }
}

template <typename E>
__global__ void __launch_bounds__(kRowThreads, 2) distill_rows_kernel(const DistillParams p) {
  pdl_prologue();
  distill_row<E, false>(p, blockIdx.x / p.cluster, 1.f);
}

// The gradient again where its weight is not 1.  The CTAs that fit at once take
// the rows in turn: most weights are 1, and as many CTAs as rows take 30 us to
// start and leave (8192 rows).
template <typename E>
__global__ void __launch_bounds__(kRowThreads, 2) distill_weighted_kernel(const DistillParams p) {
  pdl_prologue();
  const float weight = *p.weight;
  if (weight == 1.f) return;
  for (int64_t t = blockIdx.x / p.cluster; t < p.T; t += gridDim.x / p.cluster) {
    distill_row<E, true>(p, t, weight);
    __syncthreads();  // shared memory is free for the next row (clusters have one row each)
  }
}

// The mean of the row losses, added in a fixed order by one block.
constexpr int kLossThreads = 1024;
__global__ void __launch_bounds__(kLossThreads) distill_loss_kernel(const DistillParams p) {
  pdl_prologue();
  __shared__ double part[kLossThreads / 32];
  double a = 0.0;
  for (int64_t i = threadIdx.x; i < (int64_t)p.T_all * p.cluster; i += kLossThreads) a += (double)p.row_loss[i];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = a;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < kLossThreads / 32; ++i) a += part[i];
    p.loss[0] = (float)(a / (double)max(1, p.counters[0]));
  }
}

template <typename E>
void launch_rows(const DistillParams& p, cudaStream_t stream) {
  auto kern = p.weight ? distill_weighted_kernel<E> : distill_rows_kernel<E>;
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = p.cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.cluster > 1 ? 2 : 1;
  cfg.blockDim = dim3(kRowThreads, 1, 1);
  cfg.dynamicSmemBytes = (size_t)p.Kp * 12;
  cfg.stream = stream;
  const unsigned rows = p.weight && p.cluster == 1 ? std::min(p.T, 2 * num_sms()) : p.T;
  cfg.gridDim = dim3(rows * p.cluster, 1, 1);
  PB_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kern, p));
}

}  // namespace

void distill_prep(const DistillParams& p, cudaStream_t stream) {
  PB_CUDA_CHECK(cudaMemsetAsync(p.counters, 0, sizeof(int), stream));
  if (p.T == 0) return;
  launch_k(distill_prep_kernel, (p.T + kPrepWarps - 1) / kPrepWarps, 32 * kPrepWarps, 0, stream, p);
}

// a CTA per row, or a cluster while that leaves SMs idle and each CTA still has 2 vectors a thread; by all
// rows, so that the blocks of one call write their shares of row_loss alike
static int cluster_of(const DistillParams& p, bool bf16) {
  const int nvec = p.V / (bf16 ? 8 : 4);
  int cluster = 1;
  while (cluster < kMaxCluster && 2 * cluster * (int64_t)p.T_all <= 2 * num_sms() && nvec / cluster >= 4 * kRowThreads)
    cluster *= 2;
  return cluster;
}

void distill_rows(const DistillParams& p0, bool bf16, cudaStream_t stream) {
  PB_CHECK(p0.K <= kDistillMaxK && (int64_t)p0.T * kMaxCluster < ((int64_t)1 << 31), "distill: too many rows or entries");
  DistillParams p = p0;
  p.cluster = cluster_of(p, bf16);
  if (bf16)
    launch_rows<__nv_bfloat16>(p, stream);
  else
    launch_rows<float>(p, stream);
}

void distill_loss(const DistillParams& p0, bool bf16, cudaStream_t stream) {
  DistillParams p = p0;
  p.cluster = cluster_of(p, bf16);
  launch_k(distill_loss_kernel, 1, kLossThreads, 0, stream, p);
}

}  // namespace pb
