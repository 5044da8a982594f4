// Distillation from a teacher's top logits: per row t, with teacher entries
// (value, id), q = softmax(values / tau) over the entries with id >= 0 and
// p = softmax(logits / tau),
//   loss_t = tau^2 sum_k q_k (log q_k - log p_{id_k}),  mean over the N rows that count
//   d logits_v = tau (p_v - sum_k q_k [id_k = v]) / N.
//
//   distill_prep  a warp per row: q and the ids as int32, and N.
//   distill_rows  a cluster of CTAs per row; every thread holds its share of
//                 the row in registers, so that each logit is read once and
//                 its gradient written once: the kernel is bound by memory.
//
// A row of 151,936 bf16 logits is 304 KB, more than one SM's shared memory and
// too much to leave to L2 with a row per SM in flight; split over a cluster of
// 8 CTAs it is 10 16-byte vectors a thread, and three or four such CTAs fit
// an SM, so some load while others reduce and store.
#include <cuda_bf16.h>
#include <math.h>

#include <algorithm>

#include "host_util.h"
#include "objectives.cuh"
#include "ptx.cuh"

namespace pb {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kMaxCluster = 8;
constexpr int kMaxWarps = 16;

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
  const float v = p.top_bf16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p.top)[t * p.ld_top + k])
                             : reinterpret_cast<const float*>(p.top)[t * p.ld_top + k];
  return v * p.inv_tau;
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
    if (any) atomicAdd(p.counters, 1);
  }
  if (!any) return;
  float s = 0.f;
  for (int k = lane; k < p.K; k += 32) {
    const int64_t id = teacher_id(p, t, k);
    if (id >= 0) s += expf(teacher_value(p, t, k, id) - m);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (bad) s = NAN;
  const float inv = 1.f / s;
  for (int k = lane; k < p.K; k += 32) {
    const int64_t id = teacher_id(p, t, k);
    p.q[t * p.K + k] = id >= 0 ? expf(teacher_value(p, t, k, id) - m) * inv : 0.f;
    p.id[t * p.K + k] = id >= 0 && id < p.V ? (int)id : -1;
  }
}

// ---------------------------------------------------------------- student side
__device__ __forceinline__ void merge(float& m, float& s, float m2, float s2, float k2) {
  const float mn = fmaxf(m, m2);
  const float ref = mn == -INFINITY ? 0.f : mn;
  s = s * ex2((m - ref) * k2) + s2 * ex2((m2 - ref) * k2);
  m = mn;
}

__device__ __forceinline__ float2 ld_cluster_f2(const float2* p, uint32_t rank) {
  float2 v;
  const uint32_t a = mapa_shared(smem_u32(p), rank);
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(a) : "memory");
  return v;
}

template <typename E>
struct Vec;
template <>
struct Vec<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ float get(const uint4& u, int j) {
    const uint32_t w = (&u.x)[j >> 1];
    return __uint_as_float((j & 1) ? (w & 0xffff0000u) : (w << 16));
  }
  static __device__ __forceinline__ uint4 pack(const float* v) {
    return make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]),
                      pack_bf16x2(v[6], v[7]));
  }
};
template <>
struct Vec<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ float get(const uint4& u, int j) { return __uint_as_float((&u.x)[j]); }
  static __device__ __forceinline__ uint4 pack(const float* v) {
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
  }
};

// Grid: T clusters.  NV: 16-byte vectors of the row per thread.  A row may
// start at any element: up to 16 bytes in front of and behind the aligned
// vectors are taken one by one by the first CTA.
template <typename E, int NV>
__global__ void __launch_bounds__(32 * kMaxWarps) distill_rows_kernel(const DistillParams p) {
  pdl_prologue();
  using VE = Vec<E>;
  extern __shared__ __align__(16) uint8_t smem[];
  float* sq = reinterpret_cast<float*>(smem);  // [K] teacher probabilities
  float* sl = sq + p.K;                        // [K] student logits at the teacher's ids
  int* sid = reinterpret_cast<int*>(sl + p.K);  // [K]
  __shared__ float2 warp_stat[kMaxWarps];
  __shared__ float2 cta_stat;
  __shared__ float red[kMaxWarps];
  __shared__ bool s_last;

  const int C = p.cluster;
  const uint32_t rank = cluster_ctarank();
  const int64_t t = blockIdx.x / C;  // row of this block of logits
  const int64_t tg = p.row0 + t;     // row of the teacher's entries and of the loss
  const int tid = threadIdx.x, nt = blockDim.x, lane = tid & 31, warp = tid >> 5, warps = nt >> 5;
  const E* row = reinterpret_cast<const E*>(p.logits) + t * p.ld;
  E* out = p.grad ? reinterpret_cast<E*>(p.grad) + t * p.ld_grad : nullptr;
  const int mis = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(E));
  const int head = min(p.V, mis ? VE::N - mis : 0);
  const int nvec = (p.V - head) / VE::N;
  const int tail0 = head + nvec * VE::N;  // first column behind the vectors
  const int per = (nvec + C - 1) / C;
  const int v0 = (int)rank * per, v1 = min(nvec, v0 + per);
  const uint4* vin = reinterpret_cast<const uint4*>(row + head);
  uint4* vout = reinterpret_cast<uint4*>(out + head);
  // the first CTA's single columns: [0, head) by threads 0.., [tail0, V) by threads 16..
  int xcol = -1;
  if (rank == 0) {
    if (tid < head) xcol = tid;
    else if (tid >= 16 && tid < 16 + p.V - tail0) xcol = tail0 + tid - 16;
  }
  const bool live = p.live[tg] != 0;

  if (!live) {  // a row that does not count: its logits are not read, its gradient is 0
    if (out) {
      for (int i = v0 + tid; i < v1; i += nt) vout[i] = make_uint4(0u, 0u, 0u, 0u);
      if (xcol >= 0) store1(out + xcol, 0.f);
    }
    if (rank == 0 && tid == 0) p.row_loss[tg] = 0.f;
  } else {
    uint4 raw[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int v = v0 + i * nt + tid;
      if (v < v1) raw[i] = vin[v];
    }
    const float x = xcol >= 0 ? load1(row + xcol) : -INFINITY;
    // the teacher's entries; the first CTA needs every one (loss), the others those in their columns
    const int c0 = head + v0 * VE::N, c1 = head + v1 * VE::N;
    for (int k = tid; k < p.K; k += nt) {
      const int id = p.id[tg * p.K + k];
      sid[k] = id;
      sq[k] = p.q[tg * p.K + k];
      if (id >= 0 && (rank == 0 || (id >= c0 && id < c1))) sl[k] = load1(row + id);
    }
    const float k2 = kLog2e * p.inv_tau;
    float m = x;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (v0 + i * nt + tid < v1) {
#pragma unroll
        for (int j = 0; j < VE::N; ++j) m = fmaxf(m, VE::get(raw[i], j));
      }
    const float ref = m == -INFINITY ? 0.f : m;
    float s = xcol >= 0 ? ex2((x - ref) * k2) : 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (v0 + i * nt + tid < v1) {
#pragma unroll
        for (int j = 0; j < VE::N; ++j) s += ex2((VE::get(raw[i], j) - ref) * k2);
      }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float m2 = __shfl_xor_sync(0xffffffffu, m, o), s2 = __shfl_xor_sync(0xffffffffu, s, o);
      merge(m, s, m2, s2, k2);
    }
    if (lane == 0) warp_stat[warp] = make_float2(m, s);
    __syncthreads();
    m = warp_stat[0].x;
    s = warp_stat[0].y;
    for (int i = 1; i < warps; ++i) merge(m, s, warp_stat[i].x, warp_stat[i].y, k2);
    if (tid == 0) cta_stat = make_float2(m, s);
    cluster_sync();
    // every CTA merges the cluster's statistics in rank order: the same bits in all of them
    float2 st = ld_cluster_f2(&cta_stat, 0);
    m = st.x;
    s = st.y;
    for (int i = 1; i < C; ++i) {
      st = ld_cluster_f2(&cta_stat, i);
      merge(m, s, st.x, st.y, k2);
    }
    if (rank == 0) {
      const float ls = logf(s);
      float acc = 0.f;
      for (int k = tid; k < p.K; k += nt) {
        const float q = sq[k];
        // log p = (l - m) / tau - log s
        if (sid[k] >= 0 && q != 0.f) acc += q * (logf(q) - ((sl[k] - m) * p.inv_tau - ls));
        else if (isnan(q)) acc = q;
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
      if (lane == 0) red[warp] = acc;
      __syncthreads();
      if (tid == 0) {
        for (int i = 1; i < warps; ++i) acc += red[i];
        p.row_loss[tg] = p.tau * p.tau * acc;
      }
    }
    if (out) {
      const float sc = p.tau / (float)max(1, p.counters[0]);
      const float f = sc / s;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int v = v0 + i * nt + tid;
        if (v < v1) {
          float g[VE::N];
#pragma unroll
          for (int j = 0; j < VE::N; ++j) g[j] = f * ex2((VE::get(raw[i], j) - m) * k2);
          vout[v] = VE::pack(g);
        }
      }
      if (xcol >= 0) store1(out + xcol, f * ex2((x - m) * k2));
      __syncthreads();  // the plain gradients are written before the teacher's columns are corrected
      for (int k = tid; k < p.K; k += nt) {
        const int id = sid[k];
        const bool mine = id >= c0 && id < c1, single = rank == 0 && id >= 0 && (id < head || id >= tail0);
        if (mine || single) {
          float q = 0.f;  // an id that comes twice has the sum of its entries; each writes the same value
          for (int i = 0; i < p.K; ++i) q += sid[i] == id ? sq[i] : 0.f;
          store1(out + id, f * ex2((sl[k] - m) * k2) - sc * q);
        }
      }
    }
    cluster_sync();  // no CTA leaves while another may read its statistics
  }
  // the last row to finish (over all blocks of rows) adds the row losses in a fixed order
  if (rank != 0) return;
  __syncthreads();
  if (tid == 0) {
    __threadfence();
    s_last = atomicAdd(p.counters + 1, 1) == p.T_all - 1;
  }
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  __shared__ double dred[kMaxWarps];
  double a = 0.0;
  for (int i = tid; i < p.T_all; i += nt) a += (double)__ldcg(p.row_loss + i);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
  if (lane == 0) dred[warp] = a;
  __syncthreads();
  if (tid == 0) {
    for (int i = 1; i < warps; ++i) a += dred[i];
    p.loss[0] = (float)(a / (double)max(1, p.counters[0]));
  }
}

// x[i] *= g[0] unless it is 1
template <typename E>
__global__ void __launch_bounds__(256) scale_kernel(E* __restrict__ x, int64_t n, const float* __restrict__ g) {
  pdl_prologue();
  const float s = g[0];
  if (s == 1.f) return;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256)
    store1(x + i, load1(x + i) * s);
}

// Cluster size, threads and vectors per thread of a row of nvec vectors: the
// smallest cluster whose threads hold at most 10 vectors each.
struct Shape {
  int cluster, threads, nv;
};
Shape shape_of(int nvec) {
  for (int threads : {256, 512})
    for (int c = 1; c <= kMaxCluster; c *= 2)
      for (int nv : {1, 2, 4, 6, 8, 10, 16})
        if ((nv <= 10 || (threads == 512 && c == kMaxCluster)) && (int64_t)threads * c * nv >= nvec)
          if ((int64_t)((nvec + c - 1) / c) <= (int64_t)threads * nv) return {c, threads, nv};
  return {0, 0, 0};
}

template <typename E, int NV>
void launch_rows(const DistillParams& p, const Shape& sh, cudaStream_t stream) {
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = sh.cluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  cfg.gridDim = dim3((unsigned)p.T * sh.cluster, 1, 1);
  cfg.blockDim = dim3(sh.threads, 1, 1);
  cfg.dynamicSmemBytes = (size_t)p.K * 12;
  cfg.stream = stream;
  PB_CUDA_CHECK(cudaLaunchKernelEx(&cfg, distill_rows_kernel<E, NV>, p));
}

template <typename E>
void launch_rows_nv(const DistillParams& p, const Shape& sh, cudaStream_t stream) {
  switch (sh.nv) {
    case 1: return launch_rows<E, 1>(p, sh, stream);
    case 2: return launch_rows<E, 2>(p, sh, stream);
    case 4: return launch_rows<E, 4>(p, sh, stream);
    case 6: return launch_rows<E, 6>(p, sh, stream);
    case 8: return launch_rows<E, 8>(p, sh, stream);
    case 10: return launch_rows<E, 10>(p, sh, stream);
    default: return launch_rows<E, 16>(p, sh, stream);
  }
}

}  // namespace

int64_t distill_max_vocab(bool bf16) { return (int64_t)kMaxCluster * 512 * 16 * (bf16 ? 8 : 4); }

void distill_prep(const DistillParams& p, cudaStream_t stream) {
  PB_CUDA_CHECK(cudaMemsetAsync(p.counters, 0, 2 * sizeof(int), stream));
  if (p.T == 0) return;
  launch_k(distill_prep_kernel, (p.T + kPrepWarps - 1) / kPrepWarps, 32 * kPrepWarps, 0, stream, p);
}

void distill_rows(const DistillParams& p0, bool bf16, cudaStream_t stream) {
  const Shape sh = shape_of(p0.V / (bf16 ? 8 : 4));
  PB_CHECK(sh.cluster > 0 && p0.K <= kDistillMaxK, "distill: vocabulary or teacher entries out of range");
  PB_CHECK((int64_t)p0.T * sh.cluster < ((int64_t)1 << 31), "distill: too many rows for one call");
  DistillParams p = p0;
  p.cluster = sh.cluster;
  if (bf16)
    launch_rows_nv<__nv_bfloat16>(p, sh, stream);
  else
    launch_rows_nv<float>(p, sh, stream);
}

void objective_scale(void* x, int64_t n, bool bf16, const float* g, cudaStream_t stream) {
  if (n == 0) return;
  const int blocks = (int)std::min<int64_t>((n + 255) / 256, (int64_t)8 * num_sms());
  if (bf16)
    launch_k(scale_kernel<__nv_bfloat16>, blocks, 256, 0, stream, (__nv_bfloat16*)x, n, g);
  else
    launch_k(scale_kernel<float>, blocks, 256, 0, stream, (float*)x, n, g);
}

}  // namespace pb
