// Losses over token log-probabilities [B, S] (fp32): the clipped policy loss
// with a KL term and the preference loss over pairs of sequences.
//
// Both are bound by latency up to some 100k tokens (one launch each way: 8.5 + 3
// us on the GPU for 8 x 509 tokens, inside some 75 us of a call's host time), by
// memory far above (17 / 9 bytes read per token; 2M tokens: 18 + 3.4 us for the
// preference loss) and the policy loss there by its exponentials (32 + 3.6 us).  A warp sums a chunk
// of one row and writes the chunk's partial sums, and the last block to finish
// adds the partials in chunk order, so the results have the same bits on every
// run.  Tokens are worked out and added in 64 bits: advantages of both signs
// cancel, what is left is the loss, and in 32 bits it came out up to 14 times as
// far off as a plain form's (4.9e-6 against 3.4e-7 of it).  Of 2M tokens that
// takes 8 us on the GPU, which a call's host time covers.  What stands outside
// the mask is dropped by selection, never by a product: it may be anything.
#include <math.h>

#include <algorithm>

#include "host_util.h"
#include "objectives.cuh"
#include "ptx.cuh"

namespace pb {
namespace {

constexpr int kWarps = 8;          // per block when there are many units
constexpr int kAhead = 4;          // tokens a lane loads before it uses the first
constexpr int kOneBlockUnits = 32;  // up to this many units one block does it all, without a ticket

__device__ __forceinline__ double warp_add(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Sums of K doubles per thread over the block, valid in thread 0; the same
// order on every run.  sh: [32][K].
template <int K>
__device__ __forceinline__ void block_add(double (&v)[K], double (*sh)[K]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = (int)(blockDim.x >> 5);
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
  if (lane == 0)
#pragma unroll
    for (int k = 0; k < K; ++k) sh[warp][k] = v[k];
  __syncthreads();
  if (warp != 0) return;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    v[k] = lane < warps ? sh[lane][k] : 0.0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
  }
}

// True in every thread of the last block to arrive (ticket zeroed before the
// launch); the partials of all blocks are then visible.
__device__ __forceinline__ bool last_block(int* ticket) {
  if (gridDim.x == 1) {
    __syncthreads();
    return true;
  }
  __shared__ bool last;
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) last = atomicAdd(ticket, 1) == (int)gridDim.x - 1;
  __syncthreads();
  if (last) __threadfence();
  return last;
}

__global__ void __launch_bounds__(1024) policy_fwd_kernel(const PolicyParams p) {
  pdl_prologue();
  const int lane = threadIdx.x & 31;
  const int64_t units = (int64_t)p.B * p.nchunk;
  const int64_t unit = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (unit < units) {
    const int64_t b = unit / p.nchunk;
    const int64_t s0 = (unit % p.nchunk) * p.chunk;
    const int64_t s1 = min((int64_t)p.S, s0 + p.chunk);
    const float* lp = p.logp + b * p.ld_logp;
    const float* old = p.old + b * p.ld_old;
    const float* ref = p.ref ? p.ref + b * p.ld_ref : nullptr;
    const float* adv = p.adv + b * p.adv_sb;
    const uint8_t* mask = p.mask ? p.mask + b * p.ld_mask : nullptr;
    double loss = 0.0, kl = 0.0;
    int n = 0, clip = 0;
    // kAhead tokens a lane at a time: all their loads first, whatever the mask says
    // (what is outside it is dropped), then the arithmetic
    for (int64_t sb = s0 + lane; sb < s1; sb += 32 * kAhead) {
      float l[kAhead], a[kAhead], o[kAhead], rl[kAhead];
      bool on[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const int64_t s = sb + 32 * j;
        on[j] = s < s1;
        l[j] = a[j] = o[j] = rl[j] = 0.f;
        if (s < s1) {
          if (mask) on[j] = __ldg(mask + s) != 0;
          l[j] = __ldg(lp + s);
          a[j] = __ldg(adv + s * p.adv_ss);
          o[j] = __ldg(old + s);
          if (ref) rl[j] = __ldg(ref + s);
        }
      }
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const double r = exp((double)l[j] - (double)o[j]);
        const double u = r * (double)a[j];
        const double c = fmin(fmax(r, p.low), p.high) * (double)a[j];
        const bool clipped = u > c;  // false for NaN: u carries it on
        double per = clipped ? -c : -u, coef = clipped ? 0.0 : -u;
        if (ref) {
          const double x = (double)rl[j] - (double)l[j];
          const double e = expm1(x), k = e - x;  // exp(x) - 1 - x without the cancellation at small x
          if (p.kl_coef != 0.0) {  // without the term the estimate may be infinite
            per += p.kl_coef * k;
            coef -= p.kl_coef * e;
          }
          kl += on[j] ? k : 0.0;
        }
        loss += on[j] ? per : 0.0;
        n += on[j] ? 1 : 0;
        clip += on[j] && clipped ? 1 : 0;
        const int64_t s = sb + 32 * j;
        if (p.coef && s < s1) p.coef[b * p.S + s] = on[j] ? (float)coef : 0.f;
      }
    }
    loss = warp_add(loss);
    n = __reduce_add_sync(0xffffffffu, n);
    clip = __reduce_add_sync(0xffffffffu, clip);
    kl = warp_add(kl);
    if (lane == 0) {
      p.parts[unit].sums = make_double2(loss, kl);
      p.parts[unit].counts = make_int2(n, clip);
    }
  }
  if (!last_block(p.ticket)) return;
  __shared__ double sh[32][5];
  double v[5] = {0.0, 0.0, 0.0, 0.0, 0.0};  // loss, tokens, clipped, kl, rows with a token
  if (!p.per_sequence) {
    for (int64_t i = threadIdx.x; i < units; i += blockDim.x) {
      const double2 q = __ldcg(&p.parts[i].sums);
      const int2 k = __ldcg(&p.parts[i].counts);
      v[0] += q.x;
      v[1] += k.x;
      v[2] += k.y;
      v[3] += q.y;
    }
  } else {
    for (int64_t b = threadIdx.x; b < p.B; b += blockDim.x) {
      double row = 0.0, rn = 0.0;
#pragma unroll 8
      for (int c = 0; c < p.nchunk; ++c) {
        const double2 q = __ldcg(&p.parts[b * p.nchunk + c].sums);
        const int2 k = __ldcg(&p.parts[b * p.nchunk + c].counts);
        row += q.x;
        rn += k.x;
        v[2] += k.y;
        v[3] += q.y;
      }
      if (rn > 0.0) {
        v[0] += row / rn;
        v[4] += 1.0;
      }
      v[1] += rn;
      p.inv_row[b] = rn > 0.0 ? (float)(1.0 / rn) : 0.f;
    }
  }
  block_add(v, sh);
  if (threadIdx.x == 0) {
    const double per_token = 1.0 / fmax(v[1], 1.0);
    const double inv = p.per_sequence ? 1.0 / fmax(v[4], 1.0) : per_token;
    p.inv[0] = (float)inv;
    p.loss[0] = (float)(v[0] * inv);
    p.clip[0] = (float)(v[2] * per_token);
    p.kl[0] = (float)(v[3] * per_token);
  }
}

// out = coef * g * inv (* inv_row of its row)
__global__ void __launch_bounds__(kWarps * 32)
    policy_bwd_kernel(const float* __restrict__ coef, const float* __restrict__ g, const float* __restrict__ inv,
                      const float* __restrict__ inv_row, float* __restrict__ out, int B, int S, int chunk,
                      int nchunk) {
  pdl_prologue();
  const int64_t unit = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (unit >= (int64_t)B * nchunk) return;
  const int64_t b = unit / nchunk;
  const int64_t s0 = (unit % nchunk) * chunk, s1 = min((int64_t)S, s0 + chunk);
  const float w = g[0] * inv[0] * (inv_row ? inv_row[b] : 1.f);
#pragma unroll 4
  for (int64_t s = s0 + (threadIdx.x & 31); s < s1; s += 32) {
    const float c = coef[b * S + s];
    out[b * S + s] = c == 0.f ? 0.f : c * w;  // exactly 0 outside the mask, whatever g is
  }
}

__global__ void __launch_bounds__(1024) preference_fwd_kernel(const PreferenceParams p) {
  pdl_prologue();
  const int lane = threadIdx.x & 31;
  const int rows = 2 * p.P;
  const int64_t units = (int64_t)rows * p.nchunk;
  const int64_t unit = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (unit < units) {
    const int64_t b = unit / p.nchunk;
    const int64_t s0 = (unit % p.nchunk) * p.chunk;
    const int64_t s1 = min((int64_t)p.S, s0 + p.chunk);
    const float* lp = p.logp + b * p.ld_logp;
    const float* ref = p.ref ? p.ref + b * p.ld_ref : nullptr;
    const uint8_t* mask = p.mask ? p.mask + b * p.ld_mask : nullptr;
    double d = 0.0;
    int n = 0;
    for (int64_t sb = s0 + lane; sb < s1; sb += 32 * kAhead) {
      float l[kAhead], r[kAhead];
      bool on[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const int64_t s = sb + 32 * j;
        on[j] = s < s1;
        l[j] = r[j] = 0.f;
        if (s < s1) {
          if (mask) on[j] = __ldg(mask + s) != 0;
          l[j] = __ldg(lp + s);
          if (ref) r[j] = __ldg(ref + s);
        }
      }
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        d += on[j] ? (double)l[j] - (double)r[j] : 0.0;
        n += on[j] ? 1 : 0;
      }
    }
    d = warp_add(d);
    n = __reduce_add_sync(0xffffffffu, n);
    if (lane == 0) p.parts[unit] = make_double2(d, (double)n);
  }
  if (!last_block(p.ticket)) return;
  __shared__ double sh[32][1];
  double loss[1] = {0.0};
  for (int i = threadIdx.x; i < p.P; i += blockDim.x) {
    double r[2], w[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {  // the chosen row, the rejected row
      const int64_t b = i + (int64_t)k * p.P;
      double d = 0.0, n = 0.0;
#pragma unroll 8
      for (int c = 0; c < p.nchunk; ++c) {
        const double2 v = __ldcg(p.parts + b * p.nchunk + c);
        d += v.x;
        n += v.y;
      }
      w[k] = p.beta / (p.average ? fmax(n, 1.0) : 1.0);
      r[k] = w[k] * d;
      p.rewards[b] = (float)r[k];
    }
    const double gap = r[0] - r[1];
    const double t = exp(-fabs(gap)), soft = log1p(t);  // -log sigmoid(x) = soft + max(-x, 0)
    const double neg = gap < 0.0 ? -gap : 0.0, pos = gap > 0.0 ? gap : 0.0;
    const double e = p.smoothing;
    // a side that does not count enters neither: its loss may be infinite
    loss[0] += (e < 1.0 ? (1.0 - e) * (soft + neg) : 0.0) + (e > 0.0 ? e * (soft + pos) : 0.0);
    // sigmoid(-gap) and sigmoid(gap), each without cancellation
    const double small = t / (1.0 + t), big = 1.0 / (1.0 + t);
    const double s_neg = gap >= 0.0 ? small : big, s_pos = gap >= 0.0 ? big : small;
    const double dgap = (e * s_pos - (1.0 - e) * s_neg) / (double)p.P;
    p.coef[i] = (float)(w[0] * dgap);
    p.coef[i + p.P] = (float)(-w[1] * dgap);
  }
  block_add(loss, sh);
  if (threadIdx.x == 0) p.loss[0] = (float)(loss[0] / (double)p.P);
}

// out = g * coef[row] inside the mask, 0 outside
__global__ void __launch_bounds__(kWarps * 32)
    preference_bwd_kernel(const float* __restrict__ coef, const float* __restrict__ g,
                          const uint8_t* __restrict__ mask, int64_t ld_mask, float* __restrict__ out, int rows, int S,
                          int chunk, int nchunk) {
  pdl_prologue();
  const int64_t unit = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (unit >= (int64_t)rows * nchunk) return;
  const int64_t b = unit / nchunk;
  const int64_t s0 = (unit % nchunk) * chunk, s1 = min((int64_t)S, s0 + chunk);
  const float w = g[0] * coef[b];
#pragma unroll 4
  for (int64_t s = s0 + (threadIdx.x & 31); s < s1; s += 32)
    out[b * S + s] = (!mask || mask[b * ld_mask + s]) ? w : 0.f;
}

int unit_blocks(int64_t units) { return (int)((units + kWarps - 1) / kWarps); }

}  // namespace

// Tokens of a row that one warp sums: the longest that still gives each SM 16
// warps, whose loads hide one another's latency, while the last block has few
// partials to add (policy forward, 512 x 4096, inputs not in L2: 32.7 us with
// 1024 tokens a warp, 21.5 with 512, 24.7 with 256, with the
// arithmetic in 32 bits).
int objective_chunk(int64_t rows, int64_t S) {
  int chunk = 1024;
  while (chunk > 128 && rows * ((S + chunk - 1) / chunk) < (int64_t)16 * num_sms()) chunk /= 2;
  return chunk;
}

void policy_fwd(const PolicyParams& p, cudaStream_t stream) {
  const int64_t units = (int64_t)p.B * p.nchunk;
  if (units <= kOneBlockUnits) {
    launch_k(policy_fwd_kernel, 1, 32 * std::max<int>(1, (int)units), 0, stream, p);
    return;
  }
  PB_CUDA_CHECK(cudaMemsetAsync(p.ticket, 0, sizeof(int), stream));
  launch_k(policy_fwd_kernel, unit_blocks(units), 32 * kWarps, 0, stream, p);
}

void policy_bwd(const float* coef, const float* g, const float* inv, const float* inv_row, float* out, int B, int S,
                int chunk, int nchunk, cudaStream_t stream) {
  if (B == 0 || S == 0) return;
  launch_k(policy_bwd_kernel, unit_blocks((int64_t)B * nchunk), 32 * kWarps, 0, stream, coef, g, inv, inv_row, out, B,
           S, chunk, nchunk);
}

void preference_fwd(const PreferenceParams& p, cudaStream_t stream) {
  const int64_t units = (int64_t)2 * p.P * p.nchunk;
  if (units <= kOneBlockUnits) {
    launch_k(preference_fwd_kernel, 1, 32 * std::max<int>(1, (int)units), 0, stream, p);
    return;
  }
  PB_CUDA_CHECK(cudaMemsetAsync(p.ticket, 0, sizeof(int), stream));
  launch_k(preference_fwd_kernel, unit_blocks(units), 32 * kWarps, 0, stream, p);
}

void preference_bwd(const float* coef, const float* g, const uint8_t* mask, int64_t ld_mask, float* out, int rows,
                    int S, int chunk, int nchunk, cudaStream_t stream) {
  if (rows == 0 || S == 0) return;
  launch_k(preference_bwd_kernel, unit_blocks((int64_t)rows * nchunk), 32 * kWarps, 0, stream, coef, g, mask, ld_mask,
           out, rows, S, chunk, nchunk);
}

}  // namespace pb
