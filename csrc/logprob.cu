// Log-probabilities of given tokens through a language-model head, without the
// logits: logp[t] = l_id - log sum_v exp(l_v), l_v = (h_t . w_v) / temperature.
//
//   logprob_gemm    CTA-pair tcgen05 GEMM h w^T whose epilogue turns each row
//                   of an output tile into (max, sum of 2^(x - max)), x the
//                   logit in base 2, the target column left out; under a
//                   gradient it also stores E = 2^(x - group max) in 16 bits.
//   logprob_finish  per row: the target logit as its own dot product, the
//                   merge of the row's statistics, logp and the row's
//                   base-2 log-sum-exp above its maximum.
//   logprob_pack    (under a gradient, and from 768 rows on) brings the rows that
//                   have a token to the front; logprob_unpack takes their
//                   gradients back.
//   logprob_bwd     in place over E: the gradient of the logits but the target,
//                   dl_v = -c 2^(x_v - lse2), c = dlogp / temperature, and the
//                   target's own c (1 - p), in fp32.
//   logprob_unpack, logprob_own add the target's part of the gradients of h and
//                   w, c (1 - p) w_id and c (1 - p) h, in fp32: it is most of
//                   them, and as one more bf16 factor its rounding, the same in
//                   a whole row of the product, would add up to 2^-9 of it.  Where
//                   dw is bf16 a target's row was rounded once by the product (the
//                   others' part, the smaller one) and is once more with its own.
//
// Maxima are kept as they come from the tensor core, unscaled, and only
// differences of them are scaled, so no digit of an exponent is lost however
// large the logits are.
//
// The target logit is kept out of the sums and summed on its own in 64 bits,
// and logp = -log1p(sum of the others / target): the tensor core truncates as
// it accumulates (measured on a target logit of 13: 1.6e-5 low at H = 1024,
// 5e-5 at H = 4096), and where the target is nearly certain all of logp hangs
// on that logit.  The other logits enter as a sum of many, where the mean of that
// loss shows; an estimate of it is added back (kTruncation).
//
// E is relative to its group's own maximum, which is known when the tile is
// stored, while the row's log-sum-exp is not: an entry keeps 10 bits of its
// probability whatever its size (pack_e), and the backward is one multiplication
// per entry (the factor 2^(group max - lse2), shared by a group) in a pass
// bound by memory.  bf16 logits would lose |l| / 256 of the exponent instead.
#include <cuda_bf16.h>
#include <math.h>

#include <algorithm>
#include <mutex>

#include "host_util.h"
#include "objectives.cuh"
#include "ptx.cuh"

namespace pb {
namespace {

constexpr int BM_CTA = 128;  // rows of h per CTA (a pair's tile has 256)
constexpr int BK = 64;
constexpr int BN_MAX = 256;
constexpr int kThreads = 192;
constexpr int A_BYTES = BM_CTA * BK * 2;
constexpr int B_BYTES = (BN_MAX / 2) * BK * 2;
constexpr int STAGES = 7;
constexpr int SMEM_BYTES = STAGES * (A_BYTES + B_BYTES) + 1024 + 256;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// Estimate of the mean relative loss of an accumulated dot product per 16-deep
// step.  Each step truncates the running sum towards zero in its 24th bit, so a
// step loses less than 2^-23 of the sum it leaves; for one that grows evenly to
// its end half a unit a step would be 0.36 x 2^-24 of the end.  The constant is not
// derived but fitted: 0.25 to 0.28 was measured for normally distributed
// components, logits of 4 to 32, H = 512 to 4096, the spread around it a tenth to a
// third of it.  Where one early component makes the logit more is lost; where a
// late one does nothing is, and what is given back is the error: 4e-6 of the logit
// at H = 4096, as much as is lost without it in the even case.  There it takes
// logp's error against 64 bits from 2.9e-6 to 8e-8 of its norm.
constexpr double kTruncation = 0.26 / (1 << 24);

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Column groups and tiles.  A group is what one pair of statistics covers, a tile
// what one accumulator holds.  The first n_full of either are BN_MAX wide; behind
// them come narrower groups, and tiles of bn2 columns, one or more of these groups.
// For few rows that makes whole waves of wide tiles over the CTA pairs and one of
// tiles narrow enough for what is left over: 151,936 columns are 8 waves of 256 on
// 74 pairs and 384 columns, which as two wide tiles cost a ninth wave (64 rows, H
// 1024: 62.2 -> 60.1 us; 8 rows of V 10000: 12.6 -> 11.6).  The groups go by the
// vocabulary alone and the tiles by the rows too, so a row's sums are added in the
// same order, and its log-probability has the same bits, in whatever batch it comes.
__device__ __forceinline__ int tile_start(const LogprobGroups& g, int bn2, int tn) {
  return tn < g.n_full ? tn * BN_MAX : g.n_full * BN_MAX + (tn - g.n_full) * bn2;
}
__device__ __forceinline__ int tile_width(const LogprobGroups& g, int bn2, int tn) {
  return tn < g.n_full ? BN_MAX : bn2;
}

// Accumulators of columns [n0, n0 + 32): -inf past the vocabulary and at the
// row's target, so neither enters the maximum or the sum.
__device__ __forceinline__ void mask_cols(float* v, int n0, int V, int64_t id) {
  uint32_t out = 0;  // bit j: column n0 + j is masked
  if (n0 + 32 > V) out = n0 >= V ? 0xffffffffu : 0xffffffffu << (V - n0);
  const int64_t d = id - n0;
  if (d >= 0 && d < 32) out |= 1u << (int)d;
  if (out) {
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (out & (1u << j)) v[j] = -INFINITY;
  }
}

__device__ __forceinline__ float max32(const float* v) {
  float m = v[0];
#pragma unroll
  for (int j = 1; j < 32; ++j) m = fmaxf(m, v[j]);
  return m;
}

// Two values of [0, 2) in 16 bits each: a float's sign and upper exponent bit
// are 0 there, so 7 bits of exponent and 9 of mantissa remain (bf16 has 7 of
// mantissa); rounded to nearest.  Half the memory and time of fp32 between forward
// and backward, for a quarter of the error that the logits' gradient takes next, as
// the bf16 operand of both products.  NaN does not survive, nor need it: the row's
// sum has it, and with that every gradient of the row.
__device__ __forceinline__ uint32_t pack_e(float a, float b) {
  // bits 29..14, moved to the upper half with the rounding's half added
  return __byte_perm(__float_as_uint(a) * 4u + 0x8000u, __float_as_uint(b) * 4u + 0x8000u, 0x7632);
}
__device__ __forceinline__ float2 unpack_e(uint32_t u) {
  return make_float2(__uint_as_float((u << 14) & 0x3fffc000u), __uint_as_float((u >> 2) & 0x3fffc000u));
}

// 32 bytes with one store: whole sectors, though every lane is on another row.
__device__ __forceinline__ void st_32(void* p, const uint32_t* u) {
  asm volatile("st.global.cs.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(u[0]), "r"(u[1]), "r"(u[2]),
               "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7])
               : "memory");
}

// a, b -> (a - m) scale, (b - m) scale, two at a time (8192 rows, 6554 with a
// token, forward and backward: 5040 us, as with one multiply-add each and a
// rounded m scale; one at a time 5200)
__device__ __forceinline__ void scaled_diff(float& a, float& b, float m, float scale) {
  const float2 d = __fmul2_rn(__fadd2_rn(make_float2(a, b), make_float2(-m, -m)), make_float2(scale, scale));
  a = d.x;
  b = d.y;
}

// Statistics of one accumulator row (one thread) of `bn` columns from TMEM, a group:
// the maximum first (E needs one reference for the whole group), then the sum of the
// exponentials, which under a gradient (STORE) also go to E, straight from
// registers.  Staging them in shared memory for tile stores put 128 KB more per
// tile on a shared memory that the MMAs already read at its rate (8192 rows,
// 6554 with a token: 1605 us; like this 1463).  Scoring takes the same two
// passes, although a running maximum would do: the log-probabilities then are
// the same bits as in training, and a policy's ratio to itself is exactly 1.
// `release` runs after the last TMEM read of the tile's `last` group.
template <bool STORE, typename Release>
__device__ __forceinline__ float2 row_stats(uint32_t t_row, int bn, int n_base, int V, int64_t id, float scale,
                                            __nv_bfloat16* e_row, bool row_in, bool last, Release release) {
  float m = -INFINITY;
#pragma unroll 1
  for (int c = 0; c < bn; c += 32) {
    float v[32];
    tmem_ld32(t_row + c, v);
    tmem_wait_ld32(v);
    mask_cols(v, n_base + c, V, id);
    m = fmaxf(m, max32(v));
  }
  const float ref = m == -INFINITY ? 0.f : m;  // nothing but masked columns
  float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
  for (int c = 0; c < bn; c += 32) {
    float v[32];
    tmem_ld32(t_row + c, v);
    tmem_wait_ld32(v);
    if (last && c + 32 >= bn) release();
    const int n0 = n_base + c;
    mask_cols(v, n0, V, id);
#pragma unroll
    for (int j = 0; j < 32; j += 2) {
      scaled_diff(v[j], v[j + 1], ref, scale);
      v[j] = ex2(v[j]);
      v[j + 1] = ex2(v[j + 1]);
      s[j & 3] += v[j];
      s[(j & 3) + 1] += v[j + 1];
    }
    if (STORE && row_in && n0 < V) {
      uint32_t u[16];
#pragma unroll
      for (int q = 0; q < 16; ++q) u[q] = pack_e(v[2 * q], v[2 * q + 1]);
      st_32(e_row + n0, u);
      st_32(e_row + n0 + 16, u + 8);
    }
  }
  return make_float2(m, (s[0] + s[1]) + (s[2] + s[3]));
}

// Roles per CTA: warp 0 TMA producer, warp 1 TMEM allocator and (even CTA) MMA
// issuer, warps 2..5 epilogue, one output row per thread.  The accumulator is
// double buffered in TMEM, so the epilogue of one tile runs under the MMAs of
// the next.  Row tiles run innermost: every pair works on the same few column
// tiles of w, which is read from memory once.
template <bool STORE>
__global__ void __launch_bounds__(kThreads, 1)
    logprob_gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                        const __grid_constant__ CUtensorMap tmB2, __nv_bfloat16* __restrict__ e, int64_t lde,
                        const int64_t* __restrict__ ids, const int* __restrict__ count, int row0,
                        float2* __restrict__ stats, int T_all, int V, int H, int a_rows, const LogprobGroups geo,
                        int bn2, int tiles2, float scale, int* err) {
  pdl_prologue();
  const int T = count ? min(T_all, max(0, *count - row0)) : T_all;  // the rows in front that have a token
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = smem + STAGES * A_BYTES;
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(sB + STAGES * B_BYTES);
  uint64_t* empty_bar = full_bar + STAGES;
  uint64_t* tfull_bar = empty_bar + STAGES;
  uint64_t* tempty_bar = tfull_bar + 2;  // used on the even CTA (256 arrivals: both epilogues)
  uint64_t* drain_bar = tempty_bar + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain_bar + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&tfull_bar[i], 1);
      mbar_init(&tempty_bar[i], 2 * 128);
    }
    mbar_init(drain_bar, 1);
    fence_mbar_init();
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, 2 * BN_MAX);
    tmem_relinquish_pair();
  }
  if (a_rows < BM_CTA) {
    // few rows: the rest of A is multiplied too, and zeros cost the least power
    // (one row, thousands of calls in a row: 72 us, with this 66.5)
    for (int i = threadIdx.x; i < STAGES * A_BYTES / 16; i += kThreads)
      reinterpret_cast<uint4*>(sA)[i] = make_uint4(0u, 0u, 0u, 0u);
    fence_proxy_async_smem();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // barriers of both CTAs initialised before any cross-CTA use
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  const int tiles_m = (T + 2 * BM_CTA - 1) / (2 * BM_CTA);
  const int tiles_n = geo.n_full + tiles2;
  const int64_t num_tiles = (int64_t)tiles_m * tiles_n;
  const int num_kb = (H + BK - 1) / BK;
  const int n_clusters = gridDim.x >> 1;
  const int cid = blockIdx.x >> 1;

  if (warp == 0) {
    if (lane == 0) {
      // few rows: a box of the rows that are there (a box mostly out of bounds is
      // slow to fill: one row 91 us, 64 rows 61 us), and none for the odd CTA.  The
      // rest of the stage stays zero.
      const uint32_t a_bytes = a_rows < BM_CTA ? (uint32_t)a_rows * BK * 2 : 2 * A_BYTES;
      const bool load_a = a_rows == BM_CTA || leader;
      int stage = 0;
      uint32_t phase = 0;
      uint32_t issued = 0, last = 0;  // bit s: copies were issued to stage s; the parity of its last phase
      bool ok = true;
      for (int64_t w = cid; w < num_tiles && ok; w += n_clusters) {
        const int tm = (int)(w % tiles_m), tn = (int)(w / tiles_m);
        const int a_row = tm * 2 * BM_CTA + (int)rank * BM_CTA;
        const int bn = tile_width(geo, bn2, tn);
        const int b_row = tile_start(geo, bn2, tn) + (int)rank * (bn / 2);
        const CUtensorMap* map_b = tn < geo.n_full ? &tmB : &tmB2;
        const uint32_t stage_bytes = a_bytes + (uint32_t)bn * BK * 2;
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!mbar_wait(&empty_bar[stage], phase ^ 1, err)) { ok = false; break; }
          const uint32_t full_even = mapa_shared(smem_u32(&full_bar[stage]), 0);
          if (leader) mbar_arrive_expect_tx(&full_bar[stage], stage_bytes);
          if (load_a) tma_load_2d_pair(sA + stage * A_BYTES, &tmA, full_even, kb * BK, a_row);
          tma_load_2d_pair(sB + stage * B_BYTES, map_b, full_even, kb * BK, b_row);
          issued |= 1u << stage;
          last = (last & ~(1u << stage)) | (phase << stage);
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
      }
      // After an error nobody may have waited for the last copies of the pair (they
      // complete on the even CTA): do so, bounded, before the shared memory goes.
      if (leader && *((volatile int*)err) != 0) {
        const uint64_t t0 = globaltimer();
        for (int s = 0; s < STAGES; ++s)
          while ((issued >> s & 1u) && !mbar_try_wait(smem_u32(&full_bar[s]), last >> s & 1u) &&
                 globaltimer() - t0 < 100000000ull) {
          }
      }
    }
  } else if (warp == 1) {
    if (leader && lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      int local = 0;
      bool ok = true;
      for (int64_t w = cid; w < num_tiles && ok; w += n_clusters, ++local) {
        const uint32_t idesc = idesc_bf16(2 * BM_CTA, tile_width(geo, bn2, (int)(w / tiles_m)), false, false);
        const int acc = local & 1;
        const uint32_t acc_phase = (local >> 1) & 1;
        if (!mbar_wait(&tempty_bar[acc], acc_phase ^ 1, err)) break;
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + acc * BN_MAX;
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!mbar_wait(&full_bar[stage], phase, err)) { ok = false; break; }
          tc_fence_after();
          const uint32_t a_base = smem_u32(sA + stage * A_BYTES);
          const uint32_t b_base = smem_u32(sB + stage * B_BYTES);
#pragma unroll
          for (int kk = 0; kk < BK / 16; ++kk)
            mma_bf16_ss_pair(d_tmem, smem_desc_sw128(a_base + kk * 32, 16, 1024),
                             smem_desc_sw128(b_base + kk * 32, 16, 1024), idesc, (kb != 0 || kk != 0) ? 1u : 0u);
          mma_commit_pair(&empty_bar[stage], 0x3);
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
        if (ok) mma_commit_pair(&tfull_bar[acc], 0x3);
      }
    }
  } else {
    const int quarter = warp & 3;
    int local = 0;
    for (int64_t w = cid; w < num_tiles; w += n_clusters, ++local) {
      const int tm = (int)(w % tiles_m), tn = (int)(w / tiles_m);
      const int acc = local & 1;
      const uint32_t acc_phase = (local >> 1) & 1;
      if (!mbar_wait(&tfull_bar[acc], acc_phase, err)) break;
      tc_fence_after();
      const int y0 = tm * 2 * BM_CTA + (int)rank * BM_CTA + quarter * 32;
      const int t = y0 + lane;
      const uint32_t t_row = tmem_base + ((uint32_t)(quarter * 32) << 16) + acc * BN_MAX;
      const uint32_t tempty = mapa_shared(smem_u32(&tempty_bar[acc]), 0);
      auto release = [&] {
        tc_fence_before();
        mbar_arrive_cluster_relaxed(tempty);
      };
      if (y0 >= T) {  // no row of this warp is in range
        release();
        continue;
      }
      const int64_t id = t < T ? ids[t] : -1;
      const int n0 = tile_start(geo, bn2, tn);
      int width = BN_MAX, group = tn, groups = 1;
      if (tn >= geo.n_full) {
        width = 1 << geo.shift;
        group = geo.n_full + ((tn - geo.n_full) * bn2 >> geo.shift);
        groups = min(bn2 >> geo.shift, geo.n_full + geo.n_rest - group);
      }
      float2* out = stats + (int64_t)t * (geo.n_full + geo.n_rest) + group;
      for (int i = 0; i < groups; ++i) {
        const float2 st = row_stats<STORE>(t_row + i * width, width, n0 + i * width, V, id, scale, e + (int64_t)t * lde,
                                           t < T, i + 1 == groups, release);
        if (t < T) out[i] = st;
      }
    }
  }

  // On an error path the MMA issuer may have left MMAs in flight: drain them
  // (bounded) before the accumulator columns are released.
  if (warp == 1 && lane == 0 && leader && *((volatile int*)err) != 0) {
    mma_commit_pair(drain_bar, 0x1);
    const uint64_t t0 = globaltimer();
    while (!mbar_try_wait(smem_u32(drain_bar), 0) && globaltimer() - t0 < 100000000ull) {
    }
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // neither CTA leaves while the pair MMA may still read its shared memory
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, 2 * BN_MAX);
  }
}

// ---------------------------------------------------------------- finish
constexpr int kFinThreads = 128;

// One block per row of h; its log-probability goes to row perm[t] (t without
// perm).  dot in 64 bits (bf16 products are exact in fp32; eight of them are
// added in fp32, the rest in double), then the groups' statistics: with d = m -
// x_id (base 2), logp = -log(1 + s 2^d), written so that neither a large nor a
// small d loses digits.  lse: the row's maximum m, unscaled, and lse2 - m.
__global__ void __launch_bounds__(kFinThreads)
    logprob_finish_kernel(const __nv_bfloat16* __restrict__ h, int64_t ldh, const __nv_bfloat16* __restrict__ w,
                          int64_t ldw, const int64_t* __restrict__ ids, const int* __restrict__ perm,
                          const float2* __restrict__ stats, int groups, int V, int H, float scale, float scale_mma,
                          float* __restrict__ logp, float2* __restrict__ lse) {
  pdl_prologue();
  const int64_t t = blockIdx.x;
  const int64_t out = perm ? perm[t] : t;
  const int64_t id = ids[t];
  if (id < 0 || id >= V) {
    // no token: 0.  An id past the vocabulary has no log-probability: NaN.
    if (threadIdx.x == 0) {
      logp[out] = id < 0 ? 0.f : NAN;
      lse[t] = id < 0 ? make_float2(0.f, 0.f) : make_float2(NAN, NAN);
    }
    return;
  }
  double dot = 0.0;
  const uint4* hr = reinterpret_cast<const uint4*>(h + t * ldh);
  const uint4* wr = reinterpret_cast<const uint4*>(w + id * ldw);
  for (int i = threadIdx.x; i < H / 8; i += kFinThreads) {
    const uint4 a = hr[i], b = wr[i];
    const uint32_t* ap = &a.x;
    const uint32_t* bp = &b.x;
    float p = 0.f;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float2 x = unpack_bf16x2(ap[q]), y = unpack_bf16x2(bp[q]);
      p = fmaf(x.x, y.x, p);
      p = fmaf(x.y, y.y, p);
    }
    dot += (double)p;
  }
  float m = -INFINITY, s = 0.f;
  const float2* sr = stats + t * groups;
  for (int i = threadIdx.x; i < groups; i += kFinThreads) {
    const float2 v = sr[i];
    const float mn = fmaxf(m, v.x);
    if (mn == -INFINITY) {
      s += v.y;  // 0, or the NaN of a NaN logit
      continue;
    }
    s = s * ex2((m - mn) * scale_mma) + v.y * ex2((v.x - mn) * scale_mma);
    m = mn;
  }
  __shared__ double sd[kFinThreads / 32];
  __shared__ float sm[kFinThreads / 32], ss[kFinThreads / 32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    dot += __shfl_xor_sync(0xffffffffu, dot, o);
    const float m2 = __shfl_xor_sync(0xffffffffu, m, o), s2 = __shfl_xor_sync(0xffffffffu, s, o);
    const float mn = fmaxf(m, m2);
    s = mn == -INFINITY ? s + s2 : s * ex2((m - mn) * scale_mma) + s2 * ex2((m2 - mn) * scale_mma);
    m = mn;
  }
  const int wp = threadIdx.x >> 5;
  if ((threadIdx.x & 31) == 0) {
    sd[wp] = dot;
    sm[wp] = m;
    ss[wp] = s;
  }
  __syncthreads();
  if (threadIdx.x != 0) return;
#pragma unroll
  for (int i = 1; i < kFinThreads / 32; ++i) {
    dot += sd[i];
    const float mn = fmaxf(m, sm[i]);
    s = mn == -INFINITY ? s + ss[i] : s * ex2((m - mn) * scale_mma) + ss[i] * ex2((sm[i] - mn) * scale_mma);
    m = mn;
  }
  const double x_id = dot * (double)scale;
  const float d = (float)((double)m * (double)scale_mma - x_id);
  float lp, above;
  if (d <= 0.f) {
    lp = -log1pf(s * exp2f(d));
    above = -d - lp * kLog2e;
  } else {
    const float all = s + exp2f(-d);
    lp = -(d * kLn2 + logf(all));
    above = log2f(all);
  }
  if (x_id == INFINITY) lp = above = NAN;
  if (m == -INFINITY) {  // no other token
    m = 0.f;
    above = (float)x_id - lp;  // lp: 0, or NaN
  }
  logp[out] = lp;
  lse[t] = make_float2(m, above);
}

// ---------------------------------------------------------------- backward
constexpr int kBwdThreads = 256;
constexpr int kBwdUnroll = 4;

// A warp takes 256 columns of a row at a time, 8 of them per lane, which are of one
// group and have one factor.  The result is rounded to bf16, each entry on its own:
// the tensor cores multiply nothing wider at their full rate.  The target's entry, 0 in E, stays 0;
// own[t] = c (1 - p) = -c expm1(logp).
__global__ void __launch_bounds__(kBwdThreads)
    logprob_bwd_kernel(__nv_bfloat16* __restrict__ e, int64_t lde, const float2* __restrict__ stats,
                       const float2* __restrict__ lse, float scale_mma, const float* __restrict__ logp,
                       const int64_t* __restrict__ ids, const int* __restrict__ perm,
                       const int* __restrict__ count, int row0, const float* __restrict__ g, float inv_tau, int V,
                       float* __restrict__ own, const LogprobGroups geo) {
  pdl_prologue();
  const int64_t t = blockIdx.x;
  // behind the rows with a token: zeros up to the end of the last 64-deep step of
  // the head gradient's sum over rows, and nothing beyond, which no product reads
  if (t >= (max(1, *count - row0) + 63) / 64 * 64) return;
  const int64_t id = ids[t];
  const int src = perm[t];  // logp and g are in the caller's row order
  const float c = id < 0 ? 0.f : g[src] * inv_tau;
  const float2 top = lse[t];
  __nv_bfloat16* row = e + t * lde;
  const int lane = threadIdx.x & 31;
  const int warps = (int)gridDim.y * (kBwdThreads / 32);
  if (blockIdx.y == 0 && threadIdx.x == 0) own[t] = id < 0 ? 0.f : -c * expm1f(logp[src]);
  const float2* st = stats + t * (geo.n_full + geo.n_rest);
  auto scaled = [&](uint4 u, float f) {
    uint32_t* p = &u.x;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float2 x = unpack_e(p[q]);
      p[q] = pack_bf16x2(x.x * f, x.y * f);
    }
    return u;
  };
  // kBwdUnroll vectors a lane in flight
  const int windows = (V + BN_MAX - 1) / BN_MAX;
  for (int i = blockIdx.y * (kBwdThreads / 32) + (threadIdx.x >> 5); i < windows; i += kBwdUnroll * warps) {
    uint4 u[kBwdUnroll];
    float f[kBwdUnroll];
#pragma unroll
    for (int j = 0; j < kBwdUnroll; ++j) {
      const int wi = i + j * warps, col = wi * BN_MAX + lane * 8;
      if (id >= 0 && col < V) {
        u[j] = __ldcs(reinterpret_cast<const uint4*>(row + col));
        f[j] = st[wi < geo.n_full ? wi : geo.n_full + ((col - geo.n_full * BN_MAX) >> geo.shift)].x;
      }
    }
#pragma unroll
    for (int j = 0; j < kBwdUnroll; ++j) {
      const int col = (i + j * warps) * BN_MAX + lane * 8;
      if (col < V)
        *reinterpret_cast<uint4*>(row + col) =
            id < 0 ? make_uint4(0u, 0u, 0u, 0u) : scaled(u[j], -c * ex2(fmaf(f[j] - top.x, scale_mma, -top.y)));
    }
  }
}

// v += f x, x eight bf16
__device__ __forceinline__ void add_scaled(float* v, const uint4& x, float f) {
  const uint32_t* w = &x.x;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const float2 y = unpack_bf16x2(w[q]);
    v[2 * q] = fmaf(f, y.x, v[2 * q]);
    v[2 * q + 1] = fmaf(f, y.y, v[2 * q + 1]);
  }
}

// ---------------------------------------------------------------- packing
// Rows with a token first, in order, then the others: perm[i] is the row at
// place i.  The packed rows without a token are zeros, so what stands
// in them (padding, even NaN) cannot reach the head's gradient, a sum over
// rows in which their coefficient is 0.
// A block takes `rows` rows, one a warp at a time, and counts the ids before
// them itself (T ids from L2), so one launch does it all.
constexpr int kPackThreads = 256;
constexpr int kPackMaxRows = 1024;

__global__ void __launch_bounds__(kPackThreads)
    logprob_pack_kernel(const __nv_bfloat16* __restrict__ h, int64_t ldh, const int64_t* __restrict__ ids, int T,
                        int H, int rows, __nv_bfloat16* __restrict__ hp, int64_t* __restrict__ idp, int* __restrict__ perm,
                        int* __restrict__ count) {
  pdl_prologue();
  __shared__ int s_before[kPackThreads / 32], s_total[kPackThreads / 32];
  __shared__ int s_pos[kPackMaxRows];
  const int r0 = blockIdx.x * rows;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int before = 0, total = 0;
  for (int t = threadIdx.x; t < T; t += kPackThreads) {
    const int v = ids[t] >= 0 ? 1 : 0;
    total += v;
    if (t < r0) before += v;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    before += __shfl_xor_sync(0xffffffffu, before, o);
    total += __shfl_xor_sync(0xffffffffu, total, o);
  }
  if (lane == 0) {
    s_before[warp] = before;
    s_total[warp] = total;
  }
  __syncthreads();
  before = total = 0;
#pragma unroll
  for (int i = 0; i < kPackThreads / 32; ++i) {
    before += s_before[i];
    total += s_total[i];
  }
  if (warp == 0) {
    for (int i = 0; i < rows; i += 32) {
      const int t = i + lane < rows ? r0 + i + lane : T;
      const int64_t id = t < T ? ids[t] : -1;
      const uint32_t live = __ballot_sync(0xffffffffu, id >= 0);
      const int mine = before + __popc(live & ((1u << lane) - 1u));
      if (t < T) {
        const int p = id >= 0 ? mine : total + (t - mine);
        s_pos[i + lane] = p;
        perm[p] = t;
        idp[p] = id;
      }
      before += __popc(live);
    }
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) count[0] = total;
  __syncthreads();
  for (int i = warp; i < rows && r0 + i < T; i += kPackThreads / 32) {
    const int p = s_pos[i];
    const uint4* src = reinterpret_cast<const uint4*>(h + (int64_t)(r0 + i) * ldh);
    uint4* dst = reinterpret_cast<uint4*>(hp + (int64_t)p * H);
    const bool has = p < total;
#pragma unroll 4
    for (int k = lane; k < H / 8; k += 32) dst[k] = has ? src[k] : make_uint4(0u, 0u, 0u, 0u);
  }
}

// dst[perm[i]] = the sum over slices, in order, of row i of src - bf16 rows (one
// slice), or fp32 slabs - and (own) own[i] w[ids[i]], for rows with a token, 0
// for the others; a block a row.
template <typename E>
__global__ void __launch_bounds__(128)
    logprob_unpack_kernel(const E* __restrict__ src, int slices, const int* __restrict__ perm,
                          const int* __restrict__ count, int row0, int T, int H, const float* __restrict__ own,
                          const int64_t* __restrict__ ids, const __nv_bfloat16* __restrict__ w, int64_t ldw, int V,
                          __nv_bfloat16* __restrict__ dst) {
  pdl_prologue();
  const int i = blockIdx.x;
  const bool live = row0 + i < count[0];
  uint4* d = reinterpret_cast<uint4*>(dst + (int64_t)perm[i] * H);
  const int64_t slab = (int64_t)T * H;
  const int64_t id = own && live ? ids[i] : 0;
  const float f = own && live && id < V ? own[i] : 0.f;  // past the vocabulary: src is NaN already
  const uint4* wr = own && live && id < V ? reinterpret_cast<const uint4*>(w + id * ldw) : nullptr;
  for (int k = threadIdx.x; k < H / 8; k += 128) {
    uint4 u = make_uint4(0u, 0u, 0u, 0u);
    if (live) {
      if constexpr (sizeof(E) == 2) {
        u = reinterpret_cast<const uint4*>(src + (int64_t)i * H)[k];
      } else {
        float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        const uint4 x = wr ? wr[k] : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll 4
        for (int s = 0; s < slices; ++s) {
          const float4* p = reinterpret_cast<const float4*>(src + s * slab + (int64_t)i * H) + 2 * k;
          const float4 a = __ldcs(p), b = __ldcs(p + 1);
          v[0] += a.x; v[1] += a.y; v[2] += a.z; v[3] += a.w;
          v[4] += b.x; v[5] += b.y; v[6] += b.z; v[7] += b.w;
        }
        add_scaled(v, x, f);
        u = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]),
                       pack_bf16x2(v[6], v[7]));
      }
    }
    d[k] = u;
  }
}

// dw[ids[t]] += own[t] h[t] over the rows that have a token: a block a row, in
// which the first row of an id adds up all rows of that id (in the same order on
// every run) and the others leave.  The sum of all of an id's rows is kept in fp32
// and meets dw once.  Each block looks through all ids, so the time grows with
// the square of the rows; up to 8192 rows the ids stay in L1 and the loads of a
// frequent id's rows, which go out eight at a time, take longer (8192 rows of H
// 1024, 7500 ids: 56 us; one id for all rows, the worst: 703 us, 2065 one at a
// time).  64 registers: with more, fewer blocks look through the ids at a time (77:
// 63 and 582 us).
constexpr int kOwnWarps = 4;
constexpr int kOwnList = 512;
constexpr int kOwnAhead = 8;  // rows in flight
// v += own[r] h[r] for the listed rows r, in order, eight columns of them
__device__ __forceinline__ void add_rows(float* v, const __nv_bfloat16* __restrict__ h, int H,
                                         const float* __restrict__ own, const int* list, int rows) {
  if (rows == 1) {  // mostly
    const int r = list[0];
    add_scaled(v, *reinterpret_cast<const uint4*>(h + (int64_t)r * H), own[r]);
    return;
  }
  // the last rows again, times 0, where they do not fill a group
#pragma unroll 1
  for (int j = 0; j < rows; j += kOwnAhead) {
    uint4 x[kOwnAhead];
    float f[kOwnAhead];
#pragma unroll
    for (int q = 0; q < kOwnAhead; ++q) {
      const int r = list[min(j + q, rows - 1)];
      x[q] = *reinterpret_cast<const uint4*>(h + (int64_t)r * H);
      f[q] = j + q < rows ? own[r] : 0.f;
    }
#pragma unroll
    for (int q = 0; q < kOwnAhead; ++q) add_scaled(v, x[q], f[q]);
  }
}

template <typename E>
__global__ void __launch_bounds__(32 * kOwnWarps, 8)
    logprob_own_kernel(const __nv_bfloat16* __restrict__ h, const int64_t* __restrict__ ids,
                       const float* __restrict__ own, const int* __restrict__ count, int row0, int T, int V, int H,
                       E* __restrict__ dw) {
  pdl_prologue();
  __shared__ int list[kOwnWarps][kOwnList], found[kOwnWarps];
  const int n = min(T, count[0] - row0), t = blockIdx.x;
  if (t >= n) return;
  const int64_t id = ids[t];
  if (id >= V) return;  // no row of the head; the gradient is NaN already
  bool seen = false;
#pragma unroll 8
  for (int i = threadIdx.x; i < t; i += 32 * kOwnWarps) seen = seen || ids[i] == id;
  if (__syncthreads_or(seen)) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // each warp looks through a quarter of the rows from t on, 256 at a time
  const int per = (n - t + kOwnWarps - 1) / kOwnWarps;
  const int first = t + warp * per, end = min(n, first + per);
  int i = first;
  // the next rows of the id, up to kOwnList a warp; true if there may be more
  auto refill = [&] {
    int m = 0;
    while (i < end && m <= kOwnList - 256) {
      int64_t v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) v[u] = i + 32 * u + lane < end ? ids[i + 32 * u + lane] : -1;
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const uint32_t hit = __ballot_sync(0xffffffffu, v[u] == id);
        if (v[u] == id) list[warp][m + __popc(hit & ((1u << lane) - 1u))] = i + 32 * u + lane;
        m += __popc(hit);
      }
      i += 256;
    }
    if (lane == 0) found[warp] = m;
    return (bool)__syncthreads_or(i < end);
  };
  bool more = refill();
  const bool one_list = !more;
  for (int c0 = 0;;) {
    const int col = c0 + threadIdx.x * 8;
    float a[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (;;) {
      if (col < H) {
        for (int w = 0; w < kOwnWarps; ++w) add_rows(a, h + col, H, own, list[w], found[w]);
      }
      if (!more) break;
      __syncthreads();  // the list is free again
      more = refill();
    }
    if (col < H) {
      E* d = dw + id * H + col;
      if constexpr (sizeof(E) == 2) {
        uint4 u = *reinterpret_cast<uint4*>(d);
        add_scaled(a, u, 1.f);
        *reinterpret_cast<uint4*>(d) = make_uint4(pack_bf16x2(a[0], a[1]), pack_bf16x2(a[2], a[3]),
                                                  pack_bf16x2(a[4], a[5]), pack_bf16x2(a[6], a[7]));
      } else {
#pragma unroll
        for (int q = 0; q < 8; ++q) d[q] += a[q];
      }
    }
    c0 += 32 * kOwnWarps * 8;
    if (c0 >= H) return;
    if (!one_list) {  // from the first rows again for the next columns
      __syncthreads();
      i = first;
      more = refill();
    }
  }
}

template <bool STORE>
void launch_gemm(const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tb2, const LogprobParams& p,
                 int a_rows, int bn2, float scale, cudaStream_t stream) {
  auto kern = logprob_gemm_kernel<STORE>;
  static std::mutex mu;
  static int max_clusters[64] = {0};
  int dev = 0;
  PB_CUDA_CHECK(cudaGetDevice(&dev));
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = SMEM_BYTES;
  cfg.stream = stream;
  int clusters = 0;
  {
    std::lock_guard<std::mutex> lk(mu);
    if (max_clusters[dev & 63] == 0) {
      PB_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES));
      cfg.gridDim = dim3(2 * num_sms(dev) / 2, 1, 1);
      int n = 0;
      PB_CUDA_CHECK(cudaOccupancyMaxActiveClusters(&n, kern, &cfg));
      PB_CHECK(n > 0, "logprob: no cluster of two CTAs fits on this GPU");
      max_clusters[dev & 63] = n;
    }
    clusters = max_clusters[dev & 63];
  }
  const int tiles2 = (p.V - p.groups.n_full * BN_MAX + bn2 - 1) / bn2;
  const int64_t tiles = (int64_t)((p.T + 2 * BM_CTA - 1) / (2 * BM_CTA)) * (p.groups.n_full + tiles2);
  clusters = (int)std::max<int64_t>(1, std::min<int64_t>(clusters, tiles));
  cfg.gridDim = dim3(2 * clusters, 1, 1);
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  PB_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kern, ta, tb, tb2, (__nv_bfloat16*)p.e, p.lde, p.ids, p.count, p.row0, reinterpret_cast<float2*>(p.stats),
                                   p.T, p.V, p.H, a_rows, p.groups, bn2, tiles2, scale, error_word(dev)));
}

// Base-2 logit per unit of the tensor core's dot product: what its truncation
// takes is given back on average (kTruncation).
float mma_scale(float inv_tau, int H) {
  return (float)((double)kLog2e * inv_tau * (1.0 + kTruncation * ((H + 15) / 16)));
}

}  // namespace

LogprobGroups logprob_groups(int V) {
  const int pairs = std::max(1, num_sms() / 2);
  LogprobGroups g;
  g.n_full = V / BN_MAX / pairs * pairs;
  const int rest = V - g.n_full * BN_MAX;
  // the narrowest tiles, in steps of 32, of which a row tile's fit one wave; groups of the power of two in that
  int bn = 32;
  while (bn < BN_MAX && (rest + bn - 1) / bn > pairs) bn += 32;
  g.shift = 5;
  while (bn % (2 << g.shift) == 0) ++g.shift;
  g.n_rest = (rest + (1 << g.shift) - 1) >> g.shift;
  return g;
}

// Width of the tiles behind the first n_full, for T rows: the waves that they take
// times a tile's time, which goes by the operand rows that it loads (1237 rows of V
// 32003, H 2048: 120 us in tiles of 192, 92 in 256).
static int rest_width(const LogprobGroups& g, int T, int V) {
  const int64_t tiles_m = (T + 2 * BM_CTA - 1) / (2 * BM_CTA), pairs = std::max(1, num_sms() / 2);
  const int rest = V - g.n_full * BN_MAX;
  auto cost = [&](int bn) { return (tiles_m * ((rest + bn - 1) / bn) + pairs - 1) / pairs * (bn + std::min(T, 2 * BM_CTA)); };
  int best = BN_MAX;
  for (int bn = 1 << g.shift; bn < BN_MAX; bn += 1 << g.shift)
    if (cost(bn) < cost(best)) best = bn;
  return best;
}

void logprob_fwd(const LogprobParams& p, cudaStream_t stream) {
  PB_CHECK(p.T > 0 && p.V > 0 && p.H > 0, "logprob: empty problem");
  PB_CHECK(p.H % 8 == 0 && p.ldh % 8 == 0 && p.ldw % 8 == 0,
           "logprob: hidden size and row strides must be multiples of 8 elements");
  PB_CHECK((reinterpret_cast<uintptr_t>(p.h) & 15) == 0 && (reinterpret_cast<uintptr_t>(p.w) & 15) == 0,
           "logprob: h and w must be 16-byte aligned");
  const float scale = kLog2e * p.inv_tau;
  const float scale_mma = mma_scale(p.inv_tau, p.H);  // the target logit does not come from the tensor core
  const int a_rows = p.T < BM_CTA ? (p.T + 7) / 8 * 8 : BM_CTA;
  const CUtensorMap ta = make_tmap_2d_bf16(p.h, p.H, p.T, p.ldh, BK, a_rows);
  const CUtensorMap tb = make_tmap_2d_bf16(p.w, p.H, p.V, p.ldw, BK, BN_MAX / 2);
  const int bn2 = rest_width(p.groups, p.T, p.V);
  const CUtensorMap tb2 = make_tmap_2d_bf16(p.w, p.H, p.V, p.ldw, BK, bn2 / 2);
  if (p.e) {
    PB_CHECK(p.lde % 32 == 0 && (reinterpret_cast<uintptr_t>(p.e) & 63) == 0, "logprob: E must have 64-byte rows");
    launch_gemm<true>(ta, tb, tb2, p, a_rows, bn2, scale_mma, stream);
  } else {
    launch_gemm<false>(ta, tb, tb2, p, a_rows, bn2, scale_mma, stream);
  }
  launch_k(logprob_finish_kernel, p.T, kFinThreads, 0, stream, (const __nv_bfloat16*)p.h, p.ldh,
           (const __nv_bfloat16*)p.w, p.ldw, p.ids, p.perm, (const float2*)p.stats, p.groups.n(), p.V, p.H, scale,
           scale_mma, p.logp, reinterpret_cast<float2*>(p.lse));
}

void logprob_bwd(void* e, int64_t lde, const float* stats, const float* lse, const float* logp, const int64_t* ids,
                 const int* perm, const int* count, int row0, const float* g, float inv_tau, int T, int V, int H,
                 float* own, const LogprobGroups& geo, cudaStream_t stream) {
  if (T == 0) return;
  // enough blocks for every SM when there are few rows
  const int segs = std::max(1, std::min((V + 8 * BN_MAX - 1) / (8 * BN_MAX), (8 * num_sms() + T - 1) / T));
  launch_k(logprob_bwd_kernel, dim3(T, segs), kBwdThreads, 0, stream, (__nv_bfloat16*)e, lde, (const float2*)stats,
           (const float2*)lse, mma_scale(inv_tau, H), logp, ids, perm, count, row0, g, inv_tau, V, own,
           geo);
}

void logprob_pack(const void* h, int64_t ldh, const int64_t* ids, int T, int H, void* hp, int64_t* idp, int* perm,
                  int* count, cudaStream_t stream) {
  PB_CHECK(H % 8 == 0 && ldh % 8 == 0 && (reinterpret_cast<uintptr_t>(h) & 15) == 0 &&
               (reinterpret_cast<uintptr_t>(hp) & 15) == 0,
           "logprob: h must have 16-byte rows");
  // 8 rows a block up to 8192 rows; beyond, more, so that all blocks together read at most 8192 ids per row
  const int rows = std::min(kPackMaxRows, 8 * ((T + 8191) / 8192));
  launch_k(logprob_pack_kernel, (T + rows - 1) / rows, kPackThreads, 0, stream, (const __nv_bfloat16*)h, ldh, ids, T, H,
           rows, (__nv_bfloat16*)hp, idp, perm, count);
}

void logprob_unpack(const void* src, bool f32, int slices, const int* perm, const int* count, int row0, int T, int H,
                    const float* own, const int64_t* ids, const void* w, int64_t ldw, int V, void* dst,
                    cudaStream_t stream) {
  PB_CHECK(f32 || !own, "logprob: the target's part is added to fp32 sums");
  if (f32)
    launch_k(logprob_unpack_kernel<float>, T, 128, 0, stream, (const float*)src, slices, perm, count, row0, T, H, own,
             ids, (const __nv_bfloat16*)w, ldw, V, (__nv_bfloat16*)dst);
  else
    launch_k(logprob_unpack_kernel<__nv_bfloat16>, T, 128, 0, stream, (const __nv_bfloat16*)src, 1, perm, count, row0,
             T, H, own, ids, (const __nv_bfloat16*)w, ldw, V, (__nv_bfloat16*)dst);
}

void logprob_own(const void* h, const int64_t* ids, const float* own, const int* count, int row0, int T, int V, int H,
                 void* dw, bool f32, cudaStream_t stream) {
  if (f32)
    launch_k(logprob_own_kernel<float>, T, 32 * kOwnWarps, 0, stream, (const __nv_bfloat16*)h, ids, own, count, row0, T,
             V, H, (float*)dw);
  else
    launch_k(logprob_own_kernel<__nv_bfloat16>, T, 32 * kOwnWarps, 0, stream, (const __nv_bfloat16*)h, ids, own, count,
             row0, T, V, H, (__nv_bfloat16*)dw);
}

}  // namespace pb
