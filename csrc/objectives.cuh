// Launchers of the post-training objectives: token log-probabilities through
// the LM head (logprob.cu), the clipped policy and preference losses over
// token log-probabilities (objectives.cu) and distillation from a teacher's
// top logits (distill.cu).  Raw device pointers on the given stream; shapes
// are validated by the bindings.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace pb {

// ---- log-probabilities of given tokens (logprob.cu)
// h [T, H] and w [V, H] bf16; ids [T] (negative: no token, logp 0).
// stats [T, groups, 2] fp32: per row and group of vocabulary columns the maximum
// of h . w and the sum of 2^(x - x at the maximum), x the logit in base 2, target
// left out.
// e (optional, 16-bit [T, lde >= V]): 2^(x - group max), in a format of logprob.cu.
struct LogprobGroups {
  int n_full, n_rest, shift;  // n_full groups of 256 columns, then n_rest of 1 << shift
  int n() const { return n_full + n_rest; }
};
LogprobGroups logprob_groups(int V);
struct LogprobParams {
  const void* h;
  const void* w;
  const int64_t* ids;
  const int* perm;   // optional: row t's log-probability goes to logp[perm[t]]
  const int* count;  // optional: of all packed rows the first count[0] have a token, and h starts at row row0
  int row0;
  float* stats;
  float* logp;
  float* lse;  // [T, 2]: the maximum of h . w over row t's groups, the row's base-2 log-sum-exp above it
  void* e;
  int64_t ldh, ldw, lde;
  int T, V, H;
  LogprobGroups groups;
  float inv_tau;
};
void logprob_fwd(const LogprobParams& p, cudaStream_t stream);
// e becomes the gradient (bf16) of the raw logits h w^T given g = d loss / d logp,
// 0 at the target, whose gradient goes to own [T] in fp32 (row t of e has its
// logp and g in row perm[t]; e starts at packed row row0)
void logprob_bwd(void* e, int64_t lde, const float* stats, const float* lse, const float* logp, const int64_t* ids,
                 const int* perm, const int* count, int row0, const float* g, float inv_tau, int T, int V, int H,
                 float* own, const LogprobGroups& groups, cudaStream_t stream);
// hp [T, H]: the rows of h with ids >= 0 in order, then zeros; idp the ids and
// perm the rows in that order, count[0] the rows with a token
void logprob_pack(const void* h, int64_t ldh, const int64_t* ids, int T, int H, void* hp, int64_t* idp, int* perm,
                  int* count, cudaStream_t stream);
// dst[perm[i]] = row i of src [T, H] (bf16, or f32: the sum of `slices` such slabs, and of own[i] w[ids[i]] where own
// is given) for the packed rows [row0, row0 + T) with a token, 0 for the others; perm, own and ids start at row0
void logprob_unpack(const void* src, bool f32, int slices, const int* perm, const int* count, int row0, int T, int H,
                    const float* own, const int64_t* ids, const void* w, int64_t ldw, int V, void* dst,
                    cudaStream_t stream);
// dw [V, H] (fp32 or bf16, contiguous): dw[ids[t]] += own[t] h[t] over the packed rows [row0, row0 + T) with a token
void logprob_own(const void* h, const int64_t* ids, const float* own, const int* count, int row0, int T, int V, int H,
                 void* dw, bool f32, cudaStream_t stream);

// ---- losses over token log-probabilities (objectives.cu); rows b have their
// own strides, mask is bool bytes (optional).  chunk: objective_chunk(rows, S),
// nchunk = max(1, ceil(S / chunk)); parts and ticket are scratch.
int objective_chunk(int64_t rows, int64_t S);
struct PolicyPart {
  double2 sums;  // loss, kl
  int2 counts;   // tokens, clipped tokens
  int2 pad;      // to 32 bytes
};
struct PolicyParams {
  const float *logp, *old, *adv, *ref;  // ref optional
  const uint8_t* mask;
  int64_t ld_logp, ld_old, adv_sb, adv_ss, ld_ref, ld_mask;
  int B, S, chunk, nchunk;
  double low, high, kl_coef;  // the clip range [low, high] of the ratio
  bool per_sequence;         // mean over rows of the row means, else mean over tokens
  float* coef;               // optional [B, S]: d (token loss) / d logp, 0 outside the mask
  PolicyPart* parts;         // [B * nchunk]
  int* ticket;
  float *loss, *clip, *kl;  // scalars
  float *inv, *inv_row;     // gradient = coef * inv (* inv_row [B] when per_sequence)
};
void policy_fwd(const PolicyParams& p, cudaStream_t stream);
void policy_bwd(const float* coef, const float* g, const float* inv, const float* inv_row, float* out, int B, int S,
                int chunk, int nchunk, cudaStream_t stream);

// rows [0, P) are the chosen sequences, rows [P, 2P) the rejected ones
struct PreferenceParams {
  const float *logp, *ref;  // ref optional
  const uint8_t* mask;
  int64_t ld_logp, ld_ref, ld_mask;
  int P, S, chunk, nchunk;
  double beta, smoothing;
  bool average;
  double2* parts;  // [2P * nchunk]: sum, tokens
  int* ticket;
  float *loss, *rewards, *coef;  // scalar, [2P], [2P]: d loss / d (logp of a token of the row)
};
void preference_fwd(const PreferenceParams& p, cudaStream_t stream);
void preference_bwd(const float* coef, const float* g, const uint8_t* mask, int64_t ld_mask, float* out, int rows,
                    int S, int chunk, int nchunk, cudaStream_t stream);

// ---- distillation from a teacher's top logits (distill.cu)
// Teacher entries [T_all, K]: values (bf16 or fp32) and ids (int32 or int64,
// negative = absent), mask (optional bool [T_all]).  distill_prep fills q, id,
// live and counters[0] = rows that count; distill_rows then takes a block of
// T rows of logits, [row0, row0 + T), and distill_loss writes the loss of all
// blocks.  grad (optional) may be the logits themselves; the two must be
// misaligned by the same number of bytes in every row.  weight (optional): what
// the loss is multiplied with, on the device; the gradient is written again with
// it, and nothing happens where it is 1.
constexpr int kDistillMaxK = 1024;
constexpr int kDistillMaxCluster = 8;
struct DistillParams {
  const void* logits;
  void* grad;
  int64_t ld, ld_grad;
  const void *top, *ids;
  const uint8_t* mask;
  int64_t ld_top, ld_ids, ld_mask;
  bool top_bf16, ids32;
  int T, T_all, V, K, Kp, cluster;  // Kp: K rounded up to a multiple of 4
  int64_t row0;
  const int* perm;  // optional: row i of the logits is row perm[i] of the teacher's, those that count first
  int64_t* key;     // optional [T_all]: 0 for a row that counts, else -1 (what logprob_pack packs by)
  float tau, inv_tau;
  float* q;        // [T_all, Kp]
  int* id;         // [T_all, Kp]
  uint8_t* live;   // [T_all]
  float* row_loss;  // [T_all * kDistillMaxCluster]: shares of a row's loss, cluster by cluster
  int* counters;   // [1]
  float* loss;
  const float* weight;
};
void distill_prep(const DistillParams& p, cudaStream_t stream);  // T = T_all
void distill_rows(const DistillParams& p, bool bf16, cudaStream_t stream);
void distill_loss(const DistillParams& p, bool bf16, cudaStream_t stream);  // bf16: the logits' type

}  // namespace pb
