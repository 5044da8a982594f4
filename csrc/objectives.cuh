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
// stats [T, ceil(V / bn), 2] fp32: per row and tile of bn vocabulary columns
// the maximum and sum of 2^(x - max), x = l log2(e), target left out.
// e (optional, bf16 [T, lde >= V]): 2^(x - tile max).
struct LogprobParams {
  const void* h;
  const void* w;
  const int64_t* ids;
  const int* perm;  // optional: row t's log-probability goes to logp[perm[t]]
  float* stats;
  float* logp;
  float* lse2;  // base-2 log-sum-exp of row t
  void* e;
  int64_t ldh, ldw, lde;
  int T, V, H, bn;
  float inv_tau;
};
int logprob_tile_n(int T, int V);
void logprob_fwd(const LogprobParams& p, cudaStream_t stream);
// e becomes the gradient of the raw logits h w^T given g = d loss / d logp
// (row t of e has its logp and g in row perm[t])
void logprob_bwd(void* e, int64_t lde, const float* stats, const float* lse2, const float* logp, const int64_t* ids,
                 const int* perm, const float* g, float inv_tau, int T, int V, int bn, cudaStream_t stream);
// hp [T, H]: the rows of h with ids >= 0 in order, then zeros; idp the ids in
// that order, pos[t] row t's place, perm its inverse, count[0] the rows with a token
void logprob_pack(const void* h, int64_t ldh, const int64_t* ids, int T, int H, void* hp, int64_t* idp, int* perm,
                  int* pos, int* count, cudaStream_t stream);
// dst[t] = src[pos[t]] where row t has a token, else 0
void logprob_unpack(const void* src, const int* pos, const int* count, int T, int H, void* dst, cudaStream_t stream);

}  // namespace pb
