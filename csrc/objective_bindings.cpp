// Bindings of the post-training objectives (objectives.cuh).
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <algorithm>
#include <limits>
#include <string>
#include <vector>

#include "gemm.cuh"
#include "host_util.h"
#include "objectives.cuh"

namespace {

cudaStream_t cur_stream() { return at::cuda::getCurrentCUDAStream().stream(); }

constexpr int64_t kIntMax = std::numeric_limits<int>::max();

// Numbers enter error messages as strings: where the extension carries its own
// copy of the C++ runtime, streaming an integer into a message would use a
// locale of the other copy and crash instead of raising.
std::string num(int64_t n) { return std::to_string(n); }

#define CHECK_SAME_DEVICE(a, b) \
  TORCH_CHECK((a).device() == (b).device(), #a " and " #b " must be on one device, got ", (a).device().str(), " and ", (b).device().str())

bool given(const c10::optional<at::Tensor>& t) { return t.has_value() && t->defined(); }

void check_rows_bf16(const at::Tensor& t, const char* what) {
  TORCH_CHECK(t.is_cuda() && t.scalar_type() == at::kBFloat16 && t.dim() == 2 && t.stride(1) == 1, what,
              " must be a 2-D CUDA bf16 tensor with unit inner stride");
}

void check_ids(const at::Tensor& ids, int64_t T, const char* what) {
  TORCH_CHECK(ids.is_cuda() && ids.scalar_type() == at::kLong && ids.is_contiguous() && ids.numel() == T, what,
              " must be contiguous CUDA int64, one per row");
}

int* check_rows_i32(const at::Tensor& t, int64_t n, const char* what) {
  TORCH_CHECK(t.is_cuda() && t.scalar_type() == at::kInt && t.is_contiguous() && t.numel() == n, what,
              " must be contiguous CUDA int32 of ", num(n), " entries");
  return t.data_ptr<int>();
}

float* check_rows_f32(const at::Tensor& t, int64_t n, const char* what) {
  TORCH_CHECK(t.is_cuda() && t.scalar_type() == at::kFloat && t.is_contiguous() && t.numel() == n, what,
              " must be contiguous CUDA fp32 of ", num(n), " entries");
  return t.data_ptr<float>();
}

// logprob_pack(h [T, H], ids [T]) -> (packed h, packed ids, perm, count)
std::vector<at::Tensor> logprob_pack(const at::Tensor& h, const at::Tensor& ids) {
  check_rows_bf16(h, "logprob: h");
  const int64_t T = h.size(0), H = h.size(1);
  TORCH_CHECK(T >= 1 && T <= kIntMax / 2, "logprob: row count");
  check_ids(ids, T, "logprob: ids");
  CHECK_SAME_DEVICE(h, ids);
  const c10::cuda::CUDAGuard g(h.device());
  const auto i32 = h.options().dtype(at::kInt);
  at::Tensor hp = at::empty({T, H}, h.options()), idp = at::empty({T}, ids.options());
  at::Tensor perm = at::empty({T}, i32), count = at::empty({1}, i32);
  pb::logprob_pack(h.data_ptr(), h.stride(0), ids.data_ptr<int64_t>(), (int)T, (int)H, hp.data_ptr(),
                   idp.data_ptr<int64_t>(), perm.data_ptr<int>(), count.data_ptr<int>(), cur_stream());
  return {hp, idp, perm, count};
}

// logprob_unpack(src [slices * T, H] (bf16, one slice, or fp32 slabs), perm [T], count, row0, dst [T_all, H] bf16):
// dst[perm[i]] = row i of src (its slices added) where packed row row0 + i has a token, else 0; own [T] (with fp32
// slabs, the rows' ids and the head w): own[i] w[ids[i]] is added to it
void logprob_unpack(const at::Tensor& src, const at::Tensor& perm, const at::Tensor& count, int64_t row0,
                    at::Tensor& dst, const at::Tensor& own = {}, const at::Tensor& ids = {},
                    const at::Tensor& w = {}) {
  const int64_t T = perm.numel(), H = dst.size(-1);
  const bool f32 = src.scalar_type() == at::kFloat;
  TORCH_CHECK(src.is_cuda() && src.is_contiguous() && (f32 || src.scalar_type() == at::kBFloat16) && src.dim() == 2 &&
                  src.size(1) == H && H % 8 == 0 && T >= 1 && src.size(0) % T == 0 && (f32 || src.size(0) == T),
              "logprob: packed rows must be contiguous bf16 [T, H] or fp32 slabs [slices * T, H]");
  TORCH_CHECK(dst.is_contiguous() && dst.scalar_type() == at::kBFloat16 && dst.dim() == 2 && dst.size(0) >= T,
              "logprob: contiguous bf16 rows to unpack to");
  CHECK_SAME_DEVICE(src, perm);
  CHECK_SAME_DEVICE(src, count);
  CHECK_SAME_DEVICE(src, dst);
  const float* op = nullptr;
  if (own.defined()) {
    op = check_rows_f32(own, T, "logprob: own");
    check_ids(ids, T, "logprob: ids");
    check_rows_bf16(w, "logprob: w");
    for (const at::Tensor* t : {&own, &ids, &w}) CHECK_SAME_DEVICE(src, *t);
    TORCH_CHECK(w.size(1) == H && w.stride(0) % 8 == 0 && (reinterpret_cast<uintptr_t>(w.data_ptr()) & 15) == 0,
                "logprob: w must have 16-byte rows of dst's width");
  }
  const c10::cuda::CUDAGuard g(src.device());
  pb::logprob_unpack(src.data_ptr(), f32, (int)(src.size(0) / T), check_rows_i32(perm, T, "logprob: perm"),
                     check_rows_i32(count, 1, "logprob: count"), (int)row0, (int)T, (int)H, op,
                     op ? ids.data_ptr<int64_t>() : nullptr, op ? w.data_ptr() : nullptr, op ? w.stride(0) : 0,
                     op ? (int)w.size(0) : 0, dst.data_ptr(), cur_stream());
}

// logprob_fwd(h [T, H], w [V, H], ids [T], inv_tau, logp [>= T], e [T, V] or None, perm [T] or None, count [1] or
// None, row0) -> (lse [T, 2], stats [T, groups, 2]); logp of row t goes to logp[perm[t]] (logp[t] without perm).  With
// count, h holds packed rows from row row0 on, of which the first count[0] have a token.
std::vector<at::Tensor> logprob_fwd(const at::Tensor& h, const at::Tensor& w, const at::Tensor& ids, double inv_tau,
                                    at::Tensor& logp, const c10::optional<at::Tensor>& e,
                                    const c10::optional<at::Tensor>& perm, const c10::optional<at::Tensor>& count,
                                    int64_t row0) {
  check_rows_bf16(h, "logprob: h");
  check_rows_bf16(w, "logprob: w");
  const int64_t T = h.size(0), H = h.size(1), V = w.size(0);
  TORCH_CHECK(w.size(1) == H, "logprob: h has ", num(H), " columns, w has ", num(w.size(1)));
  TORCH_CHECK(T >= 1 && V >= 1 && T <= kIntMax / 2 && V <= kIntMax / 2, "logprob: row and vocabulary counts");
  check_ids(ids, T, "logprob: ids");
  TORCH_CHECK(logp.is_cuda() && logp.scalar_type() == at::kFloat && logp.is_contiguous() && logp.numel() >= T,
              "logprob: logp must be contiguous CUDA fp32, at least one entry per row");
  CHECK_SAME_DEVICE(h, w);
  CHECK_SAME_DEVICE(h, ids);
  CHECK_SAME_DEVICE(h, logp);
  const c10::cuda::CUDAGuard g(h.device());
  pb::LogprobParams p{};
  p.groups = pb::logprob_groups((int)V);
  const auto f32 = h.options().dtype(at::kFloat);
  at::Tensor lse = at::empty({T, 2}, f32), stats = at::empty({T, p.groups.n(), 2}, f32);
  p.h = h.data_ptr();
  p.w = w.data_ptr();
  p.ids = ids.data_ptr<int64_t>();
  p.stats = stats.data_ptr<float>();
  p.logp = logp.data_ptr<float>();
  p.lse = lse.data_ptr<float>();
  p.ldh = h.stride(0);
  p.ldw = w.stride(0);
  if (given(e)) {
    check_rows_bf16(*e, "logprob: e");
    CHECK_SAME_DEVICE(h, *e);
    TORCH_CHECK(e->size(0) == T && e->size(1) == V && e->stride(0) >= (V + 7) / 8 * 8,
                "logprob: e must be [T, V] with room for whole 8-column groups in each row");
    p.e = e->data_ptr();
    p.lde = e->stride(0);
  }
  if (given(perm)) {
    CHECK_SAME_DEVICE(h, *perm);
    p.perm = check_rows_i32(*perm, T, "logprob: perm");
  }
  if (given(count)) {
    CHECK_SAME_DEVICE(h, *count);
    p.count = check_rows_i32(*count, 1, "logprob: count");
    p.row0 = (int)row0;
  }
  p.T = (int)T;
  p.V = (int)V;
  p.H = (int)H;
  p.inv_tau = (float)inv_tau;
  pb::logprob_fwd(p, cur_stream());
  return {lse, stats};
}

// logprob_bwd(e [T, V], stats, lse [T, 2], ids [T], perm [T], count [1], row0, logp, g, inv_tau, H) -> own [T]: e
// becomes the gradient of h w^T but for the targets', which is own; logp and g are in the caller's row order (row
// perm[t] for row t of e)
at::Tensor logprob_bwd(at::Tensor& e, const at::Tensor& stats, const at::Tensor& lse, const at::Tensor& ids,
                 const at::Tensor& perm, const at::Tensor& count, int64_t row0, const at::Tensor& logp,
                 const at::Tensor& g, double inv_tau, int64_t H) {
  check_rows_bf16(e, "logprob: e");
  const int64_t T = e.size(0), V = e.size(1);
  TORCH_CHECK(T >= 1 && V >= 1 && T <= kIntMax / 2 && V <= kIntMax / 2, "logprob: row and vocabulary counts");
  check_ids(ids, T, "logprob: ids");
  for (const at::Tensor* t : {&stats, &lse, &ids, &perm, &count, &logp, &g}) CHECK_SAME_DEVICE(e, *t);
  TORCH_CHECK(logp.numel() == g.numel() && g.numel() >= T, "logprob: logp and g must have one entry per row");
  const c10::cuda::CUDAGuard guard(e.device());
  const pb::LogprobGroups groups = pb::logprob_groups((int)V);
  check_rows_f32(stats, T * groups.n() * 2, "logprob: stats");
  TORCH_CHECK(e.stride(0) % 8 == 0 && e.stride(0) >= (V + 7) / 8 * 8 &&
                  (reinterpret_cast<uintptr_t>(e.data_ptr()) & 15) == 0,
              "logprob: e must have 16-byte rows with room for whole 8-column groups");
  at::Tensor own = at::empty({T}, lse.options());
  pb::logprob_bwd(e.data_ptr(), e.stride(0), stats.data_ptr<float>(), check_rows_f32(lse, T * 2, "logprob: lse"),
                  check_rows_f32(logp, logp.numel(), "logprob: logp"), ids.data_ptr<int64_t>(),
                  check_rows_i32(perm, T, "logprob: perm"), check_rows_i32(count, 1, "logprob: count"), (int)row0,
                  check_rows_f32(g, g.numel(), "logprob: g"), (float)inv_tau, (int)T, (int)V, (int)H,
                  own.data_ptr<float>(), groups, cur_stream());
  return own;
}

// ---------------------------------------------------------------- policy and preference losses
const float* check_tokens(const at::Tensor& t, int64_t B, int64_t S, const char* what) {
  TORCH_CHECK(t.is_cuda() && t.scalar_type() == at::kFloat && t.dim() == 2 && t.size(0) == B && t.size(1) == S &&
                  (t.stride(1) == 1 || S <= 1),
              what, " must be CUDA fp32 [", num(B), ", ", num(S), "] with unit inner stride");
  return t.data_ptr<float>();
}

const uint8_t* check_mask(const at::Tensor& t, int64_t B, int64_t S) {
  TORCH_CHECK(t.is_cuda() && t.scalar_type() == at::kBool && t.dim() == 2 && t.size(0) == B && t.size(1) == S &&
                  (t.stride(1) == 1 || S <= 1),
              "mask must be CUDA bool [", num(B), ", ", num(S), "] with unit inner stride");
  return reinterpret_cast<const uint8_t*>(t.data_ptr<bool>());
}

struct Chunks {
  int chunk, n;
};
Chunks chunks_of(int64_t rows, int64_t S) {
  TORCH_CHECK(rows <= kIntMax && S <= kIntMax, "token log-probabilities: at most 2^31 - 1 rows and columns");
  const int chunk = pb::objective_chunk(rows, S);
  const int64_t n = std::max<int64_t>(1, (S + chunk - 1) / chunk);
  TORCH_CHECK(rows * n <= kIntMax, "token log-probabilities: too many tokens for one call");
  return {chunk, (int)n};
}

// policy_fwd(logp, old, adv, mask, ref, low, high, kl_coef, per_sequence, want_grad) ->
// (loss, clip fraction, kl, coef or None, inv, inv_row or None)
std::vector<c10::optional<at::Tensor>> policy_fwd(const at::Tensor& logp, const at::Tensor& old, const at::Tensor& adv,
                                                  const c10::optional<at::Tensor>& mask,
                                                  const c10::optional<at::Tensor>& ref, double low, double high,
                                                  double kl_coef, bool per_sequence, bool want_grad) {
  TORCH_CHECK(logp.dim() == 2, "policy_fwd: logp [B, S]");
  const int64_t B = logp.size(0), S = logp.size(1);
  pb::PolicyParams p{};
  p.logp = check_tokens(logp, B, S, "policy_fwd: logp");
  p.old = check_tokens(old, B, S, "policy_fwd: old log-probabilities");
  TORCH_CHECK(adv.is_cuda() && adv.scalar_type() == at::kFloat && adv.dim() == 2 && adv.size(0) == B &&
                  (adv.size(1) == S || adv.size(1) == 1),
              "policy_fwd: advantages must be CUDA fp32 [B, S] (any strides) or [B, 1]");
  CHECK_SAME_DEVICE(logp, old);
  CHECK_SAME_DEVICE(logp, adv);
  p.adv = adv.data_ptr<float>();
  p.ld_logp = logp.stride(0);
  p.ld_old = old.stride(0);
  p.adv_sb = adv.stride(0);
  p.adv_ss = adv.size(1) == S ? adv.stride(1) : 0;
  if (given(mask)) {
    CHECK_SAME_DEVICE(logp, *mask);
    p.mask = check_mask(*mask, B, S);
    p.ld_mask = mask->stride(0);
  }
  if (given(ref)) {
    CHECK_SAME_DEVICE(logp, *ref);
    p.ref = check_tokens(*ref, B, S, "policy_fwd: reference log-probabilities");
    p.ld_ref = ref->stride(0);
  }
  const c10::cuda::CUDAGuard g(logp.device());
  const Chunks c = chunks_of(B, S);
  p.B = (int)B;
  p.S = (int)S;
  p.chunk = c.chunk;
  p.nchunk = c.n;
  p.low = low;
  p.high = high;
  p.kl_coef = kl_coef;
  p.per_sequence = per_sequence;
  const auto f32 = logp.options();
  at::Tensor loss = at::empty({}, f32), clip = at::empty({}, f32), kl = at::empty({}, f32);
  // scratch: a PolicyPart per chunk, then the ticket
  at::Tensor scratch = at::empty({B * c.n * 8 + 1}, f32);
  at::Tensor inv = at::empty({1}, f32);
  c10::optional<at::Tensor> coef, inv_row;
  if (want_grad) coef = at::empty({B, S}, f32);
  if (per_sequence) inv_row = at::empty({B}, f32);
  p.coef = want_grad ? coef->data_ptr<float>() : nullptr;
  p.inv_row = per_sequence ? inv_row->data_ptr<float>() : nullptr;
  p.inv = inv.data_ptr<float>();
  p.loss = loss.data_ptr<float>();
  p.clip = clip.data_ptr<float>();
  p.kl = kl.data_ptr<float>();
  static_assert(sizeof(pb::PolicyPart) == 32, "scratch of policy_fwd");
  p.parts = reinterpret_cast<pb::PolicyPart*>(scratch.data_ptr<float>());
  p.ticket = reinterpret_cast<int*>(scratch.data_ptr<float>() + B * c.n * 8);
  pb::policy_fwd(p, cur_stream());
  return {loss, clip, kl, coef, inv, inv_row};
}

// policy_bwd(coef [B, S], g scalar, inv, inv_row or None) -> d loss / d logp [B, S]
at::Tensor policy_bwd(const at::Tensor& coef, const at::Tensor& g, const at::Tensor& inv,
                      const c10::optional<at::Tensor>& inv_row) {
  TORCH_CHECK(coef.dim() == 2, "policy_bwd: coef [B, S]");
  const int64_t B = coef.size(0), S = coef.size(1);
  const float* cp = check_rows_f32(coef, B * S, "policy_bwd: coef");
  const float* rp = given(inv_row) ? check_rows_f32(*inv_row, B, "policy_bwd: inv_row") : nullptr;
  CHECK_SAME_DEVICE(coef, g);
  const c10::cuda::CUDAGuard guard(coef.device());
  at::Tensor out = at::empty_like(coef);
  const Chunks c = chunks_of(B, S);
  pb::policy_bwd(cp, check_rows_f32(g, 1, "policy_bwd: g"), check_rows_f32(inv, 1, "policy_bwd: inv"), rp,
                 out.data_ptr<float>(), (int)B, (int)S, c.chunk, c.n, cur_stream());
  return out;
}

// preference_fwd(logp [2P, S], ref, mask, beta, smoothing, average) -> (loss, rewards [2P], coef [2P])
std::vector<at::Tensor> preference_fwd(const at::Tensor& logp, const c10::optional<at::Tensor>& ref,
                                       const c10::optional<at::Tensor>& mask, double beta, double smoothing,
                                       bool average) {
  TORCH_CHECK(logp.dim() == 2 && logp.size(0) >= 2 && logp.size(0) % 2 == 0, "preference_fwd: logp [2P, S], P >= 1");
  const int64_t B = logp.size(0), S = logp.size(1);
  pb::PreferenceParams p{};
  p.logp = check_tokens(logp, B, S, "preference_fwd: logp");
  p.ld_logp = logp.stride(0);
  if (given(ref)) {
    CHECK_SAME_DEVICE(logp, *ref);
    p.ref = check_tokens(*ref, B, S, "preference_fwd: reference log-probabilities");
    p.ld_ref = ref->stride(0);
  }
  if (given(mask)) {
    CHECK_SAME_DEVICE(logp, *mask);
    p.mask = check_mask(*mask, B, S);
    p.ld_mask = mask->stride(0);
  }
  const c10::cuda::CUDAGuard g(logp.device());
  const Chunks c = chunks_of(B, S);
  p.P = (int)(B / 2);
  p.S = (int)S;
  p.chunk = c.chunk;
  p.nchunk = c.n;
  p.beta = beta;
  p.smoothing = smoothing;
  p.average = average;
  const auto f32 = logp.options();
  at::Tensor loss = at::empty({}, f32), rewards = at::empty({B}, f32), coef = at::empty({B}, f32);
  at::Tensor scratch = at::empty({B * c.n * 4 + 1}, f32);
  p.parts = reinterpret_cast<double2*>(scratch.data_ptr<float>());
  p.ticket = reinterpret_cast<int*>(scratch.data_ptr<float>() + B * c.n * 4);
  p.loss = loss.data_ptr<float>();
  p.rewards = rewards.data_ptr<float>();
  p.coef = coef.data_ptr<float>();
  pb::preference_fwd(p, cur_stream());
  return {loss, rewards, coef};
}

// preference_bwd(coef [2P], g scalar, mask or None, S) -> d loss / d logp [2P, S]
at::Tensor preference_bwd(const at::Tensor& coef, const at::Tensor& g, const c10::optional<at::Tensor>& mask,
                          int64_t S) {
  const int64_t B = coef.numel();
  const float* cp = check_rows_f32(coef, B, "preference_bwd: coef");
  const uint8_t* mp = nullptr;
  int64_t ldm = 0;
  if (given(mask)) {
    CHECK_SAME_DEVICE(coef, *mask);
    mp = check_mask(*mask, B, S);
    ldm = mask->stride(0);
  }
  CHECK_SAME_DEVICE(coef, g);
  const c10::cuda::CUDAGuard guard(coef.device());
  at::Tensor out = at::empty({B, S}, coef.options());
  const Chunks c = chunks_of(B, S);
  pb::preference_bwd(cp, check_rows_f32(g, 1, "preference_bwd: g"), mp, ldm, out.data_ptr<float>(), (int)B, (int)S,
                     c.chunk, c.n, cur_stream());
  return out;
}

// ---------------------------------------------------------------- distillation
// Scratch of a distillation, one allocation of 4-byte words: q and id [T, Kp]
// (Kp: K rounded up to 4), the row losses, the count of rows, their live bytes.
struct DistillScratch {
  int64_t T, Kp;
  explicit DistillScratch(int64_t t, int64_t k) : T(t), Kp((k + 3) / 4 * 4) {}
  int64_t words() const { return T * (2 * Kp + pb::kDistillMaxCluster) + 1 + (T + 3) / 4; }
  void fill(pb::DistillParams& p, const at::Tensor& t) const {
    float* base = t.data_ptr<float>();
    p.Kp = (int)Kp;
    p.T_all = (int)T;
    p.q = base;
    p.id = reinterpret_cast<int*>(base + T * Kp);
    p.row_loss = base + 2 * T * Kp;
    p.counters = reinterpret_cast<int*>(p.row_loss + T * pb::kDistillMaxCluster);
    p.live = reinterpret_cast<uint8_t*>(p.counters + 1);
  }
};

// distill_prep(top [T, K], ids [T, K], mask [T] or None, V, inv_tau) -> scratch
at::Tensor distill_prep(const at::Tensor& top, const at::Tensor& ids, const c10::optional<at::Tensor>& mask, int64_t V,
                        double inv_tau, int64_t* key = nullptr) {
  TORCH_CHECK(top.is_cuda() && (top.scalar_type() == at::kBFloat16 || top.scalar_type() == at::kFloat) &&
                  top.dim() == 2 && (top.stride(1) == 1 || top.size(1) <= 1),
              "distill: teacher logits must be CUDA bf16 or fp32 [T, K] with unit inner stride");
  const int64_t T = top.size(0), K = top.size(1);
  TORCH_CHECK(ids.is_cuda() && (ids.scalar_type() == at::kLong || ids.scalar_type() == at::kInt) && ids.dim() == 2 &&
                  ids.size(0) == T && ids.size(1) == K && (ids.stride(1) == 1 || K <= 1),
              "distill: teacher ids must be CUDA int32 or int64, shaped as the teacher's logits, unit inner stride");
  TORCH_CHECK(K >= 1 && K <= pb::kDistillMaxK, "distill: 1 to ", num(pb::kDistillMaxK), " teacher entries a row");
  TORCH_CHECK(T <= kIntMax / 16 && V >= 1 && V <= kIntMax, "distill: row and vocabulary counts");
  CHECK_SAME_DEVICE(top, ids);
  pb::DistillParams p{};
  if (given(mask)) {
    TORCH_CHECK(mask->is_cuda() && mask->scalar_type() == at::kBool && mask->dim() == 1 && mask->numel() == T,
                "distill: mask must be CUDA bool [T]");
    CHECK_SAME_DEVICE(top, *mask);
    p.mask = reinterpret_cast<const uint8_t*>(mask->data_ptr<bool>());
    p.ld_mask = mask->stride(0);
  }
  const c10::cuda::CUDAGuard g(top.device());
  const auto f32 = top.options().dtype(at::kFloat);
  const DistillScratch sc(T, K);
  at::Tensor scratch = at::empty({sc.words()}, f32);
  sc.fill(p, scratch);
  p.top = top.data_ptr();
  p.ids = ids.data_ptr();
  p.ld_top = top.stride(0);
  p.ld_ids = ids.stride(0);
  p.top_bf16 = top.scalar_type() == at::kBFloat16;
  p.ids32 = ids.scalar_type() == at::kInt;
  p.T = (int)T;
  p.V = (int)V;
  p.K = (int)K;
  p.inv_tau = (float)inv_tau;
  p.key = key;
  pb::distill_prep(p, cur_stream());
  return scratch;
}

// Whether two [T, V] tensors of one type are misaligned by the same number of bytes in every row.
bool same_alignment(const at::Tensor& a, const at::Tensor& b) {
  auto off = [](const at::Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) & 15; };
  return (a.size(1) <= 1 || (a.stride(1) == 1 && b.stride(1) == 1)) && off(a) == off(b) &&
         (a.size(0) <= 1 || (a.stride(0) - b.stride(0)) * a.element_size() % 16 == 0);
}

// distill_rows(logits [T, V], scratch (distill_prep's of all T_all rows), T_all, K, row0, tau, grad [T, V] or None): the
// losses of rows [row0, row0 + T) and, with grad (may be logits itself), the gradient of the loss; with perm,
// row i of the logits is row perm[i] of the teacher's; with weight (a scalar), the gradient alone, times it, if it
// is not 1
void distill_rows(const at::Tensor& logits, const at::Tensor& scratch, int64_t T_all, int64_t K, int64_t row0, double tau,
                  const c10::optional<at::Tensor>& grad, const int* perm = nullptr,
                  const c10::optional<at::Tensor>& weight = c10::nullopt) {
  TORCH_CHECK(logits.is_cuda() && (logits.scalar_type() == at::kBFloat16 || logits.scalar_type() == at::kFloat) &&
                  logits.dim() == 2 && (logits.stride(1) == 1 || logits.size(1) <= 1),
              "distill: logits must be CUDA bf16 or fp32 [T, V] with unit inner stride");
  const bool bf16 = logits.scalar_type() == at::kBFloat16;
  const int64_t T = logits.size(0), V = logits.size(1);
  TORCH_CHECK(V >= 1 && V <= kIntMax, "distill: vocabulary");
  TORCH_CHECK(row0 >= 0 && row0 + T <= T_all, "distill: rows outside the teacher's");
  const DistillScratch sc(T_all, K);
  TORCH_CHECK(K >= 1 && K <= pb::kDistillMaxK, "distill: 1 to ", num(pb::kDistillMaxK), " teacher entries a row");
  CHECK_SAME_DEVICE(logits, scratch);
  check_rows_f32(scratch, sc.words(), "distill: scratch");
  if (T == 0) return;
  pb::DistillParams p{};
  sc.fill(p, scratch);
  if (given(weight)) {
    CHECK_SAME_DEVICE(logits, *weight);
    p.weight = check_rows_f32(*weight, 1, "distill: weight");
  }
  p.logits = logits.data_ptr();
  p.ld = logits.stride(0);
  if (given(grad)) {
    TORCH_CHECK(grad->scalar_type() == logits.scalar_type() && grad->sizes() == logits.sizes() &&
                    same_alignment(logits, *grad),
                "distill: grad must have logits' type, shape and alignment");
    CHECK_SAME_DEVICE(logits, *grad);
    p.grad = grad->data_ptr();
    p.ld_grad = grad->stride(0);
  }
  const c10::cuda::CUDAGuard g(logits.device());
  p.T = (int)T;
  p.V = (int)V;
  p.K = (int)K;
  p.row0 = row0;
  p.perm = perm;
  p.tau = (float)tau;
  p.inv_tau = (float)(1.0 / tau);
  pb::distill_rows(p, bf16, cur_stream());
}

// distill_loss(scratch (all rows of all blocks seen by distill_rows), T_all, K, V, bf16 logits) -> loss
at::Tensor distill_loss(const at::Tensor& scratch, int64_t T_all, int64_t K, int64_t V, bool bf16) {
  if (T_all == 0) return at::zeros({}, scratch.options());
  const c10::cuda::CUDAGuard g(scratch.device());
  at::Tensor loss = at::empty({}, scratch.options());
  pb::DistillParams p{};
  DistillScratch(T_all, K).fill(p, scratch);
  p.V = (int)V;
  p.loss = loss.data_ptr<float>();
  pb::distill_loss(p, bf16, cur_stream());
  return loss;
}

// grad_like(logits [T, V]) -> grad [T, V]: a tensor that is misaligned as logits is in every row, so that both are read
// and written in the same 16-byte vectors
at::Tensor grad_like(const at::Tensor& logits) {
  TORCH_CHECK(logits.is_cuda() && logits.dim() == 2, "grad_like: CUDA [T, V]");
  const c10::cuda::CUDAGuard g(logits.device());
  const int64_t T = logits.size(0), V = logits.size(1), unit = 16 / logits.element_size();
  const int64_t shift = (int64_t)(reinterpret_cast<uintptr_t>(logits.data_ptr()) & 15) / logits.element_size();
  const int64_t ld = V + ((logits.stride(0) - V) % unit + unit) % unit;
  return at::empty({shift + T * ld}, logits.options()).as_strided({T, V}, {ld, 1}, shift);
}

// ---------------------------------------------------------------- differentiable entry points
// The losses are calls of a few microseconds on the GPU, so their autograd
// nodes live here: a Python node costs 30 to 40 us a step in calls back into
// the interpreter (8 x 509 tokens, forward and backward: 97 us).
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

bool wants_grad(const at::Tensor& t) { return at::GradMode::is_enabled() && t.requires_grad(); }

// A dual tensor without requires_grad would pass the nodes by and lose its tangent.
void check_no_tangent(const at::Tensor& t, const char* what) {
  TORCH_CHECK(!t._fw_grad(/*level=*/0).defined(), what, ": forward-mode derivatives are not implemented");
}

// What takes no gradient takes no tangent either.
at::Tensor constant(const at::Tensor& t) { return t._fw_grad(/*level=*/0).defined() ? t.detach() : t; }
c10::optional<at::Tensor> constant(const c10::optional<at::Tensor>& t) {
  return given(t) ? c10::optional<at::Tensor>(constant(*t)) : c10::nullopt;
}

at::Tensor or_undefined(const c10::optional<at::Tensor>& t) { return given(t) ? *t : at::Tensor(); }
c10::optional<at::Tensor> or_none(const at::Tensor& t) {
  return t.defined() ? c10::optional<at::Tensor>(t) : c10::nullopt;
}

// The gradients are computed outside autograd: they cannot be differentiated again.
void check_first_order(const char* what) {
  TORCH_CHECK(!at::GradMode::is_enabled(), what, ": the gradient is not differentiable (create_graph)");
}

// Rows of a [rows, V] 16-bit block of at most max_bytes: whole 256-row tiles, one at least.
int64_t block_rows(int64_t T, int64_t V, int64_t max_bytes) {
  return std::max<int64_t>(1, std::min(T, std::max<int64_t>(256, max_bytes / (V * 2) / 256 * 256)));
}

at::Tensor rows_of(const at::Tensor& t, int64_t r0, int64_t n) { return r0 == 0 && n == t.size(0) ? t : t.narrow(0, r0, n); }

// K slices of dl @ w over the vocabulary.  A few rows make few output tiles with
// a long sum: slices spread them over the SM pairs, each into an fp32 slab that
// the unpacking adds in slice order.  The cheapest count by a wave model:
// ceil(tiles s / pairs) / s of a tile's time at 22 TFLOP/s a pair, and the
// slabs' round trip at 5 TB/s (8192 x 1024 over 151936: 1753 us in one slice,
// 1472 + 24 in 4; 333 x 4096: 860 -> 406 + 22).
int grad_rows_slices(int64_t T, int64_t H, int64_t V) {
  const int64_t pairs = std::max(1, pb::num_sms() / 2);
  const int64_t tiles = ((T + 255) / 256) * ((H + 255) / 256);
  const double t_tile = 2.0 * 256 * 256 * (double)V / 22e12;
  auto cost = [&](int64_t s) {
    return (double)((tiles * s + pairs - 1) / pairs) / s * t_tile + (s == 1 ? 0.0 : 2.0 * s * T * H * 4 / 5e12);
  };
  int best = 1;
  for (int s = 2; s <= 16 && V / s >= 1024; ++s)  // at least 16 steps of 64 a slice: none is empty
    if (cost(s) < 0.97 * cost(best)) best = s;
  return best;
}

// dl [T, V] @ w [V, H] (times factor[0]) for the rows that count: bf16 [T, H], or (several slices, or f32) fp32 slabs
// [slices * T, H]
at::Tensor grad_rows(const at::Tensor& dl, const at::Tensor& w, const at::Tensor& count, int64_t row0, bool f32,
                     const float* factor = nullptr) {
  const int64_t T = dl.size(0), V = w.size(0), H = w.size(1);
  const int slices = grad_rows_slices(T, H, V);
  at::Tensor out = at::empty({slices * T, H}, dl.options().dtype(slices == 1 && !f32 ? at::kBFloat16 : at::kFloat));
  pb::GemmParams p{};
  p.A = dl.data_ptr();
  p.B = w.data_ptr();
  p.C = out.data_ptr();
  p.lda = dl.stride(0);
  p.ldb = w.stride(0);
  p.ldc = H;
  p.M = (int)T;
  p.N = (int)H;
  p.K = (int)V;
  p.b_mn = true;
  p.alpha = 1.f;
  p.epi = slices == 1 && !f32 ? pb::kEpiStoreBf16 : pb::kEpiStoreF32;
  p.splits = slices;
  p.alpha_dev = factor;
  p.live = count.data_ptr<int>();
  p.live_row0 = (int)row0;
  pb::gemm_bf16(p, cur_stream());
  return out;
}

// out (+)= dl^T h (times factor[0]) over the rows that count; out bf16, or fp32 where several row blocks add up
void grad_head(const at::Tensor& dl, const at::Tensor& h, at::Tensor& out, bool accumulate, const at::Tensor& count,
               int64_t row0, const float* factor = nullptr) {
  pb::GemmParams p{};
  p.A = dl.data_ptr();
  p.B = h.data_ptr();
  p.C = out.data_ptr();
  p.lda = dl.stride(0);
  p.ldb = h.stride(0);
  p.ldc = out.stride(0);
  p.M = (int)out.size(0);
  p.N = (int)out.size(1);
  p.K = (int)dl.size(0);
  p.a_mn = p.b_mn = true;
  p.alpha = 1.f;
  p.epi = out.scalar_type() == at::kBFloat16 ? pb::kEpiStoreBf16 : accumulate ? pb::kEpiAccumF32 : pb::kEpiStoreF32;
  p.live = count.data_ptr<int>();
  p.live_row0 = (int)row0;
  p.live_k = true;
  p.alpha_dev = factor;
  pb::gemm_bf16(p, cur_stream());
}

// The forward keeps 16-bit exponentials of the logits (not the logits) for at
// most max_block_bytes; the backward scales them in place into the logits'
// gradient and multiplies it with the head and the hidden states.  Rows beyond
// that are scored without storing and run through the forward kernel again in
// the backward, block by block.  All of it works on packed rows: those with a
// token in front, zeros behind.
struct LogProbsNode : public torch::autograd::Function<LogProbsNode> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& h, const at::Tensor& w, const at::Tensor& ids,
                            double inv_tau, int64_t max_block_bytes) {
    const c10::cuda::CUDAGuard guard(h.device());
    const int64_t T = h.size(0), V = w.size(0);
    const auto packed = logprob_pack(h, ids);  // rows, ids, perm, count
    at::Tensor logp = at::empty({T}, h.options().dtype(at::kFloat));
    const int64_t block = block_rows(T, V, max_block_bytes);
    std::vector<at::Tensor> kept{at::empty({block, (V + 63) / 64 * 64}, h.options()).narrow(1, 0, V)};
    for (int64_t r0 = 0; r0 < T; r0 += block) {
      const int64_t n = std::min(block, T - r0);
      const auto out = logprob_fwd(rows_of(packed[0], r0, n), w, rows_of(packed[1], r0, n), inv_tau, logp,
                                   r0 == 0 ? c10::optional<at::Tensor>(kept[0]) : c10::nullopt,
                                   rows_of(packed[2], r0, n), packed[3], r0);
      if (r0 == 0) kept.push_back(out[1]);
      kept.push_back(out[0]);
    }
    // not save_for_backward: the backward overwrites the exponentials
    ctx->saved_data["kept"] = kept;
    ctx->save_for_backward({packed[0], w, packed[1], packed[2], packed[3], logp});
    ctx->saved_data["inv_tau"] = inv_tau;
    ctx->saved_data["block"] = block;
    return logp;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    check_first_order("lm_head_log_probs");
    TORCH_CHECK(ctx->saved_data.count("kept"), "lm_head_log_probs supports one backward pass per forward");
    const auto saved = ctx->get_saved_variables();
    const at::Tensor &hp = saved[0], &w = saved[1], &idp = saved[2], &perm = saved[3], &count = saved[4],
                     &logp = saved[5];
    std::vector<at::Tensor> kept = ctx->saved_data["kept"].toTensorVector();
    ctx->saved_data.erase("kept");
    const double inv_tau = ctx->saved_data["inv_tau"].toDouble();
    const int64_t block = ctx->saved_data["block"].toInt(), T = hp.size(0), V = w.size(0), H = w.size(1);
    const c10::cuda::CUDAGuard guard(hp.device());
    const at::Tensor g = grads[0].contiguous();
    at::Tensor dh, dw;
    if (ctx->needs_input_grad(0)) dh = at::empty({T, H}, hp.options());
    // one row block: the head's gradient is rounded by its product, and the rows of targets again with the target's
    // part (an fp32 product would be twice the stores, and one more pass); several blocks add up in fp32 first
    if (ctx->needs_input_grad(1)) dw = at::empty({V, H}, block >= T ? w.options() : w.options().dtype(at::kFloat));
    at::Tensor e = kept[0], stats = kept[1];
    for (int64_t r0 = 0, i = 2; r0 < T; r0 += block, ++i) {
      const int64_t n = std::min(block, T - r0);
      const at::Tensor rows = rows_of(hp, r0, n), ids = rows_of(idp, r0, n), pm = rows_of(perm, r0, n);
      if (r0) {
        e = rows_of(e, 0, n);
        at::Tensor again = at::empty_like(logp);  // the forward's logp stands
        stats = logprob_fwd(rows, w, ids, inv_tau, again, e, pm, count, r0)[1];
      }
      const at::Tensor own = logprob_bwd(e, stats, kept[i], ids, pm, count, r0, logp, g, inv_tau, H);
      if (dh.defined()) logprob_unpack(grad_rows(e, w, count, r0, true), pm, count, r0, dh, own, ids, w);
      if (dw.defined()) {
        grad_head(e, rows, dw, r0 > 0, count, r0);
        pb::logprob_own(rows.data_ptr(), ids.data_ptr<int64_t>(), own.data_ptr<float>(), count.data_ptr<int>(), (int)r0,
                        (int)n, (int)V, (int)H, dw.data_ptr(), dw.scalar_type() == at::kFloat, cur_stream());
      }
    }
    return {dh, dw.defined() ? dw.to(w.scalar_type()) : dw, at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

// Scoring packs the rows from this many on: below, packing (5 us) would save a part of one to three row tiles.
constexpr int64_t kPackRows = 768;

at::Tensor lm_head_log_probs(const at::Tensor& h, const at::Tensor& w, const at::Tensor& ids, double inv_tau,
                             int64_t max_block_bytes) {
  check_rows_bf16(h, "lm_head_log_probs: h");
  check_rows_bf16(w, "lm_head_log_probs: w");
  check_no_tangent(h, "lm_head_log_probs");
  check_no_tangent(w, "lm_head_log_probs");
  TORCH_CHECK(w.size(0) >= 1, "lm_head_log_probs: an empty vocabulary");
  if (wants_grad(h) || wants_grad(w)) return LogProbsNode::apply(h, w, ids, inv_tau, max_block_bytes);
  const c10::cuda::CUDAGuard guard(h.device());
  at::Tensor logp = at::empty({h.size(0)}, h.options().dtype(at::kFloat));
  if (h.size(0) >= kPackRows) {
    const auto packed = logprob_pack(h, ids);
    logprob_fwd(packed[0], w, packed[1], inv_tau, logp, c10::nullopt, packed[2], packed[3], 0);
  } else {
    logprob_fwd(h, w, ids, inv_tau, logp, c10::nullopt, c10::nullopt, c10::nullopt, 0);
  }
  return logp;
}

struct PolicyLossNode : public torch::autograd::Function<PolicyLossNode> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& logp, const at::Tensor& old,
                               const at::Tensor& adv, const c10::optional<at::Tensor>& mask,
                               const c10::optional<at::Tensor>& ref, double low, double high, double kl_coef,
                               bool per_sequence) {
    auto out = policy_fwd(logp, old, adv, mask, ref, low, high, kl_coef, per_sequence, true);
    ctx->save_for_backward({*out[3], *out[4], or_undefined(out[5])});
    ctx->mark_non_differentiable({*out[1], *out[2]});
    ctx->set_materialize_grads(false);
    return {*out[0], *out[1], *out[2]};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    check_first_order("policy_loss");
    const auto saved = ctx->get_saved_variables();
    variable_list grads(9);  // to logp alone
    if (g[0].defined()) grads[0] = policy_bwd(saved[0], g[0], saved[1], or_none(saved[2]));
    return grads;
  }
};

std::vector<at::Tensor> policy_loss(const at::Tensor& logp, const at::Tensor& old, const at::Tensor& adv,
                                    const c10::optional<at::Tensor>& mask, const c10::optional<at::Tensor>& ref,
                                    double low, double high, double kl_coef, bool per_sequence) {
  check_no_tangent(logp, "policy_loss");
  if (!wants_grad(logp)) {
    const auto out = policy_fwd(logp, old, adv, mask, ref, low, high, kl_coef, per_sequence, false);
    return {*out[0], *out[1], *out[2]};
  }
  return PolicyLossNode::apply(logp, constant(old), constant(adv), mask, constant(ref), low, high, kl_coef, per_sequence);
}

struct PreferenceLossNode : public torch::autograd::Function<PreferenceLossNode> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& logp, const c10::optional<at::Tensor>& ref,
                               const c10::optional<at::Tensor>& mask, double beta, double smoothing, bool average) {
    auto out = preference_fwd(logp, ref, mask, beta, smoothing, average);
    ctx->save_for_backward({out[2], or_undefined(mask)});
    ctx->saved_data["S"] = logp.size(1);
    ctx->mark_non_differentiable({out[1]});
    ctx->set_materialize_grads(false);
    return {out[0], out[1]};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    check_first_order("preference_loss");
    const auto saved = ctx->get_saved_variables();
    variable_list grads(6);
    if (g[0].defined()) grads[0] = preference_bwd(saved[0], g[0], or_none(saved[1]), ctx->saved_data["S"].toInt());
    return grads;
  }
};

std::vector<at::Tensor> preference_loss(const at::Tensor& logp, const c10::optional<at::Tensor>& ref,
                                        const c10::optional<at::Tensor>& mask, double beta, double smoothing,
                                        bool average) {
  check_no_tangent(logp, "preference_loss");
  if (!wants_grad(logp)) {
    const auto out = preference_fwd(logp, ref, mask, beta, smoothing, average);
    return {out[0], out[1]};
  }
  return PreferenceLossNode::apply(logp, constant(ref), mask, beta, smoothing, average);
}

// The gradient is written in the forward pass, from the one read of the
// logits; the backward writes it again if it comes with another weight than 1.
struct DistillationNode : public torch::autograd::Function<DistillationNode> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& logits, const at::Tensor& top,
                            const at::Tensor& ids, const c10::optional<at::Tensor>& mask, double tau) {
    const at::Tensor scratch = distill_prep(top, ids, mask, logits.size(1), 1.0 / tau), grad = grad_like(logits);
    distill_rows(logits, scratch, top.size(0), top.size(1), 0, tau, grad);
    // not save_for_backward: the backward hands the gradient out, it does not keep it
    ctx->saved_data["grad"] = grad;
    ctx->saved_data["scratch"] = scratch;
    ctx->saved_data["K"] = top.size(1);
    ctx->saved_data["tau"] = tau;
    ctx->save_for_backward({logits});
    return distill_loss(scratch, top.size(0), top.size(1), logits.size(1), logits.scalar_type() == at::kBFloat16);
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    check_first_order("distillation_loss");
    TORCH_CHECK(ctx->saved_data.count("grad"), "distillation_loss supports one backward pass per forward");
    at::Tensor logits = ctx->get_saved_variables()[0];
    const at::Tensor grad = ctx->saved_data["grad"].toTensor();
    ctx->saved_data.erase("grad");
    if (!same_alignment(logits, grad)) logits = grad_like(grad).copy_(logits);  // saved-tensor hooks may lay it out anew
    distill_rows(logits, ctx->saved_data["scratch"].toTensor(), logits.size(0), ctx->saved_data["K"].toInt(), 0,
                 ctx->saved_data["tau"].toDouble(), grad, nullptr, g[0]);
    variable_list grads(5);
    grads[0] = grad;
    return grads;
  }
};

at::Tensor distillation_loss(const at::Tensor& logits, const at::Tensor& top, const at::Tensor& ids,
                             const c10::optional<at::Tensor>& mask, double tau) {
  check_no_tangent(logits, "distillation_loss");
  if (!wants_grad(logits)) {
    const at::Tensor scratch = distill_prep(top, ids, mask, logits.size(1), 1.0 / tau);
    distill_rows(logits, scratch, top.size(0), top.size(1), 0, tau, c10::nullopt);
    return distill_loss(scratch, top.size(0), top.size(1), logits.size(1), logits.scalar_type() == at::kBFloat16);
  }
  return DistillationNode::apply(logits, top, ids, mask, tau);
}

// Distillation through the LM head: blocks of bf16 logits of the packed rows
// (those that count in front, zeros behind, as in LogProbsNode), overwritten by
// their gradient, which the backward's two products turn into those of h and w,
// times the incoming gradient before they are rounded.  The first block's logit
// gradient is kept for it (at most max_block_bytes); the logits of rows beyond are
// computed again.  bf16 logits are what the model's own head returns and what its
// cross-entropy works on (up to |logit| / 512 of a logit is lost); fp32 ones would
// take twice the memory and could not become the products' operand in place.
struct HeadDistillationNode : public torch::autograd::Function<HeadDistillationNode> {
  // logits of packed rows [r0, r0 + n) in buf's first n rows
  static at::Tensor block_logits(const at::Tensor& buf, const at::Tensor& rows, const at::Tensor& w,
                                 const at::Tensor& count, int64_t r0) {
    const at::Tensor logits = rows_of(buf, 0, rows.size(0));
    pb::GemmParams p{};
    p.A = rows.data_ptr();
    p.B = w.data_ptr();
    p.C = logits.data_ptr();
    p.lda = rows.stride(0);
    p.ldb = w.stride(0);
    p.ldc = buf.stride(0);
    p.M = (int)rows.size(0);
    p.N = (int)w.size(0);
    p.K = (int)w.size(1);
    p.alpha = 1.f;
    p.epi = pb::kEpiStoreBf16;
    p.live = count.data_ptr<int>();
    p.live_row0 = (int)r0;
    pb::gemm_bf16(p, cur_stream());
    return logits;
  }
  static at::Tensor run(AutogradContext* ctx, const at::Tensor& h, const at::Tensor& w, const at::Tensor& top,
                        const at::Tensor& ids, const c10::optional<at::Tensor>& mask, double tau, int64_t max_block_bytes) {
    const c10::cuda::CUDAGuard guard(h.device());
    const int64_t T = h.size(0), V = w.size(0), H = w.size(1), K = top.size(1);
    TORCH_CHECK(H == h.size(1) && top.size(0) == T, "lm_head_distillation: shapes");
    CHECK_SAME_DEVICE(h, w);
    CHECK_SAME_DEVICE(h, top);
    at::Tensor key = at::empty({T}, h.options().dtype(at::kLong));
    const at::Tensor scratch = distill_prep(top, ids, mask, V, 1.0 / tau, key.data_ptr<int64_t>());
    const auto packed = logprob_pack(h, key);  // rows, keys, perm, count
    const at::Tensor &hp = packed[0], &perm = packed[2], &count = packed[3];
    const int64_t block = block_rows(T, V, max_block_bytes);
    const at::Tensor buf = at::empty({block, (V + 63) / 64 * 64}, h.options()).narrow(1, 0, V);
    for (int64_t r0 = (T - 1) / block * block; r0 >= 0; r0 -= block) {  // the first block last: it stays
      const at::Tensor logits = block_logits(buf, rows_of(hp, r0, std::min(block, T - r0)), w, count, r0);
      distill_rows(logits, scratch, T, K, r0, tau, ctx && r0 == 0 ? c10::optional<at::Tensor>(logits) : c10::nullopt,
                   perm.data_ptr<int>());
    }
    if (ctx) {
      ctx->save_for_backward({hp, w, perm, count});
      ctx->saved_data["kept"] = std::vector<at::Tensor>{buf, scratch};
      ctx->saved_data["K"] = K;
      ctx->saved_data["tau"] = tau;
    }
    return distill_loss(scratch, T, K, V, true);
  }
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& h, const at::Tensor& w, const at::Tensor& top,
                            const at::Tensor& ids, const c10::optional<at::Tensor>& mask, double tau,
                            int64_t max_block_bytes) {
    return run(ctx, h, w, top, ids, mask, tau, max_block_bytes);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    check_first_order("lm_head_distillation");
    TORCH_CHECK(ctx->saved_data.count("kept"), "lm_head_distillation supports one backward pass per forward");
    const auto saved = ctx->get_saved_variables();
    const at::Tensor &hp = saved[0], &w = saved[1], &perm = saved[2], &count = saved[3];
    const std::vector<at::Tensor> kept = ctx->saved_data["kept"].toTensorVector();
    ctx->saved_data.erase("kept");
    const at::Tensor &buf = kept[0], &scratch = kept[1];
    const double tau = ctx->saved_data["tau"].toDouble();
    const int64_t K = ctx->saved_data["K"].toInt(), block = buf.size(0), T = hp.size(0), V = w.size(0), H = w.size(1);
    const c10::cuda::CUDAGuard guard(hp.device());
    CHECK_SAME_DEVICE(hp, grads[0]);
    const float* factor = check_rows_f32(grads[0], 1, "lm_head_distillation: gradient");
    at::Tensor dh, dw;
    if (ctx->needs_input_grad(0)) dh = at::empty({T, H}, hp.options());
    if (ctx->needs_input_grad(1)) dw = at::empty({V, H}, block >= T ? w.options() : w.options().dtype(at::kFloat));
    for (int64_t r0 = 0; r0 < T; r0 += block) {
      const int64_t n = std::min(block, T - r0);
      const at::Tensor rows = rows_of(hp, r0, n), dl = r0 ? block_logits(buf, rows, w, count, r0) : buf;
      if (r0) distill_rows(dl, scratch, T, K, r0, tau, dl, perm.data_ptr<int>());
      if (dh.defined()) logprob_unpack(grad_rows(dl, w, count, r0, false, factor), rows_of(perm, r0, n), count, r0, dh);
      if (dw.defined()) grad_head(dl, rows, dw, r0 > 0, count, r0, factor);
    }
    variable_list out(7);
    out[0] = dh;
    if (dw.defined()) out[1] = dw.to(w.scalar_type());
    return out;
  }
};

at::Tensor lm_head_distillation(const at::Tensor& h, const at::Tensor& w, const at::Tensor& top, const at::Tensor& ids,
                                const c10::optional<at::Tensor>& mask, double tau, int64_t max_block_bytes) {
  check_rows_bf16(h, "lm_head_distillation: h");
  check_rows_bf16(w, "lm_head_distillation: w");
  check_no_tangent(h, "lm_head_distillation");
  check_no_tangent(w, "lm_head_distillation");
  if (wants_grad(h) || wants_grad(w)) return HeadDistillationNode::apply(h, w, top, ids, mask, tau, max_block_bytes);
  return HeadDistillationNode::run(nullptr, h, w, top, ids, mask, tau, max_block_bytes);
}

}  // namespace

void register_objectives(pybind11::module& m) {
  namespace py = pybind11;
  m.def("lm_head_log_probs", &lm_head_log_probs, py::arg("h"), py::arg("w"), py::arg("ids"), py::arg("inv_tau"),
        py::arg("max_block_bytes"));
  m.def("policy_loss", &policy_loss, py::arg("logp"), py::arg("old"), py::arg("adv"), py::arg("mask"), py::arg("ref"),
        py::arg("low"), py::arg("high"), py::arg("kl_coef"), py::arg("per_sequence"));
  m.def("preference_loss", &preference_loss, py::arg("logp"), py::arg("ref"), py::arg("mask"), py::arg("beta"),
        py::arg("smoothing"), py::arg("average"));
  m.def("distillation_loss", &distillation_loss, py::arg("logits"), py::arg("top"), py::arg("ids"), py::arg("mask"),
        py::arg("tau"));
  m.def("lm_head_distillation", &lm_head_distillation, py::arg("h"), py::arg("w"), py::arg("top"), py::arg("ids"),
        py::arg("mask"), py::arg("tau"), py::arg("max_block_bytes"));
}
