// Bindings of the post-training objectives (objectives.cuh).
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <limits>
#include <vector>

#include "objectives.cuh"

namespace {

cudaStream_t cur_stream() { return at::cuda::getCurrentCUDAStream().stream(); }

constexpr int64_t kIntMax = std::numeric_limits<int>::max();

#define CHECK_SAME_DEVICE(a, b) \
  TORCH_CHECK((a).device() == (b).device(), #a " and " #b " must be on one device, got ", (a).device(), " and ", (b).device())

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
              " must be contiguous CUDA int32 of ", n, " entries");
  return t.data_ptr<int>();
}

float* check_rows_f32(const at::Tensor& t, int64_t n, const char* what) {
  TORCH_CHECK(t.is_cuda() && t.scalar_type() == at::kFloat && t.is_contiguous() && t.numel() == n, what,
              " must be contiguous CUDA fp32 of ", n, " entries");
  return t.data_ptr<float>();
}

// logprob_pack(h [T, H], ids [T]) -> (packed h, packed ids, perm, pos, count)
std::vector<at::Tensor> logprob_pack(const at::Tensor& h, const at::Tensor& ids) {
  check_rows_bf16(h, "logprob: h");
  const int64_t T = h.size(0), H = h.size(1);
  TORCH_CHECK(T >= 1 && T <= kIntMax / 2, "logprob: row count");
  check_ids(ids, T, "logprob: ids");
  CHECK_SAME_DEVICE(h, ids);
  const c10::cuda::CUDAGuard g(h.device());
  const auto i32 = h.options().dtype(at::kInt);
  at::Tensor hp = at::empty({T, H}, h.options()), idp = at::empty({T}, ids.options());
  at::Tensor perm = at::empty({T}, i32), pos = at::empty({T}, i32), count = at::empty({1}, i32);
  pb::logprob_pack(h.data_ptr(), h.stride(0), ids.data_ptr<int64_t>(), (int)T, (int)H, hp.data_ptr(),
                   idp.data_ptr<int64_t>(), perm.data_ptr<int>(), pos.data_ptr<int>(), count.data_ptr<int>(),
                   cur_stream());
  return {hp, idp, perm, pos, count};
}

// logprob_unpack(src [T, H], pos, count) -> dst [T, H]
at::Tensor logprob_unpack(const at::Tensor& src, const at::Tensor& pos, const at::Tensor& count) {
  check_rows_bf16(src, "logprob: packed rows");
  TORCH_CHECK(src.is_contiguous() && src.size(1) % 8 == 0, "logprob: packed rows must be contiguous");
  const int64_t T = src.size(0);
  CHECK_SAME_DEVICE(src, pos);
  CHECK_SAME_DEVICE(src, count);
  const c10::cuda::CUDAGuard g(src.device());
  at::Tensor dst = at::empty_like(src);
  pb::logprob_unpack(src.data_ptr(), check_rows_i32(pos, T, "logprob: pos"),
                     check_rows_i32(count, 1, "logprob: count"), (int)T, (int)src.size(1), dst.data_ptr(),
                     cur_stream());
  return dst;
}

// logprob_fwd(h [T, H], w [V, H], ids [T], inv_tau, logp [>= T], e [T, V] or None, perm [T] or None) ->
// (lse2 [T], stats [T, tiles, 2], tile width); logp of row t goes to logp[perm[t]] (logp[t] without perm)
std::tuple<at::Tensor, at::Tensor, int64_t> logprob_fwd(const at::Tensor& h, const at::Tensor& w,
                                                        const at::Tensor& ids, double inv_tau, at::Tensor& logp,
                                                        const c10::optional<at::Tensor>& e,
                                                        const c10::optional<at::Tensor>& perm) {
  check_rows_bf16(h, "logprob: h");
  check_rows_bf16(w, "logprob: w");
  const int64_t T = h.size(0), H = h.size(1), V = w.size(0);
  TORCH_CHECK(w.size(1) == H, "logprob: h has ", H, " columns, w has ", w.size(1));
  TORCH_CHECK(T >= 1 && V >= 1 && T <= kIntMax / 2 && V <= kIntMax / 2, "logprob: row and vocabulary counts");
  check_ids(ids, T, "logprob: ids");
  TORCH_CHECK(logp.is_cuda() && logp.scalar_type() == at::kFloat && logp.is_contiguous() && logp.numel() >= T,
              "logprob: logp must be contiguous CUDA fp32, at least one entry per row");
  CHECK_SAME_DEVICE(h, w);
  CHECK_SAME_DEVICE(h, ids);
  CHECK_SAME_DEVICE(h, logp);
  const c10::cuda::CUDAGuard g(h.device());
  const int bn = pb::logprob_tile_n((int)T, (int)V);
  const auto f32 = h.options().dtype(at::kFloat);
  at::Tensor lse2 = at::empty({T}, f32), stats = at::empty({T, (V + bn - 1) / bn, 2}, f32);
  pb::LogprobParams p{};
  p.h = h.data_ptr();
  p.w = w.data_ptr();
  p.ids = ids.data_ptr<int64_t>();
  p.stats = stats.data_ptr<float>();
  p.logp = logp.data_ptr<float>();
  p.lse2 = lse2.data_ptr<float>();
  p.ldh = h.stride(0);
  p.ldw = w.stride(0);
  if (e.has_value() && e->defined()) {
    check_rows_bf16(*e, "logprob: e");
    CHECK_SAME_DEVICE(h, *e);
    TORCH_CHECK(e->size(0) == T && e->size(1) == V && e->stride(0) >= (V + 7) / 8 * 8,
                "logprob: e must be [T, V] with room for whole 8-column groups in each row");
    p.e = e->data_ptr();
    p.lde = e->stride(0);
  }
  if (perm.has_value() && perm->defined()) {
    CHECK_SAME_DEVICE(h, *perm);
    p.perm = check_rows_i32(*perm, T, "logprob: perm");
  }
  p.T = (int)T;
  p.V = (int)V;
  p.H = (int)H;
  p.bn = bn;
  p.inv_tau = (float)inv_tau;
  pb::logprob_fwd(p, cur_stream());
  return {lse2, stats, bn};
}

// logprob_bwd(e [T, V], stats, lse2 [T], ids [T], perm [T], logp, g, inv_tau, bn): e becomes the gradient of h w^T;
// logp and g are in the caller's row order (row perm[t] for row t of e)
void logprob_bwd(at::Tensor& e, const at::Tensor& stats, const at::Tensor& lse2, const at::Tensor& ids,
                 const at::Tensor& perm, const at::Tensor& logp, const at::Tensor& g, double inv_tau, int64_t bn) {
  check_rows_bf16(e, "logprob: e");
  const int64_t T = e.size(0), V = e.size(1);
  check_ids(ids, T, "logprob: ids");
  for (const at::Tensor* t : {&stats, &lse2, &ids, &perm, &logp, &g}) CHECK_SAME_DEVICE(e, *t);
  TORCH_CHECK(logp.numel() == g.numel() && g.numel() >= T, "logprob: logp and g must have one entry per row");
  TORCH_CHECK(bn >= 32 && bn <= 256 && bn % 32 == 0 && stats.scalar_type() == at::kFloat && stats.is_contiguous() &&
                  stats.numel() == T * ((V + bn - 1) / bn) * 2,
              "logprob: stats must be the forward's");
  TORCH_CHECK(e.stride(0) % 8 == 0 && e.stride(0) >= (V + 7) / 8 * 8 &&
                  (reinterpret_cast<uintptr_t>(e.data_ptr()) & 15) == 0,
              "logprob: e must have 16-byte rows with room for whole 8-column groups");
  const c10::cuda::CUDAGuard guard(e.device());
  pb::logprob_bwd(e.data_ptr(), e.stride(0), stats.data_ptr<float>(), check_rows_f32(lse2, T, "logprob: lse2"),
                  check_rows_f32(logp, logp.numel(), "logprob: logp"), ids.data_ptr<int64_t>(),
                  check_rows_i32(perm, T, "logprob: perm"), check_rows_f32(g, g.numel(), "logprob: g"),
                  (float)inv_tau, (int)T, (int)V, (int)bn, cur_stream());
}

}  // namespace

void register_objectives(pybind11::module& m) {
  namespace py = pybind11;
  m.def("logprob_pack", &logprob_pack, py::arg("h"), py::arg("ids"));
  m.def("logprob_unpack", &logprob_unpack, py::arg("src"), py::arg("pos"), py::arg("count"));
  m.def("logprob_fwd", &logprob_fwd, py::arg("h"), py::arg("w"), py::arg("ids"), py::arg("inv_tau"), py::arg("logp"),
        py::arg("e") = py::none(), py::arg("perm") = py::none());
  m.def("logprob_bwd", &logprob_bwd, py::arg("e"), py::arg("stats"), py::arg("lse2"), py::arg("ids"), py::arg("perm"),
        py::arg("logp"), py::arg("g"), py::arg("inv_tau"), py::arg("bn"));
}
