// Python bindings of LayerNorm, rotary positions, expert routing and distillation from top logits (layernorm.cu,
// rotary.cu, route.cu, distill.cu); bindings.cpp adds them to the module. Every function enqueues on the current CUDA
// stream of the tensors' device and never synchronises. Scratch is allocated per call, so calls on several streams and
// captured graphs share none.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include "bindings.h"
#include "fmb_api.h"

namespace {

using torch::Tensor;
using OptTensor = c10::optional<Tensor>;

cudaStream_t cur_stream() { return at::cuda::getCurrentCUDAStream().stream(); }

int dt(const Tensor& t, const char* name) {
  if (t.scalar_type() == at::kBFloat16) return FMB_BF16;
  if (t.scalar_type() == at::kFloat) return FMB_F32;
  TORCH_CHECK(false, name, " must be bf16 or fp32, got ", t.scalar_type());
}

void ok(int rc, const char* what, int kernels) {
  TORCH_CHECK(rc == 0, "forgeminds_b200 native call '", what, "' failed with code ", rc);
  fmb_count_launches(kernels);
}

bool given(const OptTensor& t) { return t.has_value() && t->defined(); }
const void* ptr(const OptTensor& t) { return given(t) ? t->data_ptr() : nullptr; }

// a tensor that a kernel reads next to `like`: on its device, with `n` values in one piece
void beside(const Tensor& t, const Tensor& like, int64_t n, at::ScalarType type, const char* name) {
  TORCH_CHECK(t.device() == like.device(), name, " is on ", t.device(), ", not on ", like.device());
  TORCH_CHECK(t.scalar_type() == type, name, " must be ", type, ", got ", t.scalar_type());
  TORCH_CHECK(t.is_contiguous() && t.numel() == n, name, " must be contiguous with ", n, " values");
}

void rows_of(const Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
  TORCH_CHECK(t.dim() == 2 && (t.numel() == 0 || t.size(1) <= 1 || t.stride(1) == 1), name, " must be 2-D with contiguous rows");
  TORCH_CHECK(t.size(1) >= 1 && t.size(1) <= (1 << 24), name, ": rows of 1 to 2^24 values");
}

void rows_like(const Tensor& t, const Tensor& like, const char* name) {
  rows_of(t, name);
  TORCH_CHECK(t.device() == like.device() && t.scalar_type() == like.scalar_type() && t.sizes() == like.sizes(), name,
              " must have the first tensor's shape, type and device");
}

// ---- LayerNorm
// x [rows, d] (rows may be apart), w and b [d] or none, delta like x or none: (y, sum or none, stats or none)
std::vector<Tensor> layernorm_fwd(const Tensor& x, const OptTensor& delta, const OptTensor& w, const OptTensor& b, double eps,
                                  bool need_stats) {
  rows_of(x, "x");
  const int64_t rows = x.size(0), d = x.size(1);
  if (given(delta)) rows_like(*delta, x, "delta");
  const at::ScalarType wt = given(w) ? w->scalar_type() : given(b) ? b->scalar_type() : at::kFloat;
  TORCH_CHECK(wt == at::kFloat || wt == x.scalar_type(), "layer_norm: the weight must be fp32 or of the input's type");
  if (given(w)) beside(*w, x, d, wt, "w");
  if (given(b)) beside(*b, x, d, wt, "b");
  c10::cuda::CUDAGuard guard(x.device());
  Tensor y = at::empty({rows, d}, x.options()), sum, stats;
  if (given(delta)) sum = at::empty({rows, d}, x.options());
  if (need_stats) stats = at::empty({rows, 2}, x.options().dtype(at::kFloat));
  ok(fmb_layernorm_fwd(x.data_ptr(), x.stride(0), ptr(delta), given(delta) ? delta->stride(0) : 0, ptr(w), ptr(b),
                       given(delta) ? sum.data_ptr() : nullptr, y.data_ptr(), need_stats ? stats.data_ptr<float>() : nullptr, rows,
                       static_cast<int>(d), static_cast<float>(eps), dt(x, "x"), wt == at::kFloat ? FMB_F32 : FMB_BF16,
                       cur_stream()), "layernorm_fwd", rows > 0);
  return {y, sum, stats};
}

// (dx, dw or none, db or none); dw and db have the weight's type
std::vector<Tensor> layernorm_bwd(const Tensor& dy, const Tensor& x, const OptTensor& w, const Tensor& stats,
                                  const OptTensor& dres, bool need_dw, bool need_db, bool w_fp32) {
  rows_of(x, "x");
  rows_like(dy, x, "dy");
  const int64_t rows = x.size(0), d = x.size(1);
  if (given(dres)) rows_like(*dres, x, "dres");
  beside(stats, x, 2 * rows, at::kFloat, "stats");
  const at::ScalarType wt = w_fp32 ? at::kFloat : at::kBFloat16;
  TORCH_CHECK(w_fp32 || x.scalar_type() == at::kBFloat16, "layer_norm: a bf16 weight needs a bf16 input");
  if (given(w)) beside(*w, x, d, wt, "w");
  c10::cuda::CUDAGuard guard(x.device());
  Tensor dx = at::empty({rows, d}, x.options()), dw, db, partial;
  const bool cols = (need_dw || need_db) && rows > 0;
  auto wopt = x.options().dtype(wt);
  if (need_dw) dw = cols ? at::empty({d}, wopt) : at::zeros({d}, wopt);
  if (need_db) db = cols ? at::empty({d}, wopt) : at::zeros({d}, wopt);
  const int nb = fmb_layernorm_bwd_blocks(rows, static_cast<int>(d), dt(x, "x"));
  if (cols) partial = at::empty({nb, 2, d}, x.options().dtype(at::kFloat));
  ok(fmb_layernorm_bwd(dy.data_ptr(), dy.stride(0), x.data_ptr(), x.stride(0), ptr(w), stats.data_ptr<float>(), ptr(dres),
                       given(dres) ? dres->stride(0) : 0, dx.data_ptr(), cols ? partial.data_ptr<float>() : nullptr,
                       need_dw ? dw.data_ptr() : nullptr, need_db ? db.data_ptr() : nullptr, rows, static_cast<int>(d), dt(x, "x"),
                       w_fp32 ? FMB_F32 : FMB_BF16, nb, cur_stream()), "layernorm_bwd", rows > 0 ? 1 + cols : 0);
  return {dx, dw, db};
}

// ---- rotary positions
// q, k [B, T, H, D] (any strides, D in one piece; k may be none), cos / sin fp32 [table, R / 2] with equal strides,
// positions [T] or [B, T] int32 / int64 in one piece or none. Returns contiguous tensors.
std::vector<Tensor> rotary(const Tensor& q, const OptTensor& k, const Tensor& cos, const Tensor& sin, const OptTensor& positions,
                           bool interleaved, double sign) {
  auto check = [&](const Tensor& t, const char* name) {
    TORCH_CHECK(t.is_cuda() && t.device() == q.device() && t.scalar_type() == q.scalar_type(), name,
                ": CUDA tensors of one device and type required");
    TORCH_CHECK(t.dim() == 4 && (t.numel() == 0 || t.size(3) <= 1 || t.stride(3) == 1), name, " must be [B, T, H, D] with contiguous heads");
    TORCH_CHECK(t.size(0) == q.size(0) && t.size(1) == q.size(1) && t.size(3) == q.size(3), name,
                " must share q's batch, sequence and head dimensions");
  };
  check(q, "q");
  if (given(k)) check(*k, "k");
  const int64_t B = q.size(0), T = q.size(1), D = q.size(3), table = cos.size(0), R = 2 * cos.size(1);
  TORCH_CHECK(cos.dim() == 2 && cos.sizes() == sin.sizes() && cos.strides() == sin.strides() && (R <= 2 || cos.stride(1) == 1) &&
              cos.scalar_type() == at::kFloat && sin.scalar_type() == at::kFloat && cos.device() == q.device() &&
              sin.device() == q.device(), "rotary: cos and sin must be fp32 [table, R / 2] on q's device, with equal strides");
  TORCH_CHECK(R <= D && D <= (1 << 16), "rotary: the table turns ", R, " values of a head of ", D);
  TORCH_CHECK(B * T <= 0x7fffffff, "rotary: more than 2^31 tokens");
  int64_t pos_b = 0;
  int wide = 0;
  if (given(positions)) {
    wide = positions->scalar_type() == at::kLong;
    TORCH_CHECK(wide || positions->scalar_type() == at::kInt, "rotary: positions must be int32 or int64");
    TORCH_CHECK(positions->numel() == T || positions->numel() == B * T, "rotary: positions must be [T] or [B, T]");
    beside(*positions, q, positions->numel(), positions->scalar_type(), "positions");
    pos_b = positions->dim() == 2 && positions->size(0) == B ? T : 0;
    TORCH_CHECK(pos_b * B == positions->numel() || positions->numel() == T, "rotary: positions must be [T] or [B, T]");
  } else {
    TORCH_CHECK(T <= table, "rotary: a table of ", table, " positions for sequences of ", T);
  }
  c10::cuda::CUDAGuard guard(q.device());
  Tensor qo = at::empty({B, T, q.size(2), D}, q.options()), ko;
  FmbRotaryTensor qa = {q.data_ptr(), qo.data_ptr(), q.stride(0), q.stride(1), q.stride(2), static_cast<int>(q.size(2))}, ka = {};
  if (given(k)) {
    ko = at::empty({B, T, k->size(2), D}, q.options());
    ka = {k->data_ptr(), ko.data_ptr(), k->stride(0), k->stride(1), k->stride(2), static_cast<int>(k->size(2))};
  }
  if (B * T == 0 || D == 0 || qa.heads + ka.heads == 0) return {qo, ko};
  ok(fmb_rotary(&qa, &ka, cos.data_ptr<float>(), sin.data_ptr<float>(), cos.stride(0), table, ptr(positions), wide, pos_b, B,
                static_cast<int>(T), static_cast<int>(D), static_cast<int>(R), interleaved, static_cast<float>(sign), dt(q, "q"),
                cur_stream()), "rotary", 1);
  return {qo, ko};
}

// ---- distillation from top logits
void kl_check(const Tensor& student, const Tensor& values, const Tensor& index, const OptTensor& lse) {
  rows_of(student, "student");
  const int64_t rows = student.size(0);
  TORCH_CHECK(index.dim() == 2 && index.size(0) == rows && index.size(1) >= 1 && index.size(1) <= FMB_KL_MAX_KEEP,
              "kl_topk: index must be [rows, K] with K from 1 to ", FMB_KL_MAX_KEEP);
  beside(index, student, index.numel(), at::kLong, "index");
  beside(values, student, index.numel(), values.scalar_type(), "values");
  if (given(lse)) beside(*lse, student, rows, at::kFloat, "teacher_lse");
}

// (loss or none, row losses, stats, gradient or none, counts). `mean`: divided by the rows that count (`count`, or counted
// here). in_place: the gradient takes the student's place.
std::vector<Tensor> kl_topk_fwd(const Tensor& student, const Tensor& values, const Tensor& index, const OptTensor& lse, double tau,
                                bool total, bool mean, const OptTensor& count, bool need_grad, bool in_place) {
  kl_check(student, values, index, lse);
  const int64_t rows = student.size(0), V = student.size(1), K = index.size(1);
  if (given(count)) TORCH_CHECK(count->device() == student.device() && count->scalar_type() == at::kInt && count->numel() >= 1,
                                "kl_topk: count must be an int32 tensor on the student's device");
  c10::cuda::CUDAGuard guard(student.device());
  auto f32 = student.options().dtype(at::kFloat);
  Tensor row_loss = at::empty({rows}, f32), stats = at::empty({rows, 2}, f32), grad, loss;
  Tensor ws = at::empty({2}, student.options().dtype(at::kInt));
  if (need_grad) grad = in_place ? student : at::empty({rows, V}, student.options());
  if (total) loss = rows > 0 ? at::empty({}, f32) : at::zeros({}, f32);
  ok(fmb_kl_topk_fwd(student.data_ptr(), student.stride(0), values.data_ptr(),
                     reinterpret_cast<const long long*>(index.data_ptr<int64_t>()), static_cast<const float*>(ptr(lse)),
                     row_loss.data_ptr<float>(), stats.data_ptr<float>(), need_grad ? grad.data_ptr() : nullptr,
                     need_grad ? grad.stride(0) : 0, static_cast<const int*>(ptr(count)), ws.data_ptr<int>(),
                     total ? loss.data_ptr<float>() : nullptr, rows, static_cast<int>(V), static_cast<int>(K),
                     static_cast<float>(tau), mean, dt(student, "student"), dt(values, "values"), cur_stream()),
     "kl_topk_fwd", rows > 0 ? 1 + (mean && !given(count)) : 0);
  return {loss, row_loss, stats, grad, ws};
}

// Gradient for `upstream` (one fp32 number or one per row). With `done` (the gradient for an upstream of 1) the rows whose
// upstream is 1 are left as they are there, and `done` is the result; otherwise the result is new.
Tensor kl_topk_bwd(const Tensor& student, const Tensor& values, const Tensor& index, const OptTensor& lse, const Tensor& stats,
                   double tau, const OptTensor& count, const Tensor& upstream, const OptTensor& done) {
  kl_check(student, values, index, lse);
  const int64_t rows = student.size(0), V = student.size(1), K = index.size(1);
  beside(stats, student, 2 * rows, at::kFloat, "stats");
  TORCH_CHECK(upstream.numel() == 1 || upstream.numel() == rows, "kl_topk: one upstream gradient, or one per row");
  beside(upstream, student, upstream.numel(), at::kFloat, "upstream");
  if (given(done)) rows_like(*done, student, "done");
  c10::cuda::CUDAGuard guard(student.device());
  Tensor grad = given(done) ? *done : at::empty({rows, V}, student.options());
  ok(fmb_kl_topk_bwd(student.data_ptr(), student.stride(0), values.data_ptr(),
                     reinterpret_cast<const long long*>(index.data_ptr<int64_t>()), static_cast<const float*>(ptr(lse)),
                     stats.data_ptr<float>(), grad.data_ptr(), grad.stride(0), static_cast<const int*>(ptr(count)),
                     upstream.data_ptr<float>(), upstream.dim() > 0 && upstream.numel() == rows, given(done), rows,
                     static_cast<int>(V), static_cast<int>(K), static_cast<float>(tau), dt(student, "student"),
                     dt(values, "values"), cur_stream()), "kl_topk_bwd", rows > 0);
  return grad;
}

// ---- routing to experts
// (weights fp32 [N, k], idx int32 [N, k], counts int32 [E], aux fp32 or none)
std::vector<Tensor> route_fwd(const Tensor& logits, const OptTensor& bias, int64_t k, bool softmax, int64_t groups,
                              int64_t top_groups, int64_t best, bool renorm, double scale, bool need_aux, double aux_coef,
                              double z_coef) {
  rows_of(logits, "logits");
  const int64_t N = logits.size(0), E = logits.size(1);
  TORCH_CHECK(E <= FMB_ROUTE_MAX_EXPERTS && k <= FMB_ROUTE_MAX_K && groups <= 32, "route: at most ", FMB_ROUTE_MAX_EXPERTS,
              " experts, ", FMB_ROUTE_MAX_K, " of them, 32 groups");
  if (given(bias)) beside(*bias, logits, E, at::kFloat, "bias");
  c10::cuda::CUDAGuard guard(logits.device());
  auto f32 = logits.options().dtype(at::kFloat);
  auto i32 = logits.options().dtype(at::kInt);
  Tensor weights = at::empty({N, k}, f32), idx = at::empty({N, k}, i32), counts = at::empty({E}, i32), partial, aux;
  const int nb = fmb_route_blocks(N, static_cast<int>(E));
  if (need_aux) {
    partial = at::empty({nb, E + 1}, f32);
    aux = N > 0 ? at::empty({}, f32) : at::zeros({}, f32);
  }
  ok(fmb_route_fwd(logits.data_ptr(), logits.stride(0), dt(logits, "logits"), static_cast<const float*>(ptr(bias)),
                   weights.data_ptr<float>(), idx.data_ptr<int>(), counts.data_ptr<int>(),
                   need_aux ? partial.data_ptr<float>() : nullptr, need_aux ? aux.data_ptr<float>() : nullptr, N,
                   static_cast<int>(E), static_cast<int>(k), softmax, static_cast<int>(groups), static_cast<int>(top_groups),
                   static_cast<int>(best), renorm, static_cast<float>(scale), static_cast<float>(aux_coef),
                   static_cast<float>(z_coef), nb, cur_stream()), "route_fwd", N > 0 ? 1 + need_aux : 0);
  return {weights, idx, counts, aux};
}

Tensor route_bwd(const Tensor& logits, const Tensor& weights, const Tensor& idx, const Tensor& counts, const OptTensor& dweights,
                 const OptTensor& daux, bool softmax, bool renorm, double scale, double aux_coef, double z_coef) {
  rows_of(logits, "logits");
  const int64_t N = logits.size(0), E = logits.size(1);
  TORCH_CHECK(idx.dim() == 2 && idx.size(0) == N, "route: idx must be [N, k]");
  const int64_t k = idx.size(1);
  beside(idx, logits, N * k, at::kInt, "idx");
  beside(weights, logits, N * k, at::kFloat, "weights");
  beside(counts, logits, E, at::kInt, "counts");
  if (given(dweights)) beside(*dweights, logits, N * k, at::kFloat, "dweights");
  if (given(daux)) beside(*daux, logits, 1, at::kFloat, "daux");
  c10::cuda::CUDAGuard guard(logits.device());
  Tensor out = at::empty({N, E}, logits.options());
  ok(fmb_route_bwd(logits.data_ptr(), logits.stride(0), dt(logits, "logits"), weights.data_ptr<float>(), idx.data_ptr<int>(),
                   static_cast<const float*>(ptr(dweights)), static_cast<const float*>(ptr(daux)), counts.data_ptr<int>(),
                   out.data_ptr(), N, static_cast<int>(E), static_cast<int>(k), softmax, renorm, static_cast<float>(scale),
                   static_cast<float>(aux_coef), static_cast<float>(z_coef), cur_stream()), "route_bwd", N > 0);
  return out;
}

}  // namespace

void fmb_bind_rows(pybind11::module_& m) {
  m.def("layernorm_fwd", &layernorm_fwd);
  m.def("layernorm_bwd", &layernorm_bwd);
  m.def("rotary", &rotary);
  m.def("kl_topk_fwd", &kl_topk_fwd);
  m.def("kl_topk_bwd", &kl_topk_bwd);
  m.def("route_fwd", &route_fwd);
  m.def("route_bwd", &route_bwd);
  m.attr("KL_MAX_KEEP") = FMB_KL_MAX_KEEP;
  m.attr("ROUTE_MAX_EXPERTS") = FMB_ROUTE_MAX_EXPERTS;
  m.attr("ROUTE_MAX_K") = FMB_ROUTE_MAX_K;
}
