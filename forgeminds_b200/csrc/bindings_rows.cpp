// Python bindings of LayerNorm, rotary positions, expert routing and distillation from top logits (layernorm.cu,
// rotary.cu, route.cu, distill.cu); bindings.cpp adds them to the module. Every function enqueues on the current CUDA
// stream of the tensors' device and never synchronises. Scratch is allocated per call, so calls on several streams and
// captured graphs share none.
//
// The differentiable forms are autograd nodes in C++: a forward and backward pass of a few microseconds on the device is
// bound by the host, and a Python node costs it 55 us more than one of these (8192 x 1024 LayerNorm, 137 us against 79, of
// which 50 are what autograd takes for any function).
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

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

// What a user may get wrong raises ValueError, like the checks of the PyTorch path; the C++ side makes them for the kernels'
// path because they cost it a microsecond less per argument.
template <typename... P> void refuse(bool when, const P&... parts) {
  if (when) throw pybind11::value_error(c10::str(parts...));
}

// The kernels read memory by pointers: what a tensor says of itself has to be what lies there. A wrapper (DTensor, whose
// pointer is null, vmap's and torch.func's tensors), a sparse one and a view that is negated lazily are refused.
void plain(const char* op, std::initializer_list<const Tensor*> tensors) {
  for (const Tensor* t : tensors)
    if (t != nullptr && t->defined() &&
        (t->layout() != at::kStrided || t->unsafeGetTensorImpl()->is_python_dispatch() || !t->has_storage() || t->is_neg() ||
         t->_is_zerotensor()))
      throw pybind11::type_error(c10::str(op, ": the sm_100a kernels take plain strided tensors, not wrappers (DTensor, vmap), sparse "
                                              "tensors or lazily negated views"));
}

bool given(const OptTensor& t) { return t.has_value() && t->defined(); }
const Tensor* opt(const OptTensor& t) { return given(t) ? &*t : nullptr; }
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
  TORCH_CHECK(t.size(1) >= 1 && (t.size(1) <= (1 << 24) || t.numel() == 0), name, ": rows of 1 to 2^24 values");
}

// elements between rows; what a single row says about it means nothing (and may be odd, which costs the wide loads)
int64_t pitch(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

void rows_like(const Tensor& t, const Tensor& like, const char* name) {
  rows_of(t, name);
  TORCH_CHECK(t.device() == like.device() && t.scalar_type() == like.scalar_type() && t.sizes() == like.sizes(), name,
              " must have the first tensor's shape, type and device");
}

// ---- LayerNorm
// x [rows, d] (rows may be apart), w and b [d] or none, delta like x or none: (y, sum or none, stats or none). y and sum are made
// in the shape of the caller's x: a view of them, taken inside an autograd node, could not be changed in place afterwards.
std::vector<Tensor> layernorm_fwd(const Tensor& x, const OptTensor& delta, const OptTensor& w, const OptTensor& b, double eps,
                                  bool need_stats, at::IntArrayRef shape) {
  rows_of(x, "x");
  const int64_t rows = x.size(0), d = x.size(1);
  if (given(delta)) rows_like(*delta, x, "delta");
  const at::ScalarType wt = given(w) ? w->scalar_type() : given(b) ? b->scalar_type() : at::kFloat;
  TORCH_CHECK(wt == at::kFloat || wt == x.scalar_type(), "layer_norm: the weight must be fp32 or of the input's type");
  if (given(w)) beside(*w, x, d, wt, "w");
  if (given(b)) beside(*b, x, d, wt, "b");
  c10::cuda::CUDAGuard guard(x.device());
  Tensor y = at::empty(shape, x.options()), sum, stats;
  if (given(delta)) sum = at::empty(shape, x.options());
  TORCH_CHECK(y.numel() == rows * d, "layer_norm: a result of ", shape, " for ", rows, " rows of ", d);
  if (need_stats) stats = at::empty({rows, 2}, x.options().dtype(at::kFloat));
  ok(fmb_layernorm_fwd(x.data_ptr(), pitch(x), ptr(delta), given(delta) ? pitch(*delta) : 0, ptr(w), ptr(b),
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
  ok(fmb_layernorm_bwd(dy.data_ptr(), pitch(dy), x.data_ptr(), pitch(x), ptr(w), stats.data_ptr<float>(), ptr(dres),
                       given(dres) ? pitch(*dres) : 0, dx.data_ptr(), cols ? partial.data_ptr<float>() : nullptr,
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
    TORCH_CHECK(t.size(2) <= (1 << 24), name, ": more than 2^24 heads");
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
  auto step = [](const Tensor& t, int dim) { return t.size(dim) > 1 ? t.stride(dim) : 0; };       // (of one: it may be odd)
  FmbRotaryTensor qa = {q.data_ptr(), qo.data_ptr(), step(q, 0), step(q, 1), step(q, 2), static_cast<int>(q.size(2))}, ka = {};
  if (given(k)) {
    ko = at::empty({B, T, k->size(2), D}, q.options());
    ka = {k->data_ptr(), ko.data_ptr(), step(*k, 0), step(*k, 1), step(*k, 2), static_cast<int>(k->size(2))};
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
  plain("kl_topk", {&student, &values, &index, opt(lse), opt(count)});
  kl_check(student, values, index, lse);
  const int64_t rows = student.size(0), V = student.size(1), K = index.size(1);
  if (given(count)) TORCH_CHECK(count->device() == student.device() && count->scalar_type() == at::kInt && count->numel() >= 1,
                                "kl_topk: count must be an int32 tensor on the student's device");
  c10::cuda::CUDAGuard guard(student.device());
  auto f32 = student.options().dtype(at::kFloat);
  Tensor row_loss = at::empty({rows}, f32), stats = at::empty({rows, 2}, f32), grad, loss;
  Tensor ws = at::empty({FMB_KL_SCRATCH}, student.options().dtype(at::kInt));
  if (need_grad) grad = in_place ? student : at::empty({rows, V}, student.options());
  if (total) loss = rows > 0 ? at::empty({}, f32) : at::zeros({}, f32);
  ok(fmb_kl_topk_fwd(student.data_ptr(), pitch(student), values.data_ptr(),
                     reinterpret_cast<const long long*>(index.data_ptr<int64_t>()), static_cast<const float*>(ptr(lse)),
                     row_loss.data_ptr<float>(), stats.data_ptr<float>(), need_grad ? grad.data_ptr() : nullptr,
                     need_grad ? pitch(grad) : 0, static_cast<const int*>(ptr(count)), ws.data_ptr<int>(), static_cast<int>(ws.numel()),
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
  ok(fmb_kl_topk_bwd(student.data_ptr(), pitch(student), values.data_ptr(),
                     reinterpret_cast<const long long*>(index.data_ptr<int64_t>()), static_cast<const float*>(ptr(lse)),
                     stats.data_ptr<float>(), grad.data_ptr(), pitch(grad), static_cast<const int*>(ptr(count)),
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
  TORCH_CHECK(E <= FMB_ROUTE_MAX_EXPERTS && k <= FMB_ROUTE_MAX_K && groups <= FMB_ROUTE_MAX_GROUPS, "route: at most ",
              FMB_ROUTE_MAX_EXPERTS, " experts, ", FMB_ROUTE_MAX_K, " of them, ", FMB_ROUTE_MAX_GROUPS, " groups");
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
  ok(fmb_route_fwd(logits.data_ptr(), pitch(logits), dt(logits, "logits"), static_cast<const float*>(ptr(bias)),
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
  ok(fmb_route_bwd(logits.data_ptr(), pitch(logits), dt(logits, "logits"), weights.data_ptr<float>(), idx.data_ptr<int>(),
                   static_cast<const float*>(ptr(dweights)), static_cast<const float*>(ptr(daux)), counts.data_ptr<int>(),
                   out.data_ptr(), N, static_cast<int>(E), static_cast<int>(k), softmax, renorm, static_cast<float>(scale),
                   static_cast<float>(aux_coef), static_cast<float>(z_coef), cur_stream()), "route_bwd", N > 0);
  return out;
}

// ---------------------------------------------------------------------------- autograd nodes
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// The kernels carry no tangents of forward mode: a dual number is refused, whether or not it requires a gradient too.
bool has_tangent(const Tensor& t) { return c10::AutogradState::get_tls_state().get_fw_grad_mode() && t._fw_grad(0).defined(); }
bool wants_grad(std::initializer_list<const Tensor*> tensors) {
  bool any = false;
  for (const Tensor* t : tensors) {
    if (t == nullptr || !t->defined()) continue;
    TORCH_CHECK_NOT_IMPLEMENTED(!has_tangent(*t), "forgeminds_b200: this operator has no derivative in forward mode");
    any |= t->requires_grad();
  }
  return any && at::GradMode::is_enabled();
}
Tensor detached(const OptTensor& t) { return given(t) ? t->detach() : Tensor(); }
OptTensor as_opt(const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }
// an incoming gradient as memory: a lazily negated view or a tensor of zeros that has none is written out
Tensor solid(const char* op, const Tensor& g) {
  if (!g.defined()) return g;
  const Tensor t = g._is_zerotensor() ? at::zeros(g.sizes(), g.options()) : g.resolve_neg();
  plain(op, {&t});
  return t;
}
bool capturing() { return c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None; }

// The kernels' gradients are not differentiable themselves: with create_graph a second derivative raises, it is not dropped.
variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  for (auto& g : grads)
    if (g.defined()) {
      g = g.detach();
      g.set_requires_grad(true);
    }
  auto raise = std::make_shared<torch::autograd::DelayedError>(
      "forgeminds_b200: this operator's backward pass cannot be differentiated", static_cast<int64_t>(grads.size()));
  return (*raise)(std::move(grads));
}

// [rows, d] with contiguous rows: a view where the strides allow it (rows may be apart), else a copy
Tensor rows2(const Tensor& x) {
  if (x.numel() == 0) return x.reshape({x.size(-1) ? x.numel() / x.size(-1) : 0, x.size(-1)});
  const Tensor r = x.dim() == 2 ? x : x.reshape({-1, x.size(-1)});
  return r.size(1) <= 1 || r.stride(1) == 1 ? r : r.contiguous();
}
Tensor heads4(const Tensor& x) { return x.size(3) <= 1 || x.stride(3) == 1 ? x : x.contiguous(); }
Tensor f32_flat(const Tensor& t, int64_t n) { return t.to(at::kFloat).reshape({n}).contiguous(); }

// weight and bias in one type that the kernels take: fp32, or the input's
std::pair<OptTensor, OptTensor> gain(const Tensor& x, const OptTensor& w, const OptTensor& b) {
  at::ScalarType type = at::kFloat;
  const at::ScalarType first = given(w) ? w->scalar_type() : given(b) ? b->scalar_type() : at::kFloat;
  if (first == x.scalar_type() && (!given(w) || !given(b) || b->scalar_type() == first)) type = first;
  auto fit = [&](const OptTensor& t) {
    return !given(t) || (t->scalar_type() == type && t->is_contiguous()) ? t : OptTensor(t->to(type).contiguous());
  };
  return {fit(w), fit(b)};
}
Tensor shaped(const Tensor& t, const Tensor& like) { return like.dim() == 2 ? t : t.view(like.sizes()); }

void check_norm(const char* op, const Tensor& x, const OptTensor& delta, const OptTensor& w, const OptTensor& b) {
  plain(op, {&x, opt(delta), opt(w), opt(b)});
  refuse(x.dim() < 1 || x.size(-1) < 1, op, " normalises the last dimension; the input is ", x.sizes());
  if (given(delta))
    refuse(delta->sizes() != x.sizes() || delta->scalar_type() != x.scalar_type() || delta->device() != x.device(), op,
           " needs two tensors of one shape, type and device, got ", x.sizes(), " ", x.scalar_type(), " on ", x.device(), " and ",
           delta->sizes(), " ", delta->scalar_type(), " on ", delta->device());
  for (const OptTensor* t : {&w, &b})
    if (given(*t))
      refuse((*t)->dim() != 1 || (*t)->size(0) != x.size(-1) || (*t)->device() != x.device(), op, ": a weight or bias ", (*t)->sizes(),
             " on ", (*t)->device(), " does not fit rows of ", x.size(-1), " on ", x.device());
}
Tensor as_type(const Tensor& t, int64_t type) { return t.defined() ? t.to(static_cast<at::ScalarType>(type)) : t; }
int64_t type_of(const OptTensor& t) { return given(t) ? static_cast<int64_t>(t->scalar_type()) : 0; }

// `delta` given: outputs (x + delta, norm of it); else (norm)
struct LayerNormNode : public torch::autograd::Function<LayerNormNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const OptTensor& delta, const OptTensor& w,
                               const OptTensor& b, double eps) {
    ctx->set_materialize_grads(false);
    const bool add = given(delta);
    const Tensor x2 = rows2(x.detach());
    auto [wd, bd] = gain(x, w, b);
    auto out = layernorm_fwd(x2, add ? OptTensor(rows2(delta->detach())) : OptTensor(), wd, bd, eps, true, x.sizes());
    const Tensor y = out[0], sum = out[1];
    const Tensor weight = given(wd) ? (given(w) && wd->is_same(*w) ? *w : wd->detach()) : Tensor();
    if (add) ctx->save_for_backward({sum, weight, out[2]});
    else ctx->save_for_backward({x2.is_alias_of(x) && x2.sizes() == x.sizes() ? x : x2, weight, out[2]});
    const bool fp32 = (!given(wd) || wd->scalar_type() == at::kFloat) && (!given(bd) || bd->scalar_type() == at::kFloat);
    ctx->saved_data["how"] = static_cast<int64_t>(given(w)) | static_cast<int64_t>(given(b)) << 1 | static_cast<int64_t>(fp32) << 2 |
                             static_cast<int64_t>(add) << 3 | type_of(w) << 8 | type_of(b) << 16;
    return add ? variable_list{sum, y} : variable_list{y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const int64_t how = ctx->saved_data["how"].toInt();
    const bool has_w = how & 1, has_b = how & 2, add = how & 8;
    const Tensor gy = solid("layer_norm backward", add ? g[1] : g[0]), gsum = solid("layer_norm backward", add ? g[0] : Tensor());
    if (!gy.defined()) return {gsum, add ? gsum : Tensor(), Tensor(), Tensor(), Tensor()};
    const auto saved = ctx->get_saved_variables();
    const size_t first = add ? 2 : 1;
    const bool need_w = has_w && ctx->needs_input_grad(first), need_b = has_b && ctx->needs_input_grad(first + has_w);
    auto out = layernorm_bwd(rows2(gy), rows2(saved[0]), as_opt(saved[1]), saved[2],
                             gsum.defined() ? OptTensor(rows2(gsum)) : OptTensor(), need_w, need_b, how & 4);
    const Tensor dx = shaped(out[0], gy);
    return once({dx, add ? dx : Tensor(), as_type(out[1], how >> 8 & 255), as_type(out[2], how >> 16 & 255), Tensor()});
  }
};

Tensor layer_norm(const Tensor& x, const OptTensor& w, const OptTensor& b, double eps) {
  check_norm("layer_norm", x, OptTensor(), w, b);
  if (wants_grad({&x, opt(w), opt(b)})) return LayerNormNode::apply(x, OptTensor(), w, b, eps)[0];
  auto [wd, bd] = gain(x, w, b);
  return layernorm_fwd(rows2(x), OptTensor(), wd, bd, eps, false, x.sizes())[0];
}

std::tuple<Tensor, Tensor> add_layer_norm(const Tensor& x, const Tensor& delta, const OptTensor& w, const OptTensor& b, double eps) {
  check_norm("add_layer_norm", x, delta, w, b);
  if (wants_grad({&x, &delta, opt(w), opt(b)})) {
    auto out = LayerNormNode::apply(x, OptTensor(delta), w, b, eps);
    return {out[0], out[1]};
  }
  auto [wd, bd] = gain(x, w, b);
  auto out = layernorm_fwd(rows2(x), rows2(delta), wd, bd, eps, false, x.sizes());
  return {out[1], out[0]};
}

struct RotaryNode : public torch::autograd::Function<RotaryNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const OptTensor& k, const Tensor& cos, const Tensor& sin,
                               const OptTensor& positions, bool interleaved) {
    ctx->set_materialize_grads(false);
    auto out = rotary(heads4(q), given(k) ? OptTensor(heads4(*k)) : OptTensor(), cos, sin, positions, interleaved, 1.0);
    ctx->save_for_backward({cos, sin, detached(positions)});
    ctx->saved_data["interleaved"] = interleaved;
    return given(k) ? variable_list{out[0], out[1]} : variable_list{out[0]};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const Tensor gq = solid("rotary backward", g[0]), gk = g.size() > 1 ? solid("rotary backward", g[1]) : Tensor();
    if (!gq.defined() && !gk.defined()) return variable_list(6);
    const auto saved = ctx->get_saved_variables();
    const bool both = gq.defined() && gk.defined();
    auto out = rotary(heads4(gq.defined() ? gq : gk), both ? OptTensor(heads4(gk)) : OptTensor(), saved[0], saved[1],
                      as_opt(saved[2]), ctx->saved_data["interleaved"].toBool(), -1.0);      // the inverse rotation
    return once({gq.defined() ? out[0] : Tensor(), gk.defined() ? out[both ? 1 : 0] : Tensor(), Tensor(), Tensor(), Tensor(), Tensor()});
  }
};

struct RotaryTables {
  Tensor cos, sin;
  OptTensor positions;
};

// The arguments of a rotation as its kernel takes them: tables [positions, R / 2] (or [1, positions, 1, R / 2]) in fp32
RotaryTables rotary_args(const char* op, const Tensor& q, const OptTensor& k, Tensor cos, Tensor sin, const OptTensor& positions) {
  plain(op, {&q, opt(k), &cos, &sin, opt(positions)});
  refuse(q.dim() != 4 || (given(k) && k->dim() != 4), op, " needs [batch, tokens, heads, head_dim], got ", q.sizes());
  const int64_t B = q.size(0), T = q.size(1), D = q.size(3);
  if (given(k))
    refuse(k->size(0) != B || k->size(1) != T || k->size(3) != D || k->scalar_type() != q.scalar_type() || k->device() != q.device(), op,
           ": q ", q.sizes(), " ", q.scalar_type(), " on ", q.device(), " and k ", k->sizes(), " ", k->scalar_type(), " on ", k->device(),
           " differ in more than their heads");
  refuse(cos.device() != q.device() || sin.device() != q.device() || (given(positions) && positions->device() != q.device()), op,
         ": q is on ", q.device(), ", its tables or positions are not");
  refuse(cos.requires_grad() || sin.requires_grad() || has_tangent(cos) || has_tangent(sin), op,
         ": the tables are constants, but one of them requires a gradient or carries a tangent");
  if (cos.dim() == 4 && cos.size(0) == 1 && cos.size(2) == 1) {
    cos = cos.select(0, 0).select(1, 0);
    if (sin.dim() == 4) sin = sin.reshape({sin.size(1), sin.size(3)});
  }
  refuse(cos.dim() != 2 || cos.sizes() != sin.sizes() || !cos.is_floating_point(), op, ": cos and sin must be [positions, rotated / 2], got ",
         cos.sizes(), " and ", sin.sizes());
  refuse(2 * cos.size(1) > D, op, ": tables for ", 2 * cos.size(1), " values of heads of ", D);
  OptTensor at = positions;
  if (given(positions)) {
    const auto type = positions->scalar_type();
    refuse(type != at::kInt && type != at::kLong, op, ": positions must be int32 or int64, got ", type);
    const bool one = positions->dim() == 1 && positions->size(0) == T;
    const bool all = positions->dim() == 2 && positions->size(1) == T && (positions->size(0) == B || positions->size(0) == 1);
    refuse(!one && !all, op, ": positions ", positions->sizes(), " for ", B, " sequences of ", T, " tokens");
    refuse(cos.size(0) < 1, op, ": empty tables");
    if (!positions->is_contiguous()) at = positions->contiguous();
  } else {
    refuse(T > cos.size(0), op, ": tables of ", cos.size(0), " positions for sequences of ", T, " tokens");
  }
  if (cos.scalar_type() != at::kFloat || sin.scalar_type() != at::kFloat || cos.strides() != sin.strides() || cos.stride(1) != 1) {
    cos = cos.to(at::kFloat).contiguous();
    sin = sin.to(at::kFloat).contiguous();
  }
  return {cos, sin, at};
}

Tensor rotary_one(const Tensor& q, const Tensor& cos, const Tensor& sin, const OptTensor& positions, bool interleaved) {
  const auto a = rotary_args("rotary", q, OptTensor(), cos, sin, positions);
  if (wants_grad({&q})) return RotaryNode::apply(q, OptTensor(), a.cos, a.sin, a.positions, interleaved)[0];
  return rotary(heads4(q), OptTensor(), a.cos, a.sin, a.positions, interleaved, 1.0)[0];
}
std::tuple<Tensor, Tensor> rotary_qk(const Tensor& q, const Tensor& k, const Tensor& cos, const Tensor& sin,
                                     const OptTensor& positions, bool interleaved) {
  const auto a = rotary_args("rotary_qk", q, k, cos, sin, positions);
  auto out = wants_grad({&q, &k}) ? RotaryNode::apply(q, OptTensor(k), a.cos, a.sin, a.positions, interleaved)
                                  : rotary(heads4(q), heads4(k), a.cos, a.sin, a.positions, interleaved, 1.0);
  return {out[0], out[1]};
}

// The forward pass also leaves the gradient for an upstream gradient of 1, while the row is at hand; the first backward
// pass hands that tensor out after a kernel has redone the rows whose upstream gradient is another number (compared on
// the device). A second one computes it anew, and so does one in a graph capture, which may be replayed with other values.
struct KlTopkNode : public torch::autograd::Function<KlTopkNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& student, const Tensor& values, const Tensor& index, const OptTensor& lse,
                        double tau, int64_t reduction) {
    const Tensor s2 = rows2(student.detach());
    auto out = kl_topk_fwd(s2, values, index, lse, tau, reduction != 2, reduction == 0, OptTensor(), !capturing(), false);
    ctx->save_for_backward({s2.is_alias_of(student) && s2.sizes() == student.sizes() ? student : s2, values, index, detached(lse), out[2],
                            reduction == 0 ? out[4] : Tensor()});
    ctx->saved_data["tau"] = tau;
    if (out[3].defined()) ctx->saved_data["ready"] = out[3];
    return reduction == 2 ? out[1] : out[0];               // (the student is 2-D: one loss per row)
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto saved = ctx->get_saved_variables();
    OptTensor ready;
    auto at = ctx->saved_data.find("ready");
    if (at != ctx->saved_data.end()) {
      if (!capturing()) ready = at->second.toTensor();
      ctx->saved_data.erase(at);
    }
    g[0] = solid("kl_topk_logits backward", g[0]);
    const Tensor up = g[0].dim() ? f32_flat(g[0], g[0].numel()) : g[0].to(at::kFloat);
    const Tensor s2 = rows2(saved[0]);
    auto sizes = g[0].sizes().vec();
    if (g[0].dim() == 0) sizes = saved[0].sizes().vec(); else sizes.push_back(s2.size(1));
    Tensor grad = kl_topk_bwd(s2, saved[1], saved[2], as_opt(saved[3]), saved[4], ctx->saved_data["tau"].toDouble(),
                              as_opt(saved[5]), up, ready);
    return once({grad.view(sizes), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()});
  }
};

// reduction: 0 mean, 1 sum, 2 none
Tensor kl_topk(const Tensor& student, const Tensor& values, const Tensor& index, const OptTensor& lse, double tau, int64_t reduction) {
  plain("kl_topk_logits", {&student, &values, &index, opt(lse)});
  refuse(student.dim() < 1 || student.size(-1) < 1, "kl_topk_logits: student must be [.., V], got ", student.sizes());
  refuse(!(tau >= 1e-20 && tau <= 1e20), "kl_topk_logits: temperature must be from 1e-20 to 1e20, got ", tau);
  refuse((index.scalar_type() != at::kInt && index.scalar_type() != at::kLong) || !values.is_floating_point(),
         "kl_topk_logits: teacher_values must be floating-point and teacher_index int32 or int64, got ", values.scalar_type(), " and ",
         index.scalar_type());
  const auto rows = student.sizes().slice(0, student.dim() - 1);
  refuse(index.dim() != student.dim() || index.size(-1) < 1 || index.sizes() != values.sizes() ||
         index.sizes().slice(0, index.dim() - 1) != rows, "kl_topk_logits: teacher_values ", values.sizes(), " and teacher_index ",
         index.sizes(), " for rows ", rows);
  refuse(values.device() != student.device() || index.device() != student.device() || (given(lse) && lse->device() != student.device()),
         "kl_topk_logits: the student is on ", student.device(), ", the teacher is not");
  if (given(lse))
    refuse(lse->sizes() != rows || !lse->is_floating_point(), "kl_topk_logits: teacher_lse ", lse->sizes(), " ", lse->scalar_type(),
           " for rows ", rows);
  const int64_t K = index.size(-1), n = K > 0 ? index.numel() / K : 0;
  auto flat = [&](const Tensor& t) { return (t.dim() == 2 ? t : t.reshape({n, K})).contiguous(); };
  const bool taken = values.scalar_type() == at::kFloat || values.scalar_type() == at::kBFloat16;
  const Tensor v = flat(taken ? values : values.to(at::kFloat)), i = flat(index.scalar_type() == at::kLong ? index : index.to(at::kLong));
  const OptTensor l = given(lse) ? OptTensor(f32_flat(*lse, n)) : OptTensor();
  if (wants_grad({&student})) {
    const Tensor s2 = student.dim() == 2 ? student : student.reshape({n, student.size(-1)});
    Tensor out = KlTopkNode::apply(s2, v, i, l, tau, reduction);
    return reduction == 2 && student.dim() != 2 ? out.view(rows) : out;
  }
  auto out = kl_topk_fwd(rows2(student), v, i, l, tau, reduction != 2, reduction == 0, OptTensor(), false, false);
  return reduction == 2 ? out[1].view(rows) : out[0];
}

struct RouteNode : public torch::autograd::Function<RouteNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const OptTensor& bias, int64_t k, bool softmax,
                               int64_t groups, int64_t top_groups, int64_t best, bool renorm, double scale, double aux_coef,
                               double z_coef) {
    ctx->set_materialize_grads(false);
    const bool need_aux = aux_coef != 0.0 || z_coef != 0.0;
    const Tensor rows = rows2(logits.detach());
    auto out = route_fwd(rows, bias, k, softmax, groups, top_groups, best, renorm, scale, need_aux, aux_coef, z_coef);
    ctx->save_for_backward({rows.is_alias_of(logits) ? logits : rows, out[0], out[1], out[2]});
    ctx->mark_non_differentiable({out[1], out[2]});
    ctx->saved_data["softmax"] = softmax;
    ctx->saved_data["renorm"] = renorm;
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["aux"] = aux_coef;
    ctx->saved_data["z"] = z_coef;
    return need_aux ? variable_list{out[0], out[1], out[2], out[3]} : variable_list{out[0], out[1], out[2]};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    g[0] = solid("route_experts backward", g[0]);
    const Tensor daux = g.size() > 3 ? solid("route_experts backward", g[3]) : Tensor();
    if (!g[0].defined() && !daux.defined()) return variable_list(11);
    const auto saved = ctx->get_saved_variables();
    const OptTensor dw = g[0].defined() ? OptTensor(g[0].to(at::kFloat).contiguous()) : OptTensor();
    variable_list out(11);
    out[0] = route_bwd(rows2(saved[0]), saved[1], saved[2], saved[3], dw, daux.defined() ? OptTensor(f32_flat(daux, 1)) : OptTensor(),
                       ctx->saved_data["softmax"].toBool(), ctx->saved_data["renorm"].toBool(), ctx->saved_data["scale"].toDouble(),
                       ctx->saved_data["aux"].toDouble(), ctx->saved_data["z"].toDouble());
    return once(std::move(out));
  }
};

// (weights, idx, counts, aux or none)
std::tuple<Tensor, Tensor, Tensor, OptTensor> route(const Tensor& logits, const OptTensor& bias, int64_t k, bool softmax, int64_t groups,
                                                    int64_t top_groups, int64_t best, bool renorm, double scale, double aux_coef,
                                                    double z_coef) {
  plain("route_experts", {&logits, opt(bias)});
  refuse(logits.dim() != 2 || logits.size(1) < 1, "route_experts needs [tokens, experts], got ", logits.sizes());
  OptTensor steer = bias;
  if (given(bias)) {
    refuse(bias->dim() != 1 || bias->size(0) != logits.size(1) || !bias->is_floating_point() || bias->device() != logits.device(),
           "route_experts: bias ", bias->sizes(), " ", bias->scalar_type(), " on ", bias->device(), " for ", logits.size(1), " experts on ",
           logits.device());
    if (bias->scalar_type() != at::kFloat || !bias->is_contiguous()) steer = bias->to(at::kFloat).contiguous();
  }
  const bool need_aux = aux_coef != 0.0 || z_coef != 0.0;
  auto out = wants_grad({&logits})
                 ? RouteNode::apply(logits, steer, k, softmax, groups, top_groups, best, renorm, scale, aux_coef, z_coef)
                 : route_fwd(rows2(logits), steer, k, softmax, groups, top_groups, best, renorm, scale, need_aux, aux_coef, z_coef);
  return {out[0], out[1], out[2], need_aux ? OptTensor(out[3]) : OptTensor()};
}

}  // namespace

void fmb_bind_rows(pybind11::module_& m) {
  m.def("layer_norm", &layer_norm);
  m.def("add_layer_norm", &add_layer_norm);
  m.def("rotary_one", &rotary_one);
  m.def("rotary_qk", &rotary_qk);
  m.def("kl_topk", &kl_topk);
  m.def("kl_topk_fwd", &kl_topk_fwd);
  m.def("route", &route);
  m.attr("KL_MAX_KEEP") = FMB_KL_MAX_KEEP;
  m.attr("ROUTE_MAX_EXPERTS") = FMB_ROUTE_MAX_EXPERTS;
  m.attr("ROUTE_MAX_K") = FMB_ROUTE_MAX_K;
}
