// torch binding of the digital operators over the C ABI (aihwkit_b200.digital): checks of arguments, output and
// workspace tensors, autograd nodes. It sees the library through include/aihwkit_b200.h and the linker
// only, like pybind_module.cpp. In C++ because a call on a few rows is bound by the host: through ctypes and
// Python autograd nodes a norm of one row took 22 us and a training step of one 140.
#include <torch/extension.h>

#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <c10/core/AutogradState.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>

#include <algorithm>
#include <sstream>
#include <stdexcept>

#include "aihwkit_b200.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

#define REFUSE(cond, ...)                                                                          \
  do {                                                                                             \
    if (cond) {                                                                                    \
      std::ostringstream ss_;                                                                      \
      ss_ << __VA_ARGS__;                                                                          \
      throw std::runtime_error(ss_.str());                                                         \
    }                                                                                              \
  } while (0)

void check(int code) {
  if (code != 0) {
    throw std::runtime_error(ab200_last_error());
  }
}

int typeCode(const Tensor &t, const char *name) {
  switch (t.scalar_type()) {
  case at::kFloat: return AB200_DTYPE_F32;
  case at::kHalf: return AB200_DTYPE_F16;
  case at::kBFloat16: return AB200_DTYPE_BF16;
  default:
    REFUSE(true, name << " must be a float32, float16 or bfloat16 tensor, got " << t.scalar_type());
  }
  return 0;
}
// The kernels write results through plain pointers, which forward-mode differentiation and tracers do not see: a result would have
// no tangent (a derivative of zero), a trace the result's allocation and nothing that fills it.
void checkModes(std::initializer_list<const Tensor *> tensors) {
  REFUSE(torch::jit::tracer::isTracing() ||
             c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY).has_value(),
         "the digital operators cannot be traced");
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) {
    return;
  }
  for (const Tensor *t : tensors) {
    REFUSE(torch::autograd::isFwGradDefined(*t), "the digital operators have no forward-mode derivative: detach the dual tensor");
  }
}
void checkCuda(const Tensor &t, const char *name) {
  typeCode(t, name);
  REFUSE(!t.is_cuda(), name << " must be a CUDA tensor: there is no CPU compute path");
}
void checkLike(const Tensor &t, const char *name, const Tensor &x) {
  REFUSE(t.scalar_type() != x.scalar_type() || t.device() != x.device(),
         name << " must be a " << x.scalar_type() << " tensor on " << x.device() << ", got " << t.scalar_type() << " on "
              << t.device());
}
void checkSame(const Tensor &t, const char *name, const Tensor &x) {
  checkLike(t, name, x);
  REFUSE(t.sizes() != x.sizes(), name << " must have the shape " << x.sizes() << ", got " << t.sizes());
}
void checkRowsOf(const Tensor &x) {
  REFUSE(x.dim() < 1 || x.size(-1) < 1, "x must have at least one dimension and one column");
  REFUSE(x.size(-1) > INT32_MAX, "a row has at most 2^31 - 1 elements");
}
struct Random {
  double p;
  uint64_t seed;
  uint32_t call;
};
Random checkRandom(double p, const py::int_ &seed, const py::int_ &call) {
  REFUSE(!(p >= 0.0 && p <= 1.0), "the dropout probability must be between 0 and 1, got " << p);
  const unsigned long long s = PyLong_AsUnsignedLongLong(seed.ptr());
  if (PyErr_Occurred()) {
    PyErr_Clear();
    REFUSE(true, "seed must be between 0 and 2^64 - 1");
  }
  const unsigned long long c = PyLong_AsUnsignedLongLong(call.ptr());
  const bool bad = PyErr_Occurred() != nullptr;
  PyErr_Clear();
  REFUSE(bad || c > 0xffffffffULL, "call must be between 0 and 2^32 - 1");
  return {p, s, (uint32_t)c};
}

// The tensor as rows of its last dimension with one distance between them; a copy only where there is
// no such distance or a row's elements do not lie together.
struct Rows {
  Tensor t;
  const void *p = nullptr;
  int64_t ld = 0;
};
bool rowDistance(const Tensor &t, int64_t *ld) {
  const int64_t d = t.dim();
  if (d < 1 || (t.stride(d - 1) != 1 && t.size(d - 1) != 1)) {
    return false;
  }
  *ld = t.size(d - 1);
  bool first = true;
  int64_t expected = 0;
  for (int64_t i = d - 2; i >= 0; i--) {
    if (t.size(i) == 1) {
      continue;
    }
    if (first) {
      *ld = t.stride(i);
      first = false;
    } else if (t.stride(i) != expected) {
      return false;
    }
    expected = t.stride(i) * t.size(i);
  }
  return true;
}
// torch keeps the sign of some views (the imaginary part of a conjugate) apart from their memory
Tensor signedIn(const Tensor &t) { return t.defined() && t.is_neg() ? t.resolve_neg() : t; }
Rows rowsOf(const Tensor &t) {
  Rows r;
  if (!t.defined()) {
    return r;
  }
  r.t = signedIn(t);
  if (!rowDistance(r.t, &r.ld)) {
    r.t = r.t.contiguous();
    r.ld = r.t.size(-1);
  }
  r.p = r.t.data_ptr();
  return r;
}
Tensor whole(const Tensor &t) { return t.defined() ? signedIn(t).contiguous() : t; }
void *ptr(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }
void *stream() { return at::cuda::getCurrentCUDAStream().stream(); }
Tensor optional(const std::optional<Tensor> &t) { return t.has_value() ? *t : Tensor(); }
bool wantsGrad(std::initializer_list<const Tensor *> ts) {
  if (!at::GradMode::is_enabled()) {
    return false;
  }
  for (const Tensor *t : ts) {
    if (t->defined() && t->requires_grad()) {
      return true;
    }
  }
  return false;
}
// An autograd node takes a missing tensor as std::nullopt and counts only the tensors that are there
// as its inputs; Wanted gives the numbers of those that may be missing.
std::optional<Tensor> given(const Tensor &t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; }
struct Wanted {
  AutogradContext *ctx;
  size_t next;
  bool operator()(const Tensor &input) { return input.defined() && ctx->needs_input_grad(next++); }
};
// A gradient of a backward pass that is itself recorded: differentiating it raises by anything that it was made from, the
// incoming gradients and those inputs of the forward call whose places among the node's inputs are given (-1: missing). The
// node knows its inputs by their edges, whether or not it has kept their values.
Tensor once(Tensor g, const variable_list &incoming, std::initializer_list<int> places) {
  if (!g.defined() || !at::GradMode::is_enabled()) {
    return g;
  }
  torch::autograd::edge_list edges = torch::autograd::collect_next_edges(incoming);
  const auto node = torch::autograd::get_current_node();
  for (int place : places) {
    if (place >= 0) {
      edges.push_back(node->next_edge(place));
    }
  }
  if (std::any_of(edges.begin(), edges.end(), [](const torch::autograd::Edge &e) { return e.is_valid(); })) {
    torch::autograd::set_history(g, std::make_shared<torch::autograd::Error>(
                                        "the digital operators' gradients are not differentiable again", std::move(edges)));
  }
  return g;
}

// ---- dropout ----------------------------------------------------------------------------------
Tensor dropoutCompute(const Tensor &x, const Random &r, const Tensor &residual) {
  const c10::cuda::CUDAGuard guard(x.device());
  Tensor y = at::empty(x.sizes(), x.options());
  if (x.numel() > 0) {
    const int64_t cols = x.size(-1);
    const Rows xr = rowsOf(x), rr = rowsOf(residual);
    check(ab200_dropout(xr.p, xr.ld, rr.p, rr.ld, y.data_ptr(), cols, x.numel() / cols, (int)cols, typeCode(x, "x"), r.p,
                        r.seed, r.call, stream()));
  }
  return y;
}
struct Dropout : torch::autograd::Function<Dropout> {
  static Tensor forward(AutogradContext *ctx, const Tensor &x, const std::optional<Tensor> &residual, double p,
                        int64_t seed, int64_t call) {
    ctx->saved_data["residual"] = residual.has_value();
    ctx->saved_data["p"] = p;
    ctx->saved_data["seed"] = seed;
    ctx->saved_data["call"] = call;
    return dropoutCompute(x, {p, (uint64_t)seed, (uint32_t)call}, optional(residual));
  }
  static variable_list backward(AutogradContext *ctx, variable_list gs) {
    const Random r = {ctx->saved_data["p"].toDouble(), (uint64_t)ctx->saved_data["seed"].toInt(),
                      (uint32_t)ctx->saved_data["call"].toInt()};
    Tensor dx;
    if (ctx->needs_input_grad(0)) {
      dx = once(dropoutCompute(gs[0], r, Tensor()), gs, {});
    }
    const bool need_res = ctx->saved_data["residual"].toBool() && ctx->needs_input_grad(1);
    return {dx, need_res ? gs[0] : Tensor(), Tensor(), Tensor(), Tensor()};
  }
};
Tensor dropout(const Tensor &x, double p, const py::int_ &seed, const py::int_ &call,
               const std::optional<Tensor> &residual_) {
  const Tensor residual = optional(residual_);
  checkModes({&x, &residual});
  checkCuda(x, "x");
  checkRowsOf(x);
  if (residual.defined()) {
    checkSame(residual, "residual", x);
  }
  const Random r = checkRandom(p, seed, call);
  if (wantsGrad({&x, &residual})) {
    return Dropout::apply(x, given(residual), r.p, (int64_t)r.seed, (int64_t)r.call);
  }
  return dropoutCompute(x, r, residual);
}

// ---- layer norm -------------------------------------------------------------------------------
void checkNorm(const Tensor &x, const Tensor &residual, const Tensor &weight, const Tensor &bias) {
  checkModes({&x, &residual, &weight, &bias});
  checkCuda(x, "x");
  checkRowsOf(x);
  if (residual.defined()) {
    checkSame(residual, "residual", x);
  }
  const std::pair<const Tensor *, const char *> params[] = {{&weight, "weight"}, {&bias, "bias"}};
  for (const auto &q : params) {
    const Tensor &t = *q.first;
    if (t.defined()) {
      REFUSE((t.scalar_type() != x.scalar_type() && t.scalar_type() != at::kFloat) || t.device() != x.device(),
             q.second << " must be a " << x.scalar_type() << " or Float tensor on " << x.device());
      REFUSE(t.dim() != 1 || t.size(0) != x.size(-1),
             q.second << " must have the shape [" << x.size(-1) << "], got " << t.sizes());
    }
  }
  REFUSE(weight.defined() && bias.defined() && weight.scalar_type() != bias.scalar_type(),
         "weight and bias must be of one type");
}
int paramCode(const Tensor &x, const Tensor &weight, const Tensor &bias) {
  return typeCode(weight.defined() ? weight : bias.defined() ? bias : x, "weight");
}
struct NormOut {
  Tensor y, h, stats;
};
NormOut normCompute(const Tensor &x, const Tensor &residual, const Tensor &weight, const Tensor &bias, double eps,
                    const Random &r, bool want_h, bool want_stats) {
  const c10::cuda::CUDAGuard guard(x.device());
  NormOut o;
  o.y = at::empty(x.sizes(), x.options());
  const int64_t cols = x.size(-1), rows = x.numel() / cols;
  if (want_h) {
    o.h = at::empty(x.sizes(), x.options());
  }
  float *stats = nullptr;
  if (want_stats) {
    o.stats = at::empty({2, rows}, x.options().dtype(at::kFloat));
    stats = o.stats.data_ptr<float>();
  }
  const Rows xr = rowsOf(x), rr = rowsOf(residual);
  const Tensor w = whole(weight), b = whole(bias);
  check(ab200_layer_norm_forward(xr.p, xr.ld, rr.p, rr.ld, ptr(w), ptr(b), o.y.data_ptr(), cols, ptr(o.h), cols, stats,
                                 stats ? stats + rows : nullptr, rows, (int)cols, typeCode(x, "x"),
                                 paramCode(x, weight, bias), (float)eps, r.p, r.seed, r.call, stream()));
  return o;
}
struct NormGrads {
  Tensor dh, dx, dw, db;
};
NormGrads normGradCompute(const Tensor &gy, const Tensor &gh, const Tensor &h, const Tensor &residual,
                          const Tensor &weight, const Tensor &bias, const Tensor &stats, const Random &r, bool need_dh,
                          bool need_dx, bool need_dw, bool need_db) {
  const c10::cuda::CUDAGuard guard(h.device());
  const int64_t cols = h.size(-1), rows = h.numel() / cols;
  NormGrads o;
  if (need_dh) {
    o.dh = at::empty(h.sizes(), h.options());
  }
  if (need_dx) {
    o.dx = at::empty(h.sizes(), h.options());
  }
  Tensor work;
  if (need_dw || need_db) {
    long long floats = 0;
    check(ab200_layer_norm_workspace(rows, (int)cols, &floats));
    work = at::empty({(int64_t)floats}, h.options().dtype(at::kFloat));
    if (need_dw) {
      o.dw = at::empty({cols}, weight.options());
    }
    if (need_db) {
      o.db = at::empty({cols}, bias.options());
    }
  }
  const Rows gyr = rowsOf(gy), ghr = rowsOf(gh), hr = rowsOf(h), rr = rowsOf(residual);
  const Tensor w = whole(weight);
  const float *st = stats.data_ptr<float>();
  check(ab200_layer_norm_backward(gyr.p, gyr.ld, ghr.p, ghr.ld, hr.p, hr.ld, rr.p, rr.ld, ptr(w), st, st + rows, ptr(o.dh),
                                  cols, ptr(o.dx), cols, ptr(o.dw), ptr(o.db), (float *)ptr(work), rows, (int)cols,
                                  typeCode(h, "h"), paramCode(h, weight, bias), r.p, r.seed, r.call, stream()));
  return o;
}
struct LayerNorm : torch::autograd::Function<LayerNorm> {
  static Tensor forward(AutogradContext *ctx, const Tensor &x, const std::optional<Tensor> &weight_,
                        const std::optional<Tensor> &bias_, double eps) {
    const Tensor weight = optional(weight_), bias = optional(bias_);
    NormOut o = normCompute(x, Tensor(), weight, bias, eps, {0.0, 0, 0}, false, true);
    ctx->save_for_backward({x, weight, bias, o.stats});
    return o.y;
  }
  static variable_list backward(AutogradContext *ctx, variable_list gs) {
    const variable_list s = ctx->get_saved_variables();
    Wanted wanted = {ctx, 1};
    const bool need_w = wanted(s[1]), need_b = wanted(s[2]);
    const NormGrads g = normGradCompute(gs[0], Tensor(), s[0], Tensor(), s[1], s[2], s[3], {0.0, 0, 0},
                                        ctx->needs_input_grad(0), false, need_w, need_b);
    return {once(g.dh, gs, {0, s[1].defined() ? 1 : -1}), once(g.dw, gs, {0}), once(g.db, gs, {}), Tensor()};
  }
};
// h = residual + dropout(x), y = norm(h). The backward pass needs h as it went into the norm: an fp32 h is
// that; of 16-bit types x and residual are kept instead and h is summed again, since the rounded one
// would carry 2^-9 (bf16) of itself into the fp32 gradients of weight.
struct AddLayerNorm : torch::autograd::Function<AddLayerNorm> {
  static variable_list forward(AutogradContext *ctx, const Tensor &x, const Tensor &residual,
                               const std::optional<Tensor> &weight_, const std::optional<Tensor> &bias_, double eps,
                               double p, int64_t seed, int64_t call) {
    const Tensor weight = optional(weight_), bias = optional(bias_);
    ctx->set_materialize_grads(false);
    NormOut o = normCompute(x, residual, weight, bias, eps, {p, (uint64_t)seed, (uint32_t)call}, true, true);
    const bool exact = x.scalar_type() == at::kFloat;
    ctx->save_for_backward({exact ? o.h : x, exact ? Tensor() : residual, weight, bias, o.stats});
    ctx->saved_data["p"] = p;
    ctx->saved_data["seed"] = seed;
    ctx->saved_data["call"] = call;
    return {o.y, o.h};
  }
  static variable_list backward(AutogradContext *ctx, variable_list gs) {
    const variable_list s = ctx->get_saved_variables();
    const Random r = {ctx->saved_data["p"].toDouble(), (uint64_t)ctx->saved_data["seed"].toInt(),
                      (uint32_t)ctx->saved_data["call"].toInt()};
    const bool dropped = r.p > 0.0, need_x = ctx->needs_input_grad(0), need_res = ctx->needs_input_grad(1);
    Wanted wanted = {ctx, 2};
    const bool need_w = wanted(s[2]), need_b = wanted(s[3]);
    NormGrads g;
    if (gs[0].defined()) {
      g = normGradCompute(gs[0], gs[1], s[0], s[1], s[2], s[3], s[4], r, need_res || (need_x && !dropped),
                          need_x && dropped, need_w, need_b);
      const int w = s[2].defined() ? 2 : -1;
      g = {once(g.dh, gs, {0, 1, w}), once(g.dx, gs, {0, 1, w}), once(g.dw, {gs[0]}, {0, 1}), once(g.db, {gs[0]}, {})};
    } else if (gs[1].defined()) {
      g.dh = gs[1]; // the caller's own tensor, with whatever history it has
      if (need_x && dropped) {
        g.dx = once(dropoutCompute(gs[1], r, Tensor()), gs, {});
      }
    }
    variable_list out = {need_x ? (dropped ? g.dx : g.dh) : Tensor(), need_res ? g.dh : Tensor(), g.dw, g.db};
    out.resize(8);
    return out;
  }
};
Tensor layerNorm(const Tensor &x, const std::optional<Tensor> &weight_, const std::optional<Tensor> &bias_, double eps) {
  const Tensor weight = optional(weight_), bias = optional(bias_);
  checkNorm(x, Tensor(), weight, bias);
  if (wantsGrad({&x, &weight, &bias})) {
    return LayerNorm::apply(x, given(weight), given(bias), eps);
  }
  return normCompute(x, Tensor(), weight, bias, eps, {0.0, 0, 0}, false, false).y;
}
std::pair<Tensor, Tensor> addLayerNorm(const Tensor &x, const std::optional<Tensor> &residual_,
                                       const std::optional<Tensor> &weight_, const std::optional<Tensor> &bias_,
                                       double eps, double p, const py::int_ &seed, const py::int_ &call) {
  const Tensor residual = optional(residual_), weight = optional(weight_), bias = optional(bias_);
  REFUSE(!residual.defined(), "residual is missing: layer_norm is the call without one");
  checkNorm(x, residual, weight, bias);
  const Random r = checkRandom(p, seed, call);
  if (wantsGrad({&x, &residual, &weight, &bias})) {
    const variable_list o =
        AddLayerNorm::apply(x, residual, given(weight), given(bias), eps, r.p, (int64_t)r.seed, (int64_t)r.call);
    return {o[0], o[1]};
  }
  const NormOut o = normCompute(x, residual, weight, bias, eps, r, true, false);
  return {o.y, o.h};
}

// ---- low-rank adapters ------------------------------------------------------------------------
void lowRankCompute(const Tensor &base, const Tensor &x, const Tensor &a, const Tensor &b, const Tensor &scale,
                    const Tensor &ids, const Tensor &starts, const Tensor &out, const Tensor &v) {
  const int64_t k = a.size(2), n = b.size(2);
  const Rows xr = rowsOf(x), br = rowsOf(base), yr = rowsOf(out);
  check(ab200_low_rank_apply(xr.p, xr.ld, br.p, br.ld, const_cast<void *>(yr.p), yr.ld, a.data_ptr(), b.data_ptr(),
                             scale.data_ptr<float>(), ids.data_ptr<int>(), (const int32_t *)ptr(starts),
                             (int)ids.numel(), x.numel() / k, (int)k, (int)n, (int)a.size(1), (int)a.size(0),
                             typeCode(x, "x"), (float *)ptr(v), stream()));
}
struct LowRankAdd : torch::autograd::Function<LowRankAdd> {
  static Tensor forward(AutogradContext *ctx, const Tensor &base, const Tensor &x, const Tensor &a, const Tensor &b,
                        const Tensor &scale, const Tensor &ids, const std::optional<Tensor> &starts_) {
    const Tensor starts = optional(starts_);
    const c10::cuda::CUDAGuard guard(x.device());
    Tensor y = at::empty(base.sizes(), base.options()), v;
    if (b.requires_grad()) {
      v = at::empty({x.numel() / a.size(2), a.size(1)}, x.options().dtype(at::kFloat));
    }
    lowRankCompute(base, x, a, b, scale, ids, starts, y, v);
    ctx->save_for_backward({a.requires_grad() ? x : Tensor(), a, b, scale, ids, starts, v});
    ctx->saved_data["shape"] = x.sizes();
    return y;
  }
  static variable_list backward(AutogradContext *ctx, variable_list gs) {
    const variable_list s = ctx->get_saved_variables();
    const Tensor &gy = gs[0], &x = s[0], &a = s[1], &b = s[2], &scale = s[3], &ids = s[4], &starts = s[5], &v = s[6];
    const c10::cuda::CUDAGuard guard(gy.device());
    const bool need_x = ctx->needs_input_grad(1), need_a = ctx->needs_input_grad(2), need_b = ctx->needs_input_grad(3);
    const int64_t rank = a.size(1), k = a.size(2), n = b.size(2), rows = gy.numel() / n;
    Tensor dx, u, da, db;
    if (need_x) {
      dx = at::empty(ctx->saved_data["shape"].toIntVector(), gy.options());
    }
    if (need_a) {
      u = at::empty({rows, rank}, gy.options().dtype(at::kFloat));
      da = at::empty(a.sizes(), a.options());
    }
    if (need_b) {
      db = at::empty(b.sizes(), b.options());
    }
    if (need_x || need_a) {
      lowRankCompute(Tensor(), gy, b, a, scale, ids, starts, dx, u);
    }
    if (need_a || need_b) {
      long long bytes = 0;
      check(ab200_low_rank_grad_workspace(rows, (int)ids.numel(), !starts.defined(), need_a ? (int)k : 0,
                                          need_b ? (int)n : 0, (int)rank, &bytes));
      const Tensor work = at::empty({(int64_t)bytes}, gy.options().dtype(at::kByte));
      const Rows xr = rowsOf(need_a ? x : Tensor()), gr = rowsOf(gy);
      check(ab200_low_rank_grad(xr.p, xr.ld, (float *)ptr(u), ptr(da), (int)k, gr.p, gr.ld, (float *)ptr(v), ptr(db),
                                (int)n, ids.data_ptr<int>(), (const int32_t *)ptr(starts), (int)ids.numel(), rows,
                                (int)rank, (int)a.size(0), typeCode(gy, "gy"), ptr(work), stream()));
    }
    // of the inputs base, x, a, b
    return {ctx->needs_input_grad(0) ? gy : Tensor(), once(dx, gs, {2, 3}), once(da, gs, {1, 3}), once(db, gs, {1, 2}), Tensor(),
            Tensor(), Tensor()};
  }
};
// Whether two tensors may share memory: their address ranges meet, and they are not columns of one
// matrix beside each other (rows of one distance, with no element in common).
bool overlap(const Tensor &s, const Tensor &t) {
  if (s.numel() == 0 || t.numel() == 0 || s.device() != t.device()) {
    return false;
  }
  const auto span = [](const Tensor &q) {
    int64_t last = 0;
    for (int64_t i = 0; i < q.dim(); i++) {
      last += (q.size(i) - 1) * q.stride(i);
    }
    const uintptr_t p = (uintptr_t)q.data_ptr();
    return std::make_pair(p, p + (uintptr_t)((last + 1) * q.element_size()));
  };
  const auto a = span(s), b = span(t);
  if (a.first >= b.second || b.first >= a.second) {
    return false;
  }
  int64_t s_ld = 0, t_ld = 0;
  if (!rowDistance(s, &s_ld) || !rowDistance(t, &t_ld) || s_ld != t_ld || s_ld == 0) {
    return true;
  }
  const int64_t size = s.element_size(), pitch = s_ld * size;
  const int64_t between = (((int64_t)b.first - (int64_t)a.first) % pitch + pitch) % pitch;
  return between < s.size(-1) * size || between + t.size(-1) * size > pitch;
}
Tensor lowRankAdd(const Tensor &base, const Tensor &x, const Tensor &a, const Tensor &b, const Tensor &scale,
                  const Tensor &ids, const std::optional<Tensor> &starts_, const std::optional<Tensor> &out_) {
  const Tensor starts = optional(starts_), out = optional(out_);
  checkModes({&base, &x, &a, &b, &scale, &out});
  checkCuda(x, "x");
  checkLike(base, "base", x);
  checkLike(a, "a", x);
  checkLike(b, "b", x);
  REFUSE(a.dim() != 3 || b.dim() != 3 || a.size(0) != b.size(0) || a.size(1) != b.size(1),
         "a and b must be [adapters, rank, width], got " << a.sizes() << " and " << b.sizes());
  REFUSE(!a.is_contiguous() || !b.is_contiguous() || a.is_neg() || b.is_neg(), "a and b must be contiguous");
  REFUSE(a.numel() == 0 || b.numel() == 0, "at least one adapter, rank and column is needed");
  REFUSE(x.dim() < 1 || x.size(-1) != a.size(2) || base.dim() < 1 || base.size(-1) != b.size(2),
         "expected x [..., " << a.size(2) << "] and base [..., " << b.size(2) << "], got " << x.sizes() << " and "
                             << base.sizes());
  REFUSE(x.sizes().slice(0, x.dim() - 1) != base.sizes().slice(0, base.dim() - 1), "x and base need the same rows");
  REFUSE(scale.scalar_type() != at::kFloat || scale.device() != x.device() || scale.dim() != 1 ||
             scale.size(0) != a.size(0) || !scale.is_contiguous() || scale.is_neg(),
         "scale must be a contiguous Float tensor of " << a.size(0) << " values on " << x.device());
  REFUSE(wantsGrad({&scale}), "scale has no gradient here");
  const std::pair<const Tensor *, const char *> tables[] = {{&ids, "adapter_ids"}, {&starts, "row_starts"}};
  for (const auto &q : tables) {
    const Tensor &t = *q.first;
    REFUSE(t.defined() && (t.scalar_type() != at::kInt || t.device() != x.device() || t.dim() != 1 || !t.is_contiguous()),
           q.second << " must be a contiguous Int vector on " << x.device());
  }
  const int64_t rows = x.numel() / x.size(-1);
  REFUSE(!starts.defined() && ids.numel() != rows,
         "without row_starts there is one adapter id per row: " << rows << ", got " << ids.numel());
  REFUSE(starts.defined() && starts.numel() != ids.numel() + 1,
         "row_starts needs " << ids.numel() + 1 << " values, got " << starts.numel());
  REFUSE(ids.numel() > INT32_MAX || a.size(0) > INT32_MAX || a.size(1) > INT32_MAX || a.size(2) > INT32_MAX ||
             b.size(2) > INT32_MAX,
         "sizes of adapters must be below 2^31");
  const bool grad = wantsGrad({&base, &x, &a, &b});
  if (out.defined()) {
    checkSame(out, "out", base);
    // an `out` with a history of its own would keep it, and pass the result's gradient on to what it was before
    REFUSE(grad || wantsGrad({&out}), "out= is for calls without gradients");
    REFUSE((out.strides() != base.strides() || out.data_ptr() != base.data_ptr()) && overlap(out, base),
           "out may be base itself, but not a part or another view of it");
    REFUSE(overlap(out, x) || overlap(out, a) || overlap(out, b), "out must not share memory with x, a or b");
    int64_t ld = 0;
    REFUSE(out.numel() > 0 && (out.is_neg() || !rowDistance(out, &ld) || (ld < out.size(-1) && rows > 1)),
           "out must be rows of neighbouring elements with one distance between them");
  } else if (grad) {
    return LowRankAdd::apply(base, x, a, b, scale, ids, given(starts));
  }
  const c10::cuda::CUDAGuard guard(x.device());
  Tensor y = out.defined() ? out : at::empty(base.sizes(), base.options());
  lowRankCompute(base, x, a, b, scale, ids, starts, y, Tensor());
  if (out.defined() && !out.is_inference()) {
    torch::autograd::impl::bump_version(out); // as torch's own in-place operations do, for who saved it
  }
  return y;
}

} // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("dropout", &dropout);
  m.def("layer_norm", &layerNorm);
  m.def("add_layer_norm", &addLayerNorm);
  m.def("low_rank_add", &lowRankAdd);
}
