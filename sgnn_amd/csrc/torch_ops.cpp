// The typed operators (include/sgnn.h) on torch tensors: argument checks, allocation on the current stream's device
// and the autograd nodes, in C++ so that a call and its backward pass cost a few microseconds of host time each and
// neither needs the interpreter (the backward runs on autograd's own thread).  sgnn_amd/functional.py and muon.py
// document the functions; the kernels are those of libsgnn_hip.so, which bind() opens by the path the Python side
// loaded.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <dlfcn.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/utils/pybind.h>

#include <cstdarg>

#include "../../include/sgnn.h"

namespace {

using at::Tensor;
using MaybeTensor = std::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct Api {
  decltype(&sgnn_last_error) last_error;
  decltype(&sgnn_linear_workspace_bytes) linear_bytes;
  decltype(&sgnn_linear) linear;
  decltype(&sgnn_linear_bwd_workspace_bytes) linear_bwd_bytes;
  decltype(&sgnn_linear_bwd) linear_bwd;
  decltype(&sgnn_norm) norm;
  decltype(&sgnn_norm_bwd_workspace_bytes) norm_bwd_bytes;
  decltype(&sgnn_norm_bwd) norm_bwd;
  decltype(&sgnn_newton_schulz_workspace_bytes) newton_schulz_bytes;
  decltype(&sgnn_newton_schulz) newton_schulz;
} api;

void bind(const std::string& path) {
  void* lib = dlopen(path.c_str(), RTLD_NOW | RTLD_LOCAL);
  TORCH_CHECK(lib, path, ": ", dlerror());
  const auto get = [&](auto& f, const char* name) {
    f = reinterpret_cast<std::decay_t<decltype(f)>>(dlsym(lib, name));
    TORCH_CHECK(f, path, ": no ", name);
  };
  get(api.last_error, "sgnn_last_error");
  get(api.linear_bytes, "sgnn_linear_workspace_bytes");
  get(api.linear, "sgnn_linear");
  get(api.linear_bwd_bytes, "sgnn_linear_bwd_workspace_bytes");
  get(api.linear_bwd, "sgnn_linear_bwd");
  get(api.norm, "sgnn_norm");
  get(api.norm_bwd_bytes, "sgnn_norm_bwd_workspace_bytes");
  get(api.norm_bwd, "sgnn_norm_bwd");
  get(api.newton_schulz_bytes, "sgnn_newton_schulz_workspace_bytes");
  get(api.newton_schulz, "sgnn_newton_schulz");
}

void check(int status, const char* what) {
  if (status == SGNN_OK) return;
  TORCH_CHECK_VALUE(status != SGNN_ERR_INVALID, what, ": ", api.last_error(), " (status ", status, ")");
  TORCH_CHECK_NOT_IMPLEMENTED(status != SGNN_ERR_UNSUPPORTED, what, ": ", api.last_error(), " (status ", status, ")");
  TORCH_CHECK(false, what, ": ", api.last_error(), " (status ", status, ")");
}

int32_t dtype_of(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return SGNN_F32;
    case at::kBFloat16: return SGNN_BF16;
    case at::kHalf: return SGNN_F16;
    default: return -1;
  }
}
int32_t dtype_of(const Tensor& t) { return dtype_of(t.scalar_type()); }

void on_gpu(const Tensor& t, const char* name) {
  TORCH_CHECK_VALUE(t.is_cuda(), name, " must be a GPU tensor (sgnn_amd runs on MI355X only; no CPU path)");
  TORCH_CHECK_VALUE(t.layout() == at::kStrided && !t.is_neg(), name, " must be a plain strided tensor");
}
void supported(const Tensor& t, const char* name) {
  on_gpu(t, name);
  TORCH_CHECK_VALUE(dtype_of(t) >= 0, name, " must be float32, bfloat16 or float16, got ", t.scalar_type());
}
void like(const Tensor& t, const char* name, const Tensor& x) {
  on_gpu(t, name);
  TORCH_CHECK_VALUE(t.scalar_type() == x.scalar_type() && t.device() == x.device(), name, " is ", t.scalar_type(),
                    " on ", t.device(), ", expected ", x.scalar_type(), " on ", x.device());
}

// [rows, width] with unit column stride and rows that do not overlap (copied only where it is not).
Tensor rows_of(const Tensor& t) {
  Tensor r = t;
  if (t.dim() != 2) {
    int64_t rows = 1;
    for (int64_t i = 0; i + 1 < t.dim(); ++i) rows *= t.size(i);
    r = t.reshape({rows, t.size(-1)});
  }
  if ((r.stride(1) == 1 && r.stride(0) >= r.size(1)) || r.is_contiguous()) return r;
  return r.contiguous();
}
// The leading dimension of rows_of's result (a single row's stride says nothing).
int64_t ld(const Tensor& t) { return std::max(t.stride(0), t.size(1)); }

// The operators have backward derivatives alone; a tangent would be lost without a word where no node is made.
template <typename... Ts>
void reverse_mode_only(const char* what, const Ts&... ts) {
  TORCH_CHECK_NOT_IMPLEMENTED(!((ts.defined() && ts._fw_grad(/*level=*/0).defined()) || ...), what,
                              ": no forward-mode derivatives");
}

void* ptr(const Tensor& t) { return t.defined() && t.numel() ? t.data_ptr() : nullptr; }
bool wants_grad(const Tensor& t) { return t.defined() && t.requires_grad(); }

Tensor workspace(size_t bytes, const Tensor& x) {
  return bytes ? at::empty({(int64_t)bytes}, x.options().dtype(at::kByte)) : Tensor();
}
void* stream_of(const Tensor& x) { return c10::hip::getCurrentHIPStream(x.device().index()).stream(); }

MaybeTensor maybe(const Tensor& t) { return t.defined() ? MaybeTensor(t) : MaybeTensor(); }
Tensor given(const MaybeTensor& t) { return t ? *t : Tensor(); }

// The gradient that came in as rows of plain values: it may be lazily negated (the imaginary part of a conjugate) or
// sparse, whatever the output was.
Tensor grad_rows(const Tensor& g) {
  const Tensor dense = g.layout() == at::kStrided ? g : g.to_dense();
  return rows_of(dense.is_neg() ? dense.resolve_neg() : dense);
}

// Whether input i of a node (x, weight, bias, residual) wants its gradient.  `present` has a bit for each that was
// given: the node numbers those alone.
bool needs(AutogradContext* ctx, int64_t present, int i) {
  if (!(present >> i & 1)) return false;
  size_t edge = 0;
  for (int j = 0; j < i; ++j) edge += present >> j & 1;
  return ctx->needs_input_grad(edge);
}
int64_t presence(const Tensor& x, const Tensor& w, const Tensor& b, const Tensor& r) {
  return x.defined() | w.defined() << 1 | b.defined() << 2 | r.defined() << 3;
}

// The gradients of a pass that is differentiable once: where a graph of them is asked for, one that says so when it
// is used.
variable_list once(bool graph, variable_list grads) {
  if (!graph) return grads;
  at::AutoGradMode on(true);
  variable_list in;
  for (auto& g : grads)
    if (g.defined()) in.push_back(g.detach().requires_grad_(true));
  auto node = std::make_shared<torch::autograd::DelayedError>(
      "sgnn_amd.functional: the backward pass is differentiable once", (int)in.size());
  auto out = (*node)(std::move(in));
  size_t i = 0;
  for (auto& g : grads)
    if (g.defined()) g = out[i++];
  return grads;
}

// ----------------------------------------------------------------------------- linear
std::pair<Tensor, Tensor> run_linear(const Tensor& x, const Tensor& w, const Tensor& bias, const Tensor& res,
                                     int64_t act, bool need_slope) {
  const int64_t M = x.size(0), K = x.size(1), N = w.size(0);
  c10::DeviceGuard guard(x.device());
  Tensor y = at::empty({M, N}, x.options()), slope;
  if (need_slope) slope = at::empty({M, N}, x.options().dtype(at::kFloat));
  if (M && N) {
    const int32_t dt = dtype_of(x);
    const size_t nws = api.linear_bytes(dt, M, N, K);
    const Tensor ws = workspace(nws, x);
    check(api.linear(dt, M, N, K, ptr(x), ld(x), ptr(w), ld(w), ptr(bias), (int32_t)act, ptr(res), res.defined() ? ld(res) : 0,
                     slope.defined() ? slope.data_ptr<float>() : nullptr, ptr(y), N, ptr(ws), nws, stream_of(x)),
          "sgnn_linear");
  }
  return {y, slope};
}

struct LinearNode : torch::autograd::Function<LinearNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const MaybeTensor& maybe_bias,
                        const MaybeTensor& maybe_res, int64_t act) {
    const Tensor bias = given(maybe_bias), res = given(maybe_res);
    ctx->saved_data["present"] = presence(x, w, bias, res);
    ctx->saved_data["act"] = act;
    auto [y, slope] = run_linear(x, w, bias, res, act, act != SGNN_ACT_NONE);
    ctx->save_for_backward({x, w, slope});
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w = saved[1], &slope = saved[2];
    const int64_t M = x.size(0), K = x.size(1), N = w.size(0);
    const bool graph = at::GradMode::is_enabled();
    at::NoGradGuard no_grad;
    c10::DeviceGuard guard(x.device());
    const Tensor dy = grad_rows(grads[0]);
    const int64_t present = ctx->saved_data["present"].toInt();
    Tensor dx, dw, db;
    if (needs(ctx, present, 0)) dx = at::empty({M, K}, x.options());
    if (needs(ctx, present, 1)) dw = at::empty({N, K}, x.options());
    if (needs(ctx, present, 2)) db = at::empty({N}, x.options());
    if (dx.defined() || dw.defined() || db.defined()) {
      const int32_t dt = dtype_of(x) | (ctx->saved_data["act"].toInt() == SGNN_ACT_RELU ? SGNN_SLOPES_01 : 0);
      const size_t nws = api.linear_bwd_bytes(dt, M, N, K, slope.defined());
      const Tensor ws = workspace(nws, x);
      check(api.linear_bwd(dt, M, N, K, ptr(dy), ld(dy), static_cast<const float*>(ptr(slope)), ptr(x), ld(x), ptr(w), ld(w), ptr(dx), ptr(dw),
                           ptr(db), ptr(ws), nws, stream_of(x)),
            "sgnn_linear_bwd");
    }
    return once(graph, {dx, dw, db, needs(ctx, present, 3) ? grads[0] : Tensor(), Tensor()});
  }
};

Tensor linear(const Tensor& x, const Tensor& weight, const MaybeTensor& bias, const MaybeTensor& residual,
              int64_t act) {
  supported(x, "x");
  like(weight, "weight", x);
  TORCH_CHECK_VALUE(x.dim() >= 1 && weight.dim() == 2 && x.size(-1) == weight.size(1), "linear: x ", x.sizes(),
                    " does not fit weight ", weight.sizes());
  const int64_t N = weight.size(0);
  auto shape = x.sizes().vec();
  shape.back() = N;
  Tensor b, r;
  if (bias) {
    like(*bias, "bias", x);
    TORCH_CHECK_VALUE(bias->dim() == 1 && bias->size(0) == N, "linear: bias ", bias->sizes(), " does not fit weight ",
                      weight.sizes());
    b = bias->contiguous();
  }
  if (residual) {
    like(*residual, "residual", x);
    TORCH_CHECK_VALUE(residual->sizes() == at::IntArrayRef(shape), "linear: residual ", residual->sizes(),
                      ", the output is ", at::IntArrayRef(shape));
    r = rows_of(*residual);
  }
  const Tensor xr = rows_of(x), wr = rows_of(weight);
  reverse_mode_only("linear", xr, wr, b, r);
  Tensor y;
  if (at::GradMode::is_enabled() && (wants_grad(xr) || wants_grad(wr) || wants_grad(b) || wants_grad(r)))
    y = LinearNode::apply(xr, wr, maybe(b), maybe(r), act);
  else
    y = run_linear(xr, wr, b, r, act, false).first;
  return shape.size() == 2 ? y : y.view(shape);
}

// ----------------------------------------------------------------------------- layer norm
int32_t affine_type(const Tensor& x, const Tensor& w, const Tensor& b) {
  return dtype_of(w.defined() ? w : b.defined() ? b : x);
}

std::pair<Tensor, Tensor> run_norm(const Tensor& x, const Tensor& w, const Tensor& b, const Tensor& res, double eps,
                                   bool need_stats) {
  const int64_t n = x.size(0), width = x.size(1);
  c10::DeviceGuard guard(x.device());
  Tensor y = at::empty({n, width}, x.options()), stats;
  if (need_stats) stats = at::empty({2, n}, x.options().dtype(at::kFloat));
  if (n) {
    float* s = need_stats ? stats.data_ptr<float>() : nullptr;
    check(api.norm(dtype_of(x), affine_type(x, w, b), ptr(x), ld(x), n, (int32_t)width, ptr(w), ptr(b), ptr(res),
                   res.defined() ? ld(res) : 0, (float)eps, ptr(y), s, s ? s + n : nullptr, stream_of(x)),
          "sgnn_norm");
  }
  return {y, stats};
}

struct NormNode : torch::autograd::Function<NormNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const MaybeTensor& maybe_w, const MaybeTensor& maybe_b,
                        const MaybeTensor& maybe_res, double eps) {
    const Tensor w = given(maybe_w), b = given(maybe_b), res = given(maybe_res);
    ctx->saved_data["present"] = presence(x, w, b, res);
    auto [y, stats] = run_norm(x, w, b, res, eps, true);
    ctx->save_for_backward({x, w, stats});
    ctx->saved_data["affine"] = (int64_t)(w.defined() ? w : b.defined() ? b : x).scalar_type();
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w = saved[1], &stats = saved[2];
    const int64_t n = x.size(0), width = x.size(1);
    const bool graph = at::GradMode::is_enabled();
    at::NoGradGuard no_grad;
    c10::DeviceGuard guard(x.device());
    const Tensor dy = grad_rows(grads[0]);
    const auto affine_type = (at::ScalarType)ctx->saved_data["affine"].toInt();
    const auto affine = x.options().dtype(affine_type);
    const int64_t present = ctx->saved_data["present"].toInt();
    Tensor dx, dw, db;
    if (needs(ctx, present, 0)) dx = at::empty({n, width}, x.options());
    if (needs(ctx, present, 1)) dw = at::empty({width}, affine);
    if (needs(ctx, present, 2)) db = at::empty({width}, affine);
    if (dx.defined() || dw.defined() || db.defined()) {
      const size_t nws = dw.defined() || db.defined() ? api.norm_bwd_bytes(n, (int32_t)width) : 0;
      const Tensor ws = workspace(nws, x);
      const float* s = stats.data_ptr<float>();
      check(api.norm_bwd(dtype_of(x), dtype_of(affine_type), ptr(dy), ld(dy), ptr(x), ld(x),
                         s, s + n, ptr(w), n, (int32_t)width, ptr(dx), ptr(dw), ptr(db), ptr(ws), nws, stream_of(x)),
            "sgnn_norm_bwd");
    }
    return once(graph, {dx, dw, db, needs(ctx, present, 3) ? grads[0] : Tensor(), Tensor()});
  }
};

Tensor layer_norm(const Tensor& x, const MaybeTensor& weight, const MaybeTensor& bias, const MaybeTensor& residual,
                  double eps) {
  supported(x, "x");
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) <= INT32_MAX, "layer_norm: x ", x.sizes(),
                    " has no last dimension to normalise over");
  TORCH_CHECK_VALUE(eps >= 0.0, "layer_norm: eps ", eps);
  const int64_t width = x.size(-1);
  const auto affine = [&](const MaybeTensor& t, const char* name) {
    if (!t) return Tensor();
    on_gpu(*t, name);
    TORCH_CHECK_VALUE(t->device() == x.device() && (t->scalar_type() == x.scalar_type() || t->scalar_type() == at::kFloat),
                      name, " is ", t->scalar_type(), " on ", t->device(), ", expected ", x.scalar_type(),
                      " or float32 on ", x.device());
    TORCH_CHECK_VALUE(t->dim() == 1 && t->size(0) == width, "layer_norm: ", name, " ", t->sizes(), ", x is ", x.sizes());
    return t->contiguous();
  };
  const Tensor w = affine(weight, "weight"), b = affine(bias, "bias");
  TORCH_CHECK_VALUE(!w.defined() || !b.defined() || w.scalar_type() == b.scalar_type(), "layer_norm: weight and bias of two types");
  Tensor r;
  if (residual) {
    like(*residual, "residual", x);
    TORCH_CHECK_VALUE(residual->sizes() == x.sizes(), "layer_norm: residual ", residual->sizes(), ", x is ", x.sizes());
    r = rows_of(*residual);
  }
  const Tensor xr = rows_of(x);
  reverse_mode_only("layer_norm", xr, w, b, r);
  Tensor y;
  if (at::GradMode::is_enabled() && (wants_grad(xr) || wants_grad(w) || wants_grad(b) || wants_grad(r)))
    y = NormNode::apply(xr, maybe(w), maybe(b), maybe(r), eps);
  else
    y = run_norm(xr, w, b, r, eps, false).first;
  return x.dim() == 2 ? y : y.view(x.sizes());
}

// ----------------------------------------------------------------------------- newton-schulz
// given: as many outputs as inputs, or none.
std::vector<Tensor> newton_schulz(const std::vector<Tensor>& gs, const std::vector<Tensor>& given, int64_t steps,
                                  double a, double b, double c, double eps) {
  at::NoGradGuard no_grad;
  TORCH_CHECK_VALUE(steps >= 0 && steps <= INT32_MAX && eps >= 0.0, "newton_schulz: steps ", steps, ", eps ", eps);
  TORCH_CHECK_VALUE(given.empty() || given.size() == gs.size(), "newton_schulz: ", given.size(), " outputs for ",
                    gs.size(), " inputs");
  std::vector<Tensor> ins, outs;
  std::vector<sgnn_matrix> mats;
  for (size_t k = 0; k < gs.size(); ++k) {
    const Tensor& g = gs[k];
    supported(g, "g");
    like(g, "g", gs[0]);
    TORCH_CHECK_VALUE((g.dim() == 2 || g.dim() == 3) && g.size(-1) <= INT32_MAX && g.size(-2) <= INT32_MAX,
                      "newton_schulz: a matrix [m, n] or a batch [b, m, n], got ", g.sizes());
    c10::DeviceGuard guard(g.device());
    const int64_t m = g.size(-2), n = g.size(-1);
    ins.push_back((g.stride(-1) == 1 && g.stride(-2) >= n) || g.is_contiguous() ? g : g.contiguous());
    if (given.empty()) {
      outs.push_back(at::empty(g.sizes(), g.options()));
    } else {
      like(given[k], "out", g);
      TORCH_CHECK_VALUE(given[k].sizes() == g.sizes() &&
                            ((given[k].stride(-1) == 1 && given[k].stride(-2) >= n) || given[k].is_contiguous()),
                        "newton_schulz: out ", given[k].sizes(), " with strides ", given[k].strides(), " for ", g.sizes());
      const int64_t count = g.dim() == 3 ? g.size(0) : 1, row = given[k].stride(-2), batch = count > 1 ? given[k].stride(0) : 0;
      TORCH_CHECK_VALUE(count < 2 || batch >= (m - 1) * row + n || (batch >= n && row >= (count - 1) * batch + n),
                        "newton_schulz: out's matrices overlap: strides ", given[k].strides(), " for ", g.sizes());
      outs.push_back(given[k]);
      if (!given[k].is_inference()) given[k].unsafeGetTensorImpl()->bump_version();
    }
    const Tensor &in = ins.back(), &out = outs.back();
    if (g.numel() == 0) continue;
    const char* pi = static_cast<const char*>(in.data_ptr());
    char* po = static_cast<char*>(out.data_ptr());
    const int64_t count = g.dim() == 3 ? g.size(0) : 1, size = g.element_size();
    const int64_t bi = g.dim() == 3 ? in.stride(0) : 0, bo = g.dim() == 3 ? out.stride(0) : 0;
    for (int64_t i = 0; i < count; ++i)
      mats.push_back({pi + size * i * bi, po + size * i * bo, std::max(in.stride(-2), n), std::max(out.stride(-2), n),
                      (int32_t)m, (int32_t)n});
  }
  TORCH_CHECK_VALUE(mats.size() <= INT32_MAX, "newton_schulz: too many matrices");
  if (!mats.empty()) {
    const Tensor& x = gs[0];
    c10::DeviceGuard guard(x.device());
    const int32_t count = (int32_t)mats.size();
    const size_t nws = api.newton_schulz_bytes(mats.data(), count);
    const Tensor ws = workspace(nws, x);
    check(api.newton_schulz(dtype_of(x), mats.data(), count, (int32_t)steps, (float)a, (float)b, (float)c, (float)eps,
                            ptr(ws), nws, stream_of(x)),
          "sgnn_newton_schulz");
  }
  return outs;
}

}  // namespace

PYBIND11_MODULE(_torch_ops, m) {
  namespace py = pybind11;
  const auto free_gil = py::call_guard<py::gil_scoped_release>();
  m.def("bind", &bind);
  m.def("linear", &linear, free_gil);
  m.def("layer_norm", &layer_norm, free_gil);
  m.def("newton_schulz", &newton_schulz, free_gil);
}
