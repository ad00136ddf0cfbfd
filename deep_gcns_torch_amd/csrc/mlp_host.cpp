// Host side of mlp_ops: argument validity, allocation, autograd and the calls of libdgcn's C entry points (include/dgcn.h),
// in C++ because a call that a model makes once per layer and token is bound by its host side: through ctypes and a
// torch.autograd.Function in Python one row of 4096 took 12 us of which 3.8 are the launch, and a backward of a few rows
// 110 us, most of it the interpreter on autograd's thread.  No kernel lives here, and nothing of libdgcn is linked: init()
// is handed the addresses of the entry points that the ctypes binding has loaded.
//
// Each function returns None where an argument is not valid; mlp_ops then names the reason.

#include <torch/extension.h>

#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include <map>
#include <string>
#include <utility>
#include <vector>

#include "dgcn.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

constexpr int64_t kMaxNormC = 32768, kMaxK = int64_t{1} << 20;

#define ENTRY_POINTS(X) \
  X(rms_norm_fwd) X(rms_norm_num_partials) X(rms_norm_sum_bwd) X(quantize_rows_e4m3) X(linear_workspace) X(linear_act) \
  X(linear_bwd_workspace) X(linear_bwd) X(strerror)

struct {
#define X(name) decltype(&dgcn_##name) name;
  ENTRY_POINTS(X)
#undef X
} lib;

void init(const std::map<std::string, uintptr_t>& at) {
#define X(name) lib.name = reinterpret_cast<decltype(lib.name)>(at.at("dgcn_" #name));
  ENTRY_POINTS(X)
#undef X
}

void check(int rc, const char* what) {
  TORCH_CHECK(rc == 0, what, " failed (rc=", rc, "): ", lib.strerror(rc));
}

// A tensor that carries a tangent (torch.autograd.forward_ad), whatever the gradient mode: no operator here has a derivative
// for it, and a result without one would read as a derivative of zero.
bool dual(const Tensor& t) { return t.defined() && t._fw_grad(0).defined(); }
bool dual(const OptTensor& t) { return t.has_value() && dual(*t); }

// The gradients of a backward pass that has none of its own: under create_graph they are made outside the graph, and
// differentiating them again raises.
template <class Run>
variable_list once_differentiable(const char* what, const variable_list& upstream, Run run) {
  for (const Tensor& g : upstream) TORCH_CHECK(!dual(g), what, " has no forward-mode derivative");
  if (!at::GradMode::is_enabled()) return run();
  variable_list grads;
  {
    at::AutoGradMode off(false);
    grads = run();
  }
  for (Tensor& g : grads)
    if (g.defined()) g = g.detach().set_requires_grad(true);
  const auto error = std::make_shared<torch::autograd::DelayedError>(std::string(what) + " has no second derivative", grads.size());
  return (*error)(std::move(grads));
}

int row_type(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return DGCN_T_F32;
    case at::kBFloat16: return DGCN_T_BF16;
    case at::kHalf: return DGCN_T_F16;
    default: return -1;
  }
}

const void* ptr(const OptTensor& t) { return t.has_value() ? t->data_ptr() : nullptr; }

// where a call's work goes: the tensors' device, made current, and torch's current stream of it
struct Place {
  c10::DeviceGuard guard;
  void* stream;
  explicit Place(const Tensor& t) : guard(t.device()), stream(c10::hip::getCurrentHIPStream(t.get_device()).stream()) {}
};

bool on(const Tensor& t, c10::DeviceIndex d) { return t.is_cuda() && t.get_device() == d; }
bool on(const OptTensor& t, c10::DeviceIndex d) { return !t.has_value() || on(*t, d); }
bool wants(const OptTensor& t) { return t.has_value() && t->requires_grad(); }

// (rows, C) with unit stride in a row, and its row stride; rows that repeat (stride 0) are taken as they are
struct Rows {
  Tensor t;
  int64_t ld = 0;
  Rows() = default;
  explicit Rows(const Tensor& x) {
    const int64_t C = x.size(-1);
    t = x.dim() == 2 ? x : x.reshape({-1, C});
    if (C > 1 && t.stride(1) != 1) t = t.contiguous();
    ld = t.size(0) > 1 ? t.stride(0) : C;
  }
  explicit Rows(const OptTensor& x) {
    if (x.has_value()) *this = Rows(*x);
  }
  int64_t rows() const { return t.size(0); }
  const void* p() const { return t.defined() ? t.data_ptr() : nullptr; }
};

bool param_ok(const OptTensor& p, int64_t n, at::ScalarType type) {
  return !p.has_value() || (p->dim() == 1 && p->size(0) == n && (p->scalar_type() == type || p->scalar_type() == at::kFloat));
}
Tensor param(const OptTensor& p) { return p.has_value() ? (p->is_contiguous() ? *p : p->contiguous()) : Tensor(); }
const void* param_ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
int is_f32(const Tensor& t) { return t.defined() && t.scalar_type() == at::kFloat ? 1 : 0; }

std::vector<int64_t> with_last(const Tensor& x, int64_t n) {
  std::vector<int64_t> s(x.sizes().begin(), x.sizes().end());
  s.back() = n;
  return s;
}

bool same_rows(const OptTensor& r, const Tensor& x, int64_t n, at::ScalarType type) {
  if (!r.has_value()) return true;
  return r->scalar_type() == type && r->dim() == x.dim() && r->size(-1) == n && r->sizes().slice(0, x.dim() - 1) == x.sizes().slice(0, x.dim() - 1);
}

// ---- root-mean-square norm ----
struct Rms {
  Tensor y, h, q, scale, rstd;
};

Rms rms_run(const Tensor& x, const OptTensor& weight, const OptTensor& residual, double eps, bool e4m3, bool keep) {
  Rms o;
  const int64_t C = x.size(-1);
  const Rows in(x), res(residual);
  const Tensor w = param(weight);
  if (residual.has_value()) o.h = at::empty(x.sizes(), x.options());
  if (keep) o.rstd = at::empty({in.rows()}, x.options().dtype(at::kFloat));
  if (e4m3) {
    o.q = at::empty(x.sizes(), x.options().dtype(at::kFloat8_e4m3fn));
    o.scale = at::empty(x.sizes().slice(0, x.dim() - 1), x.options().dtype(at::kFloat));
  } else {
    o.y = at::empty(x.sizes(), x.options());
  }
  if (in.rows()) {
    const Place at_(x);
    check(lib.rms_norm_fwd(in.p(), in.ld, res.p(), res.ld, param_ptr(w), is_f32(w), static_cast<float>(eps), row_type(x.scalar_type()),
                           o.y.defined() ? o.y.data_ptr() : nullptr, o.h.defined() ? o.h.data_ptr() : nullptr,
                           e4m3 ? static_cast<uint8_t*>(o.q.data_ptr()) : nullptr, e4m3 ? o.scale.data_ptr<float>() : nullptr,
                           keep ? o.rstd.data_ptr<float>() : nullptr, in.rows(), static_cast<int32_t>(C), at_.stream),
          "dgcn_rms_norm_fwd");
  }
  return o;
}

struct RmsFn : torch::autograd::Function<RmsFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const OptTensor& weight, const OptTensor& residual, double eps) {
    ctx->set_materialize_grads(false);
    const Rms o = rms_run(x, weight, residual, eps, false, true);
    ctx->save_for_backward({x, weight.has_value() ? *weight : Tensor(), o.rstd, residual.has_value() ? *residual : Tensor()});
    ctx->saved_data["weight"] = weight.has_value();
    ctx->saved_data["residual"] = residual.has_value();
    if (residual.has_value()) return {o.y, o.h};
    return {o.y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    return once_differentiable("rms_norm_rows", grads, [&] { return run(ctx, grads); });
  }
  static variable_list run(AutogradContext* ctx, const variable_list& grads) {
    const bool has_w = ctx->saved_data["weight"].toBool(), has_r = ctx->saved_data["residual"].toBool();
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &weight = saved[1], &rstd = saved[2], &residual = saved[3];
    const bool need_x = ctx->needs_input_grad(0), need_w = has_w && ctx->needs_input_grad(1);
    const bool need_r = has_r && ctx->needs_input_grad(has_w ? 2 : 1);
    const Tensor g = grads[0], gh = has_r ? grads[1] : Tensor();
    Tensor dx, dw;
    if (!g.defined() || x.numel() == 0) {                     // only the sum was used: its gradient is both inputs'
      dx = gh.defined() ? gh : at::zeros_like(x);
      if (need_w) dw = at::zeros_like(weight);
    } else {
      const Rows rx(x), rg(g), rgh = gh.defined() ? Rows(gh) : Rows(), rr = has_r ? Rows(residual) : Rows();
      const int64_t rows = rx.rows();
      const int32_t C = static_cast<int32_t>(x.size(-1));
      const Tensor w = has_w ? param(weight) : Tensor();
      Tensor parts;
      if (need_x || need_r) dx = at::empty(x.sizes(), x.options());
      if (need_w) {
        dw = at::empty({C}, weight.options());
        parts = at::empty({lib.rms_norm_num_partials(rows, C), C}, x.options().dtype(at::kFloat));
      }
      if (dx.defined() || need_w) {
        const Place at_(x);
        check(lib.rms_norm_sum_bwd(rg.p(), rg.ld, rgh.p(), rgh.ld, rx.p(), rx.ld, rr.p(), rr.ld, param_ptr(w), is_f32(w), rstd.data_ptr<float>(),
                                   row_type(x.scalar_type()), dx.defined() ? dx.data_ptr() : nullptr, need_w ? dw.data_ptr() : nullptr,
                                   need_w ? parts.data_ptr<float>() : nullptr, rows, C, at_.stream),
              "dgcn_rms_norm_sum_bwd");
      }
    }
    return {need_x ? dx : Tensor(), need_w ? dw : Tensor(), need_r ? dx : Tensor(), Tensor()};
  }
};

template <bool e4m3>
py::object rms_norm(const Tensor& x, const OptTensor& weight, double eps, const OptTensor& residual) {
  const auto type = x.scalar_type();
  if (row_type(type) < 0 || x.dim() < 1 || x.size(-1) < 1 || x.size(-1) > kMaxNormC || !x.is_cuda()) return py::none();
  const auto d = x.get_device();
  if (!param_ok(weight, x.size(-1), type) || !same_rows(residual, x, x.size(-1), type) || !on(weight, d) || !on(residual, d)) return py::none();
  if (dual(x) || dual(weight) || dual(residual)) return py::none();
  if (at::GradMode::is_enabled() && (x.requires_grad() || wants(weight) || wants(residual))) {
    if constexpr (e4m3) return py::none();
    variable_list o;
    {
      py::gil_scoped_release release;
      o = RmsFn::apply(x, weight, residual, eps);
    }
    return o.size() == 2 ? py::object(py::make_tuple(o[0], o[1])) : py::cast(o[0]);
  }
  const Rms o = rms_run(x, weight, residual, eps, e4m3, false);
  if (e4m3) return residual.has_value() ? py::object(py::make_tuple(o.q, o.scale, o.h)) : py::object(py::make_tuple(o.q, o.scale));
  return residual.has_value() ? py::object(py::make_tuple(o.y, o.h)) : py::cast(o.y);
}

py::object quantize_rows(const Tensor& x) {
  if (row_type(x.scalar_type()) < 0 || x.dim() < 1 || x.size(-1) < 1 || x.size(-1) > kMaxNormC || !x.is_cuda()) return py::none();
  if (dual(x) || (at::GradMode::is_enabled() && x.requires_grad())) return py::none();
  const Rows in(x);
  Tensor q = at::empty(x.sizes(), x.options().dtype(at::kFloat8_e4m3fn));
  Tensor scale = at::empty(x.sizes().slice(0, x.dim() - 1), x.options().dtype(at::kFloat));
  if (in.rows()) {
    const Place at_(x);
    check(lib.quantize_rows_e4m3(in.p(), in.ld, row_type(x.scalar_type()), static_cast<uint8_t*>(q.data_ptr()), scale.data_ptr<float>(),
                                 in.rows(), static_cast<int32_t>(x.size(-1)), at_.stream),
          "dgcn_quantize_rows_e4m3");
  }
  return py::make_tuple(q, scale);
}

// ---- product with epilogue ----
// -> y, and what the backward keeps of the activation (keep)
std::pair<Tensor, Tensor> linear_run(const Tensor& x, const Tensor& weight, const OptTensor& sx, const OptTensor& sw, const OptTensor& bias,
                                     const OptTensor& residual, int64_t act, double slope, int in_type, at::ScalarType out, bool keep) {
  const int64_t N = weight.size(0), K = weight.size(1);
  Tensor y = at::empty(with_last(x, N), x.options().dtype(out)), z;
  if (keep && act != DGCN_ACT_NONE) z = at::empty(y.sizes(), y.options());
  if (y.numel() == 0) return {y, z};
  const Rows in(x), w(weight), res(residual);
  const Tensor b = param(bias);
  const int64_t rows = in.rows();
  // memory of this call alone, also inside a captured graph
  const size_t ws_bytes = lib.linear_workspace(in.p(), in.ld, w.p(), w.ld, in_type, rows, static_cast<int32_t>(K), static_cast<int32_t>(N));
  Tensor ws;
  if (ws_bytes) ws = at::empty({static_cast<int64_t>(ws_bytes)}, y.options().dtype(at::kByte));
  const Place at_(x);
  check(lib.linear_act(in.p(), in.ld, w.p(), w.ld, static_cast<const float*>(ptr(sx)), static_cast<const float*>(ptr(sw)), param_ptr(b), is_f32(b),
                       res.p(), res.ld, static_cast<int32_t>(act), static_cast<float>(slope), in_type, row_type(out),
                       z.defined() ? z.data_ptr() : nullptr, y.data_ptr(), rows, static_cast<int32_t>(K), static_cast<int32_t>(N),
                       ws.defined() ? ws.data_ptr() : nullptr, ws_bytes, at_.stream),
        "dgcn_linear_act");
  return {y, z};
}

struct LinearFn : torch::autograd::Function<LinearFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const OptTensor& bias, const OptTensor& residual,
                               int64_t act, double slope) {
    const bool keep = x.requires_grad() || weight.requires_grad() || wants(bias);
    const auto [y, z] = linear_run(x, weight, std::nullopt, std::nullopt, bias, residual, act, slope, row_type(x.scalar_type()), x.scalar_type(), keep);
    ctx->save_for_backward({x, weight, z});
    ctx->saved_data["act"] = act;
    ctx->saved_data["slope"] = slope;
    ctx->saved_data["bias"] = bias.has_value() ? static_cast<int64_t>(bias->scalar_type()) : int64_t{-1};
    ctx->saved_data["residual"] = residual.has_value();
    return {y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    return once_differentiable("linear_act", grads, [&] { return run(ctx, grads); });
  }
  static variable_list run(AutogradContext* ctx, const variable_list& grads) {
    const int64_t act = ctx->saved_data["act"].toInt(), bias_type = ctx->saved_data["bias"].toInt();
    const bool has_b = bias_type >= 0, has_r = ctx->saved_data["residual"].toBool();
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &weight = saved[1], &z = saved[2];
    const Tensor& g = grads[0];
    const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1), need_b = has_b && ctx->needs_input_grad(2);
    const bool need_r = has_r && ctx->needs_input_grad(has_b ? 3 : 2);
    const int64_t N = weight.size(0), K = weight.size(1);
    Tensor gx, gw, gb;
    const auto b_options = weight.options().dtype(static_cast<at::ScalarType>(has_b ? bias_type : 0));
    if (g.numel() == 0) {                                     // no rows: sums over nothing
      if (need_x) gx = at::zeros(x.sizes(), x.options());
      if (need_w) gw = at::zeros({N, K}, weight.options());
      if (need_b) gb = at::zeros({N}, b_options);
    } else if (need_x || need_w || need_b) {
      if (need_x) gx = at::empty(x.sizes(), x.options());
      if (need_w) gw = at::empty({N, K}, weight.options());
      if (need_b) gb = at::empty({N}, b_options);
      const Rows in(x), w(weight), rg(g);
      const int type = row_type(x.scalar_type());
      const int64_t rows = rg.rows();
      const size_t ws_bytes = lib.linear_bwd_workspace(rg.p(), rg.ld, in.p(), in.ld, w.p(), w.ld, static_cast<int32_t>(act), type,
                                                       need_x + 2 * need_w + 4 * need_b, rows, static_cast<int32_t>(K), static_cast<int32_t>(N));
      Tensor ws;
      if (ws_bytes) ws = at::empty({static_cast<int64_t>(ws_bytes)}, x.options().dtype(at::kByte));
      const Place at_(x);
      check(lib.linear_bwd(rg.p(), rg.ld, in.p(), in.ld, w.p(), w.ld, z.defined() ? z.data_ptr() : nullptr, static_cast<int32_t>(act),
                           static_cast<float>(ctx->saved_data["slope"].toDouble()), type, need_x ? gx.data_ptr() : nullptr,
                           need_w ? gw.data_ptr() : nullptr, need_b ? gb.data_ptr() : nullptr,
                           has_b && static_cast<at::ScalarType>(bias_type) == at::kFloat ? 1 : 0, rows, static_cast<int32_t>(K),
                           static_cast<int32_t>(N), ws.defined() ? ws.data_ptr() : nullptr, ws_bytes, at_.stream),
            "dgcn_linear_bwd");
    }
    return {gx, gw, gb, need_r ? g : Tensor(), Tensor(), Tensor()};
  }
};

bool linear_ok(const Tensor& x, const Tensor& weight, const OptTensor& bias, const OptTensor& residual, at::ScalarType out) {
  if (!x.is_cuda() || weight.dim() != 2 || x.dim() < 1) return false;
  const int64_t N = weight.size(0), K = weight.size(1);
  const auto d = x.get_device();
  return K == x.size(-1) && N >= 1 && K >= 1 && N <= kMaxK && K <= kMaxK && on(weight, d) && on(bias, d) && on(residual, d) &&
         param_ok(bias, N, out) && same_rows(residual, x, N, out) && !dual(x) && !dual(weight) && !dual(bias) && !dual(residual);
}

py::object linear_act(const Tensor& x, const Tensor& weight, const OptTensor& bias, int64_t act, const OptTensor& residual, double slope) {
  const auto type = x.scalar_type();
  if (row_type(type) < 0 || weight.scalar_type() != type || !linear_ok(x, weight, bias, residual, type)) return py::none();
  if (at::GradMode::is_enabled() && (x.requires_grad() || weight.requires_grad() || wants(bias) || wants(residual))) {
    variable_list o;
    {
      py::gil_scoped_release release;
      o = LinearFn::apply(x, weight, bias, residual, act, slope);
    }
    return py::cast(o[0]);
  }
  return py::cast(linear_run(x, weight, std::nullopt, std::nullopt, bias, residual, act, slope, row_type(type), type, false).first);
}

py::object linear_act_e4m3(const Tensor& x, const Tensor& sx, const Tensor& weight, const Tensor& sw, const OptTensor& bias, int64_t act,
                           const OptTensor& residual, at::ScalarType out, double slope) {
  if (row_type(out) < 0 || x.scalar_type() != at::kFloat8_e4m3fn || weight.scalar_type() != at::kFloat8_e4m3fn || sx.scalar_type() != at::kFloat ||
      sw.scalar_type() != at::kFloat || x.dim() < 1 || weight.dim() != 2 || sx.sizes() != x.sizes().slice(0, x.dim() - 1) ||
      sw.sizes() != weight.sizes().slice(0, 1) || !linear_ok(x, weight, bias, residual, out) || !on(sx, x.get_device()) || !on(sw, x.get_device()) ||
      dual(sx) || dual(sw))
    return py::none();
  if (at::GradMode::is_enabled() &&
      (x.requires_grad() || sx.requires_grad() || weight.requires_grad() || sw.requires_grad() || wants(bias) || wants(residual)))
    return py::none();
  return py::cast(linear_run(x, weight, sx.contiguous(), sw.contiguous(), bias, residual, act, slope, DGCN_T_E4M3, out, false).first);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
#define X(name) "dgcn_" #name,
  m.attr("ENTRY_POINTS") = std::vector<std::string>{ENTRY_POINTS(X)};
#undef X
  m.def("init", &init);
  m.def("rms_norm", &rms_norm<false>);
  m.def("rms_norm_e4m3", &rms_norm<true>);
  m.def("quantize_rows", &quantize_rows);
  m.def("linear_act", &linear_act);
  m.def("linear_act_e4m3", &linear_act_e4m3);
}
