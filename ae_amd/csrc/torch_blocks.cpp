// The operators of include/specmoe_mi355x_blocks.h for torch: argument checks, results from its allocator, the current stream, and
// autograd nodes, compiled (the module ae_amd._blocks; ae_amd/layers has the public functions). The same through ctypes and
// Python nodes took 7.8 us a call for 4.2 here (dispatch of 64 rows, no gradient; 3 of them the launch), and 81 us a training
// pass for 46: a node of Python runs in the engine's thread, and waits for the interpreter there.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/GradMode.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>

#include <cmath>
#include <sstream>

#include "../../include/specmoe_mi355x.h"
#include "../../include/specmoe_mi355x_blocks.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
namespace py = pybind11;
using Maybe = std::optional<Tensor>;

// ---- errors --------------------------------------------------------------------------------------

template <typename... Parts> std::string text(const Parts&... parts) {
  std::ostringstream s;
  (s << ... << parts);
  return s.str();
}

// A shape as Python writes it.
std::string shape_text(c10::IntArrayRef shape) {
  std::string s = "(";
  for (size_t i = 0; i < shape.size(); ++i) s += (i ? ", " : "") + std::to_string(shape[i]);
  return s + (shape.size() == 1 ? ",)" : ")");
}

std::string dtype_text(const Tensor& t) {
  py::object o = py::cast(t).attr("dtype");
  return py::str(o);
}

// A status of the library, raised as SmxError once the interpreter is at hand.
struct Failure {
  const char* name;
  int status;
};

void check(const char* name, int status) {
  if (status != SMX_OK) throw Failure{name, status};
}

template <typename Call> auto raising(Call call) -> decltype(call()) {
  try {
    py::gil_scoped_release free;  // (the allocator may wait for the GPU)
    return call();
  } catch (const Failure& f) {
    py::module_::import("ae_amd._lib").attr("check")(f.name, f.status);
    throw;
  }
}

// The same in the engine's thread.
template <typename Call> auto failing(Call call) -> decltype(call()) {
  try {
    return call();
  } catch (const Failure& f) {
    throw std::runtime_error(text(f.name, " failed with status ", f.status, ": ", smx_error_string(f.status)));
  }
}

// ---- operands ------------------------------------------------------------------------------------

int code_of(at::ScalarType t) {
  return t == at::kFloat ? 0 : t == at::kHalf ? 1 : t == at::kBFloat16 ? 2 : -1;
}

void check_dtype(const Tensor& t) {
  if (code_of(t.scalar_type()) < 0)
    throw py::type_error(text("unsupported dtype ", dtype_text(t), "; expected float32, float16 or bfloat16"));
}

void check_gpu(const Tensor& t) {
  if (!t.is_cuda()) throw py::value_error(text("expected a GPU tensor, got one on ", t.device().str()));
}

void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

void* address(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
template <typename T> T* address(const Tensor& t) { return static_cast<T*>(address(t)); }

// Elements side by side, with their sign (z.conj().imag keeps it in a flag of the tensor).
Tensor dense(const Tensor& t) { return !t.defined() || (t.is_contiguous() && !t.is_neg()) ? t : t.resolve_neg().contiguous(); }
Tensor defined(const Maybe& t) { return t.has_value() ? *t : Tensor(); }

Tensor empty(c10::IntArrayRef shape, const Tensor& like, at::ScalarType type) {
  return at::empty(shape, at::TensorOptions().dtype(type).device(like.device()));
}
Tensor scratch(size_t bytes, const Tensor& like) {
  return bytes ? empty({static_cast<int64_t>(bytes)}, like, at::kByte) : Tensor();
}

// A matrix of rows with adjacent elements, and their distance (a copy where needed).
struct Rows {
  Tensor t;
  int64_t stride = 0;

  explicit Rows(const Tensor& of) : t(of) {
    if (!t.defined()) return;
    const int64_t n = t.size(-1);
    stride = n;
    if (t.is_neg()) t = t.resolve_neg();
    if (t.is_contiguous()) return;
    if (t.dim() != 2) t = t.reshape({-1, n});
    if ((t.stride(1) != 1 && n != 1) || (t.stride(0) < n && t.size(0) > 1)) t = t.contiguous();
    if (t.size(0) > 1) stride = t.stride(0);
  }
  void* data() const { return address(t); }
};

bool records(std::initializer_list<const Tensor*> tensors) {
  if (!c10::GradMode::is_enabled()) return false;
  for (const Tensor* t : tensors)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

// Whether a trace is recorded: it would hold the allocation of a result and not the kernel that fills it.
bool traced() {
  using c10::impl::TorchDispatchModeKey, c10::impl::TorchDispatchModeTLS;
  if (torch::jit::tracer::isTracing()) return true;
  if (!TorchDispatchModeTLS::any_modes_set()) return false;
  for (const auto key : {TorchDispatchModeKey::PROXY, TorchDispatchModeKey::FAKE, TorchDispatchModeKey::FUNCTIONAL})
    if (TorchDispatchModeTLS::get_mode(key).has_value()) return true;
  return false;
}

// Refuses what the kernels would not see: traces, tensors that stand for others under a transform, and the tangents of
// forward-mode duals.
void check_plain(const char* name, at::TensorList tensors) {
  using c10::DispatchKey;
  constexpr c10::DispatchKeySet wrapped({DispatchKey::FuncTorchBatched, DispatchKey::FuncTorchGradWrapper, DispatchKey::Batched, DispatchKey::Functionalize});
  if (traced()) throw std::runtime_error(text(name, " cannot be traced"));
  for (const Tensor& t : tensors) {
    if (!t.defined()) continue;
    if (t.key_set().has_any(wrapped)) throw std::runtime_error(text(name, " does not run under vmap or another transform of torch.func"));
    if (t._fw_grad(0).defined()) throw std::runtime_error(text(name, " has no forward-mode derivative"));
  }
}

// Where a graph of the gradients themselves is recorded, they depend on deps in a way that it cannot differentiate, and says so
// if it comes to that.
struct Once : torch::autograd::Function<Once> {
  static Tensor forward(AutogradContext* ctx, const Tensor& grad, at::TensorList, std::string name) {
    ctx->saved_data["name"] = std::move(name);
    return grad;
  }
  static variable_list backward(AutogradContext* ctx, variable_list) {
    throw std::runtime_error(text(ctx->saved_data["name"].toStringRef(), " is differentiable once"));
  }
};

template <typename Make> variable_list once(const char* name, variable_list deps, Make make) {
  check_plain(name, deps);
  if (!c10::GradMode::is_enabled()) return failing(make);
  variable_list grads, some;
  {
    c10::NoGradGuard off;
    grads = failing(make);
  }
  for (const Tensor& t : deps)
    if (t.defined()) some.push_back(t);
  for (Tensor& g : grads)
    if (g.defined()) g = Once::apply(g, at::TensorList(some), std::string(name));
  return grads;
}

// ---- norms ---------------------------------------------------------------------------------------

constexpr const char* kNorm = "a norm";

at::ScalarType params_type(const Tensor& weight, const Tensor& bias, const Tensor& x) {
  return weight.defined() ? weight.scalar_type() : bias.defined() ? bias.scalar_type() : x.scalar_type();
}

void check_norm(const Tensor& x, const Tensor& weight, const Tensor& bias, double eps, const Tensor& residual) {
  if (x.dim() < 1 || x.size(-1) == 0) throw py::value_error(text("x must be [..., H], got ", shape_text(x.sizes())));
  check_dtype(x);
  if (!(eps >= 0.0)) throw py::value_error(text("eps must not be negative, got ", eps));
  const c10::IntArrayRef row(x.sizes().end() - 1, 1);
  auto one = [&](const char* name, const Tensor& t, c10::IntArrayRef shape, bool wide) {
    if (!t.defined()) return;
    if (t.sizes() != shape) throw py::value_error(text(name, " must be ", shape_text(shape), ", got ", shape_text(t.sizes())));
    if (t.device() != x.device()) throw py::value_error(text("x is on ", x.device().str(), ", ", name, " on ", t.device().str()));
    if (t.scalar_type() != x.scalar_type() && !(wide && t.scalar_type() == at::kFloat))
      throw py::type_error(text("dtype mismatch: x is ", dtype_text(x), ", ", name, " ", dtype_text(t)));
  };
  one("weight", weight, row, true);
  one("bias", bias, row, true);
  one("residual", residual, x.sizes(), false);
  if (weight.defined() && bias.defined() && weight.scalar_type() != bias.scalar_type())
    throw py::type_error(text("dtype mismatch: weight is ", dtype_text(weight), ", bias ", dtype_text(bias)));
  check_gpu(x);
}

struct NormResult { Tensor y, sum, stats; };

// y, the sum (none without a residual), and the rows' statistics where the gradient needs them.
NormResult norm_forward(int kind, const Tensor& x, const Tensor& weight, const Tensor& bias, double eps, const Tensor& residual, bool keep) {
  const c10::DeviceGuard guard(x.device());
  const int64_t h = x.size(-1), rows = x.numel() / h;
  const Rows xm(x), rm(residual);
  const Tensor w = dense(weight), b = dense(bias);
  NormResult out;
  out.y = empty(x.sizes(), x, x.scalar_type());
  if (residual.defined()) out.sum = empty(x.sizes(), x, x.scalar_type());
  if (keep) out.stats = empty({kind == SMX_NORM_RMS ? rows : 2 * rows}, x, at::kFloat);
  check("smx_norm", smx_norm(kind, xm.data(), xm.stride, rm.data(), rm.stride, code_of(x.scalar_type()), rows, h, address(w), address(b),
                             code_of(params_type(weight, bias, x)), static_cast<float>(eps), address(out.y), address(out.sum),
                             address<float>(out.stats), stream_of(x)));
  return out;
}

// Gradients of x (and the residual), the weight and the bias.
variable_list norm_backward(int kind, at::ScalarType params, const Tensor& dy, const Tensor& dsum, const Tensor& s, const Tensor& weight,
                            const Tensor& stats, bool need_x, bool need_w, bool need_b) {
  const c10::DeviceGuard guard(s.device());
  const int64_t h = s.size(-1), rows = s.numel() / h;
  Tensor dx, dw, db, ws;
  if (!dy.defined()) {  // only the sum was used
    const auto options = at::TensorOptions().dtype(params).device(s.device());
    if (need_w) dw = at::zeros({h}, options);
    if (need_b) db = at::zeros({h}, options);
    return {need_x ? dsum : Tensor(), dw, db};
  }
  const Rows sm(s), dm(dy), rm(dsum);
  const Tensor w = dense(weight);
  const int dtype = code_of(s.scalar_type());
  size_t bytes = 0;
  if (need_x) dx = empty(s.sizes(), s, s.scalar_type());
  if (need_w) dw = empty({h}, s, params);
  if (need_b) db = empty({h}, s, params);
  if (need_w || need_b) bytes = smx_norm_grad_workspace_size(kind, rows, h, dtype);
  ws = scratch(bytes, s);
  check("smx_norm_grad", smx_norm_grad(kind, dm.data(), dm.stride, rm.data(), rm.stride, sm.data(), sm.stride, dtype, rows, h, address(w),
                                       code_of(params), address<float>(stats), address(dx), address(dw), address(db), address(ws), bytes,
                                       stream_of(s)));
  return {dx, dw, db};
}

// Which of a node's operands a backward pass wants: those that are there are numbered.
struct Wanted {
  AutogradContext* ctx;
  size_t next = 0;
  bool operator()(bool there) { return there && ctx->needs_input_grad(next++); }
};

struct Norm : torch::autograd::Function<Norm> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Maybe& weight, const Maybe& bias, const Maybe& residual,
                               int64_t kind, double eps) {
    const Tensor w = defined(weight), b = defined(bias), r = defined(residual);
    const NormResult out = norm_forward(static_cast<int>(kind), x, w, b, eps, r, true);
    ctx->save_for_backward({r.defined() ? out.sum : x, w, out.stats});
    ctx->saved_data["kind"] = kind;
    ctx->saved_data["params"] = static_cast<int64_t>(params_type(w, b, x));
    ctx->saved_data["there"] = int64_t{1} * w.defined() + 2 * b.defined() + 4 * r.defined();
    ctx->set_materialize_grads(false);
    return r.defined() ? variable_list{out.y, out.sum} : variable_list{out.y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const int64_t there = ctx->saved_data["there"].toInt();
    const Tensor dy = grads[0], dsum = grads.size() > 1 ? grads[1] : Tensor();
    if (!dy.defined() && !dsum.defined()) return variable_list(6);
    Wanted wanted{ctx};
    const bool x = wanted(true), w = wanted(there & 1), b = wanted(there & 2), r = wanted(there & 4);
    const variable_list saved = ctx->get_saved_variables();  // as autograd hands them back: perhaps not at their old addresses
    const variable_list d = once(kNorm, {dy, dsum, saved[0], saved[1]}, [&] {
      return norm_backward(static_cast<int>(ctx->saved_data["kind"].toInt()), static_cast<at::ScalarType>(ctx->saved_data["params"].toInt()),
                           dy, dsum, saved[0], saved[1], saved[2], x || r, w, b);
    });
    return {x ? d[0] : Tensor(), d[1], d[2], r ? d[0] : Tensor(), Tensor(), Tensor()};
  }
};

py::object norm(int kind, const Tensor& x, const Maybe& weight, const Maybe& bias, double eps, const Maybe& residual) {
  const Tensor w = defined(weight), b = defined(bias), r = defined(residual);
  check_plain(kNorm, {x, w, b, r});
  check_norm(x, w, b, eps, r);
  const bool train = records({&x, &w, &b, &r});
  const variable_list out = raising([&] {
    if (train) return Norm::apply(x, weight, bias, residual, int64_t{kind}, eps);
    const NormResult n = norm_forward(kind, x, w, b, eps, r, false);
    return variable_list{n.y, n.sum};
  });
  return r.defined() ? py::object(py::make_tuple(out[0], out[1])) : py::cast(out[0]);
}

py::object layer_norm(const Tensor& x, const Maybe& weight, const Maybe& bias, double eps, const Maybe& residual) {
  return norm(SMX_NORM_LAYER, x, weight, bias, eps, residual);
}

py::object rms_norm(const Tensor& x, const Maybe& weight, double eps, const Maybe& residual) {
  return norm(SMX_NORM_RMS, x, weight, std::nullopt, eps, residual);
}

// ---- routing -------------------------------------------------------------------------------------

constexpr const char* kRoute = "route_experts";

struct RouteOptions {
  int64_t k;
  int scoring;
  int64_t groups, top_groups;
  bool renormalize;
  double scale;
};

void check_route(const Tensor& logits, const std::string& scoring, const Tensor& bias, const RouteOptions& o) {
  if (logits.dim() != 2) throw py::value_error(text("logits must be [T, E], got ", shape_text(logits.sizes())));
  check_dtype(logits);
  const int64_t e = logits.size(1);
  if (o.scoring < 0) throw py::value_error(text("unknown scoring '", scoring, "'; expected one of ['softmax', 'sigmoid']"));
  if (o.groups < 1 || e % o.groups != 0 || o.top_groups < 1 || o.top_groups > o.groups)
    throw py::value_error(text(e, " experts in ", o.groups, " groups, ", o.top_groups, " of them selectable"));
  if (o.k < 1 || o.k > e / o.groups * o.top_groups)
    throw py::value_error(text("top_k ", o.k, " of ", e / o.groups * o.top_groups, " selectable experts"));
  if (!std::isfinite(static_cast<float>(o.scale))) throw py::value_error(text("scale must be finite, got ", o.scale));
  if (bias.defined()) {
    if (bias.dim() != 1 || bias.size(0) != e) throw py::value_error(text("bias must be (", e, ",), got ", shape_text(bias.sizes())));
    if (bias.device() != logits.device())
      throw py::value_error(text("logits are on ", logits.device().str(), ", bias on ", bias.device().str()));
    if (!bias.is_floating_point()) throw py::type_error(text("unsupported dtype ", dtype_text(bias), " of bias"));
    if (bias.requires_grad() && c10::GradMode::is_enabled())
      throw py::value_error("bias moves the choice, not the weights: it has no gradient. Pass it detached");
  }
  check_gpu(logits);
}

// Weights, ids, places, order, offsets.
variable_list route_forward(const Tensor& logits, const Tensor& bias, const RouteOptions& o) {
  const c10::DeviceGuard guard(logits.device());
  const int64_t t = logits.size(0), e = logits.size(1);
  const Rows m(logits);
  const Tensor b = bias.defined() ? dense(bias.scalar_type() == at::kFloat ? bias : bias.to(at::kFloat)) : bias;
  Tensor weights = empty({t, o.k}, logits, at::kFloat), ids = empty({t, o.k}, logits, at::kInt), places = empty({t, o.k}, logits, at::kInt),
         order = empty({t * o.k}, logits, at::kInt), offsets = empty({e + 1}, logits, at::kLong);
  const size_t bytes = smx_route_workspace_size(t, e, o.k);
  const Tensor ws = scratch(bytes, logits);
  check("smx_route", smx_route(m.data(), m.stride, code_of(logits.scalar_type()), t, e, o.k, o.scoring, address<float>(b), o.groups,
                               o.top_groups, o.renormalize, static_cast<float>(o.scale), address<float>(weights), address<int32_t>(ids),
                               address<int32_t>(places), address<int32_t>(order), address<int64_t>(offsets), address(ws), bytes,
                               stream_of(logits)));
  return {weights, ids, places, order, offsets};
}

struct Route : torch::autograd::Function<Route> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Maybe& bias, RouteOptions o) {
    variable_list out = route_forward(logits, defined(bias), o);
    ctx->save_for_backward({logits, out[1]});
    ctx->saved_data["scoring"] = int64_t{o.scoring};
    ctx->saved_data["renormalize"] = o.renormalize;
    ctx->saved_data["scale"] = o.scale;
    ctx->mark_non_differentiable({out[1], out[2], out[3], out[4]});
    ctx->set_materialize_grads(false);
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    if (!grads[0].defined()) return variable_list(3);
    const variable_list saved = ctx->get_saved_variables();
    const Tensor logits = saved[0], ids = saved[1];
    const variable_list d = once(kRoute, {grads[0], logits}, [&]() -> variable_list {
      const c10::DeviceGuard guard(logits.device());
      const Rows m(logits);
      const Tensor dw = dense(grads[0]), grad = empty(logits.sizes(), logits, logits.scalar_type());
      check("smx_route_grad",
            smx_route_grad(address<float>(dw), m.data(), m.stride, code_of(logits.scalar_type()), logits.size(0), logits.size(1), ids.size(1),
                           static_cast<int>(ctx->saved_data["scoring"].toInt()), ctx->saved_data["renormalize"].toBool(),
                           static_cast<float>(ctx->saved_data["scale"].toDouble()), address<int32_t>(ids), address(grad), stream_of(logits)));
      return {grad};
    });
    return {d[0], Tensor(), Tensor()};
  }
};

py::tuple route_experts(const Tensor& logits, int64_t top_k, const std::string& scoring, const Maybe& bias, int64_t num_groups,
                        std::optional<int64_t> top_groups, bool renormalize, double scale) {
  check_plain(kRoute, {logits});
  const RouteOptions o{top_k, scoring == "softmax" ? SMX_SCORE_SOFTMAX : scoring == "sigmoid" ? SMX_SCORE_SIGMOID : -1, num_groups,
                       top_groups.value_or(num_groups), renormalize, scale};
  check_route(logits, scoring, defined(bias), o);
  const variable_list r = raising([&] { return records({&logits}) ? Route::apply(logits, bias, o) : route_forward(logits, defined(bias), o); });
  return py::make_tuple(r[0], r[1], r[2], r[3], r[4]);
}

// ---- rows to the experts and back ------------------------------------------------------------------

constexpr const char *kDispatch = "dispatch_rows", *kCombine = "combine_rows";

void check_matrix(const char* name, const Tensor& t) {
  if (t.dim() != 2 || t.size(1) == 0) throw py::value_error(text(name, " must be [rows, H], got ", shape_text(t.sizes())));
  check_dtype(t);
}

void check_places(const Tensor& places, const Tensor& rows) {
  if (places.scalar_type() != at::kInt || places.dim() != 2 || !places.is_contiguous() || places.is_neg())
    throw py::type_error("places must be a contiguous int32 matrix [T, k]");
  if (places.device() != rows.device())
    throw py::value_error(text("expected a GPU tensor, places is on ", places.device().str(), ", the rows on ", rows.device().str()));
  if (places.size(1) == 0) throw py::value_error("places holds no picks");
}

Tensor spread(const Tensor& x, const Tensor& places) {
  const c10::DeviceGuard guard(x.device());
  const int64_t tokens = places.size(0), k = places.size(1), h = x.size(1);
  const Rows m(x);
  Tensor rows = empty({tokens * k, h}, x, x.scalar_type());
  check("smx_dispatch_rows", smx_dispatch_rows(m.data(), m.stride, code_of(x.scalar_type()), tokens, h, address<int32_t>(places), k,
                                               address(rows), stream_of(x)));
  return rows;
}

Tensor gather(const Tensor& rows, const Tensor& places, const Tensor& weights, const Tensor& residual) {
  const c10::DeviceGuard guard(rows.device());
  const int64_t tokens = places.size(0), k = places.size(1), h = rows.size(1);
  const Rows m(rows), r(residual);
  const Tensor w = dense(weights);
  Tensor y = empty({tokens, h}, rows, rows.scalar_type());
  check("smx_combine_rows", smx_combine_rows(m.data(), m.stride, code_of(rows.scalar_type()), tokens, h, address<int32_t>(places), k,
                                             address<float>(w), r.data(), r.stride, address(y), stream_of(rows)));
  return y;
}

struct Dispatch : torch::autograd::Function<Dispatch> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& places) {
    ctx->save_for_backward({places});
    ctx->set_materialize_grads(false);
    return spread(x, places);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    if (!grads[0].defined()) return variable_list(2);
    const Tensor places = ctx->get_saved_variables()[0];
    const variable_list d = once(kDispatch, {grads[0]}, [&] { return variable_list{gather(grads[0], places, Tensor(), Tensor())}; });
    return {d[0], Tensor()};
  }
};

struct Combine : torch::autograd::Function<Combine> {
  static Tensor forward(AutogradContext* ctx, const Tensor& rows, const Tensor& places, const Maybe& weights, const Maybe& residual) {
    const Tensor w = defined(weights);
    // (the rows are read again for the weights' gradient only)
    ctx->save_for_backward({w.defined() && w.requires_grad() ? rows : Tensor(), places, w});
    ctx->saved_data["columns"] = rows.size(1);
    ctx->saved_data["there"] = int64_t{1} * w.defined() + 2 * defined(residual).defined();
    ctx->set_materialize_grads(false);
    return gather(rows, places, w, defined(residual));
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const Tensor dy = grads[0];
    if (!dy.defined()) return variable_list(4);
    const int64_t there = ctx->saved_data["there"].toInt(), h = ctx->saved_data["columns"].toInt();
    Wanted wanted{ctx};
    const bool need_rows = wanted(true);
    wanted(true);  // places
    const bool need_w = wanted(there & 1), need_r = wanted(there & 2);
    variable_list d(2);
    if (need_rows || need_w) {
      const variable_list saved = ctx->get_saved_variables();
      const Tensor rows = need_w ? saved[0] : Tensor(), places = saved[1], weights = saved[2];
      d = once(kCombine, {dy, saved[0], weights}, [&]() -> variable_list {
        const c10::DeviceGuard guard(dy.device());
        const int64_t tokens = places.size(0), k = places.size(1);
        const Rows g(dy), m(rows);
        const Tensor w = dense(weights);
        Tensor drows, dw;
        if (need_rows) drows = empty({tokens * k, h}, dy, dy.scalar_type());
        if (need_w) dw = empty({tokens, k}, dy, at::kFloat);
        check("smx_combine_rows_grad",
              smx_combine_rows_grad(g.data(), g.stride, m.data(), m.stride, code_of(dy.scalar_type()), tokens, h, address<int32_t>(places), k,
                                    address<float>(w), address(drows), address<float>(dw), stream_of(dy)));
        return {drows, dw};
      });
    }
    return {d[0], Tensor(), d[1], need_r ? dy : Tensor()};
  }
};

Tensor dispatch_rows(const Tensor& x, const Tensor& places) {
  check_plain(kDispatch, {x});
  check_matrix("x", x);
  check_places(places, x);
  if (places.size(0) != x.size(0))
    throw py::value_error(text(x.size(0), " rows of x, places of ", places.size(0), " tokens"));
  check_gpu(x);
  return raising([&] { return records({&x}) ? Dispatch::apply(x, places) : spread(x, places); });
}

Tensor combine_rows(const Tensor& rows, const Tensor& places, const Maybe& weights, const Maybe& residual) {
  const Tensor w = defined(weights), r = defined(residual);
  check_plain(kCombine, {rows, w, r});
  check_matrix("rows", rows);
  check_places(places, rows);
  const int64_t tokens = places.size(0), picks = tokens * places.size(1);
  if (rows.size(0) != picks) throw py::value_error(text("places of ", picks, " picks, ", rows.size(0), " rows"));
  if (w.defined()) {
    if (w.sizes() != places.sizes())
      throw py::value_error(text("weights must be ", shape_text(places.sizes()), ", got ", shape_text(w.sizes())));
    if (w.scalar_type() != at::kFloat) throw py::type_error(text("weights must be fp32, got ", dtype_text(w)));
  }
  if (r.defined()) {
    if (r.dim() != 2 || r.size(0) != tokens || r.size(1) != rows.size(1))
      throw py::value_error(text("residual must be (", tokens, ", ", rows.size(1), "), got ", shape_text(r.sizes())));
    if (r.scalar_type() != rows.scalar_type())
      throw py::type_error(text("dtype mismatch: rows are ", dtype_text(rows), ", residual ", dtype_text(r)));
  }
  for (const auto& [name, t] : {std::pair<const char*, const Tensor&>{"weights", w}, {"residual", r}})
    if (t.defined() && t.device() != rows.device())
      throw py::value_error(text("rows are on ", rows.device().str(), ", ", name, " on ", t.device().str()));
  check_gpu(rows);
  return raising([&] { return records({&rows, &w, &r}) ? Combine::apply(rows, places, weights, residual) : gather(rows, places, w, r); });
}

}  // namespace

PYBIND11_MODULE(_blocks, m) {
  m.def("layer_norm", torch::wrap_pybind_function(layer_norm));
  m.def("rms_norm", torch::wrap_pybind_function(rms_norm));
  m.def("route_experts", torch::wrap_pybind_function(route_experts));
  m.def("dispatch_rows", torch::wrap_pybind_function(dispatch_rows));
  m.def("combine_rows", torch::wrap_pybind_function(combine_rows));
}
