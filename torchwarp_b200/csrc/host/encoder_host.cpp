// Eager calls of the encoder operators: argument checks, allocation, autograd
// and the calls of the C ABI in one C++ module.
//
// A call on a few rows takes less time on the GPU than its host side takes in
// Python (layer norm of 4 rows: 2 us against 12; its training pass 107), so
// the host side is C++: one conversion of the arguments, no interpreter in
// the backward.  Backward passes are first order: their results carry a node
// that raises when it is differentiated.
#include <ATen/TracerMode.h>
#include <ATen/autocast_mode.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <optional>
#include <string>
#include <vector>

#include "../../../include/torchwarp_b200.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

// A C ABI call's failure; Python sees torchwarp_b200._native.NativeError.
struct NativeError : std::runtime_error {
  using std::runtime_error::runtime_error;
};

void check_status(int status, const char* what) {
  if (status != TW_OK)
    throw NativeError(std::string(what) + " failed (status " + std::to_string(status) +
                      "): " + tw_last_error());
}

// Checks compare sym_size, so that they also hold for a tracer's tensors, whose
// sizes may be symbols.
std::string text_of(const c10::SymInt& n) {
  const auto v = n.maybe_as_int();
  return v ? std::to_string(*v) : n.toSymNodeImplUnowned()->str();
}
std::string shape_of(const Tensor& t) {
  std::string s = "[";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + text_of(t.sym_size(i));
  return s + "]";
}

std::string type_of(at::ScalarType t) {
  std::string s = at::toString(t);
  return t == at::kFloat ? "float32" : t == at::kBFloat16 ? "bfloat16" : t == at::kHalf ? "float16" : s;
}

[[noreturn]] void bad_value(const std::string& msg) { throw py::value_error(msg); }
[[noreturn]] void bad_type(const std::string& msg) { throw py::type_error(msg); }

bool supported(at::ScalarType t) {
  return t == at::kFloat || t == at::kBFloat16 || t == at::kHalf;
}
void check_type(const char* name, const Tensor& t) {
  if (!supported(t.scalar_type()))
    bad_type(std::string(name) + " must be float32, bfloat16 or float16, got " +
             type_of(t.scalar_type()));
}
void check_same_type(const char* name, const Tensor& t, const Tensor& x) {
  if (t.scalar_type() != x.scalar_type())
    bad_type(std::string(name) + " must be of x's type " + type_of(x.scalar_type()) + ", got " +
             type_of(t.scalar_type()));
}
void require_cuda(const Tensor& t) {
  if (!t.is_cuda())
    throw std::runtime_error("torchwarp_b200 runs only on CUDA tensors (B200, sm_100a); got a "
                             "tensor on " + t.device().str() + ". There is no CPU fallback.");
}
// `first` and those of `others` that are there lie on one GPU.
void check_devices(const Tensor& first, std::initializer_list<const Tensor*> others) {
  require_cuda(first);
  for (const Tensor* t : others) {
    if (!t->defined()) continue;
    require_cuda(*t);
    if (t->device() != first.device())
      bad_value("all tensors must be on one device, got " + first.device().str() + " and " +
                t->device().str());
  }
}

bool wants_grad(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

// Whether a call has to go through the dispatcher: torch.jit.trace, a dispatch
// mode (make_fx, fake tensors), a transform or a tensor subclass would see only
// the allocation of an eager call's results.
bool dispatched(std::initializer_list<const Tensor*> ts) {
  if (at::tracer::impl::is_dispatch_enabled() ||
      c10::impl::TorchDispatchModeTLS::any_modes_set())
    return true;
  constexpr c10::DispatchKeySet wrapped({c10::DispatchKey::Python, c10::DispatchKey::Functionalize,
                                         c10::DispatchKey::FuncTorchBatched,
                                         c10::DispatchKey::FuncTorchGradWrapper});
  for (const Tensor* t : ts)
    if (t->defined() && t->key_set().has_any(wrapped)) return true;
  return false;
}
// The custom op of that name.
py::object op(const char* name) {
  return py::module_::import("torchwarp_b200.encoder._ops").attr(name);
}

// The operators have no forward-mode derivative: a tangent is refused, not lost.
void no_tangents(const char* name, std::initializer_list<const Tensor*> ts) {
  for (const Tensor* t : ts)
    if (t->defined() && t->_fw_grad(0).defined())
      throw std::runtime_error(std::string(name) + " has no forward-mode derivative; its "
                               "backward is first order");
}

void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

Tensor dense_like(const Tensor& x) { return at::empty(x.sizes(), x.options()); }

Tensor bytes(size_t n, const Tensor& like) {
  return n ? at::empty({(int64_t)n}, like.options().dtype(at::kByte)) : Tensor();
}

// x with its last dimension contiguous and its leading ones collapsed to rows
// `stride` elements apart: itself or a view where that is possible, else a
// copy.
struct Rows {
  Tensor t;
  int64_t stride;
};
Rows rows_of(const Tensor& x) {
  if (x.is_contiguous()) return {x, x.size(-1)};
  Tensor r = x.reshape({-1, x.size(-1)});
  if (r.stride(1) != 1 && r.size(1) != 1) r = r.contiguous();
  return {r, r.stride(0)};
}
Tensor frames_of(const Tensor& x) {
  return x.stride(2) == 1 || x.size(2) == 1 ? x : x.contiguous();
}

// Optional arguments are undefined tensors here, but std::optional where
// autograd sees them: an autograd Function counts only the tensors it is given.
OptTensor opt(const Tensor& t) { return t.defined() ? OptTensor(t) : std::nullopt; }
Tensor def(const OptTensor& t) { return t.value_or(Tensor()); }
Tensor dense(const Tensor& t) { return t.defined() ? t.contiguous() : t; }

// The entry of the element type.
#define TW_PICK(NAME, TYPE)                                                              \
  ((TYPE) == at::kFloat      ? NAME##_f32                                                \
   : (TYPE) == at::kBFloat16 ? NAME##_bf16                                               \
   : (TYPE) == at::kHalf     ? NAME##_f16                                                \
                             : throw py::type_error("no " #NAME " of " + type_of(TYPE)))

void* stream_of(const Tensor& t) {
  return (void*)c10::cuda::getCurrentCUDAStream(t.device().index()).stream();
}

// Results of a first-order backward: under create_graph they stay tied to a
// node that raises when a second derivative reaches it.
variable_list first_order(variable_list out) {
  if (!at::GradMode::is_enabled()) return out;
  std::vector<size_t> at;
  variable_list in;
  for (size_t i = 0; i < out.size(); ++i)
    if (out[i].defined()) {
      at.push_back(i);
      in.push_back(out[i].detach().requires_grad_(true));
    }
  auto node = std::make_shared<torch::autograd::DelayedError>(
      "trying to differentiate twice a function that was marked once-differentiable "
      "(a first-order native backward)", (int64_t)in.size());
  variable_list tied = (*node)(std::move(in));
  for (size_t i = 0; i < at.size(); ++i) out[at[i]] = tied[i];
  return out;
}

void check_shape_of(const char* name, const Tensor& t, const Tensor& x) {
  if (t.sym_sizes() != x.sym_sizes())
    bad_value(std::string(name) + " must have x's shape " + shape_of(x) + ", got " + shape_of(t));
}

// -------------------------------------------------------------- layer norm

void check_parameter(const char* name, const Tensor& p, const Tensor& x) {
  if (p.dim() != 1 || p.sym_size(0) != x.sym_size(-1))
    bad_value(std::string(name) + " must have shape [" + text_of(x.sym_size(-1)) + "], got " +
              shape_of(p));
  if (p.scalar_type() != x.scalar_type() && p.scalar_type() != at::kFloat)
    bad_type(std::string(name) + " must be float32 or of x's type " + type_of(x.scalar_type()) +
             ", got " + type_of(p.scalar_type()));
}

// The checks of a call, whichever way it comes: eager, or through the custom
// ops and their fakes.
void check_layer_norm(const Tensor& x, const Tensor& w, const Tensor& b, double eps) {
  check_type("x", x);
  if (x.dim() < 1 || x.sym_size(-1) == 0) bad_value("x must have shape [..., D] with D > 0");
  if (x.sym_size(-1) > INT_MAX) bad_value("x must have fewer than 2^31 columns");
  if (w.defined()) check_parameter("weight", w, x);
  if (b.defined()) check_parameter("bias", b, x);
  if (w.defined() && b.defined() && w.scalar_type() != b.scalar_type())
    bad_type("weight and bias must have one type");
  if (!(eps >= 0)) bad_value("eps must be >= 0");
  check_devices(x, {&w, &b});
}
void check_layer_norm_backward(const Tensor& dy, const Tensor& x, const Tensor& w, const Tensor& b,
                               const Tensor& stats) {
  check_shape_of("dy", dy, x);
  if (x.dim() < 1 || stats.dim() != 2 || stats.sym_size(0) != 2 ||
      stats.sym_size(1) * x.sym_size(-1) != x.sym_numel() || stats.scalar_type() != at::kFloat ||
      !stats.is_contiguous())
    bad_value("stats must be what the forward saved");
  check_layer_norm(x, w, b, 0);
  check_devices(x, {&dy, &stats});
}

std::tuple<Tensor, Tensor> layer_norm_forward(const Tensor& x, const Tensor& w, const Tensor& b,
                                              double eps, bool save) {
  const int64_t d = x.size(-1), rows = x.numel() / d;
  Tensor y = dense_like(x);
  Tensor stats = save ? at::empty({2, rows}, x.options().dtype(at::kFloat)) : Tensor();
  if (rows) {
    c10::cuda::CUDAGuard guard(x.device());
    const Rows r = rows_of(x);
    const Tensor& param = w.defined() ? w : b;
    float* mean = save ? stats.data_ptr<float>() : nullptr;
    check_status(TW_PICK(tw_layer_norm_forward, x.scalar_type())(
                     ptr(r.t), r.stride, ptr(w), ptr(b),
                     param.defined() && param.scalar_type() != x.scalar_type(), rows, (int)d, eps,
                     ptr(y), mean, save ? mean + rows : nullptr, stream_of(x)),
                 "tw_layer_norm_forward");
  }
  return {y, stats};
}

std::tuple<Tensor, Tensor, Tensor> layer_norm_backward(const Tensor& dy_in, const Tensor& x,
                                                       const Tensor& w, at::ScalarType ptype,
                                                       const Tensor& stats, bool ndx, bool ndw,
                                                       bool ndb) {
  const int64_t d = x.size(-1), rows = x.numel() / d;
  Tensor dx, dw, db;
  if (ndx) dx = dense_like(x);
  if (ndw) dw = at::empty({d}, x.options().dtype(ptype));
  if (ndb) db = at::empty({d}, x.options().dtype(ptype));
  if (ndx || ndw || ndb) {
    c10::cuda::CUDAGuard guard(x.device());
    const Rows r = rows_of(x), g = rows_of(dy_in.to(x.scalar_type()));
    const size_t n = tw_layer_norm_workspace_bytes(rows, (int)d);
    Tensor ws = bytes(n, x);
    const float* mean = stats.data_ptr<float>();
    check_status(TW_PICK(tw_layer_norm_backward, x.scalar_type())(
                     ptr(g.t), g.stride, ptr(r.t), r.stride, ptr(w), ptype != x.scalar_type(),
                     mean, mean + rows, rows, (int)d, ptr(dx), ptr(dw), ptr(db), ptr(ws), n,
                     stream_of(x)),
                 "tw_layer_norm_backward");
  }
  return {dx, dw, db};
}

struct LayerNormFn : torch::autograd::Function<LayerNormFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptTensor& weight,
                        const OptTensor& bias, double eps) {
    const Tensor w = def(weight), b = def(bias);
    auto [y, stats] = layer_norm_forward(x, w, b, eps, true);
    ctx->save_for_backward({x, w, stats});
    ctx->saved_data["ptype"] = (int64_t)(w.defined()   ? w.scalar_type()
                                         : b.defined() ? b.scalar_type()
                                                       : x.scalar_type());
    ctx->saved_data["bias"] = b.defined();
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const variable_list s = ctx->get_saved_variables();
    const bool has_w = s[1].defined(), has_b = ctx->saved_data["bias"].toBool();
    auto [dx, dw, db] = layer_norm_backward(
        g[0], s[0], s[1], (at::ScalarType)ctx->saved_data["ptype"].toInt(), s[2],
        ctx->needs_input_grad(0), has_w && ctx->needs_input_grad(1),
        has_b && ctx->needs_input_grad(1 + has_w));
    return first_order({dx, dw, db, Tensor()});
  }
};

Tensor layer_norm(const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps) {
  Tensor w = def(weight), b = def(bias);
  no_tangents("layer_norm", {&x, &w, &b});
  if (dispatched({&x, &w, &b}))
    return op("layer_norm")(x, weight, bias, eps)
        .cast<std::pair<Tensor, Tensor>>().first;
  check_layer_norm(x, w, b, eps);
  w = dense(w);
  b = dense(b);
  if (wants_grad({&x, &w, &b})) return LayerNormFn::apply(x, opt(w), opt(b), eps);
  return std::get<0>(layer_norm_forward(x, w, b, eps, false));
}

// ------------------------------------------------------------------ linear

// A tensor's shape is x's but for its last dimension, `n`.
bool rows_like(const Tensor& t, const Tensor& x, const c10::SymInt& n) {
  bool same = t.dim() == x.dim() && t.sym_size(-1) == n;
  for (int64_t i = 0; same && i + 1 < x.dim(); ++i) same = t.sym_size(i) == x.sym_size(i);
  return same;
}

void check_linear(const Tensor& x, const Tensor& w, const Tensor& b, const Tensor& r) {
  check_type("x", x);
  if (w.dim() != 2 || w.sym_size(0) == 0 || w.sym_size(1) == 0)
    bad_value("weight must have shape [N, K] with N, K > 0");
  const c10::SymInt n = w.sym_size(0), k = w.sym_size(1);
  if (x.dim() < 1 || x.sym_size(-1) != k)
    bad_value("x must have shape [..., " + text_of(k) + "], got " + shape_of(x));
  if (b.defined() && (b.dim() != 1 || b.sym_size(0) != n))
    bad_value("bias must have shape [" + text_of(n) + "], got " + shape_of(b));
  if (r.defined() && !rows_like(r, x, n))
    bad_value("residual must have the result's shape [..., " + text_of(n) + "], got " +
              shape_of(r));
  check_same_type("weight", w, x);
  if (b.defined()) check_same_type("bias", b, x);
  if (r.defined()) check_same_type("residual", r, x);
  check_devices(x, {&w, &b, &r});
}
void check_linear_backward(const Tensor& dy, const Tensor& x, const Tensor& w, const Tensor& z,
                           int64_t act) {
  if (x.dim() < 1 || w.dim() != 2 || !rows_like(dy, x, w.sym_size(0)))
    bad_value("dy must have the result's shape, got " + shape_of(dy));
  if (act && (!z.defined() || z.dim() != 2 || z.sym_size(0) * w.sym_size(1) != x.sym_numel() ||
              z.sym_size(1) != w.sym_size(0) || z.scalar_type() != x.scalar_type() ||
              !z.is_contiguous()))
    bad_value("z must be what the forward saved");
  check_linear(x, w, Tensor(), Tensor());
  check_devices(x, {&dy, &z});
}

// 1 when a row of 16-bit elements may start off a 16-byte boundary.
int unaligned(const Rows& r) {
  return ((uintptr_t)r.t.data_ptr() & 15) != 0 || (r.stride & 7) != 0 || r.stride < r.t.size(-1);
}

std::tuple<Tensor, Tensor> linear_forward(const Tensor& x, const Tensor& w, const Tensor& bias,
                                          const Tensor& res, int64_t act, bool save) {
  const int64_t n = w.size(0), k = w.size(1), m = x.numel() / k;
  std::vector<int64_t> shape = x.sizes().vec();
  shape.back() = n;
  Tensor y = at::empty(shape, x.options());
  Tensor z = save && act ? at::empty({m, n}, x.options()) : Tensor();
  if (m) {
    TORCH_CHECK(m <= INT_MAX && n <= INT_MAX && k <= INT_MAX, "linear: a size is too large");
    c10::cuda::CUDAGuard guard(x.device());
    const Rows xr = rows_of(x), wr = rows_of(w);
    Rows rr{Tensor(), 0};
    if (res.defined()) rr = rows_of(res);
    const size_t bytes_needed = tw_linear_workspace_bytes(
        (int)m, (int)n, (int)k, (int)x.element_size(), (int)act, 0, unaligned(xr) | unaligned(wr));
    Tensor ws = bytes(bytes_needed, x);
    check_status(TW_PICK(tw_linear_forward, x.scalar_type())(
                     ptr(xr.t), xr.stride, ptr(wr.t), wr.stride, ptr(bias), ptr(rr.t), rr.stride,
                     (int)m, (int)n, (int)k, (int)act, ptr(y), ptr(z), ptr(ws), bytes_needed,
                     stream_of(x)),
                 "tw_linear_forward");
  }
  return {y, z};
}

std::tuple<Tensor, Tensor, Tensor> linear_backward(const Tensor& dy_in, const Tensor& x,
                                                   const Tensor& w, const Tensor& z, int64_t act,
                                                   bool ndx, bool ndw, bool ndb) {
  const int64_t n = w.size(0), k = w.size(1), m = x.numel() / k;
  Tensor dx, dw, db;
  if (ndx) dx = dense_like(x);
  if (ndw) dw = dense_like(w);
  if (ndb) db = at::empty({n}, x.options());
  if (ndx || ndw || ndb) {
    TORCH_CHECK(m <= INT_MAX, "linear: a size is too large");
    c10::cuda::CUDAGuard guard(x.device());
    const Rows g = rows_of(dy_in.to(x.scalar_type())), xr = rows_of(x), wr = rows_of(w);
    const size_t bytes_needed = tw_linear_workspace_bytes(
        (int)m, (int)n, (int)k, (int)x.element_size(), (int)act, 1,
        unaligned(xr) | unaligned(wr) | unaligned(g));
    Tensor ws = bytes(bytes_needed, x);
    check_status(TW_PICK(tw_linear_backward, x.scalar_type())(
                     ptr(g.t), g.stride, ptr(xr.t), xr.stride, ptr(wr.t), wr.stride, ptr(z), (int)m,
                     (int)n, (int)k, (int)act, ptr(dx), ptr(dw), ptr(db), ptr(ws), bytes_needed,
                     stream_of(x)),
                 "tw_linear_backward");
  }
  return {dx, dw, db};
}

struct LinearFn : torch::autograd::Function<LinearFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w,
                        const OptTensor& bias, const OptTensor& residual, int64_t act) {
    auto [y, z] = linear_forward(x, w, def(bias), def(residual), act, true);
    ctx->save_for_backward({x, w, z});
    ctx->saved_data["act"] = act;
    ctx->saved_data["bias"] = bias.has_value();
    ctx->saved_data["residual"] = residual.has_value();
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const variable_list s = ctx->get_saved_variables();
    const bool has_b = ctx->saved_data["bias"].toBool();
    const bool has_r = ctx->saved_data["residual"].toBool();
    auto [dx, dw, db] = linear_backward(g[0], s[0], s[1], s[2], ctx->saved_data["act"].toInt(),
                                        ctx->needs_input_grad(0), ctx->needs_input_grad(1),
                                        has_b && ctx->needs_input_grad(2));
    variable_list out = first_order({dx, dw, db});
    out.push_back(has_r && ctx->needs_input_grad(2 + has_b) ? g[0] : Tensor());
    out.push_back(Tensor());
    return out;
  }
};

Tensor linear(Tensor x, Tensor w, const OptTensor& bias, const OptTensor& residual, int64_t act) {
  Tensor b = bias.value_or(Tensor()), r = residual.value_or(Tensor());
  if (at::autocast::is_autocast_enabled(at::kCUDA)) {
    // torch's own rule and cache: float64 and integers keep their type (and are
    // refused), a weight is cast once a region
    const at::ScalarType t = at::autocast::get_autocast_dtype(at::kCUDA);
    for (Tensor* v : {&x, &w, &b, &r})
      if (v->defined()) *v = at::autocast::cached_cast(t, *v, at::kCUDA);
  }
  no_tangents("linear", {&x, &w, &b, &r});
  if (dispatched({&x, &w, &b, &r}))
    return op("linear")(x, w, opt(b), opt(r), act)
        .cast<std::pair<Tensor, Tensor>>().first;
  check_linear(x, w, b, r);
  b = dense(b);
  if (wants_grad({&x, &w, &b, &r})) return LinearFn::apply(x, w, opt(b), opt(r), act);
  return std::get<0>(linear_forward(x, w, b, r, act, false));
}

// -------------------------------------------------------------- gated scan

void check_gate(const Tensor& gate, const Tensor& x) {
  check_shape_of("gate", gate, x);
  check_same_type("gate", gate, x);
}
void check_state(const char* name, const Tensor& state, const Tensor& x) {
  const c10::SymInt batch = x.sym_size(0), dim = x.sym_size(-1);
  if (state.dim() != 2 || state.sym_size(0) != batch || state.sym_size(1) != dim)
    bad_value(std::string(name) + " must have shape [" + text_of(batch) + ", " + text_of(dim) +
              "], got " + shape_of(state));
}
void check_gated_scan(const Tensor& x, const Tensor& gate, const Tensor& h0,
                      const Tensor& lengths) {
  check_type("x", x);
  if (x.dim() != 3 || x.sym_size(2) == 0)
    bad_value("x must have shape [batch, time, feature] with features");
  check_gate(gate, x);
  if (h0.defined()) {
    check_state("state", h0, x);
    if (h0.scalar_type() != at::kFloat)
      bad_type("state must be float32, got " + type_of(h0.scalar_type()));
  }
  if (lengths.defined()) {
    if (lengths.dim() != 1 || lengths.sym_size(0) != x.sym_size(0))
      bad_value("lengths must have shape [" + text_of(x.sym_size(0)) + "], got " +
                shape_of(lengths));
    if (lengths.scalar_type() != at::kLong && lengths.scalar_type() != at::kInt)
      bad_type("lengths must be int64 or int32, got " + type_of(lengths.scalar_type()));
  }
  check_devices(x, {&gate, &h0, &lengths});
}
void check_gated_scan_backward(const Tensor& dy, const Tensor& dstate, const Tensor& x,
                               const Tensor& gate, const Tensor& lengths, const Tensor& carry) {
  if (dy.defined()) check_shape_of("dy", dy, x);
  if (x.dim() == 3 && dstate.defined()) check_state("dstate", dstate, x);
  if (carry.scalar_type() != at::kByte || !carry.is_contiguous())  // its size: the C ABI
    bad_value("carry must be what the forward saved");
  check_gated_scan(x, gate, Tensor(), lengths);
  check_devices(x, {&dy, &dstate, &carry});
}
// lengths as the kernels read them.
Tensor whole_lengths(const Tensor& lengths) {
  return lengths.defined() ? lengths.to(at::kLong).contiguous() : lengths;
}

int dim32(int64_t v) {
  TORCH_CHECK(v <= INT_MAX, "gated_scan: a size is too large");
  return (int)v;
}

std::tuple<Tensor, Tensor, Tensor> gated_scan_forward(const Tensor& x_in, const Tensor& gate_in,
                                                      const Tensor& h0_in, const Tensor& lengths,
                                                      bool save) {
  const int64_t b = x_in.size(0), t = x_in.size(1), d = x_in.size(2);
  Tensor y = dense_like(x_in);
  Tensor state = at::empty({b, d}, x_in.options().dtype(at::kFloat));
  // the saved states, and behind them the call's own scratch
  const int es = (int)x_in.element_size();
  const size_t scratch = tw_gated_scan_workspace_bytes(dim32(b), dim32(t), dim32(d), es);
  const size_t n = save ? tw_gated_scan_carry_bytes((int)b, (int)t, (int)d, es) : scratch;
  Tensor carry = bytes(n, x_in);
  if (b) {
    c10::cuda::CUDAGuard guard(x_in.device());
    const Tensor x = frames_of(x_in), gate = frames_of(gate_in);
    const Tensor h0 = h0_in.defined() ? h0_in.contiguous() : h0_in;
    check_status(TW_PICK(tw_gated_scan_forward, x.scalar_type())(
                     ptr(x), x.stride(0), x.stride(1), ptr(gate), gate.stride(0), gate.stride(1),
                     (const float*)ptr(h0), (const int64_t*)ptr(lengths), dim32(b), dim32(t),
                     dim32(d), ptr(y), state.data_ptr<float>(), ptr(carry), n, stream_of(x)),
                 "tw_gated_scan_forward");
  }
  if (save && !carry.defined()) carry = at::empty({0}, x_in.options().dtype(at::kByte));
  if (save && scratch) carry = carry.narrow(0, 0, (int64_t)(n - scratch));
  return {y, state, carry};
}

// dL/dy or dL/dstate may be undefined: zero.
std::tuple<Tensor, Tensor, Tensor> gated_scan_backward(const Tensor& dy_in, const Tensor& dstate_in,
                                                       const Tensor& x_in, const Tensor& gate_in,
                                                       const Tensor& lengths, const Tensor& carry) {
  const int64_t b = x_in.size(0), t = x_in.size(1), d = x_in.size(2);
  Tensor dx = dense_like(x_in), dgate = dense_like(x_in);
  Tensor dh0 = at::empty({b, d}, x_in.options().dtype(at::kFloat));
  if (b) {
    c10::cuda::CUDAGuard guard(x_in.device());
    const Tensor x = frames_of(x_in), gate = frames_of(gate_in);
    const Tensor dy =
        dy_in.defined() ? frames_of(dy_in.to(x.scalar_type())) : at::zeros_like(dx);
    const Tensor ds =
        dstate_in.defined() ? dstate_in.to(at::kFloat).contiguous() : dstate_in;
    const size_t n = tw_gated_scan_workspace_bytes(dim32(b), dim32(t), dim32(d),
                                                   (int)x.element_size());
    Tensor ws = bytes(n, x);
    check_status(TW_PICK(tw_gated_scan_backward, x.scalar_type())(
                     ptr(dy), dy.stride(0), dy.stride(1), (const float*)ptr(ds), ptr(x),
                     x.stride(0), x.stride(1), ptr(gate), gate.stride(0), gate.stride(1),
                     (const int64_t*)ptr(lengths), ptr(carry), (size_t)carry.numel(), dim32(b),
                     dim32(t), dim32(d), ptr(dx), ptr(dgate), dh0.data_ptr<float>(), ptr(ws), n,
                     stream_of(x)),
                 "tw_gated_scan_backward");
  }
  return {dx, dgate, dh0};
}

struct GatedScanFn : torch::autograd::Function<GatedScanFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& gate,
                               const OptTensor& h0, const OptTensor& lengths) {
    auto [y, state, carry] = gated_scan_forward(x, gate, def(h0), def(lengths), true);
    ctx->save_for_backward({x, gate, def(lengths), carry});
    ctx->saved_data["state"] = h0.has_value();
    ctx->set_materialize_grads(false);
    return {y, state};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    if (!g[0].defined() && !g[1].defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
    const variable_list s = ctx->get_saved_variables();
    auto [dx, dgate, dh0] = gated_scan_backward(g[0], g[1], s[0], s[1], s[2], s[3]);
    return first_order({dx, dgate, ctx->saved_data["state"].toBool() ? dh0 : Tensor(), Tensor()});
  }
};

std::tuple<Tensor, Tensor> gated_scan(const Tensor& x, const Tensor& gate, const OptTensor& state,
                                      const OptTensor& lengths_in) {
  const Tensor h0 = def(state), n = def(lengths_in);
  no_tangents("gated_scan", {&x, &gate, &h0});
  if (dispatched({&x, &gate, &h0, &n})) {
    auto out = op("gated_scan")(x, gate, state, lengths_in)
                   .cast<std::tuple<Tensor, Tensor, Tensor>>();
    return {std::get<0>(out), std::get<1>(out)};
  }
  check_gated_scan(x, gate, h0, n);
  const Tensor lengths = whole_lengths(n);
  if (wants_grad({&x, &gate, &h0})) {
    variable_list out = GatedScanFn::apply(x, gate, opt(h0), opt(lengths));
    return {out[0], out[1]};
  }
  auto [y, last, carry] = gated_scan_forward(x, gate, h0, lengths, false);
  return {y, last};
}

void check_gated_scan_step(const Tensor& x, const Tensor& gate, const Tensor& state) {
  check_type("x", x);
  if (x.dim() != 2 || x.size(1) == 0)
    bad_value("x must have shape [batch, feature] with features");
  check_gate(gate, x);
  if (!state.defined()) bad_value("state must be a [B,D] tensor: it is updated in place");
  check_state("state", state, x);
  if (state.scalar_type() != at::kFloat)
    bad_type("state must be float32, got " + type_of(state.scalar_type()));
  if (!state.is_contiguous()) bad_value("state must be contiguous: it is updated in place");
  check_devices(x, {&gate, &state});
  if (wants_grad({&x, &gate, &state}))
    throw std::runtime_error("gated_scan_step is not differentiable; use gated_scan, or no_grad");
}

Tensor gated_scan_step_forward(const Tensor& x, const Tensor& gate, const Tensor& state) {
  const int64_t b = x.size(0), d = x.size(1);
  Tensor y = dense_like(x);
  if (b) {
    c10::cuda::CUDAGuard guard(x.device());
    const Rows xr = rows_of(x), gr = rows_of(gate);
    check_status(TW_PICK(tw_gated_scan_step, x.scalar_type())(
                     ptr(xr.t), xr.stride, ptr(gr.t), gr.stride, state.data_ptr<float>(), dim32(b),
                     dim32(d), ptr(y), stream_of(x)),
                 "tw_gated_scan_step");
  }
  return y;
}

Tensor gated_scan_step(const Tensor& x, const Tensor& gate, const OptTensor& state_in) {
  const Tensor state = def(state_in);
  no_tangents("gated_scan_step", {&x, &gate, &state});
  check_gated_scan_step(x, gate, state);
  if (dispatched({&x, &gate, &state})) return op("gated_scan_step")(x, gate, state).cast<Tensor>();
  const Tensor y = gated_scan_step_forward(x, gate, state);
  // written through a raw pointer: autograd has to see the change
  if (!state.is_inference()) state.unsafeGetTensorImpl()->bump_version();
  return y;
}

// ------------------------------------------------------------------ AdamW

// One AdamW step (or, CHECK, its checks alone) over `params`, which had `sizes` values each when the flat
// buffers of their states were made, one after the other on boundaries of 256
// values; a parameter without a gradient is left out, and with none at all
// nothing is done.
template <bool CHECK>
void adamw_step(const std::vector<Tensor>& params, const std::vector<int64_t>& sizes,
                int64_t bits, const Tensor& m, const OptTensor& ms, const Tensor& v,
                const OptTensor& vs, const Tensor& step, double lr, const OptTensor& lr_tensor,
                double beta1, double beta2, double eps, double weight_decay, int64_t seed) {
  TORCH_CHECK(params.size() == sizes.size(), "adamw_step: one size a parameter");
  std::vector<uint64_t> table;
  std::vector<Tensor> keep;
  table.reserve(4 * params.size());
  const at::ScalarType type = params.empty() ? at::kFloat : params[0].scalar_type();
  int64_t offset = 0;
  bool any = false;
  for (size_t i = 0; i < params.size(); offset += (sizes[i] + 255) / 256 * 256, ++i) {
    const Tensor& p = params[i];
    Tensor g = p.grad();
    if (g.defined() && (p.numel() != sizes[i] || g.numel() != sizes[i]))
      bad_value("a parameter has " + std::to_string(p.numel()) + " values and its gradient " +
                std::to_string(g.numel()) + ", where its states were made for " +
                std::to_string(sizes[i]));
    any = any || g.defined();
    if (!g.defined() || p.numel() == 0) continue;
    if (p.scalar_type() != type || g.scalar_type() != type || g.layout() != at::kStrided)
      bad_type("a gradient must be dense and of its parameter's type " + type_of(type) + ", got " +
               type_of(g.scalar_type()));
    if (!p.is_contiguous()) bad_value("parameters must be contiguous");
    if (p.device() != m.device() || g.device() != m.device())
      bad_value("parameters and gradients must stay on the device of their states, " +
                m.device().str());
    if (!g.is_contiguous()) {
      g = g.contiguous();
      keep.push_back(g);
    }
    table.insert(table.end(), {(uint64_t)p.data_ptr(), (uint64_t)g.data_ptr(), (uint64_t)p.numel(),
                               (uint64_t)offset});
  }
  if (!any) return;  // no step
  const at::ScalarType kind = bits == 8 ? at::kFloat8_e4m3fn : at::kFloat;
  for (const Tensor* t : {&m, &v})
    TORCH_CHECK(t->is_cuda() && t->is_contiguous() && t->scalar_type() == kind &&
                    t->numel() >= offset,
                "adamw_step: the states are too short or of another type");
  for (const OptTensor* t : {&ms, &vs})
    TORCH_CHECK(t->has_value() == (bits == 8) &&
                    (bits != 8 || ((*t)->is_cuda() && (*t)->is_contiguous() &&
                                   (*t)->scalar_type() == at::kFloat &&
                                   (*t)->numel() * 256 >= offset)),
                "adamw_step: the scales are too short or of another type");
  TORCH_CHECK(step.is_cuda() && step.numel() == 2, "adamw_step: the step is two int32 values");
  const float* lr_device = nullptr;
  if (lr_tensor.has_value()) {
    const Tensor& t = *lr_tensor;
    if (t.device() != m.device() || t.scalar_type() != at::kFloat || t.numel() != 1)
      bad_value("lr must be a number or one float32 value on " + m.device().str());
    lr_device = t.data_ptr<float>();
  }
  if (CHECK) return;
  c10::cuda::CUDAGuard guard(m.device());
  check_status(TW_PICK(tw_adamw_step, type)(
                   table.data(), (int)(table.size() / 4), (int)bits, ptr(m),
                   (float*)ptr(ms.value_or(Tensor())), ptr(v), (float*)ptr(vs.value_or(Tensor())),
                   step.data_ptr<int>(), lr, lr_device, beta1, beta2, eps, weight_decay,
                   (size_t)(uint32_t)seed, stream_of(m)),
               "tw_adamw_step");
  for (const Tensor& p : params)
    if (p.grad().defined() && !p.is_inference()) p.unsafeGetTensorImpl()->bump_version();
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  static PyObject* native =
      py::object(py::module_::import("torchwarp_b200._native").attr("NativeError")).release().ptr();
  py::register_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const NativeError& e) {
      PyErr_SetString(native, e.what());
    }
  });
  m.def("layer_norm", &layer_norm);
  m.def("linear", &linear);
  m.def("gated_scan", &gated_scan);
  m.def("gated_scan_step", &gated_scan_step);
  m.def("adamw_step", &adamw_step<false>);
  m.def("adamw_check", &adamw_step<true>);
  // whether two sequences hold the same objects, in one order
  m.def("same_objects", [](const py::tuple& a, const py::list& b) {
    bool same = a.size() == b.size();
    for (size_t i = 0; same && i < a.size(); ++i)
      same = PyTuple_GET_ITEM(a.ptr(), i) == PyList_GET_ITEM(b.ptr(), i);
    return same;
  });
  // without autograd, for the custom ops
  m.def("layer_norm_forward", [](const Tensor& x, const OptTensor& w, const OptTensor& b,
                                 double eps, bool save) {
    const Tensor weight = def(w), bias = def(b);
    no_tangents("layer_norm", {&x, &weight, &bias});
    check_layer_norm(x, weight, bias, eps);
    auto [y, stats] = layer_norm_forward(x, dense(weight), dense(bias), eps, save);
    return std::make_tuple(y, opt(stats));
  });
  m.def("layer_norm_backward", [](const Tensor& dy, const Tensor& x, const OptTensor& w,
                                  const OptTensor& b, const Tensor& stats) {
    check_layer_norm_backward(dy, x, def(w), def(b), stats);
    const Tensor p = w.has_value() ? *w : def(b);
    return layer_norm_backward(dy, x, dense(def(w)),
                               p.defined() ? p.scalar_type() : x.scalar_type(), stats, true, true,
                               true);
  });
  m.def("linear_forward", [](const Tensor& x, const Tensor& w, const OptTensor& b,
                             const OptTensor& r, int64_t act, bool save) {
    const Tensor bias = def(b), residual = def(r);
    no_tangents("linear", {&x, &w, &bias, &residual});
    check_linear(x, w, bias, residual);
    auto [y, z] = linear_forward(x, w, dense(bias), residual, act, save);
    return std::make_tuple(y, opt(z));
  });
  m.def("linear_backward", [](const Tensor& dy, const Tensor& x, const Tensor& w,
                              const OptTensor& z, int64_t act) {
    check_linear_backward(dy, x, w, def(z), act);
    return linear_backward(dy, x, w, def(z), act, true, true, true);
  });
  m.def("gated_scan_forward", [](const Tensor& x, const Tensor& g, const OptTensor& h0,
                                 const OptTensor& n, bool save) {
    const Tensor state = def(h0);
    no_tangents("gated_scan", {&x, &g, &state});
    check_gated_scan(x, g, state, def(n));
    auto [y, last, carry] = gated_scan_forward(x, g, state, whole_lengths(def(n)), save);
    return std::make_tuple(y, last, save ? opt(carry) : std::nullopt);
  });
  m.def("gated_scan_backward", [](const OptTensor& dy, const OptTensor& ds, const Tensor& x,
                                  const Tensor& g, const OptTensor& n, const Tensor& carry) {
    check_gated_scan_backward(def(dy), def(ds), x, g, def(n), carry);
    return gated_scan_backward(def(dy), def(ds), x, g, whole_lengths(def(n)), carry);
  });
  m.def("gated_scan_step_forward", [](const Tensor& x, const Tensor& g, const Tensor& state) {
    no_tangents("gated_scan_step", {&x, &g, &state});
    check_gated_scan_step(x, g, state);
    return gated_scan_step_forward(x, g, state);
  });
  // and for their fakes
  m.def("check_layer_norm", [](const Tensor& x, const OptTensor& w, const OptTensor& b,
                               double eps) { check_layer_norm(x, def(w), def(b), eps); });
  m.def("check_layer_norm_backward",
        [](const Tensor& dy, const Tensor& x, const OptTensor& w, const OptTensor& b,
           const Tensor& stats) { check_layer_norm_backward(dy, x, def(w), def(b), stats); });
  m.def("check_linear", [](const Tensor& x, const Tensor& w, const OptTensor& b,
                           const OptTensor& r) { check_linear(x, w, def(b), def(r)); });
  m.def("check_linear_backward", [](const Tensor& dy, const Tensor& x, const Tensor& w,
                                    const OptTensor& z, int64_t act) {
    check_linear_backward(dy, x, w, def(z), act);
  });
  m.def("check_gated_scan", [](const Tensor& x, const Tensor& g, const OptTensor& h0,
                               const OptTensor& n) { check_gated_scan(x, g, def(h0), def(n)); });
  m.def("check_gated_scan_step", [](const Tensor& x, const Tensor& g, const Tensor& state) {
    check_gated_scan_step(x, g, state);
  });
  m.def("check_gated_scan_backward",
        [](const OptTensor& dy, const OptTensor& ds, const Tensor& x, const Tensor& g,
           const OptTensor& n, const Tensor& carry) {
          check_gated_scan_backward(def(dy), def(ds), x, g, def(n), carry);
        });
}
