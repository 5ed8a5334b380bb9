// Binding of the expert operators for torch tensors: argument checks, output
// and workspace allocation, the current stream, and torch.autograd.
//
// These calls last a few microseconds when a token at a time is answered, of
// which a Python binding and a Python autograd function would be the larger
// part: that is why this part of the library's binding is compiled.  It calls
// the C entry points of include/einjax_hip.h and computes nothing itself.
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/util/Exception.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <optional>
#include <string>
#include <tuple>
#include <vector>

#include "../../include/einjax_hip.h"

namespace py = pybind11;

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;

// ---- checks ------------------------------------------------------------------

// Raised as NotImplementedError.  A C++ exception that holds no Python state:
// gradients are computed on autograd's thread, which does not hold Python's lock.
[[noreturn]] void not_implemented(const std::string &msg) {
  C10_THROW_ERROR(NotImplementedError, msg);
}

void check(int status, const char *what) {
  if (status == EJ_OK) return;
  const std::string msg = std::string(what) + ": " + ej_last_error();
  switch (status) {
    case EJ_E_INVAL:
    case EJ_E_RANGE: throw py::value_error(msg);
    case EJ_E_UNSUPPORTED: not_implemented(msg);
    default: throw std::runtime_error("HIP error in " + msg);
  }
}

std::string str(c10::IntArrayRef s) {
  std::string r = "(";
  for (size_t i = 0; i < s.size(); ++i) r += (i ? ", " : "") + std::to_string(s[i]);
  return r + ")";
}

Tensor on_gpu(py::handle h, const char *what) {
  if (!THPVariable_Check(h.ptr()) || !THPVariable_Unpack(h.ptr()).is_cuda())
    throw py::type_error(std::string(what) + " must be a torch tensor on the GPU");
  return THPVariable_Unpack(h.ptr());
}

Tensor on_gpu_of(const Tensor &ref, py::handle h, const char *what) {
  Tensor t = on_gpu(h, what);
  if (t.get_device() != ref.get_device())
    throw py::value_error(std::string(what) + " is on " + t.device().str() + ", expected " +
                          ref.device().str());
  return t;
}

// EJ_* code of a value type, -1 for others.
int code_of(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return EJ_F32;
    case at::kBFloat16: return EJ_BF16;
    case at::kHalf: return EJ_F16;
    default: return -1;
  }
}

std::string name_of(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return "torch.float32";
    case at::kBFloat16: return "torch.bfloat16";
    case at::kHalf: return "torch.float16";
    default: return c10::toString(t);
  }
}

int value_code(const Tensor &t, const char *what) {
  const int c = code_of(t.scalar_type());
  if (c < 0)
    throw py::type_error(std::string(what) + " must be float32, bfloat16 or float16, got " +
                         name_of(t.scalar_type()));
  return c;
}

// int32, contiguous, of the given shape.
Tensor index(Tensor t, c10::IntArrayRef shape, const char *what) {
  if (t.sizes() != shape)
    throw py::value_error(std::string(what) + " has shape " + str(t.sizes()) + ", expected " +
                          str(shape));
  if (t.scalar_type() != at::kInt) {
    if (t.scalar_type() != at::kLong)
      throw py::type_error(std::string(what) + " must be int32 or int64, got " +
                           name_of(t.scalar_type()));
    t = t.to(at::kInt);
  }
  return t.is_contiguous() ? t : t.contiguous();
}

// t [n, m] with unit stride along its rows and rows that do not overlap
// (itself if it is so already).
Tensor rows_of(const Tensor &t) {
  if (t.is_contiguous()) return t;
  const int64_t n = t.size(0), m = t.size(1);
  if ((m <= 1 || t.stride(1) == 1) && (n <= 1 || t.stride(0) >= m)) return t;
  return t.contiguous();
}

int64_t row_stride(const Tensor &t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

int32_t int32_of(int64_t v, const char *what) {
  if (v < INT32_MIN || v > INT32_MAX)
    throw py::value_error(std::string(what) + " = " + std::to_string(v) + " passes 32 bits");
  return static_cast<int32_t>(v);
}

const void *ptr(const Tensor &t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void *mut(const Tensor &t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }
const int32_t *ints(const Tensor &t) { return static_cast<const int32_t *>(ptr(t)); }
int32_t *mut_ints(const Tensor &t) { return static_cast<int32_t *>(mut(t)); }
const float *floats(const Tensor &t) { return static_cast<const float *>(ptr(t)); }
float *mut_floats(const Tensor &t) { return static_cast<float *>(mut(t)); }

// The operands' device made current, and its current stream.
struct Launch {
  c10::OptionalDeviceGuard guard;
  ej_stream_t stream;
  explicit Launch(const Tensor &ref) {
    if (c10::hip::current_device() != ref.get_device()) guard.reset_device(ref.device());
    stream = c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(ref.get_device()).stream();
  }
};

Tensor workspace(const Tensor &ref, size_t bytes) {
  return bytes ? at::empty({static_cast<int64_t>(bytes)}, ref.options().dtype(at::kByte))
               : Tensor();
}

// Gradients are first order: with create_graph, differentiating one again
// raises instead of passing for a constant.
variable_list first_order(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list out;
  for (Tensor &g : grads) {
    if (!g.defined()) {
      out.push_back(g);
      continue;
    }
    auto err = std::make_shared<torch::autograd::DelayedError>(
        "the gradients of the expert operators are first order: they cannot be differentiated "
        "again",
        1);
    Tensor v = g.detach();
    v.set_requires_grad(true);
    out.push_back((*err)({v})[0]);
  }
  return out;
}

bool wants_grad(const Tensor &t) { return t.requires_grad() && at::GradMode::is_enabled(); }

// A dual tensor's tangent would be dropped, which is a derivative of zero.
template <class... Operands>
void no_tangents(const Operands &...t) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
  if ((... || (t.defined() && t._fw_grad(0).defined())))
    not_implemented("the expert operators have no forward-mode derivatives: an operand is a dual "
                    "tensor");
}

// ---- routing -------------------------------------------------------------------

struct Routing {
  Tensor weights, experts, offsets, rows, slots;
  py::tuple tuple() const { return py::make_tuple(weights, experts, offsets, rows, slots); }
};

Routing empty_routing(const Tensor &ref, int64_t T, int64_t k, int64_t E) {
  const auto opt = at::TensorOptions().device(ref.device()).dtype(at::kInt);
  Routing r;
  r.offsets = at::empty({E + 1}, opt);
  r.rows = at::empty({T * k}, opt);
  r.slots = at::empty({T, k}, opt);
  return r;
}

Tensor route_workspace(const Tensor &ref, int64_t T, int64_t E, size_t *bytes) {
  check(ej_expert_route_workspace_size(T, int32_of(E, "experts"), bytes),
        "ej_expert_route_workspace_size");
  return workspace(ref, *bytes);
}

Routing run_route(const Tensor &given, int64_t k, bool renorm) {
  const int code = value_code(given, "logits");
  no_tangents(given);
  const Tensor logits = rows_of(given);
  const int64_t T = logits.size(0), E = logits.size(1);
  Launch on(logits);
  size_t bytes;
  const Tensor ws = route_workspace(logits, T, E, &bytes);
  Routing r = empty_routing(logits, T, k, E);
  r.weights = at::empty({T, k}, logits.options().dtype(at::kFloat));
  r.experts = at::empty({T, k}, r.rows.options());
  check(ej_expert_route(ptr(logits), code, T, static_cast<int32_t>(E),
                        std::max(row_stride(logits), E), static_cast<int32_t>(k), renorm,
                        mut_floats(r.weights), mut_ints(r.experts), mut_ints(r.offsets),
                        mut_ints(r.rows), mut_ints(r.slots), mut(ws), bytes, on.stream),
        "ej_expert_route");
  return r;
}

Tensor run_route_vjp(const Tensor &given, const Tensor &experts, const Tensor &grad, bool renorm) {
  const int code = value_code(given, "logits");
  no_tangents(given, grad);
  const Tensor logits = rows_of(given);
  const int64_t T = logits.size(0), E = logits.size(1), k = experts.size(1);
  const Tensor g = grad.to(at::kFloat).contiguous();
  Launch on(logits);
  Tensor out = at::empty({T, E}, logits.options());
  check(ej_expert_route_vjp(ptr(logits), code, T, int32_of(E, "experts"),
                            std::max(row_stride(logits), E), int32_of(k, "k"), renorm,
                            ints(experts), floats(g), mut(out), on.stream),
        "ej_expert_route_vjp");
  return out;
}

struct RouteFunction : public Function<RouteFunction> {
  static Tensor forward(AutogradContext *ctx, const Tensor &logits, int64_t k, bool renorm,
                        Routing *made) {
    *made = run_route(logits, k, renorm);
    ctx->saved_data["renorm"] = renorm;
    ctx->save_for_backward({logits, made->experts});
    return made->weights;
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    return first_order({run_route_vjp(saved[0], saved[1], grads[0],
                                      ctx->saved_data["renorm"].toBool()),
                        Tensor(), Tensor(), Tensor()});
  }
};

py::tuple route(py::handle logits_, int64_t k, bool renorm) {
  const Tensor logits = on_gpu(logits_, "logits");
  if (logits.dim() != 2)
    throw py::value_error("logits must be [tokens, experts], got shape " + str(logits.sizes()));
  value_code(logits, "logits");
  if (k < 1 || k > std::max<int64_t>(logits.size(1), 1))
    throw py::value_error("k = " + std::to_string(k) + ", expected 1 to the number of experts, " +
                          std::to_string(logits.size(1)));
  if (!wants_grad(logits)) return run_route(logits, k, renorm).tuple();
  Routing made;
  made.weights = RouteFunction::apply(logits, k, renorm, &made);
  return made.tuple();
}

Tensor route_vjp(py::handle logits_, py::handle experts_, py::handle grad_, bool renorm) {
  const Tensor logits = on_gpu(logits_, "logits");
  Tensor experts = on_gpu_of(logits, experts_, "experts");
  const Tensor grad = on_gpu_of(logits, grad_, "grad_weights");
  if (logits.dim() != 2 || experts.dim() != 2 || experts.size(0) != logits.size(0))
    throw py::value_error("logits " + str(logits.sizes()) + " and experts " +
                          str(experts.sizes()) + " must be [tokens, experts] and [tokens, k]");
  if (grad.sizes() != experts.sizes())
    throw py::value_error("grad_weights has shape " + str(grad.sizes()) + ", expected " +
                          str(experts.sizes()));
  experts = index(experts, experts.sizes(), "experts");
  return run_route_vjp(logits, experts, grad, renorm);
}

py::tuple group(py::handle experts_, int64_t E, py::handle weights_) {
  Tensor experts = on_gpu(experts_, "experts");
  if (experts.dim() != 2)
    throw py::value_error("experts must be [tokens, k], got shape " + str(experts.sizes()));
  const int64_t T = experts.size(0), k = experts.size(1);
  Tensor weights;
  if (weights_.is_none()) {
    weights = at::ones({T, k}, experts.options().dtype(at::kFloat));
  } else {
    weights = on_gpu_of(experts, weights_, "weights");
    if (weights.sizes() != experts.sizes() || weights.scalar_type() != at::kFloat)
      throw py::value_error("weights must be float32 " + str(experts.sizes()) + ", got " +
                            name_of(weights.scalar_type()) + " " + str(weights.sizes()));
  }
  // no wrapping of values past 32 bits into the range
  if (experts.scalar_type() == at::kLong) experts = experts.clamp(-1, E);
  experts = index(experts, {T, k}, "experts");
  // The library groups no more picks than experts.  There may be more, of
  // experts elsewhere: then for groups that stay empty behind those that are here.
  const int64_t groups = E >= 1 ? std::max(E, k) : E;
  if (groups > E) experts = experts.masked_fill(experts.ge(E), -1);
  Launch on(experts);
  size_t bytes;
  const Tensor ws = route_workspace(experts, T, groups, &bytes);
  Routing r = empty_routing(experts, T, k, groups);
  r.weights = weights;
  r.experts = experts;
  check(ej_expert_group(ints(experts), T, int32_of(k, "k"), static_cast<int32_t>(groups),
                        mut_ints(r.offsets), mut_ints(r.rows), mut_ints(r.slots), mut(ws), bytes,
                        on.stream),
        "ej_expert_group");
  if (groups > E) r.offsets = r.offsets.narrow(0, 0, E + 1);
  return r.tuple();
}

// ---- back to tokens ----------------------------------------------------------------

Tensor run_combine(const Tensor &given, const Tensor &slots, const Tensor &weights,
                   at::ScalarType out_type) {
  no_tangents(given, weights);
  const Tensor y = rows_of(given);
  const int64_t T = slots.size(0), n = y.size(1);
  Launch on(y);
  Tensor out = at::empty({T, n}, y.options().dtype(out_type));
  check(ej_expert_combine(ptr(y), value_code(y, "y"), y.size(0), row_stride(y), floats(weights),
                          ints(slots), T, int32_of(slots.size(1), "k"), int32_of(n, "n"), mut(out),
                          code_of(out_type), on.stream),
        "ej_expert_combine");
  return out;
}

variable_list run_combine_vjp(const Tensor &y_, const Tensor &slots, const Tensor &offsets,
                              const Tensor &weights, const Tensor &grad_, bool need_y,
                              bool need_w) {
  no_tangents(y_, weights, grad_);
  const Tensor y = rows_of(y_), grad = rows_of(grad_);
  const int64_t T = slots.size(0), n = y.size(1);
  Launch on(y);
  const Tensor gy = need_y ? at::empty(y.sizes(), y.options()) : Tensor();
  const Tensor gw = need_w ? at::empty(slots.sizes(), y.options().dtype(at::kFloat)) : Tensor();
  check(ej_expert_combine_vjp(ptr(y), value_code(y, "y"), y.size(0), row_stride(y),
                              floats(weights), ints(slots), ints(offsets),
                              int32_of(offsets.size(0) - 1, "experts"), T,
                              int32_of(slots.size(1), "k"), int32_of(n, "n"), ptr(grad),
                              row_stride(grad), mut(gy), mut_floats(gw), on.stream),
        "ej_expert_combine_vjp");
  return {gy, gw};
}

struct CombineFunction : public Function<CombineFunction> {
  static Tensor forward(AutogradContext *ctx, const Tensor &y, const Tensor &weights,
                        const Tensor &slots, const Tensor &offsets) {
    ctx->save_for_backward({y, weights, slots, offsets});
    return run_combine(y, slots, weights, y.scalar_type());
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    variable_list g = run_combine_vjp(s[0], s[2], s[3], s[1], grads[0], ctx->needs_input_grad(0),
                                      ctx->needs_input_grad(1));
    return first_order({g[0], g[1], Tensor(), Tensor()});
  }
};

struct CombineArgs {
  Tensor y, weights, slots, offsets;
};

CombineArgs combine_args(py::handle y_, py::handle weights_, py::handle slots_,
                         py::handle offsets_) {
  CombineArgs a;
  a.y = on_gpu(y_, "y");
  a.weights = on_gpu_of(a.y, weights_, "weights");
  a.slots = on_gpu_of(a.y, slots_, "slots");
  a.offsets = on_gpu_of(a.y, offsets_, "offsets");
  if (a.slots.dim() != 2 || a.offsets.dim() != 1 || a.offsets.size(0) < 1)
    throw py::value_error("slots must be [tokens, k] and offsets [experts + 1], got shapes " +
                          str(a.slots.sizes()) + " and " + str(a.offsets.sizes()));
  if (a.y.dim() != 2 || a.y.size(0) != a.slots.numel())
    throw py::value_error("y has shape " + str(a.y.sizes()) + ", expected [" +
                          std::to_string(a.slots.numel()) + ", n]: a row for each slot of the "
                          "routing");
  value_code(a.y, "y");
  if (a.weights.scalar_type() != at::kFloat || a.weights.sizes() != a.slots.sizes())
    throw py::value_error("weights must be float32 " + str(a.slots.sizes()) + ", got " +
                          name_of(a.weights.scalar_type()) + " " + str(a.weights.sizes()));
  a.weights = a.weights.contiguous();
  a.slots = index(a.slots, a.slots.sizes(), "slots");
  a.offsets = index(a.offsets, a.offsets.sizes(), "offsets");
  return a;
}

Tensor combine(py::handle y, py::handle weights, py::handle slots, py::handle offsets) {
  const CombineArgs a = combine_args(y, weights, slots, offsets);
  if (!wants_grad(a.y) && !wants_grad(a.weights))
    return run_combine(a.y, a.slots, a.weights, a.y.scalar_type());
  return CombineFunction::apply(a.y, a.weights, a.slots, a.offsets);
}

py::tuple combine_vjp(py::handle y, py::handle weights, py::handle slots, py::handle offsets,
                      py::handle grad_, bool need_y, bool need_w) {
  const CombineArgs a = combine_args(y, weights, slots, offsets);
  const Tensor grad = on_gpu_of(a.y, grad_, "grad_out");
  if (grad.dim() != 2 || grad.size(0) != a.slots.size(0) || grad.size(1) != a.y.size(1))
    throw py::value_error("grad_out has shape " + str(grad.sizes()) + ", expected " +
                          str({a.slots.size(0), a.y.size(1)}));
  at::NoGradGuard no_grad;
  variable_list g = run_combine_vjp(a.y, a.slots, a.offsets, a.weights,
                                    grad.to(a.y.scalar_type()), need_y, need_w);
  return py::make_tuple(need_y ? py::cast(g[0]) : py::none(),
                        need_w ? py::cast(g[1]) : py::none());
}

// ---- grouped products ------------------------------------------------------------------

// What a product reads of its groups: offsets int32 [E + 1] (undefined: one
// group of every slot), the row of x for each slot (undefined: the slot
// itself) and, where rows are gathered, the slots of each row.
struct Groups {
  Tensor offsets, rows, slots;
  int64_t n_slots = 0;
};

// rows and slots of a routing, or None for offsets alone.
Groups groups_of(const Tensor &x, int64_t E, py::handle offsets_, py::handle rows_,
                 py::handle slots_, bool gather) {
  Groups g;
  g.offsets = on_gpu_of(x, offsets_, "offsets");
  if (rows_.is_none()) {
    if (gather)
      throw py::value_error("gather=True needs an ExpertRouting: offsets alone do not say which "
                            "rows the slots take");
    g.offsets = index(g.offsets, {E + 1}, "offsets");
    g.n_slots = x.size(0);
    return g;
  }
  if (g.offsets.dim() != 1 || g.offsets.size(0) != E + 1)
    throw py::value_error("the routing has " + std::to_string(g.offsets.numel() - 1) +
                          " experts, the weights have " + std::to_string(E));
  g.offsets = index(g.offsets, {E + 1}, "offsets");
  const Tensor rows = on_gpu_of(x, rows_, "rows"), slots = on_gpu_of(x, slots_, "slots");
  if (slots.dim() != 2 || slots.numel() != rows.numel())
    throw py::value_error("the routing has slots " + str(slots.sizes()) + " and " +
                          std::to_string(rows.numel()) + " rows");
  g.n_slots = rows.numel();
  const int64_t want = gather ? slots.size(0) : g.n_slots;
  if (x.size(0) != want)
    throw py::value_error("x has " + std::to_string(x.size(0)) + " rows, expected " +
                          std::to_string(want) +
                          (gather ? " (tokens of the routing)" : " (slots of the routing)"));
  if (gather) {
    g.rows = index(rows, {g.n_slots}, "rows");
    g.slots = index(slots, slots.sizes(), "slots");
  }
  return g;
}

struct Order {
  Tensor w;
  int32_t order;
  int64_t group, row;  // strides
};

// How w [E, k, n] lies in memory; a copy if neither k nor n is contiguous.
Order weight_order(Tensor w) {
  const int64_t E = w.size(0), k = w.size(1), n = w.size(2);
  if (w.is_contiguous()) return {w, EJ_W_KN, k * n, n};
  for (int order : {EJ_W_KN, EJ_W_NK}) {
    const bool kn = order == EJ_W_KN;
    const int64_t rows = kn ? k : n, cols = kn ? n : k;
    const int64_t row = rows > 1 ? w.stride(kn ? 1 : 2) : std::max<int64_t>(cols, 1);
    const int64_t group = E > 1 ? w.stride(0) : rows * row;
    if ((cols <= 1 || w.stride(kn ? 2 : 1) == 1) && row >= cols && group >= rows * row)
      return {w, order, group, row};
  }
  return {w.contiguous(), EJ_W_KN, k * n, n};
}

ej_grouped_desc describe(const Tensor &x, int code, int out_code, const Order &o, int64_t E,
                         int64_t k, int64_t n, int64_t n_slots, int64_t out_stride) {
  ej_grouped_desc d = {};
  d.dtype = code;
  d.out_dtype = out_code;
  d.w_order = o.order;
  d.n_groups = int32_of(E, "groups");
  d.k = int32_of(k, "k");
  d.n = int32_of(n, "n");
  d.n_slots = n_slots;
  d.n_rows = x.size(0);
  d.x_stride = std::max(row_stride(x), k);
  d.w_group = o.group;
  d.w_stride = o.row;
  d.out_stride = out_stride;
  return d;
}

// out[s] = x[row of s] w[group of s], zero in slots of no group; with scales,
// 8-bit operands (w in rows of k).
Tensor run_product(const Tensor &x_, const Order &o, int64_t k, int64_t n, const Groups &g,
                   at::ScalarType out_type, const Tensor &x_scale = Tensor(),
                   const Tensor &w_scale = Tensor()) {
  no_tangents(x_, o.w, x_scale, w_scale);
  const Tensor x = rows_of(x_);
  const int code = x_scale.defined() ? EJ_I8 : code_of(x.scalar_type());
  Launch on(x);
  Tensor out = at::empty({g.n_slots, n}, x.options().dtype(out_type));
  const ej_grouped_desc d =
      describe(x, code, code_of(out_type), o, o.w.size(0), k, n, g.n_slots, n);
  size_t bytes;
  check(ej_grouped_gemm_workspace_size(&d, &bytes), "ej_grouped_gemm_workspace_size");
  const Tensor ws = workspace(x, bytes);
  check(ej_grouped_gemm(&d, ptr(x), ints(g.rows), ints(g.offsets), ptr(o.w), floats(x_scale),
                        floats(w_scale), mut(out), mut(ws), bytes, on.stream),
        "ej_grouped_gemm");
  return out;
}

Tensor product(const Tensor &x, const Tensor &w, const Groups &g, at::ScalarType out_type) {
  return run_product(x, weight_order(w), w.size(1), w.size(2), g, out_type);
}

// Gradient to w [E, k, n], in the order w lies in.
Tensor weight_gradient(const Tensor &x_, const Tensor &w, const Groups &g, const Tensor &grad_) {
  no_tangents(x_, grad_);
  const Tensor x = rows_of(x_), grad = rows_of(grad_);
  const int64_t E = w.size(0), k = w.size(1), n = w.size(2);
  Order o = weight_order(w);
  Launch on(x);
  const bool kn = o.order == EJ_W_KN;
  Tensor gw = kn ? at::empty({E, k, n}, w.options())
                 : at::empty({E, n, k}, w.options()).transpose(1, 2);
  o.group = k * n;
  o.row = kn ? n : k;
  const int code = code_of(x.scalar_type());
  const ej_grouped_desc d =
      describe(x, code, code, o, E, k, n, g.n_slots, std::max(row_stride(grad), n));
  size_t bytes;
  check(ej_grouped_gemm_dw_workspace_size(&d, &bytes), "ej_grouped_gemm_dw_workspace_size");
  const Tensor ws = workspace(x, bytes);
  check(ej_grouped_gemm_dw(&d, ptr(x), ints(g.rows), ints(g.offsets), ptr(grad), mut(gw), mut(ws),
                           bytes, on.stream),
        "ej_grouped_gemm_dw");
  return gw;
}

variable_list product_vjp(const Tensor &x, const Tensor &w, const Groups &g, const Tensor &grad_,
                          bool need_x, bool need_w) {
  at::NoGradGuard no_grad;
  // an fp32 cotangent of 16-bit operands is rounded to their type: both
  // gradients are 16-bit products with fp32 sums
  const Tensor grad = grad_.to(x.scalar_type());
  Tensor gx, gw;
  if (need_x) {
    Groups slots;
    slots.offsets = g.offsets;
    slots.n_slots = g.n_slots;
    // gathered rows: each slot's gradient stays in fp32 until a token's slots
    // are summed, so that the sum is rounded once
    gx = product(grad, w.transpose(1, 2), slots, g.rows.defined() ? at::kFloat : x.scalar_type());
    if (g.rows.defined()) gx = run_combine(gx, g.slots, Tensor(), x.scalar_type());
  }
  if (need_w) gw = weight_gradient(x, w, g, grad);
  return {gx, gw};
}

struct ProductFunction : public Function<ProductFunction> {
  static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &w, const Groups *g,
                        int64_t out_type) {
    variable_list saved = {x, w, g->offsets};
    if (g->rows.defined()) {
      saved.push_back(g->rows);
      saved.push_back(g->slots);
    }
    ctx->save_for_backward(saved);
    ctx->saved_data["n_slots"] = g->n_slots;
    return product(x, w, *g, static_cast<at::ScalarType>(out_type));
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    Groups g;
    g.offsets = s[2];
    if (s.size() > 3) {
      g.rows = s[3];
      g.slots = s[4];
    }
    g.n_slots = ctx->saved_data["n_slots"].toInt();
    variable_list v = product_vjp(s[0], s[1], g, grads[0], ctx->needs_input_grad(0),
                                  ctx->needs_input_grad(1));
    return first_order({v[0], v[1], Tensor(), Tensor()});
  }
};

// The result's type: x's, or float32.
at::ScalarType check_product(const Tensor &x, const Tensor &w, py::handle out_dtype) {
  if (x.dim() != 2 || w.dim() != 3 || x.size(1) != w.size(1))
    throw py::value_error("x " + str(x.sizes()) + " and w " + str(w.sizes()) +
                          " must be [rows, k] and [groups, k, n]");
  if (x.scalar_type() != w.scalar_type() || code_of(x.scalar_type()) < 0)
    throw py::type_error("x and w must share float32, bfloat16 or float16, got " +
                         name_of(x.scalar_type()) + " and " + name_of(w.scalar_type()));
  if (out_dtype.is_none()) return x.scalar_type();
  const at::ScalarType t = py::cast<at::ScalarType>(out_dtype);
  if (t != at::kFloat && t != x.scalar_type())
    throw py::type_error("out_dtype must be float32 or " + name_of(x.scalar_type()) + ", got " +
                         name_of(t));
  return t;
}

// The gradient to gathered rows is the sum of each token's slots.
void check_picks(const Tensor &slots) {
  if (slots.size(1) < 1 || slots.size(1) > EJ_MAX_PICKS)
    not_implemented("the gradient to gathered rows adds 1 to " + std::to_string(EJ_MAX_PICKS) +
                    " slots of a token, the routing has " + std::to_string(slots.size(1)));
}

Tensor grouped_matmul(py::handle x_, py::handle w_, py::handle offsets, py::handle rows,
                      py::handle slots, bool gather, py::handle out_dtype) {
  const Tensor x = on_gpu(x_, "x"), w = on_gpu_of(x, w_, "w");
  const at::ScalarType t = check_product(x, w, out_dtype);
  const Groups g = groups_of(x, w.size(0), offsets, rows, slots, gather);
  if (!wants_grad(x) && !wants_grad(w)) return product(x, w, g, t);
  // refused now, not when the gradient is asked for
  if (wants_grad(x) && g.slots.defined()) check_picks(g.slots);
  return ProductFunction::apply(x, w, &g, static_cast<int64_t>(t));
}

py::tuple grouped_matmul_vjp(py::handle x_, py::handle w_, py::handle offsets, py::handle rows,
                             py::handle slots, bool gather, py::handle grad_, bool need_x,
                             bool need_w) {
  const Tensor x = on_gpu(x_, "x"), w = on_gpu_of(x, w_, "w");
  check_product(x, w, py::none());
  const Groups g = groups_of(x, w.size(0), offsets, rows, slots, gather);
  if (need_x && g.slots.defined()) check_picks(g.slots);
  const Tensor grad = on_gpu_of(x, grad_, "grad_out");
  if (grad.dim() != 2 || grad.size(0) != g.n_slots || grad.size(1) != w.size(2))
    throw py::value_error("grad_out has shape " + str(grad.sizes()) + ", expected " +
                          str({g.n_slots, w.size(2)}));
  variable_list v = product_vjp(x, w, g, grad, need_x, need_w);
  return py::make_tuple(need_x ? py::cast(v[0]) : py::none(),
                        need_w ? py::cast(v[1]) : py::none());
}

// ---- 8-bit integers -----------------------------------------------------------------------

py::tuple quantize_rows(py::handle x_) {
  const Tensor given = on_gpu(x_, "x"), x = given.detach();
  no_tangents(given);
  const int code = value_code(x, "x");
  if (x.dim() < 1) throw py::value_error("x must have at least one dimension");
  const int64_t n = x.size(-1);
  const auto lead = x.sizes().slice(0, x.dim() - 1);
  int64_t m = 1;
  for (int64_t s : lead) m *= s;
  const Tensor flat = rows_of(x.dim() == 2 ? x : x.reshape({m, n}));
  Launch on(x);
  Tensor q = at::empty(x.sizes(), x.options().dtype(at::kChar));
  Tensor scale = at::empty(lead, x.options().dtype(at::kFloat));
  check(ej_quantize_rows(ptr(flat), code, m, std::max(row_stride(flat), n), int32_of(n, "n"),
                         static_cast<int8_t *>(mut(q)), mut_floats(scale), on.stream),
        "ej_quantize_rows");
  return py::make_tuple(q, scale);
}

Tensor int8_matmul(py::handle q_, py::handle q_scale_, py::handle w_, py::handle w_scale_,
                   py::handle offsets, py::handle rows, py::handle slots, bool gather,
                   at::ScalarType out_type) {
  const Tensor q = on_gpu(q_, "q");
  Tensor q_scale = on_gpu_of(q, q_scale_, "q_scale"), w = on_gpu_of(q, w_, "w");
  Tensor w_scale = on_gpu_of(q, w_scale_, "w_scale");
  if (q.scalar_type() != at::kChar || w.scalar_type() != at::kChar)
    throw py::type_error("q and w must be int8, got " + name_of(q.scalar_type()) + " and " +
                         name_of(w.scalar_type()));
  if (q_scale.scalar_type() != at::kFloat || w_scale.scalar_type() != at::kFloat)
    throw py::type_error("scales must be float32, got " + name_of(q_scale.scalar_type()) +
                         " and " + name_of(w_scale.scalar_type()));
  if (code_of(out_type) < 0)
    throw py::type_error("out_dtype must be float32, bfloat16 or float16, got " +
                         name_of(out_type));
  if (q.dim() != 2) throw py::value_error("q must be [rows, k], got shape " + str(q.sizes()));
  const bool dense = offsets.is_none();
  if (dense && w.dim() == 2) {
    w = w.unsqueeze(0);
    w_scale = w_scale.unsqueeze(0);
  }
  if (w.dim() != 3)
    throw py::value_error("w must be [groups, n, k] (or [n, k] without groups), got shape " +
                          str(w.sizes()));
  const int64_t E = w.size(0), n = w.size(1), k = w.size(2);
  if (q.size(1) != k)
    throw py::value_error("q has rows of " + std::to_string(q.size(1)) + ", w of " +
                          std::to_string(k));
  if (q_scale.dim() != 1 || q_scale.size(0) != q.size(0) || w_scale.dim() != 2 ||
      w_scale.size(0) != E || w_scale.size(1) != n)
    throw py::value_error("scales have shapes " + str(q_scale.sizes()) + " and " +
                          str(w_scale.sizes()) + ", expected " + str({q.size(0)}) + " and " +
                          str({E, n}));
  Groups g;
  if (dense) {
    if (gather || E != 1)
      throw py::value_error("more than one weight matrix, or gather=True, needs groups");
    g.n_slots = q.size(0);
  } else {
    g = groups_of(q, E, offsets, rows, slots, gather);
  }
  // rows of k, as they lie where they can be read so
  Order o{w, EJ_W_NK, E > 1 ? w.stride(0) : 0, n > 1 ? w.stride(1) : std::max<int64_t>(k, 1)};
  if (E <= 1) o.group = n * o.row;
  if (!((k <= 1 || w.stride(2) == 1) && o.row >= k && o.group >= n * o.row)) {
    o.w = w.contiguous();
    o.row = std::max<int64_t>(k, 1);
    o.group = n * o.row;
  }
  return run_product(q, o, k, n, g, out_type, q_scale.contiguous(), w_scale.contiguous());
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.doc() = "Expert operators for torch tensors over libejhip.so.";
  py::register_local_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const c10::NotImplementedError &e) {
      PyErr_SetString(PyExc_NotImplementedError, e.what_without_backtrace());
    }
  });
  m.def("route", &route);
  m.def("route_vjp", &route_vjp);
  m.def("group", &group);
  m.def("combine", &combine);
  m.def("combine_vjp", &combine_vjp);
  m.def("grouped_matmul", &grouped_matmul);
  m.def("grouped_matmul_vjp", &grouped_matmul_vjp);
  m.def("quantize_rows", &quantize_rows);
  m.def("int8_matmul", &int8_matmul);
  m.def("rows_of", &rows_of);
  m.def("weight_order", [](const Tensor &w) {
    const Order o = weight_order(w);
    return py::make_tuple(o.w, o.order, o.group, o.row);
  });
}
