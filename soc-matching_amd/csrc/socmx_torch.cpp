// socmx_torch.cpp -- the layer operators and AdamW on torch tensors: argument checks, allocations, autograd nodes.
//
// The kernels are libsocmx.so's, through its C ABI (include/socmx.h); this module is what stands between a Python call and a launch,
// in C++ because at small sizes that is what a call costs: a training call of layer norm through Python autograd functions and ctypes
// took 143 us on the host for 40 us of GPU time, most of it in the engine's worker thread, where Python runs cold.
// Memory comes from torch's allocator, launches go to the current stream of the tensors' device.
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <dlfcn.h>
#include <hip/hip_runtime_api.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include <algorithm>
#include <sstream>
#include <unordered_set>

#include "../../include/socmx.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef c10::optional<Tensor> Maybe;

// ---- the C ABI, found in the library that socmx/_lib.py has loaded -----------------------------------------------------------
#define SOCMX_ABI(X)                                                                                                               \
  X(socmx_layer_norm_fwd) X(socmx_layer_norm_bwd_workspace_floats) X(socmx_layer_norm_bwd) X(socmx_gated_scan_sizes)                 \
  X(socmx_gated_scan_fwd) X(socmx_gated_scan_bwd) X(socmx_gated_scan_step) X(socmx_adamw_step) X(socmx_adamw_step_counts) \
  X(socmx_adamw_state_values)
#define SOCMX_DECLARE(F) decltype(&::F) F;
struct Abi { SOCMX_ABI(SOCMX_DECLARE) } abi;
PyObject* socmx_error = nullptr;             // socmx._lib.SocmxError

struct Refusal : std::runtime_error { using std::runtime_error::runtime_error; };

template <typename... A>
[[noreturn]] void refuse(const A&... parts) {
  std::ostringstream s;
  (s << ... << parts);
  throw Refusal(s.str());
}

void check(int status, const char* what) {
  if (status == 0) return;
  static const char* kinds[] = {"null pointer", "bad dimension", "unknown problem kind or element type", "workspace too small", "does not fit in LDS"};
  refuse(what, " failed with status ", status, " (", status < 0 && status >= -5 ? kinds[-status - 1] : status < 0 ? "invalid argument" : "hipError_t", ")");
}

void bind_library(const std::string& path, py::object error) {
  void* lib = dlopen(path.c_str(), RTLD_NOW | RTLD_LOCAL);
  if (!lib) throw std::runtime_error(std::string("socmx: ") + dlerror());
#define SOCMX_FIND(F)                                                                                       \
  abi.F = reinterpret_cast<decltype(abi.F)>(dlsym(lib, #F));                                                  \
  if (!abi.F) throw std::runtime_error(path + " does not export " #F ": stale build?");
  SOCMX_ABI(SOCMX_FIND)
  socmx_error = error.release().ptr();
}

// ---- tensors -------------------------------------------------------------------------------------------------------------------
int element_type(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return SOCMX_F32;
    case at::kBFloat16: return SOCMX_BF16;
    case at::kHalf: return SOCMX_F16;
    default: return -1;
  }
}

std::string shape(const Tensor& t) {
  std::ostringstream s;
  s << "(";
  for (int64_t i = 0; i < t.dim(); ++i) s << (i ? ", " : "") << t.size(i);
  s << (t.dim() == 1 ? ",)" : ")");
  return s.str();
}

void on_gpu(const char* what, const Tensor& first) {
  if (!first.is_cuda()) refuse(what, ": tensors on the GPU are needed, got ", first.device(), " (there is no CPU path)");
}

void beside(const char* what, const Tensor& first, const Maybe& t) {
  if (t && t->device() != first.device()) refuse(what, ": tensors on ", first.device(), " and on ", t->device());
}

// A trace would record the allocations of a call and none of its launches: what it made would return memory that nobody has written.
void not_traced(const char* what) {
  if (torch::jit::tracer::isTracing() || c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY))
    refuse(what, ": cannot be traced");
}

// Forward-mode derivatives have no rule here: a dual tensor would lose its tangent without a word.
void no_tangent(const char* what, std::initializer_list<const Tensor*> inputs) {
  for (const Tensor* t : inputs)
    if (t->defined() && t->_fw_grad(/*level=*/0).defined())
      refuse(what, ": forward-mode derivatives are not implemented, and an input has a tangent");
}
const Tensor* given(const Maybe& t) {
  static const Tensor none;
  return t ? &*t : &none;
}

void floating(const char* what, const Tensor& t) {
  if (element_type(t) < 0) refuse(what, ": float32, bfloat16 or float16 is needed, got ", t.scalar_type());
}

void* pointer(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
template <typename T>
T* pointer_as(const Tensor& t) { return static_cast<T*>(pointer(t)); }

Tensor empty(at::IntArrayRef size, at::ScalarType type, const at::Device& dev) {
  return at::empty(size, at::TensorOptions().dtype(type).device(dev));
}

// what a call wrote in place: a graph that has saved it refuses its backward
void written(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

Tensor floats(int64_t n, const at::Device& dev) { return n ? empty({n}, at::kFloat, dev) : Tensor(); }

// the device of the tensors made current, and its current stream
struct Launch {
  c10::DeviceGuard guard;
  void* stream;
  explicit Launch(const at::Device& dev) : guard(dev) {
    stream = c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(dev.index()).stream();
  }
};

// the number of the capture that a stream is part of, or 0
unsigned long long capture_of(void* stream) {
  hipStreamCaptureStatus s = hipStreamCaptureStatusNone;
  unsigned long long id = 0;
  return hipStreamGetCaptureInfo(static_cast<hipStream_t>(stream), &s, &id) == hipSuccess && s == hipStreamCaptureStatusActive ? id : 0;
}
// (the default stream is never captured, and not asked while another one is)
bool joined(const c10::Stream& s, unsigned long long capture) {
  return s.id() != 0 && capture_of(c10::hip::HIPStreamMasqueradingAsCUDA(s).stream()) == capture;
}

// A leaf's gradient node keeps the stream of the first autograd graph that used the leaf, for as long as any graph of it lives.  torch
// makes that stream wait for a backward on another one; inside a capture that draws it into the graph, and closing the capture ends
// the process.  Such a forward is refused while it is captured, before there is a backward: for every leaf that leads to its inputs, by
// whatever operations.
void refuse_foreign_leaves(const char* what, const at::Device& dev, std::initializer_list<Tensor> inputs) {
  if (!at::GradMode::is_enabled()) return;
  const unsigned long long capture = capture_of(Launch(dev).stream);
  if (capture == 0) return;
  const c10::Stream here = c10::impl::VirtualGuardImpl(dev.type()).getStream(dev);
  std::vector<std::shared_ptr<torch::autograd::Node>> todo;
  std::unordered_set<torch::autograd::Node*> seen;
  auto visit = [&](const std::shared_ptr<torch::autograd::Node>& node) {
    if (node && seen.insert(node.get()).second) todo.push_back(node);
  };
  for (const Tensor& t : inputs)
    if (t.defined() && t.requires_grad()) visit(t.is_leaf() ? torch::autograd::impl::try_get_grad_accumulator(t) : t.grad_fn());
  while (!todo.empty()) {
    const auto node = todo.back();
    todo.pop_back();
    for (const auto& edge : node->next_edges()) visit(edge.function);
    if (!dynamic_cast<torch::autograd::AccumulateGrad*>(node.get())) continue;
    const auto first = node->stream();
    if (first && *first != here && !joined(*first, capture))
      refuse(what, ": an autograd graph of the same leaf, built on another stream, is alive: drop what keeps it (the outputs of an eager "
                   "iteration) before capturing");
  }
}

// What a backward returns cannot be differentiated again.  Under create_graph it gets a node that raises and that lies on the way to
// everything the backward depends on -- the gradients it got, and whatever the node that runs has a way to: all of the forward's inputs, also
// those of which the forward saved a copy or nothing -- so that a second derivative raises and does not leave terms out.
variable_list once(const char* what, variable_list out, const variable_list& upstream) {
  if (!at::GradMode::is_enabled()) return out;
  torch::autograd::edge_list edges;
  for (const Tensor& t : upstream)
    if (t.defined() && t.requires_grad()) edges.push_back(torch::autograd::impl::gradient_edge(t));
  if (const auto node = torch::autograd::get_current_node())
    for (const auto& edge : node->next_edges())
      if (edge.is_valid()) edges.push_back(edge);
  if (edges.empty()) return out;
  const auto node = std::make_shared<torch::autograd::Error>(std::string(what) + ": its backward is not differentiable", std::move(edges));
  for (Tensor& t : out) {
    if (!t.defined()) continue;
    t = t.detach();
    torch::autograd::set_history(t, node);
  }
  return out;
}

// ---- layer norm -------------------------------------------------------------------------------------------------------------------
// `t` as rows of its last dimension, each dense, at one distance from the next: a view where the strides allow it
Tensor rows_of(const Tensor& t) {
  const int64_t cols = t.size(-1);
  Tensor r = t.dim() == 2 ? t : t.reshape({-1, cols});
  return cols > 1 && r.stride(1) != 1 ? r.contiguous() : r;
}

int norm_weight_type(const Tensor& x, const Tensor& w, const Tensor& b) { return element_type(w.defined() ? w : b.defined() ? b : x); }

Tensor norm_forward(const Tensor& x, const Tensor& w, const Tensor& b, double eps, Tensor* stats) {
  const Tensor r = rows_of(x);
  const int64_t rows = r.size(0), cols = r.size(1);
  Tensor y = empty(x.sizes(), x.scalar_type(), x.device());
  if (stats) *stats = empty({2, rows}, at::kFloat, x.device());
  if (rows) {
    const Launch l(x.device());
    float* s = stats ? stats->data_ptr<float>() : nullptr;
    check(abi.socmx_layer_norm_fwd(element_type(x), norm_weight_type(x, w, b), pointer(r), rows, cols, r.stride(0), pointer(w), pointer(b),
                                   (float)eps, pointer(y), s, s ? s + rows : nullptr, l.stream), "socmx_layer_norm_fwd");
  }
  return y;
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Maybe& w0, const Maybe& b0, double eps) {
    const Tensor w = w0 ? w0->contiguous() : Tensor(), b = b0 ? b0->contiguous() : Tensor();
    Tensor stats;
    Tensor y = norm_forward(x, w, b, eps, &stats);
    ctx->save_for_backward({x, w, stats});
    ctx->saved_data["weight"] = w.defined();
    ctx->saved_data["bias"] = b.defined();
    ctx->saved_data["wtype"] = (int64_t)(w.defined() ? w : b.defined() ? b : x).scalar_type();
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    no_tangent("layer_norm", {&grads[0]});
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w = saved[1], &stats = saved[2];
    const auto wtype = static_cast<at::ScalarType>(ctx->saved_data["wtype"].toInt());
    const Tensor r = rows_of(x), d = rows_of(grads[0]);
    const int64_t rows = r.size(0), cols = r.size(1);
    const at::Device dev = x.device();
    // (needs_input_grad counts the tensors that were given)
    const bool has_w = ctx->saved_data["weight"].toBool(), has_b = ctx->saved_data["bias"].toBool();
    const bool need_w = has_w && ctx->needs_input_grad(1), need_b = has_b && ctx->needs_input_grad(1 + has_w);
    Tensor dx, dw, db, ws;
    if (ctx->needs_input_grad(0)) dx = empty(x.sizes(), x.scalar_type(), dev);
    if (need_w) dw = empty({cols}, wtype, dev);
    if (need_b) db = empty({cols}, wtype, dev);
    if (rows == 0) {
      if (need_w) dw.zero_();
      if (need_b) db.zero_();
      return once("layer_norm", {dx, dw, db, Tensor()}, grads);
    }
    const int type = element_type(x), wkind = wtype == at::kFloat ? SOCMX_F32 : type;
    if (need_w || need_b) ws = floats(abi.socmx_layer_norm_bwd_workspace_floats(type, rows, cols), dev);
    {
      const Launch l(dev);
      const float* s = stats.data_ptr<float>();
      check(abi.socmx_layer_norm_bwd(type, wkind, pointer(r), rows, cols, r.stride(0), pointer(d), d.stride(0), pointer(w), s, s + rows,
                                     pointer(dx), pointer(dw), pointer(db), pointer_as<float>(ws), l.stream), "socmx_layer_norm_bwd");
    }
    return once("layer_norm", {dx, dw, db, Tensor()}, grads);
  }
};

Tensor layer_norm(const Tensor& x, const Maybe& weight, const Maybe& bias, double eps) {
  const char* what = "layer_norm";
  not_traced(what);
  no_tangent(what, {&x, given(weight), given(bias)});
  if (x.dim() < 1 || x.size(-1) < 1) refuse(what, ": the last dimension is empty or missing, got shape ", shape(x));
  on_gpu(what, x);
  beside(what, x, weight);
  beside(what, x, bias);
  floating(what, x);
  const int64_t cols = x.size(-1);
  for (const auto& [name, t] : {std::pair<const char*, const Maybe&>("weight", weight), std::pair<const char*, const Maybe&>("bias", bias)}) {
    if (!t) continue;
    if (t->dim() != 1 || t->size(0) != cols) refuse(what, ": ", name, " is (", cols, ",) for this input, got ", shape(*t));
    if (t->scalar_type() != x.scalar_type() && t->scalar_type() != at::kFloat)
      refuse(what, ": ", name, " is of the input's type ", x.scalar_type(), " or float32, got ", t->scalar_type());
  }
  if (weight && bias && weight->scalar_type() != bias->scalar_type())
    refuse(what, ": weight and bias of two types, ", weight->scalar_type(), " and ", bias->scalar_type());
  if (!(eps >= 0.0)) refuse(what, ": eps ", eps, " is negative");
  const Tensor w = weight.value_or(Tensor()), b = bias.value_or(Tensor());
  if (!at::GradMode::is_enabled() || !(x.requires_grad() || (weight && w.requires_grad()) || (bias && b.requires_grad()))) {
    at::NoGradGuard off;
    return norm_forward(x, weight ? w.contiguous() : w, bias ? b.contiguous() : b, eps, nullptr);
  }
  refuse_foreign_leaves(what, x.device(), {x, w, b});
  return LayerNorm::apply(x, weight, bias, eps);
}

// ---- gated scan --------------------------------------------------------------------------------------------------------------------
Tensor dense_last(const Tensor& t) { return t.size(-1) <= 1 || t.stride(-1) == 1 ? t : t.contiguous(); }

// a new tensor of `t`'s shape with steps outside rows, or rows outside steps, as in `t`: whichever it has further apart.  (No view of another
// tensor: what a node returns as a view may not be changed in place.)
Tensor laid_like(const Tensor& t) {
  const int64_t T = t.size(0), B = t.size(1), D = t.size(2);
  const bool rows_outside = t.stride(0) < t.stride(1);
  return at::empty_strided({T, B, D}, {rows_outside ? D : B * D, rows_outside ? T * D : D, 1}, t.options().requires_grad(false));
}

socmx_scan descriptor(const Tensor& x, const Tensor& a, const Tensor& lengths, bool reverse) {
  socmx_scan s = {};
  s.type = element_type(x);
  s.gate_type = element_type(a);
  s.T = (int32_t)x.size(0); s.B = (int32_t)x.size(1); s.D = (int32_t)x.size(2); s.G = (int32_t)a.size(2);
  s.reverse = reverse;
  s.x_stride_t = x.stride(0); s.x_stride_b = x.stride(1); s.gate_stride_t = a.stride(0); s.gate_stride_b = a.stride(1);
  s.lengths = pointer_as<const int32_t>(lengths);
  return s;
}

// no step, or no row: the state is what it was
bool no_steps(const Tensor& x) { return x.size(0) == 0 || x.size(1) == 0; }

std::pair<Tensor, Tensor> scan_forward(const Tensor& x, const Tensor& a, const Tensor& initial, const Tensor& lengths, bool reverse,
                                       Tensor* states) {
  const at::Device dev = x.device();
  if (no_steps(x)) return {laid_like(x), initial.defined() ? initial.clone() : at::zeros({x.size(1), x.size(2)}, x.options().dtype(at::kFloat).requires_grad(false))};
  const socmx_scan s = descriptor(x, a, lengths, reverse);
  int64_t n_states, n_ws, n_bwd;
  check(abi.socmx_gated_scan_sizes(&s, &n_states, &n_ws, &n_bwd), "socmx_gated_scan_sizes");
  Tensor h = laid_like(x), final_state = empty({x.size(1), x.size(2)}, at::kFloat, dev);
  const Tensor ws = floats(n_ws, dev);
  if (states) *states = floats(n_states, dev);
  const Launch l(dev);
  check(abi.socmx_gated_scan_fwd(&s, pointer(x), pointer(a), pointer_as<float>(initial), pointer(h), h.stride(0), h.stride(1),
                                 final_state.data_ptr<float>(), states ? states->data_ptr<float>() : nullptr, pointer_as<float>(ws),
                                 l.stream), "socmx_gated_scan_fwd");
  return {h, final_state};
}

struct GatedScan : torch::autograd::Function<GatedScan> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x0, const Tensor& a0, const Maybe& initial, const Maybe& lengths0,
                               bool reverse) {
    const Tensor x = dense_last(x0), a = dense_last(a0);
    const Tensor lengths = lengths0.value_or(Tensor());
    Tensor states;
    auto [h, final_state] = scan_forward(x, a, initial ? initial->contiguous() : Tensor(), lengths, reverse, &states);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({x, a, states, lengths});
    ctx->saved_data["reverse"] = reverse;
    ctx->saved_data["initial"] = initial.has_value();
    return {h, final_state};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    no_tangent("gated_scan", {&grads[0], &grads[1]});
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &a = saved[1], &states = saved[2], &lengths = saved[3];
    const at::Device dev = x.device();
    const bool need_initial = ctx->saved_data["initial"].toBool() && ctx->needs_input_grad(2);
    Tensor dx = laid_like(x), da = laid_like(a), dinitial;
    if (need_initial) dinitial = empty({x.size(1), x.size(2)}, at::kFloat, dev);
    if (no_steps(x)) {
      if (need_initial && grads[1].defined()) dinitial.copy_(grads[1]);
      else if (need_initial) dinitial.zero_();
      return once("gated_scan", {dx, da, dinitial, Tensor(), Tensor()}, grads);
    }
    const socmx_scan s = descriptor(x, a, lengths, ctx->saved_data["reverse"].toBool());
    int64_t n_states, n_fwd, n_ws;
    check(abi.socmx_gated_scan_sizes(&s, &n_states, &n_fwd, &n_ws), "socmx_gated_scan_sizes");
    const Tensor ws = floats(n_ws, dev);
    const Tensor dh = grads[0].defined() ? dense_last(grads[0]) : Tensor(), dfinal = grads[1].defined() ? grads[1].contiguous() : Tensor();
    {
      const Launch l(dev);
      check(abi.socmx_gated_scan_bwd(&s, pointer(x), pointer(a), states.data_ptr<float>(), pointer(dh), dh.defined() ? dh.stride(0) : 0,
                                     dh.defined() ? dh.stride(1) : 0, pointer_as<float>(dfinal), pointer(dx), dx.stride(0), dx.stride(1),
                                     pointer(da), da.stride(0), da.stride(1), pointer_as<float>(dinitial), pointer_as<float>(ws), l.stream),
            "socmx_gated_scan_bwd");
    }
    return once("gated_scan", {dx, da, dinitial, Tensor(), Tensor()}, grads);
  }
};

void check_scan(const char* what, const Tensor& x, const Tensor& a, int64_t dims) {
  if (x.dim() != dims || a.dim() != dims)
    refuse(what, ": x and log_decay have ", dims, " dimensions, got ", shape(x), " and ", shape(a));
  on_gpu(what, x);
  beside(what, x, a);
  floating(what, x);
  if (a.scalar_type() != x.scalar_type() && a.scalar_type() != at::kFloat)
    refuse(what, ": log_decay is of x's type ", x.scalar_type(), " or float32, got ", a.scalar_type());
  for (int64_t i = 0; i + 1 < dims; ++i)
    if (a.size(i) != x.size(i))
      refuse(what, ": log_decay ", shape(a), " does not go with x ", shape(x), " (expand() shares a gate between steps or rows)");
  const int64_t D = x.size(-1), G = a.size(-1);
  if (D < 1 || G < 1 || D % G) refuse(what, ": ", G, " gates do not divide ", D, " channels");
  if (D > INT32_MAX || x.size(0) > INT32_MAX || x.size(-2) > INT32_MAX) refuse(what, ": x ", shape(x), " is too large");
}

std::pair<Tensor, Tensor> gated_scan(const Tensor& x, const Tensor& a, const Maybe& initial, const Maybe& lengths, bool reverse) {
  const char* what = "gated_scan";
  not_traced(what);
  no_tangent(what, {&x, &a, given(initial)});
  check_scan(what, x, a, 3);
  const int64_t B = x.size(1), D = x.size(2);
  beside(what, x, initial);
  beside(what, x, lengths);
  if (initial && (initial->dim() != 2 || initial->size(0) != B || initial->size(1) != D || initial->scalar_type() != at::kFloat))
    refuse(what, ": initial is (", B, ", ", D, ") float32, got ", shape(*initial), " ", initial->scalar_type());
  if (lengths && (lengths->dim() != 1 || lengths->size(0) != B || lengths->scalar_type() != at::kInt))
    refuse(what, ": lengths is (", B, ",) int32, got ", shape(*lengths), " ", lengths->scalar_type());
  const Tensor first = initial.value_or(Tensor()), n = lengths ? lengths->contiguous() : Tensor();
  if (!at::GradMode::is_enabled() || !(x.requires_grad() || a.requires_grad() || (initial && first.requires_grad()))) {
    at::NoGradGuard off;
    return scan_forward(dense_last(x), dense_last(a), initial ? first.contiguous() : first, n, reverse, nullptr);
  }
  refuse_foreign_leaves(what, x.device(), {x, a, first});
  const variable_list out = GatedScan::apply(x, a, initial, lengths ? Maybe(n) : Maybe(), reverse);
  return {out[0], out[1]};
}

// whether a dense row of `s` (rows apart) and a dense row of `t` (rows at any distance) have memory in common
bool rows_meet(const Tensor& s, const Tensor& t) {
  if (s.numel() == 0 || t.numel() == 0) return false;
  const int64_t s_size = s.size(1) * s.element_size(), t_size = t.size(1) * t.element_size(), s_step = s.stride(0) * s.element_size();
  const int64_t t_step = t.stride(0) * t.element_size(), last = t.size(0) - 1;
  const int64_t gap = static_cast<const char*>(s.data_ptr()) - static_cast<const char*>(t.data_ptr());      // from t's first byte to s's
  if (gap >= last * t_step + t_size || -gap >= (s.size(0) - 1) * s_step + s_size) return false;
  for (int64_t i = 0; i < s.size(0); ++i) {
    const int64_t lo = gap + i * s_step, hi = lo + s_size;      // row i of s, in bytes behind t's first one
    // t's row j begins at j t_step: the first one that ends behind lo
    const int64_t j = t_step == 0 || lo < t_size ? 0 : (lo - t_size) / t_step + 1;
    if (j <= last && j * t_step < hi && j * t_step + t_size > lo) return true;
  }
  return false;
}

Tensor gated_scan_step(const Tensor& state, const Tensor& x0, const Tensor& a0) {
  const char* what = "gated_scan_step";
  not_traced(what);
  no_tangent(what, {&state, &x0, &a0});
  const bool wants_grad = at::GradMode::is_enabled() && (x0.requires_grad() || a0.requires_grad());
  const at::NoGradGuard off;
  check_scan(what, x0, a0, 2);
  beside(what, x0, state);
  const int64_t B = x0.size(0), D = x0.size(1);
  if (state.dim() != 2 || state.size(0) != B || state.size(1) != D || state.scalar_type() != at::kFloat || (D > 1 && state.stride(1) != 1))
    refuse(what, ": state is (", B, ", ", D, ") float32 with dense rows, got ", shape(state), " ", state.scalar_type(), " strides ", state.strides());
  if (state.requires_grad()) refuse(what, ": state is updated in place and must not require a gradient");
  if (B > 1 && state.stride(0) < D) refuse(what, ": the rows of state overlap (stride ", state.stride(0), ")");
  if (wants_grad) refuse(what, ": x or log_decay requires a gradient, and a step has none: detach them or take the step under no_grad");
  const Tensor x = dense_last(x0), a = dense_last(a0);
  for (const Tensor* t : {&x, &a})
    if (rows_meet(state, *t)) refuse(what, ": state shares memory with x or log_decay");
  Tensor h = empty({B, D}, x.scalar_type(), x.device());
  if (B) {
    const Launch l(x.device());
    check(abi.socmx_gated_scan_step(element_type(x), element_type(a), (int32_t)B, (int32_t)D, (int32_t)a.size(1), pointer(x), x.stride(0),
                                    pointer(a), a.stride(0), state.data_ptr<float>(), state.stride(0), pointer(h), l.stream),
          "socmx_gated_scan_step");
    written(state);
  }
  return h;
}

// ---- AdamW -------------------------------------------------------------------------------------------------------------------------
typedef std::vector<Tensor> Tensors;

struct Span {                                // the memory of a dense tensor
  uintptr_t begin;
  uint64_t bytes : 63, written : 1;
  Span(const void* p, uint64_t size, bool w) : begin(reinterpret_cast<uintptr_t>(p)), bytes(size), written(w) {}
};

// whether any of them that is written shares memory with another one
bool shared(std::vector<Span>& spans) {
  std::sort(spans.begin(), spans.end(), [](const Span& a, const Span& b) { return a.begin < b.begin; });
  uintptr_t any = 0, written = 0;            // how far those in front reach
  for (const Span& s : spans) {
    if (s.begin < (s.written ? any : written)) return true;
    any = std::max<uintptr_t>(any, s.begin + s.bytes);
    if (s.written) written = std::max<uintptr_t>(written, s.begin + s.bytes);
  }
  return false;
}

constexpr int64_t kBlock = 256;

// steps: one tensor with a count for each of the params, or `counts`: a tensor of one element for each
void adamw_update(const Tensors& params, const Tensors& grads, const Tensors& ms, const Tensors& vs, const Tensor& steps, const Tensors* counts, double lr,
                  double b1, double b2, double eps, double weight_decay, const c10::optional<Tensors>& scales, const c10::optional<Tensors>& masters) {
  const char* what = "adamw_step";
  not_traced(what);
  const size_t count = params.size();
  auto same = [&](const char* name, size_t n) { if (n != count) refuse(what, ": ", count, " params and ", n, " ", name); };
  same("grads", grads.size());
  same("exp_avgs", ms.size());
  same("exp_avg_sqs", vs.size());
  if (counts) same("steps", counts->size());
  if (scales) same("scales", scales->size());
  if (masters) same("masters", masters->size());
  if (count == 0) return;
  const at::Device dev = params[0].device();
  const at::ScalarType type = params[0].scalar_type();
  on_gpu(what, params[0]);
  if (element_type(params[0]) < 0) refuse(what, ": float32, bfloat16 or float16 weights are needed, got ", type);
  if (masters && type == at::kFloat) refuse(what, ": float32 weights have no masters");
  if (!(b1 >= 0.0 && b1 < 1.0 && b2 >= 0.0 && b2 < 1.0)) refuse(what, ": betas (", b1, ", ", b2, ") outside [0, 1)");
  if (!counts && (steps.dim() != 1 || steps.size(0) != (int64_t)count || steps.scalar_type() != at::kFloat || steps.device() != dev || !steps.is_contiguous()))
    refuse(what, ": steps is a dense (", count, ",) float32 on ", dev, ", got ", shape(steps), " ", steps.scalar_type(), " on ", steps.device());
  const at::ScalarType mt = scales ? at::kChar : at::kFloat, vt = scales ? at::kByte : at::kFloat;
  if (torch::autograd::ForwardADLevel::try_get_by_idx(0))          // (no level is open, no tensor has a tangent)
    for (size_t i = 0; i < count; ++i) no_tangent(what, {&params[i], &grads[i], &ms[i], &vs[i]});
  std::vector<socmx_adamw_tensor> rows(count);
  const int64_t bytes = params[0].element_size();
  std::vector<Span> spans;
  spans.reserve(7 * count + 1);
  std::vector<float*> at;
  if (counts)
    for (size_t i = 0; i < count; ++i) {
      const Tensor& t = (*counts)[i];
      if (t.numel() != 1 || t.scalar_type() != at::kFloat || t.device() != dev)
        refuse(what, ": the step count of tensor ", i, " is one float32 on ", dev, ", got ", shape(t), " ", t.scalar_type(), " on ", t.device());
      at.push_back(t.data_ptr<float>());
      spans.emplace_back(at.back(), 4, true);
    }
  else
    spans.emplace_back(pointer(steps), 4 * count, true);
  for (size_t i = 0; i < count; ++i) {
    const Tensor &p = params[i], &g = grads[i], &m = ms[i], &v = vs[i];
    const Tensor s = scales ? (*scales)[i] : Tensor(), w = masters ? (*masters)[i] : Tensor();
    const int64_t n = p.numel();
    if (p.scalar_type() != type || g.scalar_type() != type || m.scalar_type() != mt || v.scalar_type() != vt || (masters && w.scalar_type() != at::kFloat))
      refuse(what, ": tensor ", i, " has types ", p.scalar_type(), ", ", g.scalar_type(), ", ", m.scalar_type(), ", ", v.scalar_type(),
             "; wanted ", type, ", ", type, ", ", mt, ", ", vt, masters ? ", and a float32 master" : "");
    if (g.numel() != n || m.numel() != n || v.numel() != n || (masters && w.numel() != n))
      refuse(what, ": the sizes of tensor ", i, " differ: ", n, " weights, ", g.numel(), " gradients, ", m.numel(), " and ", v.numel(), " states");
    if (scales && (s.dim() != 2 || s.size(0) != (n + kBlock - 1) / kBlock || s.size(1) != 2 || s.scalar_type() != at::kFloat))
      refuse(what, ": the scales of tensor ", i, " are (", (n + kBlock - 1) / kBlock, ", 2) float32, got ", shape(s), " ", s.scalar_type());
    // (any order of the dimensions in memory, the same for all: the update goes by memory)
    const bool plain = p.is_contiguous();
    for (const Tensor* t : {&p, &g, &m, &v, &s, &w}) {
      if (!t->defined()) continue;
      const bool alike = plain || t == &s ? t->is_contiguous()
                                          : t->is_non_overlapping_and_dense() && t->sizes() == p.sizes() && t->strides() == p.strides();
      if (t->device() != dev || !alike)
        refuse(what, ": tensor ", i, " has a part on ", t->device(), " with strides ", t->strides(), " beside ", p.strides(), "; dense ones on ", dev,
               ", laid out alike, are needed");
    }
    rows[i] = socmx_adamw_tensor{pointer(p), pointer(g), pointer(m), pointer(v), pointer_as<float>(s), pointer_as<float>(w), n};
    if (n) {
      const int64_t state = n * (scales ? 1 : 4);
      spans.emplace_back(rows[i].p, n * bytes, true);
      spans.emplace_back(rows[i].grad, n * bytes, false);
      spans.emplace_back(rows[i].exp_avg, state, true);
      spans.emplace_back(rows[i].exp_avg_sq, state, true);
      if (scales) spans.emplace_back(rows[i].scale, 8 * s.size(0), true);
      if (masters) spans.emplace_back(rows[i].master, 4 * n, true);
    }
  }
  if (shared(spans)) refuse(what, ": memory of one of the tensors, states, masters or counts is another tensor's too (gradients may be shared among themselves)");
  const Tensor ws = floats(4 * (int64_t)count, dev);
  const Launch l(dev);
  const int type_id = element_type(params[0]), bits = scales ? 8 : 32;
  if (counts)
    check(abi.socmx_adamw_step_counts(type_id, bits, rows.data(), (int32_t)count, at.data(), ws.data_ptr<float>(), lr, b1, b2, eps, weight_decay,
                                      l.stream), "socmx_adamw_step_counts");
  else
    check(abi.socmx_adamw_step(type_id, bits, rows.data(), (int32_t)count, steps.data_ptr<float>(), ws.data_ptr<float>(), lr, b1, b2, eps,
                               weight_decay, l.stream), "socmx_adamw_step");
  if (!counts) written(steps);
  for (size_t i = 0; i < count; ++i) {
    if (counts) written((*counts)[i]);
    written(params[i]);
    written(ms[i]);
    written(vs[i]);
    if (scales) written((*scales)[i]);
    if (masters) written((*masters)[i]);
  }
}

void adamw_step(const Tensors& params, const Tensors& grads, const Tensors& ms, const Tensors& vs, const Tensor& steps, double lr, double b1,
                double b2, double eps, double weight_decay, const c10::optional<Tensors>& scales, const c10::optional<Tensors>& masters) {
  adamw_update(params, grads, ms, vs, steps, nullptr, lr, b1, b2, eps, weight_decay, scales, masters);
}

void adamw_step_counts(const Tensors& params, const Tensors& grads, const Tensors& ms, const Tensors& vs, const Tensors& steps, double lr, double b1,
                       double b2, double eps, double weight_decay, const c10::optional<Tensors>& scales, const c10::optional<Tensors>& masters) {
  adamw_update(params, grads, ms, vs, Tensor(), &steps, lr, b1, b2, eps, weight_decay, scales, masters);
}

// a dense tensor of its own over a part of a buffer's storage (which lives as long as one of them does)
Tensor part_of(const Tensor& flat, int64_t offset, at::IntArrayRef sizes) {
  Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(flat.storage()), flat.key_set(), flat.dtype());
  t.unsafeGetTensorImpl()->set_storage_offset(offset);
  t.unsafeGetTensorImpl()->set_sizes_contiguous(sizes);
  return t;
}

std::pair<Tensors, Tensors> adamw_state_values(const Tensors& ms, const Tensors& vs, const Tensors& scales) {
  const char* what = "adamw_state_values";
  not_traced(what);
  const size_t count = ms.size();
  if (vs.size() != count || scales.size() != count) refuse(what, ": ", count, ", ", vs.size(), " and ", scales.size(), " tensors");
  std::pair<Tensors, Tensors> out;
  if (count == 0) return out;
  const at::Device dev = ms[0].device();
  on_gpu(what, ms[0]);
  out.first.reserve(count);
  out.second.reserve(count);
  int64_t total = 0, at = 0;           // (one allocation for all first, one for all second moments, each at a multiple of 64 bytes)
  for (const Tensor& m : ms) total += (m.numel() + 15) / 16 * 16;
  const Tensor flat_m = empty({total}, at::kFloat, dev), flat_v = empty({total}, at::kFloat, dev);
  std::vector<socmx_adamw_state> rows;
  for (size_t i = 0; i < count; ++i) {
    const Tensor &m = ms[i], &v = vs[i], &s = scales[i];
    const int64_t n = m.numel(), blocks = (n + kBlock - 1) / kBlock;
    if (m.scalar_type() != at::kChar || v.scalar_type() != at::kByte || v.sizes() != m.sizes())
      refuse(what, ": state ", i, " is int8 and uint8 codes of one shape, got ", m.scalar_type(), " ", shape(m), ", ", v.scalar_type(), " ", shape(v));
    if (s.dim() != 2 || s.size(0) != blocks || s.size(1) != 2 || s.scalar_type() != at::kFloat)
      refuse(what, ": the scales of state ", i, " are (", blocks, ", 2) float32, got ", shape(s), " ", s.scalar_type());
    for (const Tensor* t : {&m, &v, &s})
      if (t->device() != dev || !t->is_contiguous()) refuse(what, ": state ", i, " is not dense, or not on ", dev);
    out.first.push_back(part_of(flat_m, at, m.sizes()));
    out.second.push_back(part_of(flat_v, at, m.sizes()));
    at += (n + 15) / 16 * 16;
    if (n)
      rows.push_back(socmx_adamw_state{pointer(m), pointer(v), s.data_ptr<float>(), out.first.back().data_ptr<float>(),
                                       out.second.back().data_ptr<float>(), n});
  }
  if (!rows.empty()) {
    const Launch l(dev);
    check(abi.socmx_adamw_state_values(rows.data(), (int32_t)rows.size(), l.stream), "socmx_adamw_state_values");
  }
  return out;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  py::register_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const Refusal& e) {
      PyErr_SetString(socmx_error ? socmx_error : PyExc_RuntimeError, e.what());
    }
  });
  m.def("bind_library", &bind_library);
  m.def("layer_norm", &layer_norm);
  m.def("gated_scan", &gated_scan);
  m.def("gated_scan_step", &gated_scan_step);
  m.def("adamw_step", &adamw_step);
  m.def("adamw_step_counts", &adamw_step_counts);
  m.def("adamw_state_values", &adamw_state_values);
}
