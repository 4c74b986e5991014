// The plain calls of ops.w4_linear, ops.gated_linear and ops.sandwich_norm, and the last two's gradients, without Python in between: with a
// row or a few hundred they are over on the GPU in 4 - 40 us, and from Python the checks, allocations and launches of one call took 15 - 35 us,
// a forward and a backward pass 140.
//
// A function returns None for any call that is not of the plain kind (another type, device or layout, a tensor subclass, a mode that
// watches tensor functions, no rows, a wrong argument): the Python function then goes its general way, which also raises what there is to raise.
#include "host_call.h"

#include <ATen/PythonTorchFunctionTLS.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <array>
#include <atomic>

#include "../../include/ksana_b200.h"

namespace ksana_host {
namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// set by setup()
struct Library {
  decltype(&ksb_w4_linear) w4 = nullptr;
  decltype(&ksb_gated_linear) gated = nullptr;
  decltype(&ksb_gated_linear_saved) gated_saved = nullptr;
  decltype(&ksb_gated_linear_workspace) gated_workspace = nullptr;
  decltype(&ksb_gated_linear_backward) gated_backward = nullptr;
  decltype(&ksb_sandwich_norm) norm = nullptr;
  decltype(&ksb_sandwich_norm_workspace) norm_workspace = nullptr;
  decltype(&ksb_sandwich_norm_backward) norm_backward = nullptr;
  decltype(&ksb_last_error) last_error = nullptr;
  PyObject* error = nullptr;  // the library's exception
} lib;

std::atomic<int64_t> kernels{0};  // that the calls here have queued

// Kernels queued by a call, or its refusal, for which alone the interpreter is taken: in the engine's thread that takes 4 us.
void count(int rc, const char* what) {
  if (rc >= 0) {
    kernels += rc;
    return;
  }
  PyGILState_STATE gil = PyGILState_Ensure();
  PyErr_Format(lib.error, "%s failed (rc=%d): %s", what, rc, lib.last_error());
  python_error e;
  e.persist();
  PyGILState_Release(gil);
  throw e;
}

int dtype_of(const Tensor& t) { return t.scalar_type() == at::kBFloat16 ? KSB_BF16 : KSB_FP16; }
bool aligned(const Tensor& t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0; }
cudaStream_t stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }
Tensor bytes(int64_t n, const Tensor& like) { return at::empty({n}, like.options().dtype(at::kByte)); }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// Whether plain calls may take this way at all just now.
bool watched() {
  return lib.error == nullptr || at::impl::torch_function_mode_enabled() || c10::impl::TorchDispatchModeTLS::any_modes_set() || torch::jit::tracer::isTracing();
}
// A forward-mode derivative goes with the tensor, whether or not it requires a gradient.
bool has_tangent(const Tensor& t) { return t._fw_grad(0).defined(); }
// A tensor argument, or none (undefined) where that is allowed.  False: not a plain one.
bool take(PyObject* o, bool optional, Tensor& t) {
  if (o == Py_None) return optional;
  if (!plain_tensor(o)) return false;
  t = THPVariable_Unpack(o);
  return !has_tangent(t);
}
// x [.., K] of a half type on the current GPU: rows a constant distance apart, on 16-byte boundaries
bool rows(const Tensor& x, int64_t& M, int64_t& K, int64_t& ld) {
  const int64_t dim = x.dim();
  if (dim < 1 || !x.is_cuda() || x.device().index() != c10::cuda::current_device() || (x.scalar_type() != at::kBFloat16 && x.scalar_type() != at::kHalf)) return false;
  K = x.size(-1);
  if (K < 1 || x.numel() == 0 || !aligned(x)) return false;
  M = x.numel() / K;
  if (x.is_contiguous()) {
    ld = K;
    return true;
  }
  if (dim != 2 || x.stride(1) != 1 || x.stride(0) % 8 != 0 || x.stride(0) < K) return false;
  ld = x.stride(0);
  return true;
}
// a dense vector or matrix like x
bool like(const Tensor& t, const Tensor& x, at::ScalarType type) { return t.device() == x.device() && t.scalar_type() == type && aligned(t); }
std::vector<int64_t> with_last(const Tensor& x, int64_t n) {
  std::vector<int64_t> s = x.sizes().vec();
  s.back() = n;
  return s;
}
// an incoming gradient as contiguous rows
Tensor dense(const Tensor& d) {
  if (!d.defined()) return d;
  TORCH_CHECK(!has_tangent(d), "the operators of a gated half have no forward-mode derivatives");
  Tensor c = d.contiguous();
  return aligned(c) ? c : c.clone();
}
// Which of a function's tensor arguments (some of them absent) this backward pass asks gradients of.
int64_t asked(AutogradContext* ctx, int64_t there) {
  int64_t need = 0;
  for (int64_t i = 0, edge = 0; there >> i; ++i)
    if (there >> i & 1) need |= static_cast<int64_t>(ctx->needs_input_grad(edge++)) << i;
  return need;
}
// Gradients that raise when they are differentiated again: with create_graph they would count as constants.
constexpr const char* AGAIN = "the operators of a gated half have no second derivatives";
variable_list last_derivatives(variable_list&& out, bool again) {
  const auto node = again ? torch::autograd::get_current_node() : nullptr;
  for (Tensor& g : out) {
    if (!node || !g.defined()) continue;
    torch::autograd::edge_list inputs = node->next_edges();
    torch::autograd::create_gradient_edge(g, std::shared_ptr<torch::autograd::Node>(new torch::autograd::Error(AGAIN, std::move(inputs)), torch::autograd::deleteNode));
  }
  return std::move(out);
}
// A leaf's accumulation node keeps the stream that it was made on for as long as any graph of the leaf lives.  One of the default stream cannot take
// part in a capture, and its failure inside the engine can end the process; here it is an error of this call, ahead of any launch.
// Leaves whose gradients the pass does not ask for take no part.
void leaves_can_be_captured() {
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  if (cudaStreamIsCapturing(c10::cuda::getCurrentCUDAStream().stream(), &status) != cudaSuccess || status == cudaStreamCaptureStatusNone) return;
  const auto node = torch::autograd::get_current_node();
  if (!node) return;
  for (size_t i = 0; i < node->num_outputs(); ++i) {
    const auto& edge = node->next_edge(i);
    if (!edge.function || !dynamic_cast<torch::autograd::AccumulateGrad*>(edge.function.get()) || !node->task_should_compute_output(i)) continue;
    const auto stream = edge.function->stream();
    TORCH_CHECK(!stream || !stream->device().is_cuda() || c10::cuda::CUDAStream(*stream) != c10::cuda::getDefaultCUDAStream(stream->device_index()),
                "a backward pass is captured while a graph of the same leaves that was made on the default stream is alive: release its outputs first");
  }
}
PyObject* none() { Py_RETURN_NONE; }

// ---------------------------------------------------------------------------------------------- 4-bit Linear

// (x, weight, weight_scale, weight_zero, bias, out_features)
PyObject* w4_linear(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Tensor x, weight, scale, zero, bias;
  if (n != 6 || watched() || !take(args[0], false, x) || !take(args[1], false, weight) || !take(args[2], false, scale) || !take(args[3], true, zero) ||
      !take(args[4], true, bias))
    return none();
  int64_t M, K, ld, N;
  if (!rows(x, M, K, ld) || weight.dim() != 3 || scale.dim() != 3) return none();
  if (at::GradMode::is_enabled() && (x.requires_grad() || scale.requires_grad() || (bias.defined() && bias.requires_grad()))) return none();
  if (args[5] == Py_None) {
    N = bias.defined() ? bias.numel() : weight.size(0) * 16;
  } else {
    if (!PyLong_Check(args[5])) return none();
    N = PyLong_AsLongLong(args[5]);
    if (N == -1 && PyErr_Occurred()) PyErr_Clear();
  }
  const int64_t groups = scale.size(1), nt = (N + 15) / 16, group = groups > 0 ? K / groups : 0;
  if (N < 1 || !like(weight, x, at::kByte) || !weight.is_contiguous() || weight.size(0) != nt || weight.size(1) != (K + 63) / 64 || weight.size(2) != 512 ||
      (group != 32 && group != 64 && group != 128) || group * groups != K || !like(scale, x, x.scalar_type()) || !scale.is_contiguous() || scale.size(0) != nt || scale.size(2) != 16 ||
      (zero.defined() && (!like(zero, x, at::kByte) || !zero.is_contiguous() || !zero.sizes().equals(scale.sizes()))) ||
      (bias.defined() && (bias.device() != x.device() || bias.scalar_type() != x.scalar_type() || bias.dim() != 1 || bias.size(0) != N || bias.stride(0) != 1)))
    return none();
  Tensor out = at::empty(with_last(x, N), x.options());
  const int rc = lib.w4(x.data_ptr(), dtype_of(x), M, K, ld, weight.data_ptr(), scale.data_ptr(), ptr(zero), static_cast<int>(group), ptr(bias), N, out.data_ptr(), N, stream_of(x));
  count(rc, "ksb_w4_linear");
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------------------------------------- gated projections

struct GatedShape {
  int64_t M, F, K, ldx, ldg, ldu;
};
bool gated_shape(const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& bg, const Tensor& bu, GatedShape& s) {
  int64_t K;
  if (wg.dim() != 2 || wu.dim() != 2 || !rows(x, s.M, s.K, s.ldx) || !rows(wg, s.F, K, s.ldg) || K != s.K || !rows(wu, s.F, K, s.ldu)) return false;
  if (!wu.sizes().equals(wg.sizes()) || wg.scalar_type() != x.scalar_type() || wu.scalar_type() != x.scalar_type() || s.F % 8 != 0 || s.K % 8 != 0) return false;
  for (const Tensor* b : {&bg, &bu})
    if (b->defined() && (!like(*b, x, x.scalar_type()) || b->dim() != 1 || b->size(0) != s.F || b->stride(0) != 1)) return false;
  return true;
}
Tensor gated_run(const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& bg, const Tensor& bu, int act, const GatedShape& s, const Tensor& saved) {
  Tensor h = at::empty(with_last(x, s.F), x.options());
  count(lib.gated(x.data_ptr(), s.ldx, wg.data_ptr(), s.ldg, wu.data_ptr(), s.ldu, ptr(bg), ptr(bu), dtype_of(x), s.M, s.F, s.K, act, h.data_ptr(), ptr(saved), stream_of(x)),
        "ksb_gated_linear");
  return h;
}

struct GatedLinear : torch::autograd::Function<GatedLinear> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& wg, const Tensor& wu, const std::optional<Tensor>& bg, const std::optional<Tensor>& bu, int64_t act) {
    const Tensor b0 = bg.value_or(Tensor()), b1 = bu.value_or(Tensor());
    GatedShape s;
    TORCH_CHECK(gated_shape(x, wg, wu, b0, b1, s), "gated_linear: the tensors changed under the call");
    const Tensor saved = bytes(lib.gated_saved(s.M, s.F), x);
    const Tensor h = gated_run(x, wg, wu, b0, b1, static_cast<int>(act), s, saved);
    ctx->save_for_backward({x, wg, wu, saved});
    ctx->saved_data["act"] = act;
    ctx->saved_data["there"] = static_cast<int64_t>(7 | b0.defined() << 3 | b1.defined() << 4);
    return h;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    leaves_can_be_captured();
    const bool again = at::GradMode::is_enabled();
    at::NoGradGuard no_grad;
    variable_list out(6);
    if (!grads[0].defined()) return out;
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &wg = saved[1], &wu = saved[2], dh = dense(grads[0]);
    GatedShape s;
    const Tensor no;
    TORCH_CHECK(gated_shape(x, wg, wu, no, no, s), "gated_linear: the saved tensors are not those of the call");
    const int64_t need = asked(ctx, ctx->saved_data["there"].toInt());
    const std::array<std::vector<int64_t>, 5> shapes{x.sizes().vec(), {s.F, s.K}, {s.F, s.K}, {s.F}, {s.F}};
    for (int i = 0; i < 5; ++i)
      if (need >> i & 1) out[i] = at::empty(shapes[i], x.options());
    const Tensor ws = bytes(lib.gated_workspace(s.M, s.F, s.K), x);
    ksb_gated_linear_grads a{};
    a.x = x.data_ptr(); a.w_gate = wg.data_ptr(); a.w_up = wu.data_ptr(); a.saved = saved[3].data_ptr(); a.dh = dh.data_ptr();
    a.dx = ptr(out[0]); a.dw_gate = ptr(out[1]); a.dw_up = ptr(out[2]); a.db_gate = ptr(out[3]); a.db_up = ptr(out[4]);
    a.M = s.M; a.F = s.F; a.K = s.K; a.ldx = s.ldx; a.ldg = s.ldg; a.ldu = s.ldu; a.lddh = s.F;
    a.dtype = dtype_of(x); a.act = static_cast<int>(ctx->saved_data["act"].toInt());
    count(lib.gated_backward(&a, ws.data_ptr(), stream_of(x)), "ksb_gated_linear_backward");
    return last_derivatives(std::move(out), again);
  }
};

std::optional<Tensor> maybe(const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; }
bool wants_grad(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

// (x, w_gate, w_up, b_gate, b_up, act)
PyObject* gated_linear(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Tensor x, wg, wu, bg, bu;
  if (n != 6 || watched() || !take(args[0], false, x) || !take(args[1], false, wg) || !take(args[2], false, wu) || !take(args[3], true, bg) || !take(args[4], true, bu) ||
      !PyLong_Check(args[5]))
    return none();
  const int act = static_cast<int>(PyLong_AsLong(args[5]));
  GatedShape s;
  if (!gated_shape(x, wg, wu, bg, bu, s)) return none();
  if (wants_grad({&x, &wg, &wu, &bg, &bu})) return THPVariable_Wrap(GatedLinear::apply(x, wg, wu, maybe(bg), maybe(bu), static_cast<int64_t>(act)));
  return THPVariable_Wrap(gated_run(x, wg, wu, bg, bu, act, s, Tensor()));
  END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------------------------------------- norms on both sides

enum NormTensor { X, Y, GATE, SCALE, SHIFT, POST, PRE, NORM_TENSORS };
typedef std::array<Tensor, NORM_TENSORS> NormTensors;

// How many rows a modulation tensor has for x, and the distance between them; 0: not one of the plain kind.
int64_t modulation_rows(const Tensor& t, const Tensor& x, int64_t& stride) {
  const int64_t C = x.size(-1), lead = x.dim() - 1;
  stride = 0;
  if (!like(t, x, x.scalar_type()) || t.dim() < 1 || t.size(-1) != C || t.stride(-1) != 1) return 0;
  if (t.numel() == C) return 1;
  int64_t n = 0, axes = 0;  // axes: those that tell rows apart
  if (t.dim() == 2) {
    n = t.size(0);
    axes = 1;
    if (!(lead == 1 ? n > 0 && x.size(0) % n == 0 : n == x.size(0))) return 0;
  } else if (t.dim() == x.dim()) {
    n = 1;
    while (axes < lead && t.size(axes) == x.size(axes)) n *= t.size(axes++);
    for (int64_t i = axes; i < lead; ++i)
      if (t.size(i) != 1) return 0;
  } else {
    return 0;
  }
  if (!t.is_contiguous()) {
    if (axes != 1) return 0;
    stride = t.stride(0);
  } else {
    stride = C;
  }
  return stride % 8 == 0 ? n : 0;
}

struct NormCall {
  ksb_sandwich_norm_args a{};
  bool pre = true;
};
// Fills a call's arguments; false: not one of the plain kind.
bool norm_call(const NormTensors& t, double residual_scale, bool pre, bool layer, double eps, NormCall& c) {
  ksb_sandwich_norm_args& a = c.a;
  c.pre = pre;
  if (!rows(t[X], a.M, a.C, a.ldx) || a.C % 8 != 0 || a.C > KSB_NORM_MAX_C || a.M > KSB_NORM_MAX_M) return false;
  if (t[Y].defined()) {
    int64_t M, C;
    if (!t[Y].sizes().equals(t[X].sizes()) || t[Y].scalar_type() != t[X].scalar_type() || !rows(t[Y], M, C, a.ldy)) return false;
  } else if (!pre || t[GATE].defined() || t[POST].defined()) {
    return false;
  }
  if (!pre && (t[SCALE].defined() || t[SHIFT].defined() || t[PRE].defined())) return false;
  for (int i : {POST, PRE})
    if (t[i].defined() && (!like(t[i], t[X], at::kFloat) || t[i].dim() != 1 || t[i].size(0) != a.C || t[i].stride(0) != 1)) return false;
  a.mod_rows = 1;
  int64_t n[3], stride[3];
  for (int i = 0; i < 3; ++i) {
    const Tensor& m = t[GATE + i];
    n[i] = 1;
    stride[i] = 0;
    if (!m.defined()) continue;
    n[i] = modulation_rows(m, t[X], stride[i]);
    if (n[i] == 0 || (n[i] != 1 && a.mod_rows != 1 && a.mod_rows != n[i])) return false;
    a.mod_rows = std::max(a.mod_rows, n[i]);
  }
  a.gate_stride = n[0] == 1 ? 0 : stride[0];
  a.scale_stride = n[1] == 1 ? 0 : stride[1];
  a.shift_stride = n[2] == 1 ? 0 : stride[2];
  a.x = t[X].data_ptr(); a.y = ptr(t[Y]); a.gate = ptr(t[GATE]); a.scale = ptr(t[SCALE]); a.shift = ptr(t[SHIFT]);
  a.post_w = static_cast<const float*>(ptr(t[POST])); a.pre_w = static_cast<const float*>(ptr(t[PRE]));
  a.dtype = dtype_of(t[X]); a.layer = layer; a.eps = static_cast<float>(eps); a.residual_scale = static_cast<float>(residual_scale);
  return true;
}
// (r, h), undefined where there is none
std::pair<Tensor, Tensor> norm_run(const NormTensors& t, NormCall& c, const Tensor& stats) {
  Tensor r, h;
  if (t[Y].defined()) r = at::empty(t[X].sizes(), t[X].options());
  if (c.pre) h = at::empty(t[X].sizes(), t[X].options());
  c.a.stats = static_cast<float*>(ptr(stats));
  count(lib.norm(&c.a, ptr(r), ptr(h), stream_of(t[X])), "ksb_sandwich_norm");
  return {r, h};
}

struct SandwichNorm : torch::autograd::Function<SandwichNorm> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const std::optional<Tensor>& y, const std::optional<Tensor>& gate, const std::optional<Tensor>& scale,
                               const std::optional<Tensor>& shift, const std::optional<Tensor>& post, const std::optional<Tensor>& pre_w, double residual_scale, bool pre, bool layer,
                               double eps) {
    const Tensor no;
    const NormTensors t{x, y.value_or(no), gate.value_or(no), scale.value_or(no), shift.value_or(no), post.value_or(no), pre_w.value_or(no)};
    NormCall c;
    TORCH_CHECK(norm_call(t, residual_scale, pre, layer, eps, c), "sandwich_norm: the tensors changed under the call");
    const Tensor stats = at::empty({c.a.M, 4}, x.options().dtype(at::kFloat));
    auto [r, h] = norm_run(t, c, stats);
    ctx->set_materialize_grads(false);
    variable_list save(t.begin(), t.end());
    save.push_back(stats);
    ctx->save_for_backward(save);
    int64_t there = 0;
    for (int i = 0; i < NORM_TENSORS; ++i) there |= static_cast<int64_t>(t[i].defined()) << i;
    ctx->saved_data["there"] = there;
    ctx->saved_data["residual_scale"] = residual_scale;
    ctx->saved_data["pre"] = pre;
    ctx->saved_data["layer"] = layer;
    ctx->saved_data["eps"] = eps;
    variable_list out;
    if (r.defined()) out.push_back(r);
    if (h.defined()) out.push_back(h);
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    leaves_can_be_captured();
    const bool again = at::GradMode::is_enabled();
    at::NoGradGuard no_grad;
    variable_list out(NORM_TENSORS + 4);
    const auto saved = ctx->get_saved_variables();
    NormTensors t;
    std::copy_n(saved.begin(), static_cast<int>(NORM_TENSORS), t.begin());
    const bool pre = ctx->saved_data["pre"].toBool(), behind = t[Y].defined();
    const Tensor dr = behind ? dense(grads[0]) : Tensor(), dh = pre ? dense(grads[behind ? 1 : 0]) : Tensor();
    if (!dr.defined() && !dh.defined()) return out;
    NormCall c;
    TORCH_CHECK(norm_call(t, ctx->saved_data["residual_scale"].toDouble(), pre, ctx->saved_data["layer"].toBool(), ctx->saved_data["eps"].toDouble(), c),
                "sandwich_norm: the saved tensors are not those of the call");
    c.a.stats = static_cast<float*>(saved[NORM_TENSORS].data_ptr());
    const int64_t need = asked(ctx, ctx->saved_data["there"].toInt());
    const Tensor& x = t[X];
    for (int i = 0; i < NORM_TENSORS; ++i) {
      // without dh, what belongs to the norm behind the sum has no gradient
      const bool there = i == X || (i == Y || i == GATE || i == POST ? behind : dh.defined());
      if (!(need >> i & 1) || !there) continue;
      if (i == POST || i == PRE) out[i] = at::empty({c.a.C}, x.options().dtype(at::kFloat));
      else if (i < GATE) out[i] = at::empty(x.sizes(), x.options());
      else out[i] = at::empty(t[i].sizes(), x.options());
    }
    ksb_sandwich_norm_grads g{};
    for (int i = GATE; i <= SHIFT; ++i)  // one row for rows that others of the call tell apart
      if (t[i].defined() && c.a.mod_rows > 1 && t[i].numel() == c.a.C) g.one_row |= 1 << (i - GATE);
    g.dr = ptr(dr); g.dh = ptr(dh); g.lddr = g.lddh = c.a.C;
    g.dx = ptr(out[X]); g.dy = ptr(out[Y]); g.dgate = ptr(out[GATE]); g.dscale = ptr(out[SCALE]); g.dshift = ptr(out[SHIFT]);
    g.dpost_w = static_cast<float*>(ptr(out[POST])); g.dpre_w = static_cast<float*>(ptr(out[PRE]));
    const Tensor ws = bytes(lib.norm_workspace(c.a.M, c.a.C, c.a.mod_rows), x);
    count(lib.norm_backward(&c.a, &g, ws.data_ptr(), stream_of(x)), "ksb_sandwich_norm_backward");
    return last_derivatives(std::move(out), again);
  }
};

// (x, y, gate, scale, shift, post_weight, pre_weight, residual_scale, pre, layer, eps) -> (r or None, h or None)
PyObject* sandwich_norm(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != NORM_TENSORS + 4 || watched()) return none();
  NormTensors t;
  for (int i = 0; i < NORM_TENSORS; ++i)
    if (!take(args[i], i != X, t[i])) return none();
  if (!PyFloat_Check(args[7]) || !PyBool_Check(args[8]) || !PyBool_Check(args[9]) || !PyFloat_Check(args[10])) return none();
  const double residual_scale = PyFloat_AS_DOUBLE(args[7]), eps = PyFloat_AS_DOUBLE(args[10]);
  const bool pre = args[8] == Py_True, layer = args[9] == Py_True;
  NormCall c;
  if (!norm_call(t, residual_scale, pre, layer, eps, c)) return none();
  Tensor r, h;
  if (wants_grad({&t[X], &t[Y], &t[GATE], &t[SCALE], &t[SHIFT], &t[POST], &t[PRE]})) {
    variable_list out = SandwichNorm::apply(t[X], maybe(t[Y]), maybe(t[GATE]), maybe(t[SCALE]), maybe(t[SHIFT]), maybe(t[POST]), maybe(t[PRE]), residual_scale, pre, layer, eps);
    if (t[Y].defined()) r = out[0];
    if (pre) h = out.back();
  } else {
    std::tie(r, h) = norm_run(t, c, Tensor());
  }
  Ref pr(nullptr), ph(nullptr);
  pr.p = r.defined() ? THPVariable_Wrap(r) : (Py_INCREF(Py_None), Py_None);
  ph.p = h.defined() ? THPVariable_Wrap(h) : (Py_INCREF(Py_None), Py_None);
  if (!pr.p || !ph.p) return nullptr;
  return PyTuple_Pack(2, pr.p, ph.p);
  END_HANDLE_TH_ERRORS
}

// For a backward pass that runs in Python.
PyObject* check_captured_leaves(PyObject*, PyObject*) {
  HANDLE_TH_ERRORS
  leaves_can_be_captured();
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

PyObject* queued(PyObject*, PyObject*) { return PyLong_FromLongLong(kernels); }

// setup(the library's exception, addresses of the nine entries above in their order)
PyObject* setup(PyObject*, PyObject* args) {
  PyObject* error;
  unsigned long long at[9];
  if (!PyArg_ParseTuple(args, "O(KKKKKKKKK)", &error, at, at + 1, at + 2, at + 3, at + 4, at + 5, at + 6, at + 7, at + 8)) return nullptr;
  lib.w4 = reinterpret_cast<decltype(lib.w4)>(at[0]);
  lib.gated = reinterpret_cast<decltype(lib.gated)>(at[1]);
  lib.gated_saved = reinterpret_cast<decltype(lib.gated_saved)>(at[2]);
  lib.gated_workspace = reinterpret_cast<decltype(lib.gated_workspace)>(at[3]);
  lib.gated_backward = reinterpret_cast<decltype(lib.gated_backward)>(at[4]);
  lib.norm = reinterpret_cast<decltype(lib.norm)>(at[5]);
  lib.norm_workspace = reinterpret_cast<decltype(lib.norm_workspace)>(at[6]);
  lib.norm_backward = reinterpret_cast<decltype(lib.norm_backward)>(at[7]);
  lib.last_error = reinterpret_cast<decltype(lib.last_error)>(at[8]);
  Py_INCREF(error);
  Py_XSETREF(lib.error, error);  // the last: see watched
  Py_RETURN_NONE;
}

PyCFunction fast(PyObject* (*f)(PyObject*, PyObject* const*, Py_ssize_t)) { return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)); }

}  // namespace

PyMethodDef op_methods[] = {{"setup", setup, METH_VARARGS, nullptr},
                            {"queued", queued, METH_NOARGS, nullptr},
                            {"check_captured_leaves", check_captured_leaves, METH_NOARGS, nullptr},
                            {"w4_linear", fast(w4_linear), METH_FASTCALL, nullptr},
                            {"gated_linear", fast(gated_linear), METH_FASTCALL, nullptr},
                            {"sandwich_norm", fast(sandwich_norm), METH_FASTCALL, nullptr},
                            {nullptr, nullptr, 0, nullptr}};

}  // namespace ksana_host
