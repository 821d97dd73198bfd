// Ordinary eager calls without Python between the launches: the checks of a call, its allocations, the C-ABI entry points,
// the autograd nodes of the two losses and the optimiser's calls, as an extension module of CPython over torch's C++ interface.
//
// A small step is host work: with the same steps in Python (ctypes, torch.empty, an autograd.Function whose backward takes the
// interpreter's lock on autograd's device thread) B=64, K=32, F=4096, D=256 fp32 takes 160 us (TopK) and 195 us
// (hierarchical) for 35-45 us of kernels; the figures with this module stand at the entry points in ops.py.
//
// A function here returns None for a call that is not its business (tensors that are not plain, something around the call that
// has to see the ops, arguments that a check refuses): the caller then goes through the ops, which see, resolve or refuse it.
// A backward whose surroundings or gradient are not plain calls back into ops.py with what was saved.
#include <dlfcn.h>

#include <atomic>
#include <cmath>
#include <optional>
#include <vector>

#include <ATen/ATen.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/pybind.h>

#include "../../include/flexsae_amd.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Variable;
using torch::autograd::variable_list;

// ---- the library ---------------------------------------------------------------------------
#define FLEXSAE_ENTRIES(X)                                                                                              \
  X(abi_version) X(fwd_workspace_bytes) X(topk_fwd_best_workspace_bytes) X(topk_fwd) X(hier_fwd)                        \
  X(topk_bwd_from_indices_workspace_bytes) X(topk_bwd_from_indices) X(hier_bwd_workspace_bytes) X(hier_bwd)             \
  X(hier_fwd_bwd_workspace_bytes_flags) X(hier_step) X(finish_grads)                                                    \
  X(grad_norm_workspace_bytes) X(grad_norm) X(adamw_step) X(adamw_check) X(adamw8_moments)                              \
  X(layer_norm_fwd) X(layer_norm_bwd_workspace_bytes) X(layer_norm_bwd) X(lookup_fwd) X(lookup_bwd_workspace_bytes)     \
  X(lookup_bwd) X(distill_workspace_bytes) X(distill_fwd) X(distill_bwd)
struct Library {
#define X(name) decltype(&flexsae_##name) name = nullptr;
  FLEXSAE_ENTRIES(X)
#undef X
} lib;

// What the Python side keeps: callbacks, the flags of the devices (never freed: the interpreter is gone when statics are) and
// settings.
PyObject *general_backward = nullptr;  // (kind, grad, saved, needs, numbers, dW) -> (gradients, dW left)
PyObject *raise_status = nullptr;      // (status, entry point)
constexpr int kMaxDevices = 64;
Tensor *const status_flags = new Tensor[kMaxDevices];
std::atomic<int> topk_bwd_flags{0};
std::atomic<bool> lists_in_python{false};  // a shared_pair_list() block is active: backwards look there first

[[noreturn]] void throw_python() {  // what the interpreter has raised
  if (!PyErr_Occurred()) PyErr_SetString(PyExc_TypeError, "unexpected result of a callback");
  python_error e;
  e.persist();
  throw e;
}

void check(int status, const char *entry) {
  if (status == FLEXSAE_OK) return;
  pybind11::gil_scoped_acquire gil;
  PyObject *r = PyObject_CallFunction(raise_status, "is", status, entry);
  Py_XDECREF(r);
  throw_python();
}

// ---- which calls ---------------------------------------------------------------------------
// A tensor on the GPU whose values are its memory and which nothing but autograd looks at.
bool plain_tensor(const Tensor &t) {
  static const uint64_t usual =
      (c10::DispatchKeySet(c10::DispatchKey::CUDA) | c10::DispatchKeySet(c10::DispatchKey::AutogradCUDA) |
       c10::DispatchKeySet(c10::DispatchKey::ADInplaceOrView) | c10::DispatchKeySet(c10::DispatchKey::AutocastCUDA))
          .raw_repr();
  return t.defined() && t.is_cuda() && (t.key_set().raw_repr() & ~usual) == 0 && !t._fw_grad(0).defined();
}

// Nothing around the call that has to see the ops: modes, transforms, tracers.
bool plain_surroundings() {
  static const c10::DispatchKeySet watching(
      {c10::DispatchKey::FuncTorchDynamicLayerFrontMode, c10::DispatchKey::FuncTorchDynamicLayerBackMode,
       c10::DispatchKey::Functionalize, c10::DispatchKey::Python, c10::DispatchKey::PreDispatch, c10::DispatchKey::Tracer,
       c10::DispatchKey::FuncTorchBatched, c10::DispatchKey::FuncTorchVmapMode});
  return c10::impl::TorchDispatchModeTLS::stack_len() == 0 && !c10::impl::TorchDispatchModeTLS::any_modes_set() &&
         at::impl::PythonTorchFunctionTLS::stack_len() == 0 &&
         !c10::impl::tls_local_dispatch_key_set().included_.has_any(watching);
}

bool plain_backward(const Tensor &grad) {
  return !c10::GradMode::is_enabled() && plain_tensor(grad) && plain_surroundings();
}

int dtype_of(c10::ScalarType t) {
  switch (t) {
    case c10::ScalarType::Float: return FLEXSAE_F32;
    case c10::ScalarType::BFloat16: return FLEXSAE_BF16;
    case c10::ScalarType::Half: return FLEXSAE_F16;
    default: return -1;
  }
}

struct Inputs {
  Tensor indices, weight, vals, bias, target;
};

// The checks of _validate in ops.py (which says what is wrong with what fails here).  A bias that is not defined is not asked for.
bool usable(const Inputs &in) {
  for (const Tensor *t : {&in.indices, &in.weight, &in.vals, &in.bias, &in.target})
    if (t->defined() || t != &in.bias)
      if (!plain_tensor(*t) || t->device() != in.weight.device() || t->dim() != (t == &in.bias ? 1 : 2)) return false;
  const int64_t B = in.indices.size(0), K = in.indices.size(1), F = in.weight.size(0), D = in.weight.size(1);
  if (in.vals.size(0) != B || in.vals.size(1) != K || (in.bias.defined() && in.bias.size(0) != D) || in.target.size(0) != B ||
      in.target.size(1) != D)
    return false;
  if (B < 1 || K < 1 || F < 1 || D < 1 || F >= (int64_t{1} << 31) || D >= (int64_t{1} << 29) ||
      B > ((int64_t{1} << 32) - 1) / K)
    return false;
  if (in.indices.scalar_type() != c10::ScalarType::Long) return false;
  for (const Tensor *t : {&in.weight, &in.vals, &in.bias, &in.target})
    if (t->defined() && dtype_of(t->scalar_type()) < 0) return false;
  const int device = in.weight.device().index();
  return device >= 0 && device < kMaxDevices && status_flags[device].defined();
}

// What hooks have handed back for the saved tensors of a backward may be anything.
bool usable_fp32(const Tensor &t, const Tensor &weight, at::IntArrayRef sizes) {
  return plain_tensor(t) && t.device() == weight.device() && t.sizes() == sizes && t.scalar_type() == c10::ScalarType::Float;
}

// ... of a backward of its own: indices, weight, vals, resid
bool usable_saved(const variable_list &saved) {
  return usable({saved[0], saved[1], saved[2], Tensor(), saved[3]}) && saved[3].scalar_type() == c10::ScalarType::Float;
}

// ... of a step: its inputs
bool usable_inputs(const variable_list &saved) { return usable({saved[0], saved[1], saved[2], saved[3], saved[4]}); }

flexsae_shape shape_of(const Tensor &indices, const Tensor &weight, const Tensor &vals, int bias_dtype, int target_dtype) {
  return {indices.size(0), indices.size(1), weight.size(0), weight.size(1), dtype_of(weight.scalar_type()),
          dtype_of(vals.scalar_type()), bias_dtype, target_dtype};
}

flexsae_shape shape_of(const Inputs &in) {
  return shape_of(in.indices, in.weight, in.vals, dtype_of(in.bias.scalar_type()), dtype_of(in.target.scalar_type()));
}

// Contiguous and 16-byte aligned, as the vector accesses of the kernels need.
Tensor prepared(const Tensor &t) {
  const Tensor c = t.contiguous();
  return reinterpret_cast<uintptr_t>(c.data_ptr()) % 16 ? c.clone() : c;
}

Inputs prepared(const Inputs &in) {
  return {prepared(in.indices), prepared(in.weight), prepared(in.vals), prepared(in.bias), prepared(in.target)};
}

Tensor make(const Tensor &like, at::IntArrayRef sizes, c10::ScalarType type) {
  return at::empty(sizes, like.options().dtype(type).requires_grad(false));
}

Tensor make_workspace(const Tensor &like, size_t bytes) {
  return make(like, {static_cast<int64_t>(bytes)}, c10::ScalarType::Byte);
}

int *flag_of(const Tensor &t) { return status_flags[t.device().index()].data_ptr<int>(); }
void *stream_of(const Tensor &t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
bool capturing(const Tensor &t) {
  const c10::DeviceGuard guard(t.device());
  return c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None;
}
// The graph that the tensor's current stream is captured into: 0 for none, else a number of its own.
int64_t capture_of(const Tensor &t) {
  const c10::DeviceGuard guard(t.device());
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  unsigned long long id = 0;
  const hipError_t rc = hipStreamGetCaptureInfo(c10::hip::getCurrentHIPStream(t.device().index()).stream(), &status, &id);
  TORCH_CHECK(rc == hipSuccess, "hipStreamGetCaptureInfo: ", hipGetErrorString(rc));
  return status == hipStreamCaptureStatusNone ? 0 : static_cast<int64_t>(id) + 1;
}
const int64_t *index_ptr(const Tensor &t) { return t.const_data_ptr<int64_t>(); }
float *f32(const Tensor &t) { return t.data_ptr<float>(); }

// The upstream gradient as one fp32 number on the device.
Tensor grad_scalar(const Tensor &grad, const c10::Device &device) {
  const Tensor g = grad.detach();
  if (g.scalar_type() == c10::ScalarType::Float && g.device() == device && g.numel() == 1) return g;
  return g.to(device, c10::ScalarType::Float).reshape({1}).contiguous();
}

// ---- the steps -----------------------------------------------------------------------------
// (loss, resid)
std::pair<Tensor, Tensor> forward(bool topk, const Inputs &given) {
  const c10::DeviceGuard guard(given.weight.device());
  const Inputs in = prepared(given);
  const flexsae_shape s = shape_of(in);
  const size_t bytes = topk ? lib.topk_fwd_best_workspace_bytes(&s) : lib.fwd_workspace_bytes(&s);
  const Tensor workspace = make_workspace(in.weight, bytes);
  Tensor loss = make(in.weight, {}, c10::ScalarType::Float);
  Tensor resid = make(in.weight, {s.B, s.D}, c10::ScalarType::Float);
  check((topk ? lib.topk_fwd : lib.hier_fwd)(&s, index_ptr(in.indices), in.weight.data_ptr(), in.vals.data_ptr(),
                                             in.bias.data_ptr(), in.target.data_ptr(), f32(loss), f32(resid),
                                             workspace.data_ptr(), bytes, flag_of(in.weight), stream_of(in.weight)),
        topk ? "flexsae_topk_fwd" : "flexsae_hier_fwd");
  return {loss, resid};
}

// (dW, dvals, dbias), dvals and dbias times grad (undefined: one) in the leaves' types; dW_unit (undefined: none) times it in
// the weight's, in place where it has that type and is to be
std::tuple<Tensor, Tensor, Tensor> finish(const Tensor &grad, const Tensor &weight, const Tensor &dW_unit, const Tensor &dvals,
                                          c10::ScalarType vals_type, const Tensor &dbias, c10::ScalarType bias_type,
                                          bool in_place = true) {
  const Tensor g = grad.defined() ? grad_scalar(grad, weight.device()) : Tensor();
  Tensor dW;
  if (dW_unit.defined())
    dW = in_place && dW_unit.scalar_type() == weight.scalar_type() ? dW_unit : make(weight, dW_unit.sizes(), weight.scalar_type());
  Tensor out_v = make(weight, dvals.sizes(), vals_type), out_b = make(weight, dbias.sizes(), bias_type);
  check(lib.finish_grads(dW.defined() ? dW.data_ptr() : nullptr, dtype_of(weight.scalar_type()),
                         dW.defined() ? dW_unit.data_ptr() : nullptr,
                         dtype_of((dW.defined() ? dW_unit : weight).scalar_type()), dW.defined() ? dW.numel() : 0,
                         out_v.data_ptr(), dtype_of(vals_type), f32(dvals), dvals.numel(), out_b.data_ptr(),
                         dtype_of(bias_type), f32(dbias), dbias.numel(), g.defined() ? f32(g) : nullptr, stream_of(weight)),
        "flexsae_finish_grads");
  return {dW, out_v, out_b};
}

// How a training step of the hierarchical loss runs: what ops.py has decided about it.
struct StepPlan {
  bool need_dw;
  int64_t slice_cols;
  int64_t flags;     // of the call
  int64_t ws_flags;  // of the workspace query
  Tensor stats;      // pinned memory for what the pair list says about the indices (undefined: not wanted) ...
  int64_t tag;       // ... and the mark that it has arrived
};

struct Step {
  Tensor loss, dvals, dbias, dW;
};

// grad (undefined: the unit gradient, of fp16 weights in fp32): dW is the gradient for it in the weight's type.
// step: dW is not formed, the weights move by it.
Step hier_step(const Inputs &given, const StepPlan &p, const Tensor &grad = Tensor(), const Tensor &step = Tensor()) {
  const c10::DeviceGuard guard(given.weight.device());
  const Inputs in = prepared(given);
  const flexsae_shape s = shape_of(in);
  const size_t bytes = lib.hier_fwd_bwd_workspace_bytes_flags(&s, p.slice_cols, static_cast<int>(p.ws_flags));
  const Tensor workspace = make_workspace(in.weight, bytes);
  const bool half = in.weight.scalar_type() == c10::ScalarType::Half;
  const auto type = half && !grad.defined() ? c10::ScalarType::Float : in.weight.scalar_type();
  Step r;
  r.loss = make(in.weight, {}, c10::ScalarType::Float);
  if (p.need_dw && !step.defined()) r.dW = make(in.weight, {s.F, s.D}, type);
  r.dvals = make(in.weight, {s.B, s.K}, c10::ScalarType::Float);
  r.dbias = make(in.weight, {s.D}, c10::ScalarType::Float);
  const Tensor g = grad.defined() ? grad_scalar(grad, in.weight.device()) : Tensor();
  const Tensor by = step.defined() ? grad_scalar(step, in.weight.device()) : Tensor();
  const int status = lib.hier_step(
      &s, index_ptr(in.indices), in.weight.data_ptr(), in.vals.data_ptr(), in.bias.data_ptr(), in.target.data_ptr(),
      g.defined() ? f32(g) : nullptr, by.defined() ? f32(by) : nullptr, f32(r.loss),
      r.dW.defined() ? r.dW.data_ptr() : nullptr, dtype_of(type), f32(r.dvals), f32(r.dbias), workspace.data_ptr(), bytes,
      static_cast<int>(p.flags) | (p.need_dw ? 0 : FLEXSAE_BWD_NO_DW),
      p.stats.defined() ? static_cast<uint32_t *>(p.stats.data_ptr()) : nullptr, static_cast<uint32_t>(p.tag),
      flag_of(in.weight), stream_of(in.weight));
  // (a call that was refused, here or by an allocation above, has left the weights alone)
  if (step.defined() && (status == FLEXSAE_OK || status == FLEXSAE_ERR_LAUNCH))
    torch::autograd::impl::bump_version(given.weight);
  check(status, "flexsae_hier_step");
  return r;
}

// ---- autograd ------------------------------------------------------------------------------
enum Kind { kTopk = 0, kHier = 1, kSliced = 2, kLate = 3 };

void save_plan(AutogradContext *ctx, const StepPlan &plan) {
  ctx->saved_data["need_dw"] = static_cast<int64_t>(plan.need_dw);
  ctx->saved_data["cols"] = plan.slice_cols;
  ctx->saved_data["flags"] = plan.flags;
  ctx->saved_data["ws_flags"] = plan.ws_flags;
}

StepPlan saved_plan(AutogradContext *ctx) {
  return {ctx->saved_data["need_dw"].toInt() != 0, ctx->saved_data["cols"].toInt(), ctx->saved_data["flags"].toInt(),
          ctx->saved_data["ws_flags"].toInt(), Tensor(), 0};
}

// A backward that is not plain, by ops.py; dW: the unit gradient, which it may take or leave.
variable_list backward_in_python(AutogradContext *ctx, Kind kind, const Tensor &grad, const variable_list &saved,
                                 std::initializer_list<int64_t> numbers, Tensor *dW, size_t n_inputs) {
  pybind11::gil_scoped_acquire gil;
  auto tuple_of = [](size_t n, auto item) {
    auto t = pybind11::reinterpret_steal<pybind11::object>(PyTuple_New(static_cast<Py_ssize_t>(n)));
    for (size_t i = 0; i < n; ++i) PyTuple_SET_ITEM(t.ptr(), static_cast<Py_ssize_t>(i), item(i));
    return t;
  };
  const auto py_saved = tuple_of(saved.size(), [&](size_t i) { return THPVariable_Wrap(saved[i]); });
  const auto py_needs = tuple_of(5, [&](size_t i) { return PyBool_FromLong(ctx->needs_input_grad(i)); });
  const auto py_numbers = tuple_of(numbers.size(), [&](size_t i) { return PyLong_FromLongLong(numbers.begin()[i]); });
  const auto py_grad = pybind11::reinterpret_steal<pybind11::object>(THPVariable_Wrap(grad));
  const auto py_dw = dW && dW->defined() ? pybind11::reinterpret_steal<pybind11::object>(THPVariable_Wrap(*dW))
                                         : pybind11::reinterpret_borrow<pybind11::object>(Py_None);
  const auto r = pybind11::reinterpret_steal<pybind11::object>(
      PyObject_CallFunction(general_backward, "iOOOOO", static_cast<int>(kind), py_grad.ptr(), py_saved.ptr(),
                            py_needs.ptr(), py_numbers.ptr(), py_dw.ptr()));
  if (!r.ptr()) throw_python();
  PyObject *const grads = PyTuple_GetItem(r.ptr(), 0), *const left = PyTuple_GetItem(r.ptr(), 1);
  if (!grads || !left || !PyTuple_Check(grads) || PyTuple_GET_SIZE(grads) != 5) throw_python();
  if (dW) *dW = left == Py_None ? Tensor() : THPVariable_Unpack(left);
  variable_list out(n_inputs);
  for (Py_ssize_t i = 0; i < 5; ++i) {
    PyObject *const g = PyTuple_GET_ITEM(grads, i);
    if (g != Py_None) out[static_cast<size_t>(i)] = THPVariable_Unpack(g);
  }
  return out;
}

struct TopkLoss : torch::autograd::Function<TopkLoss> {
  static Variable forward(AutogradContext *ctx, const Variable &indices, const Variable &weight, const Variable &vals,
                          const Variable &bias, const Variable &target) {
    auto [loss, resid] = ::forward(true, {indices, weight, vals, bias, target});
    ctx->save_for_backward({indices, weight, vals, resid});
    ctx->set_materialize_grads(false);
    ctx->saved_data["bias"] = static_cast<int64_t>(bias.scalar_type());
    ctx->saved_data["target"] = static_cast<int64_t>(target.scalar_type());
    return loss;
  }

  static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &grad = grads[0];
    if (!grad.defined()) return variable_list(5);
    const int64_t bias_type = ctx->saved_data["bias"].toInt(), target_type = ctx->saved_data["target"].toInt();
    if (!plain_backward(grad) || lists_in_python || !usable_saved(saved))
      return backward_in_python(ctx, kTopk, grad, saved,
                                {dtype_of(static_cast<c10::ScalarType>(bias_type)),
                                 dtype_of(static_cast<c10::ScalarType>(target_type))},
                                nullptr, 5);
    const Tensor indices = prepared(saved[0]), weight = prepared(saved[1]), vals = prepared(saved[2]), resid = prepared(saved[3]);
    const c10::DeviceGuard guard(weight.device());
    const Tensor g = grad_scalar(grad, weight.device());
    const flexsae_shape s = shape_of(indices, weight, vals, FLEXSAE_F32, FLEXSAE_F32);
    // (the slice width only sizes the partial sums of frequent latents: up to 256 MiB of them)
    const int64_t per_col = s.B * s.K / 32 * 4, cols = (int64_t{256} << 20) / (per_col > 1 ? per_col : 1);
    const size_t bytes = lib.topk_bwd_from_indices_workspace_bytes(&s, cols > 1 ? cols : 1);
    const auto leaf_bias = static_cast<c10::ScalarType>(bias_type);
    Tensor dW = at::empty_like(weight);
    Tensor dvals = make(weight, {s.B, s.K}, vals.scalar_type()), dbias = make(weight, {s.D}, leaf_bias);
    const Tensor workspace = make_workspace(weight, bytes);
    check(lib.topk_bwd_from_indices(&s, index_ptr(indices), weight.data_ptr(), vals.data_ptr(), f32(resid), f32(g),
                                    dW.data_ptr(), s.weight_dtype, dvals.data_ptr(), s.vals_dtype, dbias.data_ptr(),
                                    dtype_of(leaf_bias), workspace.data_ptr(), bytes, topk_bwd_flags, flag_of(weight),
                                    stream_of(weight)),
          "flexsae_topk_bwd_from_indices");
    Tensor dtarget;
    if (ctx->needs_input_grad(4))
      dtarget = (resid * (grad.to(c10::ScalarType::Float) * (-2.0 / static_cast<double>(s.B * s.D))))
                    .to(static_cast<c10::ScalarType>(target_type));
    return {Tensor(), dW, dvals, dbias, dtarget};
  }
};

struct HierLoss : torch::autograd::Function<HierLoss> {
  static Variable forward(AutogradContext *ctx, const Variable &indices, const Variable &weight, const Variable &vals,
                          const Variable &bias, const Variable &target, int64_t slice_cols) {
    auto [loss, resid] = ::forward(false, {indices, weight, vals, bias, target});
    ctx->save_for_backward({indices, weight, vals, resid});
    ctx->set_materialize_grads(false);
    ctx->saved_data["bias"] = static_cast<int64_t>(bias.scalar_type());
    ctx->saved_data["cols"] = slice_cols;
    return loss;
  }

  static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &grad = grads[0];
    if (!grad.defined()) return variable_list(6);
    const auto leaf_bias = static_cast<c10::ScalarType>(ctx->saved_data["bias"].toInt());
    if (!plain_backward(grad) || lists_in_python || !usable_saved(saved))
      return backward_in_python(ctx, kHier, grad, saved, {dtype_of(leaf_bias)}, nullptr, 6);
    const Tensor indices = prepared(saved[0]), weight = prepared(saved[1]), vals = prepared(saved[2]), resid = prepared(saved[3]);
    const c10::DeviceGuard guard(weight.device());
    const Tensor g = grad_scalar(grad, weight.device());
    const flexsae_shape s = shape_of(indices, weight, vals, FLEXSAE_F32, FLEXSAE_F32);
    const size_t bytes = lib.hier_bwd_workspace_bytes(&s, ctx->saved_data["cols"].toInt());
    const Tensor workspace = make_workspace(weight, bytes);
    Tensor dW = at::empty_like(weight);
    Tensor dvals = make(weight, {s.B, s.K}, c10::ScalarType::Float), dbias = make(weight, {s.D}, c10::ScalarType::Float);
    check(lib.hier_bwd(&s, index_ptr(indices), weight.data_ptr(), vals.data_ptr(), f32(resid), f32(g), dW.data_ptr(),
                       s.weight_dtype, f32(dvals), f32(dbias), workspace.data_ptr(), bytes, 0, flag_of(weight),
                       stream_of(weight)),
          "flexsae_hier_bwd");
    if (vals.scalar_type() != c10::ScalarType::Float || leaf_bias != c10::ScalarType::Float)
      std::tie(std::ignore, dvals, dbias) = finish(Tensor(), weight, Tensor(), dvals, vals.scalar_type(), dbias, leaf_bias);
    return {Tensor(), dW, dvals, dbias, Tensor(), Tensor()};
  }
};

struct SlicedLoss : torch::autograd::Function<SlicedLoss> {
  static Variable forward(AutogradContext *ctx, const Variable &indices, const Variable &weight, const Variable &vals,
                          const Variable &bias, const Variable &target, const StepPlan &plan) {
    Step r = hier_step({indices, weight, vals, bias, target}, plan);
    ctx->save_for_backward({indices, weight, vals, bias, target, r.dvals, r.dbias});
    ctx->set_materialize_grads(false);
    // the unit gradient is no saved tensor: the backward scales it in place and hands the very buffer on
    if (plan.need_dw) {
      ctx->saved_data["dW"] = r.dW;
      ctx->saved_data["capture"] = capture_of(weight);
    }
    save_plan(ctx, plan);
    return r.loss;
  }

  static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
    auto saved = ctx->get_saved_variables();
    const Tensor &grad = grads[0];
    if (!grad.defined()) return variable_list(6);
    const auto at = ctx->saved_data.find("dW");
    // That of a graph which this backward is no part of is read alone: its replays write it again.  That of an eager forward is not
    // for a graph: every replay would scale it again, or read memory that is another's by then.
    const int64_t from = at != ctx->saved_data.end() ? ctx->saved_data["capture"].toInt() : 0;
    const bool mine = at != ctx->saved_data.end() && from == capture_of(at->second.toTensor());
    Tensor dW = mine || from != 0 ? at->second.toTensor() : Tensor();
    const StepPlan plan = saved_plan(ctx);
    if (!plain_backward(grad) || (lists_in_python && !dW.defined()) || !usable_inputs(saved) ||
        !usable_fp32(saved[5], saved[1], saved[2].sizes()) || !usable_fp32(saved[6], saved[1], saved[3].sizes()) ||
        (dW.defined() && dW.device() != saved[1].device())) {
      if (!mine) dW = Tensor();
      auto out = backward_in_python(ctx, kSliced, grad, saved, {plan.need_dw, plan.flags}, &dW, 6);
      if (mine && !dW.defined()) ctx->saved_data.erase("dW");
      return out;
    }
    Tensor dvals = prepared(saved[5]), dbias = prepared(saved[6]);
    const bool in_place = mine || !dW.defined();
    if (ctx->needs_input_grad(1)) {
      TORCH_CHECK(plan.need_dw, "the step ran without dW but weight requires a gradient");
      if (mine) ctx->saved_data.erase("dW");  // the buffer now belongs to whoever receives the gradient
      if (!dW.defined()) {                    // a second backward through a retained graph: the buffer went with the first one
        Step again = hier_step({saved[0], saved[1], saved[2], saved[3], saved[4]}, plan);
        dW = again.dW;
        dvals = again.dvals;
        dbias = again.dbias;
      }
    } else {
      dW = Tensor();
    }
    const c10::DeviceGuard guard(saved[1].device());
    auto [w, v, b] = finish(grad, saved[1], dW, dvals, saved[2].scalar_type(), dbias, saved[3].scalar_type(), in_place);
    return {Tensor(), w, v, b, Tensor(), Tensor()};
  }
};

// The loss alone in the forward, the step with the upstream gradient in the backward (_late_step in ops.py).
struct LateLoss : torch::autograd::Function<LateLoss> {
  static Variable forward(AutogradContext *ctx, const Variable &indices, const Variable &weight, const Variable &vals,
                          const Variable &bias, const Variable &target, const StepPlan &plan) {
    auto [loss, resid] = ::forward(false, {indices, weight, vals, bias, target});
    ctx->save_for_backward({indices, weight, vals, bias, target});
    ctx->set_materialize_grads(false);
    save_plan(ctx, plan);
    if (plan.stats.defined()) ctx->saved_data["stats"] = plan.stats;
    ctx->saved_data["tag"] = plan.tag;
    return loss;
  }

  static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &grad = grads[0];
    if (!grad.defined()) return variable_list(6);
    StepPlan plan = saved_plan(ctx);
    if (!plain_backward(grad) || lists_in_python || !usable_inputs(saved))
      return backward_in_python(ctx, kLate, grad, saved, {plan.need_dw, plan.flags}, nullptr, 6);
    const auto at = ctx->saved_data.find("stats");
    // (a graph under capture would write them again at every replay, as those of the forward's step)
    if (at != ctx->saved_data.end() && !capturing(saved[1])) {
      plan.stats = at->second.toTensor();
      plan.tag = ctx->saved_data["tag"].toInt();
      ctx->saved_data.erase("stats");
    }
    const Step r = hier_step({saved[0], saved[1], saved[2], saved[3], saved[4]}, plan, grad);
    const c10::DeviceGuard guard(saved[1].device());
    auto [w, v, b] = finish(grad, saved[1], Tensor(), r.dvals, saved[2].scalar_type(), r.dbias, saved[3].scalar_type());
    return {Tensor(), r.dW, v, b, Tensor(), Tensor()};
  }
};

// ---- the module ----------------------------------------------------------------------------
bool take_inputs(PyObject *const *args, Inputs &in) {
  Tensor *const to[5] = {&in.indices, &in.weight, &in.vals, &in.bias, &in.target};
  for (int i = 0; i < 5; ++i) {
    if (!THPVariable_CheckExact(args[i])) return false;
    *to[i] = THPVariable_Unpack(args[i]);
  }
  return plain_surroundings() && usable(in);
}

int64_t number(PyObject *o) {
  const int64_t v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw_python();
  return v;
}

bool arguments(Py_ssize_t n, Py_ssize_t want) {
  if (n == want) return true;
  PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", want, n);
  return false;
}

// topk_loss(indices, weight, vals, bias, target) -> loss
PyObject *py_topk_loss(PyObject *, PyObject *const *args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Inputs in;
  if (!arguments(n, 5)) return nullptr;
  if (!take_inputs(args, in)) Py_RETURN_NONE;
  Tensor loss;
  {
    pybind11::gil_scoped_release no_gil;
    const bool grad = c10::GradMode::is_enabled() && (in.weight.requires_grad() || in.vals.requires_grad() ||
                                                      in.bias.requires_grad() || in.target.requires_grad());
    loss = grad ? TopkLoss::apply(in.indices, in.weight, in.vals, in.bias, in.target) : forward(true, in).first;
  }
  return THPVariable_Wrap(loss);
  END_HANDLE_TH_ERRORS
}

// hier_loss(indices, weight, vals, bias, target, slice_cols) -> loss: forward, and a backward of its own
PyObject *py_hier_loss(PyObject *, PyObject *const *args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Inputs in;
  if (!arguments(n, 6)) return nullptr;
  if (!take_inputs(args, in)) Py_RETURN_NONE;
  const int64_t cols = number(args[5]);
  Tensor loss;
  {
    pybind11::gil_scoped_release no_gil;
    const bool grad = c10::GradMode::is_enabled() && (in.weight.requires_grad() || in.vals.requires_grad() ||
                                                      in.bias.requires_grad() || in.target.requires_grad());
    loss = grad ? HierLoss::apply(in.indices, in.weight, in.vals, in.bias, in.target, cols) : forward(false, in).first;
  }
  return THPVariable_Wrap(loss);
  END_HANDLE_TH_ERRORS
}

// need_dw (or the step of an update), slice_cols, flags, ws_flags, stats, tag
constexpr Py_ssize_t kPlanArguments = 6;
StepPlan take_plan(PyObject *const *args, bool need_dw) {
  StepPlan plan = {need_dw, number(args[1]), number(args[2]), number(args[3]), Tensor(), number(args[5])};
  if (THPVariable_Check(args[4])) plan.stats = THPVariable_Unpack(args[4]);
  return plan;
}

template <typename Loss>
PyObject *step_loss(PyObject *const *args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Inputs in;
  if (!arguments(n, 5 + kPlanArguments)) return nullptr;
  if (!take_inputs(args, in)) Py_RETURN_NONE;
  const StepPlan plan = take_plan(args + 5, number(args[5]) != 0);
  Tensor loss;
  {
    pybind11::gil_scoped_release no_gil;
    loss = Loss::apply(in.indices, in.weight, in.vals, in.bias, in.target, plan);
  }
  return THPVariable_Wrap(loss);
  END_HANDLE_TH_ERRORS
}

// hier_sliced(indices, weight, vals, bias, target, need_dw, slice_cols, flags, ws_flags, stats, tag) -> loss: the training step
PyObject *py_hier_sliced(PyObject *, PyObject *const *args, Py_ssize_t n) { return step_loss<SlicedLoss>(args, n); }
// hier_late(the same): the loss, and the step in the backward
PyObject *py_hier_late(PyObject *, PyObject *const *args, Py_ssize_t n) { return step_loss<LateLoss>(args, n); }

// hier_sgd(indices, weight, vals, bias, target, step, slice_cols, flags, ws_flags, stats, tag) -> (loss, dvals, dbias)
PyObject *py_hier_sgd(PyObject *, PyObject *const *args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Inputs in;
  if (!arguments(n, 5 + kPlanArguments)) return nullptr;
  if (!take_inputs(args, in) || !THPVariable_CheckExact(args[5])) Py_RETURN_NONE;
  const Tensor step = THPVariable_Unpack(args[5]);
  if (!plain_tensor(step) || in.weight.is_inference() || !in.weight.is_contiguous() ||
      reinterpret_cast<uintptr_t>(in.weight.data_ptr()) % 16 || in.weight.size(1) % 4 || in.indices.size(1) > 256)
    Py_RETURN_NONE;
  const StepPlan plan = take_plan(args + 5, true);
  Step r;
  {
    pybind11::gil_scoped_release no_gil;
    const c10::AutoGradMode no_grad(false);
    in.vals = in.vals.detach();
    in.bias = in.bias.detach();
    r = hier_step(in, plan, Tensor(), step);
  }
  return Py_BuildValue("NNN", THPVariable_Wrap(r.loss), THPVariable_Wrap(r.dvals), THPVariable_Wrap(r.dbias));
  END_HANDLE_TH_ERRORS
}

// ---- the optimiser -------------------------------------------------------------------------
// The tensors of a list or tuple, each plain and of `device` (undefined: the first one's); false: not this module's business.  The
// list keeps them: these functions hold the interpreter's lock and run no Python code once they have taken tensors, and have no
// reference of their own (a step of 192 tiny tensors is host work: 30 us; 55 with references, with checks for forward gradients,
// which optim.py has made, and 48 tensors a launch).
using Tensors = std::vector<const Tensor *>;
bool take_tensors(PyObject *o, Tensors &out, c10::optional<c10::Device> &device) {
  static const uint64_t usual =
      (c10::DispatchKeySet(c10::DispatchKey::CUDA) | c10::DispatchKeySet(c10::DispatchKey::AutogradCUDA) |
       c10::DispatchKeySet(c10::DispatchKey::ADInplaceOrView) | c10::DispatchKeySet(c10::DispatchKey::AutocastCUDA))
          .raw_repr();
  if (!PyList_CheckExact(o) && !PyTuple_CheckExact(o)) return false;
  const Py_ssize_t n = PySequence_Fast_GET_SIZE(o);
  PyObject **const items = PySequence_Fast_ITEMS(o);
  out.reserve(static_cast<size_t>(n));
  for (Py_ssize_t i = 0; i < n; ++i) {
    if (!THPVariable_CheckExact(items[i])) return false;
    const Tensor &t = THPVariable_Unpack(items[i]);
    if (!t.defined() || !t.is_cuda() || (t.key_set().raw_repr() & ~usual) != 0 || (device && t.device() != *device)) return false;
    if (!device) device = t.device();
    out.push_back(&t);
  }
  return true;
}

// A tensor that a call changes: its memory as it is.
bool changeable(const Tensor &t) { return t.is_contiguous() && !t.is_inference(); }

double real(PyObject *o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw_python();
  return v;
}

// The numbers of a list or tuple, or a number by itself; false: something else.  Reading one may run Python code (__float__, and a
// tensor's waits for its device without the interpreter's lock), which may change any list: numbers are read before tensors are
// taken.
struct Reals {
  std::vector<double> values;
  bool one = false;

  bool take(PyObject *o) {
    if (PyList_CheckExact(o) || PyTuple_CheckExact(o)) {
      for (Py_ssize_t i = 0; i < PySequence_Fast_GET_SIZE(o); ++i) {
        const auto item = pybind11::reinterpret_borrow<pybind11::object>(PySequence_Fast_GET_ITEM(o, i));
        values.push_back(real(item.ptr()));
      }
      return true;
    }
    one = PyFloat_Check(o) || PyLong_Check(o);
    if (one) values.push_back(real(o));
    return one;
  }
  bool serve(size_t n) const { return one || values.size() == n; }
  float at(size_t i) const { return static_cast<float>(values[one ? 0 : i]); }
};

// One fp32 number of `device`; None: none.
bool take_scalar(PyObject *o, const c10::Device &device, Tensor &out) {
  if (o == Py_None) return true;
  if (!THPVariable_Check(o)) return false;
  out = THPVariable_Unpack(o);
  return plain_tensor(out) && out.device() == device && out.scalar_type() == c10::ScalarType::Float && out.numel() == 1;
}

// grad_norm(grads) -> norm
PyObject *py_grad_norm(PyObject *, PyObject *const *args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!arguments(n, 1)) return nullptr;
  Tensors grads;
  c10::optional<c10::Device> device;
  if (!plain_surroundings() || !take_tensors(args[0], grads, device) || grads.empty()) Py_RETURN_NONE;
  const c10::AutoGradMode no_grad(false);
  const c10::DeviceGuard guard(*device);
  std::vector<flexsae_grad> list;
  list.reserve(grads.size());
  std::vector<Tensor> copies;
  for (const Tensor *g : grads) {
    const int dtype = dtype_of(g->scalar_type());
    if (dtype < 0) Py_RETURN_NONE;
    if (!g->is_contiguous()) {
      copies.push_back(g->contiguous());
      list.push_back({copies.back().const_data_ptr(), g->numel(), dtype});
    } else {
      list.push_back({g->const_data_ptr(), g->numel(), dtype});
    }
  }
  const auto count = static_cast<int64_t>(list.size());
  const size_t bytes = lib.grad_norm_workspace_bytes(count);
  const c10::DataPtr workspace = c10::GetAllocator(c10::DeviceType::CUDA)->allocate(bytes);  // (of the current stream, as tensors')
  const Tensor norm = make(*grads[0], {}, c10::ScalarType::Float);
  check(lib.grad_norm(list.data(), count, f32(norm), workspace.get(), bytes, stream_of(norm)), "flexsae_grad_norm");
  return THPVariable_Wrap(norm);
  END_HANDLE_TH_ERRORS
}

// A step of AdamW: bits, params, grads, state0s, state1s, masters, counter, lr, weight_decay, beta1, beta2, eps, grad_scale,
// grad_norm, max_norm, unit_rows.  All numbers are read before any tensor is taken, and everything is looked at before the launch.
constexpr Py_ssize_t kAdamwArguments = 16;
class AdamwCall {
 public:
  void read_numbers(PyObject *const *args) {
    eight_ = number(args[0]) == 8;
    unit_ = number(args[15]) != 0;
    device_lr_ = THPVariable_Check(args[7]);
    numbers_ = (device_lr_ || lrs_.take(args[7])) && weight_decays_.take(args[8]);
    config_ = {real(args[9]), real(args[10]), real(args[11]), static_cast<float>(real(args[12])), static_cast<float>(real(args[14])),
               nullptr, nullptr, nullptr, eight_ ? 8 : 32, unit_ ? FLEXSAE_ADAMW_UNIT_ROWS : 0};
  }

  // False: not this module's business.  (Runs no Python code.)
  bool take(PyObject *const *args) {
    Tensors grads;
    if (!numbers_ || !take_tensors(args[1], params_, device_) || params_.empty() || !take_tensors(args[2], grads, device_) ||
        !take_tensors(args[3], s0_, device_) || !take_tensors(args[4], s1_, device_) ||
        (args[5] != Py_None && !take_tensors(args[5], masters_, device_)))
      return false;
    const size_t count = params_.size();
    if (grads.size() != count || s0_.size() != count || s1_.size() != count || (args[5] != Py_None && masters_.size() != count) ||
        (!device_lr_ && !lrs_.serve(count)) || !weight_decays_.serve(count) || !THPVariable_Check(args[6]))
      return false;
    counter_ = &THPVariable_Unpack(args[6]);
    if (!plain_tensor(*counter_) || counter_->device() != *device_ || counter_->scalar_type() != c10::ScalarType::Long ||
        counter_->numel() != 2 || !changeable(*counter_))
      return false;
    if ((device_lr_ && !take_scalar(args[7], *device_, lr_)) || !take_scalar(args[13], *device_, norm_)) return false;
    const c10::AutoGradMode no_grad(false);
    const c10::DeviceGuard guard(*device_);
    list_.resize(count);
    for (size_t i = 0; i < count; ++i) {
      const Tensor &p = *params_[i], &g = *grads[i], &a = *s0_[i], &b = *s1_[i];
      const int dtype = dtype_of(p.scalar_type());
      if (dtype < 0 || g.scalar_type() != p.scalar_type() || g.sizes() != p.sizes() || !changeable(p) || !changeable(a) ||
          !changeable(b) || (unit_ && p.dim() < 2))
        return false;
      const int64_t numel = p.numel(), cols = unit_ ? p.size(-1) : numel, rows = unit_ ? (cols ? numel / cols : 0) : 1;
      if (eight_) {
        const at::IntArrayRef sizes = a.sizes();
        if (a.scalar_type() != c10::ScalarType::Byte || b.scalar_type() != c10::ScalarType::Float || a.dim() != p.dim() + 1 ||
            sizes.back() != 2 || sizes.slice(0, sizes.size() - 1) != p.sizes() || b.dim() != 3 || b.size(0) != rows ||
            b.size(1) != (cols + 255) / 256 || b.size(2) != 2 || reinterpret_cast<uintptr_t>(b.const_data_ptr()) % 8 ||
            reinterpret_cast<uintptr_t>(a.const_data_ptr()) % 2)
          return false;
      } else if (a.scalar_type() != c10::ScalarType::Float || b.scalar_type() != c10::ScalarType::Float || a.sizes() != p.sizes() ||
                 b.sizes() != p.sizes()) {
        return false;
      }
      void *master = nullptr;
      if (!masters_.empty() && dtype != FLEXSAE_F32) {
        if (masters_[i]->scalar_type() != c10::ScalarType::Float || masters_[i]->sizes() != p.sizes() || !changeable(*masters_[i]))
          return false;
        master = masters_[i]->data_ptr();
      }
      if (!g.is_contiguous()) copies_.push_back(g.contiguous());
      list_[i] = {p.data_ptr(), (g.is_contiguous() ? g : copies_.back()).const_data_ptr(), master, a.data_ptr(), b.data_ptr(), rows, cols,
                  device_lr_ ? 1.f : lrs_.at(i), weight_decays_.at(i), dtype};
    }
    config_.grad_norm = norm_.defined() ? f32(norm_) : nullptr;
    config_.lr = lr_.defined() ? f32(lr_) : nullptr;
    config_.counter = counter_->data_ptr<int64_t>();
    return true;
  }

  int check_alone() const { return lib.adamw_check(list_.data(), static_cast<int64_t>(list_.size()), &config_); }

  int launch() {
    const c10::DeviceGuard guard(*device_);
    const int status = lib.adamw_step(list_.data(), static_cast<int64_t>(list_.size()), &config_, stream_of(*counter_));
    if (status == FLEXSAE_OK || status == FLEXSAE_ERR_LAUNCH) {
      for (const auto *changed : {&params_, &s0_, &s1_})
        for (const Tensor *t : *changed) t->unsafeGetTensorImpl()->bump_version();
      for (size_t i = 0; i < masters_.size(); ++i)  // (that of an fp32 parameter is ignored)
        if (list_[i].master != nullptr) masters_[i]->unsafeGetTensorImpl()->bump_version();
      counter_->unsafeGetTensorImpl()->bump_version();
    }
    return status;
  }

 private:
  bool eight_ = false, unit_ = false, device_lr_ = false, numbers_ = false;
  Reals lrs_, weight_decays_;
  flexsae_adamw_config config_{};
  Tensors params_, s0_, s1_, masters_;
  c10::optional<c10::Device> device_;
  const Tensor *counter_ = nullptr;
  Tensor lr_, norm_;
  std::vector<flexsae_adamw_tensor> list_;
  std::vector<Tensor> copies_;  // of gradients that are not contiguous
};

// adamw(the arguments of an AdamwCall) -> True
PyObject *py_adamw(PyObject *, PyObject *const *args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!arguments(n, kAdamwArguments)) return nullptr;
  if (!plain_surroundings()) Py_RETURN_NONE;
  AdamwCall call;
  call.read_numbers(args);
  if (!call.take(args)) Py_RETURN_NONE;
  const int status = call.launch();
  if (status == FLEXSAE_ERR_INVALID_ARGUMENT) Py_RETURN_NONE;  // nothing was launched; optim.py says what is wrong
  check(status, "flexsae_adamw_step");
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

// adamw_all([the arguments of an AdamwCall, as a tuple, ...]) -> True: all of the steps, or, where one is refused, none
PyObject *py_adamw_all(PyObject *, PyObject *const *args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!arguments(n, 1)) return nullptr;
  if (!plain_surroundings() || !PyList_CheckExact(args[0])) Py_RETURN_NONE;
  std::vector<pybind11::object> tuples;
  for (Py_ssize_t i = 0; i < PyList_GET_SIZE(args[0]); ++i) {
    tuples.push_back(pybind11::reinterpret_borrow<pybind11::object>(PyList_GET_ITEM(args[0], i)));
    if (!PyTuple_CheckExact(tuples.back().ptr()) || PyTuple_GET_SIZE(tuples.back().ptr()) != kAdamwArguments) Py_RETURN_NONE;
  }
  std::vector<AdamwCall> calls(tuples.size());
  for (size_t i = 0; i < calls.size(); ++i) calls[i].read_numbers(PySequence_Fast_ITEMS(tuples[i].ptr()));
  for (size_t i = 0; i < calls.size(); ++i)
    if (!calls[i].take(PySequence_Fast_ITEMS(tuples[i].ptr()))) Py_RETURN_NONE;
  for (const AdamwCall &call : calls) {
    const int status = call.check_alone();
    if (status == FLEXSAE_ERR_INVALID_ARGUMENT) Py_RETURN_NONE;
    check(status, "flexsae_adamw_check");
  }
  for (AdamwCall &call : calls) check(call.launch(), "flexsae_adamw_step");
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

// adamw8_moments(codes, absmax, dtype) -> (exp_avgs, exp_avg_sqs)
PyObject *py_adamw8_moments(PyObject *, PyObject *const *args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!arguments(n, 3)) return nullptr;
  const int64_t dtype = number(args[2]);
  Tensors codes, absmax;
  std::vector<Tensor> m, v;
  c10::optional<c10::Device> device;
  if (!plain_surroundings() || !take_tensors(args[0], codes, device) || codes.empty() || !take_tensors(args[1], absmax, device) ||
      absmax.size() != codes.size() || dtype < 0 || dtype > 2)
    Py_RETURN_NONE;
  const c10::DeviceGuard guard(*device);
  std::vector<flexsae_adamw8_state> list(codes.size());
  const c10::ScalarType type = dtype == FLEXSAE_F32    ? c10::ScalarType::Float
                               : dtype == FLEXSAE_BF16 ? c10::ScalarType::BFloat16
                                                       : c10::ScalarType::Half;
  for (size_t i = 0; i < codes.size(); ++i) {
    const Tensor &c = *codes[i], &a = *absmax[i];
    if (c.scalar_type() != c10::ScalarType::Byte || a.scalar_type() != c10::ScalarType::Float || c.dim() < 1 || c.size(-1) != 2 ||
        a.dim() != 3 || a.size(2) != 2 || !c.is_contiguous() || !a.is_contiguous() ||
        reinterpret_cast<uintptr_t>(c.const_data_ptr()) % 2 || reinterpret_cast<uintptr_t>(a.const_data_ptr()) % 8)
      Py_RETURN_NONE;
    const int64_t rows = a.size(0), cols = rows ? c.numel() / 2 / rows : 0;
    if (rows * cols != c.numel() / 2 || (rows && a.size(1) != (cols + 255) / 256)) Py_RETURN_NONE;
    m.push_back(make(c, c.sizes().slice(0, c.dim() - 1), type));
    v.push_back(make(c, c.sizes().slice(0, c.dim() - 1), type));
    list[i] = {c.const_data_ptr(), a.const_data_ptr<float>(), m[i].data_ptr(), v[i].data_ptr(), rows, cols};
  }
  check(lib.adamw8_moments(list.data(), static_cast<int64_t>(list.size()), static_cast<int>(dtype), stream_of(*codes[0])),
        "flexsae_adamw8_moments");
  auto list_of = [](const std::vector<Tensor> &tensors) {
    auto l = pybind11::reinterpret_steal<pybind11::object>(PyList_New(static_cast<Py_ssize_t>(tensors.size())));
    for (size_t i = 0; i < tensors.size(); ++i) PyList_SET_ITEM(l.ptr(), static_cast<Py_ssize_t>(i), THPVariable_Wrap(tensors[i]));
    return l;
  };
  return Py_BuildValue("NN", list_of(m).release().ptr(), list_of(v).release().ptr());
  END_HANDLE_TH_ERRORS
}

// ---- around a dictionary in a model ----------------------------------------------------------
#include "eager_lm.hpp"

// set_flag(device, flag)
PyObject *py_set_flag(PyObject *, PyObject *const *args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!arguments(n, 2)) return nullptr;
  const int64_t device = number(args[0]);
  if (device >= 0 && device < kMaxDevices && THPVariable_Check(args[1])) status_flags[device] = THPVariable_Unpack(args[1]);
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// settings(topk_bwd_flags, lists_in_python)
PyObject *py_settings(PyObject *, PyObject *const *args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!arguments(n, 2)) return nullptr;
  topk_bwd_flags = static_cast<int>(number(args[0]));
  lists_in_python = number(args[1]) != 0;
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// init(path of the library, general_backward, raise_status)
PyObject *py_init(PyObject *, PyObject *const *args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!arguments(n, 3)) return nullptr;
  const char *const path = PyUnicode_AsUTF8(args[0]);
  if (!path) return nullptr;
  void *const handle = dlopen(path, RTLD_NOW | RTLD_LOCAL);
  if (!handle) return PyErr_Format(PyExc_OSError, "%s", dlerror());
#define X(name)                                                                                                  \
  if (!(lib.name = reinterpret_cast<decltype(lib.name)>(dlsym(handle, "flexsae_" #name))))                       \
    return PyErr_Format(PyExc_OSError, "%s does not export flexsae_" #name, path);
  FLEXSAE_ENTRIES(X)
#undef X
  if (lib.abi_version() != FLEXSAE_ABI_VERSION) return PyErr_Format(PyExc_OSError, "%s has another ABI version", path);
  Py_INCREF(args[1]);
  Py_INCREF(args[2]);
  general_backward = args[1];
  raise_status = args[2];
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

#define FLEXSAE_METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_##name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FLEXSAE_METHOD(init),       FLEXSAE_METHOD(set_flag),    FLEXSAE_METHOD(settings),
                         FLEXSAE_METHOD(topk_loss),  FLEXSAE_METHOD(hier_loss),   FLEXSAE_METHOD(hier_sliced),
                         FLEXSAE_METHOD(hier_late),  FLEXSAE_METHOD(hier_sgd),    FLEXSAE_METHOD(grad_norm),
                         FLEXSAE_METHOD(adamw),      FLEXSAE_METHOD(adamw_all),   FLEXSAE_METHOD(adamw8_moments),
                         FLEXSAE_METHOD(layer_norm), FLEXSAE_METHOD(embedding_lookup), FLEXSAE_METHOD(distillation_loss),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_eager", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

// build_id, torch_version: what the module was built from and against, for whoever loads it to compare
PyMODINIT_FUNC PyInit__eager() {
  PyObject *const m = PyModule_Create(&module);
  if (m && (PyModule_AddStringConstant(m, "build_id", FLEXSAE_BUILD_ID) < 0 ||
            PyModule_AddStringConstant(m, "torch_version", FLEXSAE_TORCH_VERSION) < 0)) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
