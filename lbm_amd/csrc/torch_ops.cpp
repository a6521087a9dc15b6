// Host path of the training operators: argument checks, outputs, descriptors and autograd nodes around lbm_hip_norm_forward,
// lbm_hip_norm_backward and lbm_hip_dropout.  A training step of the tracker's sizes calls them for a few microseconds of GPU work each,
// forty times a step: the same path in Python took 16 us a forward and, in the thread that autograd runs a GPU's nodes in, 35 us a
// backward call.  No kernels here; the entry points come as addresses from the library that lbm_amd/hip.py has loaded.
#include <initializer_list>
#include <mutex>
#include <optional>
#include <string>
#include <tuple>

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/utils/pybind.h>

#include "../../include/lbm_hip.h"

namespace {

using at::Tensor;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

struct Api {
  decltype(&lbm_hip_norm_forward) forward = nullptr;
  decltype(&lbm_hip_norm_backward) backward = nullptr;
  decltype(&lbm_hip_dropout) dropout = nullptr;
  decltype(&lbm_hip_norm_workspace_bytes) workspace_bytes = nullptr;
  decltype(&lbm_hip_last_error) last_error = nullptr;
  PyObject* error = nullptr;                     // lbm_amd.hip.HipError
} api;

// HipError(message); python_error crosses the autograd engine's threads and is restored in the caller's
[[noreturn]] void fail(const std::string& message) {
  pybind11::gil_scoped_acquire gil;
  PyErr_SetString(api.error, message.c_str());
  python_error e;
  e.persist();
  throw e;
}
std::string text(const Tensor& t) {
  std::string s = "(";
  for (const auto n : t.sizes()) s += (s.size() > 1 ? ", " : "") + std::to_string(n);
  return s + ") " + c10::toString(t.scalar_type()) + " on " + t.device().str();
}

int elem_type(const Tensor& t, const char* what) {
  TORCH_CHECK(api.forward != nullptr, "lbm_amd._torch_ops is used through lbm_amd.hip.ops()");
  if (!t.is_cuda()) fail(std::string(what) + ": expected a GPU tensor, got " + text(t));
  if (!t.has_storage()) fail(std::string(what) + ": expected a plain dense tensor (no torch.func transform, no sparse layout), got " + text(t));
  switch (t.scalar_type()) {
    case at::kFloat: return LBM_TYPE_F32;
    case at::kHalf: return LBM_TYPE_F16;
    case at::kBFloat16: return LBM_TYPE_BF16;
    default: fail(std::string(what) + ": expected float32, float16 or bfloat16, got " + text(t));
  }
}

// a view that torch negates when it reads it (the imaginary part of a conjugate): a copy
Tensor as_stored(const Tensor& t) { return t.is_neg() ? t.resolve_neg() : t; }

// Rows of the last dimension at one stride are used where they lie, any other layout is copied; ld: elements between rows
Tensor as_rows(const Tensor& given, int64_t& ld) {
  const Tensor t = as_stored(given);
  const int64_t n = t.size(-1);
  ld = n;
  if (t.is_contiguous()) return t;
  if (t.stride(-1) == 1 && t.numel() > 0) {
    int64_t row = 0, reach = 0;                  // stride of the innermost dimension of rows; what the next outer one must have
    bool one = true;
    for (int64_t i = t.dim() - 2; i >= 0 && one; --i) {
      if (t.size(i) == 1) continue;
      if (row == 0) row = t.stride(i);
      else one = t.stride(i) == reach;
      reach = t.stride(i) * t.size(i);
      one = one && row > 0;
    }
    if (row == 0) row = n;
    if (one && row >= n && row < (int64_t{1} << 31)) {
      ld = row;
      return t;
    }
  }
  return t.contiguous();
}

struct Drop {
  double p = 0.0;
  uint64_t seed = 0, offset = 0;
  Tensor seed_dev;                               // defined: read by the kernel in place of seed
  const void* address() const { return seed_dev.defined() ? seed_dev.const_data_ptr() : nullptr; }
};
void check_seed(const char* what, const Tensor& seed, c10::Device device) {
  if (!seed.has_storage() || seed.scalar_type() != at::kLong || seed.numel() != 1 || seed.device() != device)
    fail(std::string(what) + ": a seed tensor holds one int64 on the operands' device, got " + text(seed));
}
Drop make_drop(const char* what, double p, uint64_t seed, const std::optional<Tensor>& seed_dev, uint64_t offset, const Tensor& x) {
  Drop d;
  if (!(p >= 0.0 && p <= 1.0)) fail(std::string(what) + ": p = " + std::to_string(p) + " is not a probability");
  d.p = p;
  d.seed = seed;
  d.offset = offset;
  if (seed_dev.has_value() && seed_dev->defined()) {
    d.seed_dev = *seed_dev;
    check_seed(what, d.seed_dev, x.device());
  }
  return d;
}

struct Operands {
  Tensor x, residual, weight;                    // dense or at a row stride
  bool bias = false;
  const void* bias_ptr = nullptr;
  Tensor bias_dense;
  int64_t rows = 0, cols = 0, ld_x = 0, ld_r = 0;
  int x_type = 0, r_type = 0, p_type = 0;
  at::ScalarType p_scalar = at::kFloat;
};
Tensor param(const char* what, const Tensor& p, const Operands& o) {
  if (p.dim() != 1 || p.size(0) != o.cols || p.device() != o.x.device())
    fail(std::string(what) + ": weight / bias are (" + std::to_string(o.cols) + ") on " + o.x.device().str() + ", got " + text(p));
  return as_stored(p).contiguous();
}
Operands operands(const char* what, const Tensor& x, const Tensor& residual, const Tensor& weight, const Tensor& bias) {
  Operands o;
  o.x_type = o.r_type = o.p_type = elem_type(x, what);
  o.p_scalar = x.scalar_type();
  if (x.dim() < 1 || x.size(-1) < 1) fail(std::string(what) + ": x needs a last dimension of at least one element, got " + text(x));
  o.cols = x.size(-1);
  o.rows = x.numel() / o.cols;
  o.x = as_rows(x, o.ld_x);
  if (residual.defined()) {
    o.r_type = elem_type(residual, what);
    if (residual.sizes() != x.sizes() || residual.device() != x.device()) fail(std::string(what) + ": the residual is " + text(residual) + ", x " + text(x));
    if (o.r_type != o.x_type && o.r_type != LBM_TYPE_F32) fail(std::string(what) + ": the residual's type must be x's or float32, got " + text(residual) + " beside " + text(x));
    o.residual = as_rows(residual, o.ld_r);
  }
  if (weight.defined()) {
    o.p_type = elem_type(weight, what);
    o.p_scalar = weight.scalar_type();
    o.weight = param(what, weight, o);
  }
  if (bias.defined()) {
    const int type = elem_type(bias, what);
    if (weight.defined() && type != o.p_type) fail(std::string(what) + ": weight and bias differ in type");
    o.p_type = type;
    o.p_scalar = bias.scalar_type();
    o.bias_dense = param(what, bias, o);
    o.bias = true;
  }
  if (o.p_type != o.x_type && o.p_type != LBM_TYPE_F32) fail(std::string(what) + ": the type of weight and bias must be x's or float32");
  return o;
}

const void* address(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void* address_mut(const Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }
lbm_stream_t stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
void checked(int rc, const char* what) {
  if (rc != 0) fail(std::string(what) + ": " + api.last_error());
}

void describe(lbm_hip_norm_desc& d, const Operands& o, double eps, const Drop& drop) {
  d = lbm_hip_norm_desc{};
  d.x = address(o.x);
  d.residual = address(o.residual);
  d.weight = address(o.weight);
  d.rows = o.rows;
  d.cols = o.cols;
  d.ld_x = o.ld_x;
  d.ld_residual = o.ld_r;
  d.x_type = o.x_type;
  d.res_type = o.r_type;
  d.param_type = o.p_type;
  d.eps = (float)eps;
  d.p = drop.p;
  d.seed = drop.seed;
  d.offset = drop.offset;
  d.seed_dev = drop.address();
}

// -> y, and fp32 [2, rows] mean and rstd when asked for
std::tuple<Tensor, Tensor> run_forward(const Operands& o, double eps, const Drop& drop, bool want_stats) {
  const c10::DeviceGuard guard(o.x.device());
  const Tensor& like = o.residual.defined() ? o.residual : o.x;
  Tensor y = at::empty(o.x.sizes(), like.options()), stats;
  lbm_hip_norm_desc d;
  describe(d, o, eps, drop);
  d.bias = address(o.bias_dense);
  d.y = y.mutable_data_ptr();
  if (want_stats) {
    stats = at::empty({2, o.rows}, o.x.options().dtype(at::kFloat));
    d.mean = (float*)stats.mutable_data_ptr();
    d.rstd = d.mean + o.rows;
  }
  checked(api.forward(&d, stream_of(o.x)), "lbm_hip_norm_forward");
  return {y, stats};
}
// -> dx, dresidual, dweight, dbias, undefined where not wanted or absent
variable_list run_backward(const Operands& o, double eps, const Drop& drop, const Tensor& dy, const float* mean, const float* rstd,
                           bool want_x, bool want_r, bool want_w, bool want_b) {
  const c10::DeviceGuard guard(o.x.device());
  variable_list out(4);
  lbm_hip_norm_desc d;
  describe(d, o, eps, drop);
  const Tensor rows_dy = as_rows(dy, d.ld_dy);
  d.dy = address(rows_dy);
  d.mean = const_cast<float*>(mean);
  d.rstd = const_cast<float*>(rstd);
  if (want_x) out[0] = at::empty(o.x.sizes(), o.x.options());
  if (want_r && o.residual.defined()) out[1] = at::empty(o.x.sizes(), o.residual.options());
  if (want_w && o.weight.defined()) out[2] = at::empty({o.cols}, o.x.options().dtype(o.p_scalar));
  if (want_b && o.bias) out[3] = at::empty({o.cols}, o.x.options().dtype(o.p_scalar));
  d.dx = address_mut(out[0]);
  d.dresidual = address_mut(out[1]);
  d.dweight = address_mut(out[2]);
  d.dbias = address_mut(out[3]);
  Tensor workspace;
  if (out[2].defined() || out[3].defined()) {
    d.workspace_bytes = api.workspace_bytes(o.rows, o.cols);
    workspace = at::empty({(int64_t)d.workspace_bytes}, o.x.options().dtype(at::kByte));
    d.workspace = workspace.mutable_data_ptr();
  }
  checked(api.backward(&d, stream_of(o.x)), "lbm_hip_norm_backward");
  return out;
}
Tensor run_dropout(const Tensor& x, const Drop& drop) {
  const int type = elem_type(x, "dropout");
  const c10::DeviceGuard guard(x.device());
  const Tensor dense = as_stored(x).contiguous();
  Tensor y = at::empty(x.sizes(), x.options());
  checked(api.dropout(address(dense), y.mutable_data_ptr(), x.numel(), type, drop.p, drop.seed, drop.address(), drop.offset, stream_of(x)), "lbm_hip_dropout");
  return y;
}

// ---- autograd --------------------------------------------------------------------------------------------------------
SavedVariable saved(const Tensor& t) { return SavedVariable(t, /*is_output=*/false); }

// A captured backward pass that would run on into an eager graph on the default stream: that stream cannot wait inside the capture, and the
// process would end there.  Asked before the node hands its gradients on; the engine has made the node's stream the current one.
void refuse_captured_into_eager(const char* what, Node& node, const std::vector<bool>& wanted) {
  const auto mine = node.stream();
  if (!mine.has_value() || mine->id() == 0 || c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
  for (size_t i = 0; i < node.num_outputs(); ++i) {
    const auto& next = node.next_edge(i).function;
    if (!next || !wanted[i]) continue;
    const auto stream = next->stream();
    if (stream.has_value() && stream->id() == 0)
      fail(std::string(what) + ": the captured backward pass would run on into an eager graph on the default stream (" + next->name() + "): capture all of the graph or detach");
  }
}

struct NormBackward : public Node {
  SavedVariable x, residual, weight, seed;
  Tensor stats;
  bool bias = false;
  at::ScalarType p_scalar = at::kFloat;
  int p_type = 0;
  double eps = 0.0;
  Drop drop;                                     // its seed tensor is in `seed`, which notices in-place changes

  variable_list apply(variable_list&& grads) override {
    const std::lock_guard<std::mutex> lock(mutex_);
    if (c10::GradMode::is_enabled())             // create_graph: a result without a graph would drop the second derivatives in silence
      fail("the gradients of layer_norm and dropout_add_layer_norm are not differentiable (create_graph=True)");
    if (!grads[0].defined()) return variable_list(4);
    refuse_captured_into_eager("norm_backward", *this, {task_should_compute_output(0), task_should_compute_output(1), task_should_compute_output(2), task_should_compute_output(3)});
    const Tensor tx = x.unpack(), tr = residual.unpack(), tw = weight.unpack(), ts = seed.unpack();
    // hooks on saved tensors may return anything; the kernels take every size and type from x and residual, and the statistics from the forward pass
    const Tensor& dy = grads[0];
    elem_type(dy, "norm_backward");
    const Tensor& like = tr.defined() ? tr : tx;
    if (dy.sizes() != tx.sizes() || dy.scalar_type() != like.scalar_type() || dy.device() != tx.device() || (tw.defined() && tw.scalar_type() != p_scalar))
      fail("norm_backward: a saved tensor came back with another size, type or device: x " + text(tx) + ", the forward pass's result was like " + text(dy));
    Operands o = operands("norm_backward", tx, tr, tw, Tensor());
    o.bias = bias;
    o.p_type = p_type;
    o.p_scalar = p_scalar;
    Drop d = drop;
    d.seed_dev = ts;
    if (ts.defined()) check_seed("norm_backward", ts, dy.device());
    const float* mean = (const float*)stats.const_data_ptr();
    return run_backward(o, eps, d, dy, mean, mean + o.rows, task_should_compute_output(0), task_should_compute_output(1),
                        task_should_compute_output(2), task_should_compute_output(3));
  }
  void release_variables() override {
    const std::lock_guard<std::mutex> lock(mutex_);
    x.reset_data();
    residual.reset_data();
    weight.reset_data();
    seed.reset_data();
    stats.reset();
  }
  std::string name() const override { return "LbmNormBackward"; }
};

Tensor dropout(const Tensor& x, const Drop& drop);
struct DropoutBackward : public Node {
  SavedVariable seed;
  Drop drop;
  variable_list apply(variable_list&& grads) override {
    const std::lock_guard<std::mutex> lock(mutex_);
    if (!grads[0].defined()) return variable_list(1);
    refuse_captured_into_eager("dropout_backward", *this, {task_should_compute_output(0)});
    Drop d = drop;
    d.seed_dev = seed.unpack();
    if (d.seed_dev.defined()) check_seed("dropout_backward", d.seed_dev, grads[0].device());
    return {dropout(grads[0], d)};
  }
  void release_variables() override {
    const std::lock_guard<std::mutex> lock(mutex_);
    seed.reset_data();
  }
  std::string name() const override { return "LbmDropoutBackward"; }
};

bool wants_grad(const Tensor& t) { return t.defined() && t.requires_grad(); }

// What a graph of these operators would get wrong without an error: forward-mode derivatives, which they do not carry on; and a step
// captured while an eager graph on the default stream still holds the leaves -- the backward pass would make that stream wait
// inside the capture, which the default stream cannot.  `inputs`: x first, whose device's stream the operator runs on.
void refuse(const char* what, std::initializer_list<const Tensor*> inputs, bool grad) {
  for (const Tensor* t : inputs)
    if (t->defined() && t->_fw_grad(0).defined()) fail(std::string(what) + ": forward-mode derivatives are not supported");
  // (the default stream cannot capture, and asking it while another stream does is an error)
  const c10::Device device = (*inputs.begin())->device();
  if (!grad || c10::hip::getCurrentHIPStream(device.index()).id() == 0) return;
  const c10::DeviceGuard guard(device);
  if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
  for (const Tensor* t : inputs) {
    if (!wants_grad(*t) || !t->is_leaf()) continue;
    const auto leaf = torch::autograd::impl::try_get_grad_accumulator(*t);
    if (!leaf) continue;
    const auto stream = leaf->stream();
    if (stream.has_value() && stream->id() == 0)
      fail(std::string(what) + ": captured while an eager graph on the default stream still holds the leaf " + text(*t) + ": release that graph first");
  }
}

Tensor dropout(const Tensor& x, const Drop& drop) {
  std::shared_ptr<DropoutBackward> node;
  const bool grad = c10::GradMode::is_enabled() && wants_grad(x);
  refuse("dropout", {&x}, grad);
  if (grad) {
    node = std::shared_ptr<DropoutBackward>(new DropoutBackward(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(x));
    node->seed = saved(drop.seed_dev);
    node->drop = drop;
    node->drop.seed_dev = Tensor();
  }
  Tensor y;
  {
    const c10::AutoGradMode off(false);
    y = run_dropout(x, drop);
  }
  if (node) torch::autograd::set_history(y, node);
  return y;
}

Tensor norm(const char* what, const Tensor& x, const Tensor& residual, const Tensor& weight, const Tensor& bias, double eps, const Drop& drop) {
  for (const Tensor* t : {&x, &residual, &weight, &bias})
    if (t->defined()) elem_type(*t, what);       // before refuse(), which asks the GPU
  const bool grad = c10::GradMode::is_enabled() && (wants_grad(x) || wants_grad(residual) || wants_grad(weight) || wants_grad(bias));
  refuse(what, {&x, &residual, &weight, &bias}, grad);
  std::tuple<Tensor, Tensor> r;
  Operands o;
  {
    const c10::AutoGradMode off(false);
    o = operands(what, x, residual, weight, bias);
    r = run_forward(o, eps, drop, grad);
  }
  Tensor y = std::get<0>(r);
  if (grad) {
    auto node = std::shared_ptr<NormBackward>(new NormBackward(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(x, residual, weight, bias));
    node->x = saved(x);
    node->residual = saved(residual);
    node->weight = saved(weight);
    node->seed = saved(drop.seed_dev);
    node->stats = std::get<1>(r);
    node->bias = o.bias;
    node->p_scalar = o.p_scalar;
    node->p_type = o.p_type;
    node->eps = eps;
    node->drop = drop;
    node->drop.seed_dev = Tensor();
    torch::autograd::set_history(y, node);
  }
  return y;
}

Tensor get(const std::optional<Tensor>& t) { return t.has_value() ? *t : Tensor(); }
using Maybe = std::optional<Tensor>;

}  // namespace

PYBIND11_MODULE(_torch_ops, m) {
  m.doc() = "host path of lbm_amd's training operators";
  m.def("bind", [](uintptr_t forward, uintptr_t backward, uintptr_t drop, uintptr_t workspace, uintptr_t last_error, py::object error) {
    api.forward = reinterpret_cast<decltype(api.forward)>(forward);
    api.backward = reinterpret_cast<decltype(api.backward)>(backward);
    api.dropout = reinterpret_cast<decltype(api.dropout)>(drop);
    api.workspace_bytes = reinterpret_cast<decltype(api.workspace_bytes)>(workspace);
    api.last_error = reinterpret_cast<decltype(api.last_error)>(last_error);
    api.error = error.release().ptr();
  });
  // differentiable
  m.def("dropout", [](const Tensor& x, double p, uint64_t seed, const Maybe& seed_dev, uint64_t offset) -> Tensor {
    HANDLE_TH_ERRORS
    const py::gil_scoped_release no_gil;         // allocations and launches may wait
    elem_type(x, "dropout");
    return dropout(x, make_drop("dropout", p, seed, seed_dev, offset, x));
    END_HANDLE_TH_ERRORS_PYBIND
  });
  m.def("norm", [](const Tensor& x, const Maybe& residual, const Maybe& weight, const Maybe& bias, double eps, double p, uint64_t seed,
                   const Maybe& seed_dev, uint64_t offset) -> Tensor {
    HANDLE_TH_ERRORS
    const py::gil_scoped_release no_gil;         // allocations and launches may wait
    const char* what = residual.has_value() ? "dropout_add_layer_norm" : "layer_norm";
    return norm(what, x, get(residual), get(weight), get(bias), eps, make_drop(what, p, seed, seed_dev, offset, x));
    END_HANDLE_TH_ERRORS_PYBIND
  });
  // single passes
  m.def("dropout_pass", [](const Tensor& x, double p, uint64_t seed, const Maybe& seed_dev, uint64_t offset) -> Tensor {
    HANDLE_TH_ERRORS
    const py::gil_scoped_release no_gil;         // allocations and launches may wait
    const c10::AutoGradMode off(false);
    elem_type(x, "dropout");
    return run_dropout(x, make_drop("dropout", p, seed, seed_dev, offset, x));
    END_HANDLE_TH_ERRORS_PYBIND
  });
  m.def("norm_forward", [](const Tensor& x, const Maybe& residual, const Maybe& weight, const Maybe& bias, double eps, double p, uint64_t seed,
                           const Maybe& seed_dev, uint64_t offset, bool want_stats) -> std::tuple<Tensor, Tensor> {
    HANDLE_TH_ERRORS
    const py::gil_scoped_release no_gil;         // allocations and launches may wait
    const c10::AutoGradMode off(false);
    const Operands o = operands("norm_forward", x, get(residual), get(weight), get(bias));
    return run_forward(o, eps, make_drop("norm_forward", p, seed, seed_dev, offset, x), want_stats);
    END_HANDLE_TH_ERRORS_PYBIND
  });
  m.def("norm_backward", [](const Tensor& dy, const Tensor& x, const Tensor& mean, const Tensor& rstd, const Maybe& residual, const Maybe& weight,
                            const Maybe& bias, double eps, double p, uint64_t seed, const Maybe& seed_dev, uint64_t offset, bool want_x,
                            bool want_r, bool want_w, bool want_b) -> variable_list {
    HANDLE_TH_ERRORS
    const py::gil_scoped_release no_gil;         // allocations and launches may wait
    const c10::AutoGradMode off(false);
    const Operands o = operands("norm_backward", x, get(residual), get(weight), get(bias));
    const Tensor& like = residual.has_value() ? *residual : x;
    if (dy.sizes() != x.sizes() || dy.scalar_type() != like.scalar_type() || dy.device() != x.device())
      fail("norm_backward: dy is " + text(dy) + ", the forward pass's result was like " + text(like));
    for (const Tensor* t : {&mean, &rstd})
      if (t->scalar_type() != at::kFloat || t->numel() != o.rows || t->device() != x.device() || !t->is_contiguous())
        fail("norm_backward: mean and rstd are the dense fp32 statistics of norm_forward, one a row; got " + text(*t));
    return run_backward(o, eps, make_drop("norm_backward", p, seed, seed_dev, offset, x), dy, (const float*)mean.const_data_ptr(),
                        (const float*)rstd.const_data_ptr(), want_x, want_r, want_w, want_b);
    END_HANDLE_TH_ERRORS_PYBIND
  });
}
