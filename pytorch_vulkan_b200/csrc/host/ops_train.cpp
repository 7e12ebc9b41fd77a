// What a transformer's training step needs beside its layers: the softmax
// cross entropy of a linear layer over a large vocabulary, the AdamW step
// over many tensors (torch's _fused_adam_ / _fused_adamw_, and the 8-bit
// state of pytorch_vulkan_b200.optim.AdamW) and the learned relative position
// bias, as ops of the `ocl` namespace with their gradients.  The reference
// had none of them: its optimizers fell into one mul_/add_ launch per tensor and
// operation (src/pointwise_ops.cpp:115-234,407-434).
#include <torch/csrc/autograd/custom_function.h>
#include <torch/extension.h>

#include "ocl.h"

namespace ocl {

// ------------------------------------------------------------------ AdamW
static bool adam_type(c10::ScalarType t) { return t == at::kFloat || t == at::kHalf || t == at::kBFloat16; }

// memory order of `t` is that of `p`: the flat walk pairs their elements
static bool same_layout(const at::Tensor& t, const at::Tensor& p) {
  return t.sizes().equals(p.sizes()) && t.is_non_overlapping_and_dense() && (t.strides().equals(p.strides()) ||
         (t.is_contiguous() && p.is_contiguous()));
}

static at::Tensor grad_like(const at::Tensor& g, const at::Tensor& p) {
  if (same_layout(g, p)) return g;
  at::Tensor c = empty_strided_dev(p.sizes(), p.strides(), p.scalar_type(), p.device().index());
  copy_into(c, g, false);
  return c;
}

static void check_param(const at::Tensor& p, const at::Tensor& g, int dev, c10::ScalarType type, size_t i) {
  TORCH_CHECK(is_ocl(p) && p.device().index() == dev && is_ocl(g) && g.device().index() == dev,
              "ocl AdamW: parameter ", i, " and its gradient have to be on ocl:", dev);
  TORCH_CHECK(adam_type(p.scalar_type()) && p.scalar_type() == type && g.scalar_type() == type,
              "ocl AdamW: parameters and gradients of one type (fp32, fp16 or bf16) expected, got ", p.scalar_type(),
              " and ", g.scalar_type(), " at ", i);
  TORCH_CHECK(g.sizes().equals(p.sizes()), "ocl AdamW: gradient ", i, " has another shape than its parameter");
  TORCH_CHECK(p.is_non_overlapping_and_dense(), "ocl AdamW: parameter ", i, " has gaps or overlaps in memory");
}

static float* step_ptr(const at::Tensor& t, int dev, size_t i) {
  TORCH_CHECK(is_ocl(t) && t.device().index() == dev && t.scalar_type() == at::kFloat && t.numel() == 1,
              "ocl AdamW: step ", i, " has to be one fp32 value on ocl:", dev);
  return t.data_ptr<float>();
}

static const float* scalar_ptr(const std::optional<at::Tensor>& t, int dev, const char* what) {
  if (!t.has_value() || !t->defined()) return nullptr;
  TORCH_CHECK(is_ocl(*t) && t->device().index() == dev && t->scalar_type() == at::kFloat && t->numel() == 1,
              "ocl _fused_adam: ", what, " has to be one fp32 value on ocl:", dev);
  return t->data_ptr<float>();
}

static void fused_adam(bool decoupled, at::TensorList self, at::TensorList grads, at::TensorList exp_avgs,
                       at::TensorList exp_avg_sqs, at::TensorList max_exp_avg_sqs, at::TensorList state_steps, double lr,
                       const float* lr_device, double beta1, double beta2, double weight_decay, double eps,
                       bool amsgrad, bool maximize, const std::optional<at::Tensor>& grad_scale,
                       const std::optional<at::Tensor>& found_inf) {
  if (self.empty()) return;
  const size_t n = self.size();
  TORCH_CHECK(grads.size() == n && exp_avgs.size() == n && exp_avg_sqs.size() == n && state_steps.size() == n &&
                  (!amsgrad || max_exp_avg_sqs.size() == n),
              "ocl _fused_adam: lists of one length expected");
  const int dev = self[0].device().index();
  const c10::ScalarType type = self[0].scalar_type(), state = exp_avgs[0].scalar_type();
  DeviceScope scope(dev);
  OCL_OP(decoupled ? "_fused_adamw_" : "_fused_adam_", dev);
  std::vector<pvb2_adamw_tensor> ts(n);
  std::vector<at::Tensor> copies;  // gradients laid out unlike their parameters
  const bool scaled = grad_scale.has_value() && grad_scale->defined();
  for (size_t i = 0; i < n; ++i) {
    check_param(self[i], grads[i], dev, type, i);
    // a gradient that is unscaled is written back, so no copy will do
    TORCH_CHECK(!scaled || same_layout(grads[i], self[i]),
                "ocl _fused_adam: gradient ", i, " is laid out unlike its parameter");
    const at::Tensor g = grad_like(grads[i], self[i]);
    if (!g.is_same(grads[i])) copies.push_back(g);
    pvb2_adamw_tensor& t = ts[i];
    memset(&t, 0, sizeof(t));
    auto held = [&](const at::Tensor& x) {
      TORCH_CHECK(is_ocl(x) && x.device().index() == dev && x.scalar_type() == state && same_layout(x, self[i]),
                  "ocl _fused_adam: moments ", i, " have to be of one type and laid out as their parameter");
      return x.data_ptr();
    };
    t.param = self[i].data_ptr();
    t.grad = g.data_ptr();
    t.exp_avg = held(exp_avgs[i]);
    t.exp_avg_sq = held(exp_avg_sqs[i]);
    if (amsgrad) t.max_exp_avg_sq = held(max_exp_avg_sqs[i]);
    t.step = step_ptr(state_steps[i], dev, i);
    t.numel = self[i].numel();
  }
  TORCH_CHECK(state == at::kFloat || state == type, "ocl _fused_adam: moments of the parameters' type or fp32 expected");
  pvb2_adamw_desc d;
  memset(&d, 0, sizeof(d));
  d.param_dtype = dtype_code(type);
  d.state_dtype = dtype_code(state);
  d.decoupled = decoupled ? 1 : 0;
  d.maximize = maximize ? 1 : 0;
  d.amsgrad = amsgrad ? 1 : 0;
  d.lr = lr;
  d.beta1 = beta1;
  d.beta2 = beta2;
  d.eps = eps;
  d.weight_decay = weight_decay;
  d.lr_device = lr_device;
  d.grad_scale = scalar_ptr(grad_scale, dev, "grad_scale");
  d.found_inf = scalar_ptr(found_inf, dev, "found_inf");
  Workspace ws(pvb2_adamw_workspace_size((int)n), dev);
  OCL_CHECK(pvb2_adamw_multi(&d, (int)n, ts.data(), ws.get(), ws.bytes, stream_for(dev)));
}

template <bool DECOUPLED>
static void fused_adam_(at::TensorList self, at::TensorList grads, at::TensorList exp_avgs, at::TensorList exp_avg_sqs,
                        at::TensorList max_exp_avg_sqs, at::TensorList state_steps, double lr, double beta1,
                        double beta2, double weight_decay, double eps, bool amsgrad, bool maximize,
                        const std::optional<at::Tensor>& grad_scale, const std::optional<at::Tensor>& found_inf) {
  fused_adam(DECOUPLED, self, grads, exp_avgs, exp_avg_sqs, max_exp_avg_sqs, state_steps, lr, nullptr, beta1, beta2,
             weight_decay, eps, amsgrad, maximize, grad_scale, found_inf);
}

template <bool DECOUPLED>
static void fused_adam_tensor_lr_(at::TensorList self, at::TensorList grads, at::TensorList exp_avgs,
                                  at::TensorList exp_avg_sqs, at::TensorList max_exp_avg_sqs,
                                  at::TensorList state_steps, const at::Tensor& lr, double beta1, double beta2,
                                  double weight_decay, double eps, bool amsgrad, bool maximize,
                                  const std::optional<at::Tensor>& grad_scale,
                                  const std::optional<at::Tensor>& found_inf) {
  if (self.empty()) return;
  // a learning rate in host memory is a number; one on the device is read there
  const bool host = lr.device().is_cpu();
  fused_adam(DECOUPLED, self, grads, exp_avgs, exp_avg_sqs, max_exp_avg_sqs, state_steps,
             host ? lr.item().toDouble() : 0.0, host ? nullptr : scalar_ptr(lr, self[0].device().index(), "lr"), beta1,
             beta2, weight_decay, eps, amsgrad, maximize, grad_scale, found_inf);
}

// The optimizer's Python objects, read here since a loop in Python over the
// parameters costs more than the launch: tensors, and the dict of a
// parameter's state.
static const at::Tensor& py_tensor(PyObject* o, const char* what) {
  TORCH_CHECK(o && THPVariable_Check(o), "ocl AdamW: ", what, " is not a tensor");
  return THPVariable_Unpack(o);
}

// a key of a state's dict, made once
struct StateKey {
  const char* name;
  PyObject* key;
  explicit StateKey(const char* n) : name(n), key(PyUnicode_InternFromString(n)) {}
};

struct AdamState {  // of one parameter
  PyObject* dict = nullptr;
  // (a key's hash and comparison are a string's: no Python code runs here)
  const at::Tensor& get(const StateKey& k) const { return py_tensor(PyDict_GetItemWithError(dict, k.key), k.name); }
};

// objects that stay alive until this goes
struct PyHeld {
  std::vector<PyObject*> objects;
  explicit PyHeld(size_t n) { objects.reserve(n); }
  PyHeld(const PyHeld&) = delete;
  ~PyHeld() {
    for (PyObject* o : objects) Py_DECREF(o);
  }
  void hold(PyObject* o) {
    objects.push_back(o);
    Py_INCREF(o);
  }
};

struct StateKeys {
  StateKey step{"step"}, exp_avg{"exp_avg"}, exp_avg_sq{"exp_avg_sq"}, exp_avg_code{"exp_avg_code"},
      exp_avg_rms_code{"exp_avg_rms_code"}, exp_avg_scale{"exp_avg_scale"}, exp_avg_rms_scale{"exp_avg_rms_scale"};
};
static const StateKeys& state_keys() {
  static const StateKeys* keys = new StateKeys;  // outlives the interpreter's objects
  return *keys;
}

// undefined state: an empty or a missing dict.  A tensor's hash is Python code,
// in which anything may happen to the program's lists, gradients and states,
// from another thread too: whatever was found before is held.
static bool adam_state(const pybind11::dict& state, PyObject* p, AdamState* s, PyHeld& held) {
  s->dict = PyDict_GetItemWithError(state.ptr(), p);
  if (!s->dict && PyErr_Occurred()) throw pybind11::error_already_set();
  if (!s->dict) return false;
  held.hold(s->dict);
  TORCH_CHECK(PyDict_Check(s->dict), "ocl AdamW: a parameter's state is not a dict");
  return PyDict_Size(s->dict) > 0;
}

// How a tensor of the state lies in memory: as its parameter; as its parameter,
// or in a row if the parameter does (codes; their order is the parameter's
// memory order, which a row says only of a contiguous one); in a row.
enum class Held { kAsParam, kCodes, kRow };

static void* adam_held(const at::Tensor& x, const at::Tensor& p, c10::ScalarType want, int64_t numel, Held how,
                       const char* what) {
  auto row = [&] { return x.dim() == 1 && x.is_contiguous(); };
  const bool fits = how == Held::kRow     ? row()
                    : how == Held::kCodes ? (row() && p.is_contiguous()) || same_layout(x, p)
                                          : same_layout(x, p);
  TORCH_CHECK(is_ocl(x) && x.device() == p.device() && x.scalar_type() == want && x.numel() == numel && fits,
              "ocl AdamW: ", what, " of the state does not fit its parameter (shape, type, device or memory order)");
  return x.data_ptr();
}

// the pointers of a parameter's 8-bit moments
static void adam_codes(const AdamState& s, const at::Tensor& p, pvb2_adamw_tensor& t) {
  const StateKeys& keys = state_keys();
  const int64_t n = p.numel(), blocks = (n + 255) / 256;
  t.exp_avg = adam_held(s.get(keys.exp_avg_code), p, at::kByte, n, Held::kCodes, "exp_avg_code");
  t.exp_avg_sq = adam_held(s.get(keys.exp_avg_rms_code), p, at::kByte, n, Held::kCodes, "exp_avg_rms_code");
  t.exp_avg_scale = (float*)adam_held(s.get(keys.exp_avg_scale), p, at::kFloat, blocks, Held::kRow, "exp_avg_scale");
  t.exp_avg_sq_scale =
      (float*)adam_held(s.get(keys.exp_avg_rms_scale), p, at::kFloat, blocks, Held::kRow, "exp_avg_rms_scale");
}

// One step of pytorch_vulkan_b200.optim.AdamW over the parameters of a group
// that have a gradient: counts the steps, then updates, one call for each
// device and type among them.  Parameters that have no state yet are returned
// and nothing is done.  Python code runs while the states are looked up, and
// not from there to the launches: gradients are read then, and need no count
// (211 parameters: 59 us a call, 54 where the states were not held either, 71
// where all are pybind11 objects and each gradient is counted up and down); one
// that has gone by then has no part in the step.
static pybind11::list adamw_step(const pybind11::list& params, const pybind11::dict& state, int64_t bits, double lr,
                                 double beta1, double beta2, double eps, double weight_decay, bool maximize) {
  const bool codes = bits == 8;
  pybind11::list missing;
  struct Item {
    const at::Tensor *p, *g;  // of an object in `list`, and its gradient
    AdamState state;
    bool done;
  };
  const pybind11::tuple list(params);
  PyHeld held(list.size());
  std::vector<Item> items;
  items.reserve(list.size());
  for (const pybind11::handle h : list) {
    const at::Tensor& p = py_tensor(h.ptr(), "a parameter");
    if (!p.grad().defined()) continue;
    items.push_back({&p, nullptr, {}, false});
    if (!adam_state(state, h.ptr(), &items.back().state, held)) missing.append(h);
  }
  if (missing.size() || items.empty()) return missing;
  for (Item& it : items) {
    it.g = &it.p->grad();
    it.done = !it.g->defined();
    TORCH_CHECK(it.done || !it.g->is_sparse(), "ocl AdamW: sparse gradients are not supported");
  }
  // everything is checked before anything is launched
  struct Call {
    int dev;
    c10::ScalarType type;
    std::vector<pvb2_adamw_tensor> ts;
  };
  std::vector<Call> calls;
  std::vector<at::Tensor> copies;  // gradients laid out unlike their parameters
  for (size_t first = 0; first < items.size(); ++first) {
    if (items[first].done) continue;
    const at::Tensor& lead = *items[first].p;
    TORCH_CHECK(is_ocl(lead), "ocl AdamW: parameter ", first, " is on ", lead.device());
    const int dev = lead.device().index();
    const c10::ScalarType type = lead.scalar_type();
    DeviceScope scope(dev);
    calls.push_back({dev, type, {}});
    std::vector<pvb2_adamw_tensor>& ts = calls.back().ts;
    ts.reserve(items.size() - first);
    for (size_t i = first; i < items.size(); ++i) {
      Item& it = items[i];
      const at::Tensor& p = *it.p;
      if (it.done || p.device() != lead.device() || p.scalar_type() != type) continue;
      it.done = true;
      check_param(p, *it.g, dev, type, i);
      const at::Tensor* g = it.g;
      if (!same_layout(*g, p)) {
        copies.push_back(grad_like(*g, p));
        g = &copies.back();
      }
      pvb2_adamw_tensor t;
      memset(&t, 0, sizeof(t));
      t.numel = p.numel();
      t.param = p.data_ptr();
      t.grad = g->data_ptr();
      if (codes) {
        adam_codes(it.state, p, t);
      } else {
        t.exp_avg = adam_held(it.state.get(state_keys().exp_avg), p, at::kFloat, t.numel, Held::kAsParam, "exp_avg");
        t.exp_avg_sq =
            adam_held(it.state.get(state_keys().exp_avg_sq), p, at::kFloat, t.numel, Held::kAsParam, "exp_avg_sq");
      }
      t.step = step_ptr(it.state.get(state_keys().step), dev, i);
      ts.push_back(t);
    }
  }
  for (const Call& call : calls) {
    DeviceScope scope(call.dev);
    OCL_OP("adamw_step", call.dev);
    const int n = (int)call.ts.size();
    pvb2_adamw_desc d;
    memset(&d, 0, sizeof(d));
    d.param_dtype = dtype_code(call.type);
    d.state_dtype = codes ? PVB2_U8 : PVB2_F32;
    d.decoupled = 1;
    d.maximize = maximize ? 1 : 0;
    d.increment_step = 1;
    d.lr = lr;
    d.beta1 = beta1;
    d.beta2 = beta2;
    d.eps = eps;
    d.weight_decay = weight_decay;
    Workspace ws(pvb2_adamw_workspace_size(n), call.dev);
    OCL_CHECK(pvb2_adamw_multi(&d, n, call.ts.data(), ws.get(), ws.bytes, stream_for(call.dev)));
  }
  for (const Item& it : items)
    if (it.g->defined()) it.p->unsafeGetTensorImpl()->bump_version();
  return missing;
}

// the moments that the 8-bit states of `params` (those that have one) stand
// for, into fp32 tensors laid out like them
static void adamw8_values(const pybind11::list& params, const pybind11::dict& state,
                          const std::vector<at::Tensor>& exp_avgs, const std::vector<at::Tensor>& exp_avg_sqs) {
  std::vector<at::Tensor> ps;
  std::vector<AdamState> states;
  const pybind11::tuple list(params);
  PyHeld held(list.size());
  for (const pybind11::handle h : list) {
    AdamState s;
    if (!adam_state(state, h.ptr(), &s, held)) continue;
    ps.push_back(py_tensor(h.ptr(), "a parameter"));
    states.push_back(s);
  }
  TORCH_CHECK_VALUE(exp_avgs.size() == ps.size() && exp_avg_sqs.size() == ps.size(), ps.size(),
                    " parameters have a state, got ", exp_avgs.size(), " and ", exp_avg_sqs.size(), " tensors");
  std::vector<char> done(ps.size(), 0);
  for (size_t first = 0; first < ps.size(); ++first) {
    if (done[first]) continue;
    const int dev = ps[first].device().index();
    DeviceScope scope(dev);
    OCL_OP("adamw8_values", dev);
    std::vector<pvb2_adamw_tensor> ts;
    for (size_t i = first; i < ps.size(); ++i) {
      if (done[i] || ps[i].device() != ps[first].device()) continue;
      done[i] = 1;
      pvb2_adamw_tensor t;
      memset(&t, 0, sizeof(t));
      t.numel = ps[i].numel();
      adam_codes(states[i], ps[i], t);
      t.param = adam_held(exp_avgs[i], ps[i], at::kFloat, t.numel, Held::kAsParam, "the tensor for a first moment");
      t.grad = adam_held(exp_avg_sqs[i], ps[i], at::kFloat, t.numel, Held::kAsParam, "the tensor for a second moment");
      ts.push_back(t);
    }
    OCL_CHECK(pvb2_adamw8_values((int)ts.size(), ts.data(), stream_for(dev)));
  }
  for (size_t i = 0; i < ps.size(); ++i) {
    exp_avgs[i].unsafeGetTensorImpl()->bump_version();
    exp_avg_sqs[i].unsafeGetTensorImpl()->bump_version();
  }
}

// ------------------------------------------------------- clipping by the norm
// The norm of the gradients of `params` (those that have one) as one vector:
// norm_type 1, 2, or 0 for the maximum; with `scale` they are scaled to it.
static at::Tensor clip_grad_norm(const pybind11::list& params, double max_norm, int64_t norm_type, bool scale) {
  const pybind11::tuple list(params);
  std::vector<at::Tensor> grads;
  std::vector<pvb2_grad> gs;
  grads.reserve(list.size());
  gs.reserve(list.size());
  for (const pybind11::handle h : list) {
    const at::Tensor& g = py_tensor(h.ptr(), "a parameter").grad();
    if (!g.defined()) continue;
    const size_t i = grads.size();
    TORCH_CHECK(!g.is_sparse() && is_ocl(g) && adam_type(g.scalar_type()),
                "ocl clip_grad_norm_: fp32, fp16 or bf16 gradients on ocl expected, got ", g.scalar_type(), " on ", g.device(),
                " at ", i);
    TORCH_CHECK(grads.empty() || g.device() == grads[0].device(), "ocl clip_grad_norm_: gradients on ", grads[0].device(),
                " and ", g.device());
    TORCH_CHECK(g.is_non_overlapping_and_dense(), "ocl clip_grad_norm_: gradient ", i, " has gaps or overlaps in memory");
    grads.push_back(g);
    gs.push_back({g.numel() ? g.data_ptr() : nullptr, g.numel(), dtype_code(g.scalar_type())});
  }
  if (grads.empty()) return at::zeros({}, at::kFloat);
  const int dev = grads[0].device().index();
  DeviceScope scope(dev);
  OCL_OP("clip_grad_norm_", dev);
  at::Tensor norm = empty({}, at::kFloat, dev);
  const int n = (int)gs.size();
  Workspace ws(pvb2_clip_grad_norm_workspace_size(n), dev);
  OCL_CHECK(pvb2_clip_grad_norm(n, gs.data(), (int)norm_type, scale ? 1 : 0, max_norm, (float*)norm.data_ptr(), ws.get(),
                                ws.bytes, stream_for(dev)));
  if (scale)
    for (const at::Tensor& g : grads) g.unsafeGetTensorImpl()->bump_version();
  return norm;
}

// -------------------------------------------------- relative position bias
static pvb2_relative_bias_desc bias_desc(c10::ScalarType type, int64_t buckets, int64_t heads, int64_t q_len,
                                         int64_t k_len, bool bidirectional, int64_t max_distance, int64_t q_offset) {
  TORCH_CHECK(type == at::kFloat || type == at::kHalf || type == at::kBFloat16,
              "ocl relative_position_bias: fp32, fp16 or bf16 expected, got ", type);
  const int64_t most = std::numeric_limits<int32_t>::max();
  TORCH_CHECK(buckets <= most && heads <= most, "ocl relative_position_bias: table too large");
  pvb2_relative_bias_desc d;
  memset(&d, 0, sizeof(d));
  d.H = (int32_t)heads;
  d.num_buckets = (int32_t)buckets;
  d.bidirectional = bidirectional ? 1 : 0;
  d.dtype = dtype_code(type);
  d.Lq = q_len;
  d.Lk = k_len;
  d.max_distance = max_distance;
  d.q_offset = q_offset;
  return d;
}

static at::Tensor relative_position_bias(const at::Tensor& table, int64_t q_len, int64_t k_len, bool bidirectional,
                                         int64_t max_distance, int64_t q_offset) {
  TORCH_CHECK(is_ocl(table) && table.dim() == 2, "ocl relative_position_bias: table [num_buckets, heads] on ocl expected");
  TORCH_CHECK(q_len >= 0 && k_len >= 0, "ocl relative_position_bias: lengths below zero");
  const int dev = table.device().index();
  DeviceScope scope(dev);
  OCL_OP("relative_position_bias", dev);
  const pvb2_relative_bias_desc d = bias_desc(table.scalar_type(), table.size(0), table.size(1), q_len, k_len,
                                              bidirectional, max_distance, q_offset);
  const at::Tensor t = contiguous(table);
  at::Tensor out = empty({1, table.size(1), q_len, k_len}, table.scalar_type(), dev);
  OCL_CHECK(pvb2_relative_bias_fwd(&d, t.data_ptr(), out.data_ptr(), stream_for(dev)));
  return out;
}

static at::Tensor relative_position_bias_backward(const at::Tensor& grad, int64_t num_buckets, bool bidirectional,
                                                  int64_t max_distance, int64_t q_offset) {
  TORCH_CHECK(is_ocl(grad) && grad.dim() == 4,
              "ocl relative_position_bias_backward: grad [batch, heads, q_len, k_len] on ocl expected");
  const int dev = grad.device().index();
  DeviceScope scope(dev);
  OCL_OP("relative_position_bias_backward", dev);
  const pvb2_relative_bias_desc d = bias_desc(grad.scalar_type(), num_buckets, grad.size(1), grad.size(2), grad.size(3),
                                              bidirectional, max_distance, q_offset);
  at::Tensor out = empty({num_buckets, grad.size(1)}, grad.scalar_type(), dev);
  Workspace ws(pvb2_relative_bias_bwd_workspace_size(&d, grad.size(0)), dev);
  const pvb2_tensor g = desc(grad);
  OCL_CHECK(pvb2_relative_bias_bwd(&d, &g, out.data_ptr(), ws.get(), ws.bytes, stream_for(dev)));
  return out;
}

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// the backward passes below are kernels, not differentiable ops
static void no_double_backward(const char* op) {
  TORCH_CHECK(!at::GradMode::is_enabled(), "ocl ", op, ": the backward pass cannot be differentiated again");
}

struct RelativeBias : public torch::autograd::Function<RelativeBias> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& table, int64_t q_len, int64_t k_len,
                            bool bidirectional, int64_t max_distance, int64_t q_offset) {
    at::AutoDispatchBelowADInplaceOrView below;
    ctx->saved_data["buckets"] = table.size(0);
    ctx->saved_data["bidirectional"] = bidirectional;
    ctx->saved_data["max_distance"] = max_distance;
    ctx->saved_data["q_offset"] = q_offset;
    return relative_position_bias(table, q_len, k_len, bidirectional, max_distance, q_offset);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    no_double_backward("relative_position_bias");
    at::Tensor g;
    if (grads[0].defined())
      g = relative_position_bias_backward(grads[0], ctx->saved_data["buckets"].toInt(),
                                          ctx->saved_data["bidirectional"].toBool(),
                                          ctx->saved_data["max_distance"].toInt(), ctx->saved_data["q_offset"].toInt());
    const at::Tensor none;
    return {g, none, none, none, none, none};
  }
};

static at::Tensor relative_position_bias_autograd(const at::Tensor& table, int64_t q_len, int64_t k_len,
                                                  bool bidirectional, int64_t max_distance, int64_t q_offset) {
  TORCH_CHECK(table.dim() == 2, "ocl relative_position_bias: table [num_buckets, heads] expected");
  return RelativeBias::apply(table, q_len, k_len, bidirectional, max_distance, q_offset);
}

// ------------------------------------------------- linear cross entropy
// [rows, length] with unit stride along the length; 16-bit rows that lie 16
// bytes apart begin on 16-byte boundaries.  Anything else is copied.
static at::Tensor ce_operand(const at::Tensor& t) {
  const int64_t R = t.size(0), C = t.size(1);
  const bool rows = (C == 1 || t.stride(1) == 1) && (R <= 1 || t.stride(0) >= C);
  const bool aligned = t.scalar_type() == at::kFloat || (R > 1 && t.stride(0) % 8 != 0) ||
                       (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0;
  if (rows && aligned) return t;
  at::Tensor c = empty(t.sizes(), t.scalar_type(), t.device().index());
  copy_into(c, t, false);
  return c;
}

static pvb2_linear_ce_desc ce_desc(const at::Tensor& x, const at::Tensor& w, int64_t ignore_index, int64_t reduction,
                                   double label_smoothing) {
  pvb2_linear_ce_desc d;
  memset(&d, 0, sizeof(d));
  d.N = x.size(0);
  d.D = x.size(1);
  d.V = w.size(0);
  d.ldx = x.stride(0);
  d.ldw = w.stride(0);
  d.ignore_index = ignore_index;
  d.label_smoothing = label_smoothing;
  d.dtype = dtype_code(x.scalar_type());
  d.reduction = (int32_t)reduction;
  return d;
}

static void ce_check(const at::Tensor& input, const at::Tensor& weight, const at::Tensor& target,
                     const std::optional<at::Tensor>& bias) {
  const char* op = "ocl linear_cross_entropy: ";
  TORCH_CHECK(is_ocl(input) && is_ocl(weight) && is_ocl(target), op, "input, weight and target on ocl expected, got ",
              input.device(), ", ", weight.device(), " and ", target.device());
  const int dev = input.device().index();
  TORCH_CHECK(weight.device().index() == dev && target.device().index() == dev, op, "tensors on one device expected");
  TORCH_CHECK(adam_type(input.scalar_type()) && weight.scalar_type() == input.scalar_type(), op,
              "input and weight of one type (fp32, fp16 or bf16) expected, got ", input.scalar_type(), " and ",
              weight.scalar_type());
  TORCH_CHECK(input.dim() >= 1 && weight.dim() == 2 && input.size(-1) == weight.size(1), op,
              "input [..., features] and weight [classes, features] expected, got ", input.sizes(), " and ",
              weight.sizes());
  TORCH_CHECK(weight.size(0) > 0 && weight.size(1) > 0, op, "no classes or no features");
  TORCH_CHECK(target.scalar_type() == at::kLong && target.sizes().equals(input.sizes().slice(0, input.dim() - 1)), op,
              "int64 target shaped like the input without its features expected, got ", target.scalar_type(), " ",
              target.sizes());
  if (bias.has_value() && bias->defined())
    TORCH_CHECK(is_ocl(*bias) && bias->device().index() == dev && bias->scalar_type() == input.scalar_type() &&
                    bias->dim() == 1 && bias->size(0) == weight.size(0),
                op, "bias [classes] of the input's type expected");
}

// bytes that a forward pass may keep for its backward pass
static size_t ce_keep_budget() {
  const char* e = getenv("B200_CE_KEEP_MB");
  const double mb = e ? atof(e) : 2048.0;
  return mb > 0 ? (size_t)(std::min(mb, 1e9) * 1048576.0) : 0;
}

struct CeForward {
  at::Tensor loss, lse, count;  // lse: of each row; count: rows that have a loss, and the operands' scales
  at::Tensor kept;              // what the backward pass takes, of the first `entries` classes (undefined: none)
  int64_t entries = 0;
};

static CeForward linear_cross_entropy_forward(const at::Tensor& input, const at::Tensor& weight,
                                              const at::Tensor& target, const std::optional<at::Tensor>& bias,
                                              int64_t ignore_index, int64_t reduction, double label_smoothing,
                                              bool keep) {
  ce_check(input, weight, target, bias);
  TORCH_CHECK(reduction >= 0 && reduction <= 2, "ocl linear_cross_entropy: unknown reduction");
  const int dev = input.device().index();
  DeviceScope scope(dev);
  OCL_OP("linear_cross_entropy", dev);
  const at::Tensor x = ce_operand(input.reshape({-1, input.size(-1)})), w = ce_operand(weight);
  const at::Tensor t = contiguous(target);
  at::Tensor b;
  if (bias.has_value() && bias->defined()) b = contiguous(*bias);
  pvb2_linear_ce_desc d = ce_desc(x, w, ignore_index, reduction, label_smoothing);
  CeForward r;
  if (keep) {
    const size_t bytes = pvb2_linear_ce_keep(&d, ce_keep_budget());
    if (bytes) {
      try {
        r.kept = empty({(int64_t)bytes}, at::kByte, dev);
      } catch (const c10::Error&) {  // no memory for it: the backward pass does without
        d.kept = 0;
      }
    }
    r.entries = d.kept;
  }
  at::Tensor loss = reduction == PVB2_LOSS_NONE ? empty(target.sizes(), at::kFloat, dev) : empty({}, at::kFloat, dev);
  at::Tensor lse = empty({d.N}, at::kFloat, dev), count = empty({3}, at::kFloat, dev);
  Workspace ws(pvb2_linear_ce_fwd_workspace_size(&d), dev);
  OCL_CHECK(pvb2_linear_ce_fwd(&d, x.data_ptr(), w.data_ptr(), b.defined() ? b.data_ptr() : nullptr,
                               (const int64_t*)t.data_ptr(), (float*)loss.data_ptr(), (float*)lse.data_ptr(),
                               (float*)count.data_ptr(), r.kept.defined() ? r.kept.data_ptr() : nullptr, ws.get(),
                               ws.bytes, stream_for(dev)));
  r.loss = loss;
  r.lse = lse;
  r.count = count;
  return r;
}

static std::tuple<at::Tensor, at::Tensor, at::Tensor> linear_cross_entropy_backward(
    const at::Tensor& grad, const at::Tensor& input, const at::Tensor& weight, const at::Tensor& target,
    const std::optional<at::Tensor>& bias, const at::Tensor& lse, const at::Tensor& count, const at::Tensor& kept,
    int64_t entries, int64_t ignore_index, int64_t reduction, double label_smoothing, std::array<bool, 3> mask) {
  ce_check(input, weight, target, bias);
  const int dev = input.device().index();
  const int64_t rows = target.numel();
  TORCH_CHECK(is_ocl(grad) && grad.scalar_type() == at::kFloat && grad.numel() == (reduction == 0 ? rows : 1) &&
                  is_ocl(lse) && lse.scalar_type() == at::kFloat && lse.numel() == rows && lse.is_contiguous() &&
                  is_ocl(count) && count.scalar_type() == at::kFloat && count.numel() == 3 && count.is_contiguous(),
              "ocl linear_cross_entropy_backward: gradient or saved tensors do not fit");
  DeviceScope scope(dev);
  OCL_OP("linear_cross_entropy_backward", dev);
  const at::Tensor x = ce_operand(input.reshape({-1, input.size(-1)})), w = ce_operand(weight);
  // one number for all rows, as the sum of the losses sends back: that of a sum,
  // which needs one G instead of two (8192 x 4096 -> 32768 bf16 with nothing
  // kept: 7.0 ms against 8.5)
  bool one = reduction == PVB2_LOSS_NONE && rows > 0;
  for (int64_t k = 0; k < grad.dim(); ++k) one = one && (grad.size(k) == 1 || grad.stride(k) == 0);
  if (one) reduction = PVB2_LOSS_SUM;
  const at::Tensor t = contiguous(target), g = one ? grad : contiguous(grad);
  const bool has_bias = bias.has_value() && bias->defined();
  at::Tensor b;
  if (has_bias) b = contiguous(*bias);
  pvb2_linear_ce_desc d = ce_desc(x, w, ignore_index, reduction, label_smoothing);
  d.kept = entries;
  at::Tensor dx, dw, db;
  if (mask[0]) dx = empty(input.sizes(), input.scalar_type(), dev);
  if (mask[1]) dw = empty(weight.sizes(), weight.scalar_type(), dev);
  if (mask[2] && has_bias) db = empty({d.V}, input.scalar_type(), dev);
  Workspace ws(pvb2_linear_ce_bwd_workspace_size(&d), dev);
  OCL_CHECK(pvb2_linear_ce_bwd(&d, x.data_ptr(), w.data_ptr(), has_bias ? b.data_ptr() : nullptr,
                               (const int64_t*)t.data_ptr(), (const float*)lse.data_ptr(),
                               (const float*)count.data_ptr(), kept.defined() ? kept.data_ptr() : nullptr,
                               (const float*)g.data_ptr(),
                               dx.defined() ? dx.data_ptr() : nullptr, dw.defined() ? dw.data_ptr() : nullptr,
                               db.defined() ? db.data_ptr() : nullptr, ws.get(), ws.bytes, stream_for(dev)));
  return {dx, dw, db};
}

static at::Tensor linear_cross_entropy(const at::Tensor& input, const at::Tensor& weight, const at::Tensor& target,
                                       const std::optional<at::Tensor>& bias, int64_t ignore_index, int64_t reduction,
                                       double label_smoothing) {
  return linear_cross_entropy_forward(input, weight, target, bias, ignore_index, reduction, label_smoothing, false).loss;
}

struct LinearCrossEntropy : public torch::autograd::Function<LinearCrossEntropy> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& input, const at::Tensor& weight,
                            const at::Tensor& target, const std::optional<at::Tensor>& bias, int64_t ignore_index,
                            int64_t reduction, double label_smoothing) {
    at::AutoDispatchBelowADInplaceOrView below;
    const CeForward r =
        linear_cross_entropy_forward(input, weight, target, bias, ignore_index, reduction, label_smoothing, true);
    ctx->save_for_backward({input, weight, target, bias.value_or(at::Tensor()), r.lse, r.count, r.kept});
    ctx->saved_data["entries"] = r.entries;
    ctx->saved_data["ignore_index"] = ignore_index;
    ctx->saved_data["reduction"] = reduction;
    ctx->saved_data["label_smoothing"] = label_smoothing;
    return r.loss;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    no_double_backward("linear_cross_entropy");
    const at::Tensor none;
    if (!grads[0].defined()) return {none, none, none, none, none, none, none};
    const variable_list s = ctx->get_saved_variables();
    const bool has_bias = s[3].defined();
    // needs_input_grad counts the tensors that were passed: input, weight, target, bias
    const std::array<bool, 3> mask = {ctx->needs_input_grad(0), ctx->needs_input_grad(1),
                                      has_bias && ctx->needs_input_grad(3)};
    at::Tensor dx, dw, db;
    std::tie(dx, dw, db) = linear_cross_entropy_backward(
        grads[0], s[0], s[1], s[2], has_bias ? std::optional<at::Tensor>(s[3]) : std::nullopt, s[4], s[5], s[6],
        ctx->saved_data["entries"].toInt(), ctx->saved_data["ignore_index"].toInt(), ctx->saved_data["reduction"].toInt(),
        ctx->saved_data["label_smoothing"].toDouble(), mask);
    return {dx, dw, none, db, none, none, none};
  }
};

static at::Tensor linear_cross_entropy_autograd(const at::Tensor& input, const at::Tensor& weight,
                                                const at::Tensor& target, const std::optional<at::Tensor>& bias,
                                                int64_t ignore_index, int64_t reduction, double label_smoothing) {
  auto any = [&](auto f) { return f(input) || f(weight) || (bias.has_value() && bias->defined() && f(*bias)); };
  // a tangent (forward mode, for which requires_grad says nothing) goes to the function too, which refuses it
  const bool grads = (at::GradMode::is_enabled() && any([](const at::Tensor& t) { return t.requires_grad(); })) ||
                     any([](const at::Tensor& t) { return t._fw_grad(0).defined(); });
  if (!grads) {
    at::AutoDispatchBelowADInplaceOrView below;
    return linear_cross_entropy(input, weight, target, bias, ignore_index, reduction, label_smoothing);
  }
  return LinearCrossEntropy::apply(input, weight, target, bias, ignore_index, reduction, label_smoothing);
}

}  // namespace ocl

TORCH_LIBRARY(ocl, m) {
  m.def("linear_cross_entropy(Tensor input, Tensor weight, Tensor target, Tensor? bias, int ignore_index, "
        "int reduction, float label_smoothing) -> Tensor");
  m.def("relative_position_bias(Tensor table, int q_len, int k_len, bool bidirectional, int max_distance, "
        "int q_offset) -> Tensor");
  m.def("relative_position_bias_backward(Tensor grad, int num_buckets, bool bidirectional, int max_distance, "
        "int q_offset) -> Tensor");
}

TORCH_LIBRARY_IMPL(ocl, PrivateUse1, m) {
  m.impl("linear_cross_entropy", &ocl::linear_cross_entropy);
  m.impl("relative_position_bias", &ocl::relative_position_bias);
  m.impl("relative_position_bias_backward", &ocl::relative_position_bias_backward);
}

TORCH_LIBRARY_IMPL(ocl, AutogradPrivateUse1, m) {
  m.impl("linear_cross_entropy", &ocl::linear_cross_entropy_autograd);
  m.impl("relative_position_bias", &ocl::relative_position_bias_autograd);
}

TORCH_LIBRARY_IMPL(aten, PrivateUse1, m) {
  m.impl("_fused_adam_", &ocl::fused_adam_<false>);
  m.impl("_fused_adam_.tensor_lr", &ocl::fused_adam_tensor_lr_<false>);
  m.impl("_fused_adamw_", &ocl::fused_adam_<true>);
  m.impl("_fused_adamw_.tensor_lr", &ocl::fused_adam_tensor_lr_<true>);
}

void register_train_bindings(pybind11::module& m) {
  m.def("impl_adamw_step", &ocl::adamw_step, "one AdamW step over a group's parameters");
  m.def("impl_clip_grad_norm", &ocl::clip_grad_norm, "the gradients' norm, and their scaling to it");
  m.def("impl_adamw8_values", &ocl::adamw8_values, "the moments that 8-bit codes stand for");
}
