// The host side of dropout, norm, residual_norm and fp8_linear for PyTorch: argument checks, outputs and workspaces from
// PyTorch's allocator on the current stream, and autograd nodes, over the C ABI of libpack3d_b200.so.
// In Python these cost more than the kernels of a small call (a training step of residual_norm on 39 rows:
// 179 us, of which 25 us kernels); the functions here are called with positional arguments by
// pack3d_b200.residual and pack3d_b200.fp8, whose docstrings describe them.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <string>

#include "pack3d_b200.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

constexpr int64_t kMaxDim = 16384;

// ------------------------------------------------------------------------------- arguments
int dtype_code(at::ScalarType t) {
  return t == at::kFloat ? P3D_F32 : t == at::kHalf ? P3D_F16 : t == at::kBFloat16 ? P3D_BF16 : -1;
}

Tensor tensor_or_none(PyObject *o, const char *what) {
  if (o == Py_None) return Tensor();
  TORCH_CHECK_VALUE(THPVariable_Check(o), what, " must be a tensor");
  return THPVariable_Unpack(o);
}
Tensor tensor(PyObject *o, const char *what) {
  TORCH_CHECK_VALUE(THPVariable_Check(o), what, " must be a tensor");
  return THPVariable_Unpack(o);
}
double number(PyObject *o, const char *what) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    TORCH_CHECK_VALUE(false, what, " must be a number");
  }
  return v;
}
bool is_word(PyObject *o, const char *word) {
  return PyUnicode_Check(o) && PyUnicode_CompareWithASCIIString(o, word) == 0;
}

void check_cuda(const Tensor &x) {
  TORCH_CHECK_VALUE(x.is_cuda() && dtype_code(x.scalar_type()) >= 0, "b200 backend requires CUDA fp32/fp16/bf16 tensors");
  TORCH_CHECK_VALUE(at::cuda::getDeviceProperties(x.device().index())->major == 10,
                    "b200 backend targets compute capability 10.x (sm_100a) devices");
}
void check_input(const Tensor &x, const char *what) {
  TORCH_CHECK_VALUE(x.dim() >= 1, what, " needs at least one dimension");
  check_cuda(x);
  TORCH_CHECK_VALUE(x.size(-1) >= 1 && x.size(-1) <= kMaxDim, what, ": the last dimension must be 1 to ", kMaxDim, ", got ",
                    x.size(-1));
}
void check_vector(const Tensor &t, const Tensor &x, const char *what) {
  if (!t.defined()) return;
  TORCH_CHECK_VALUE(t.dim() == 1 && t.size(0) == x.size(-1), what, ": parameters must have shape [", x.size(-1), "], got ",
                    t.sizes());
  TORCH_CHECK_VALUE(t.device() == x.device(), what, ": parameters and input must be on the same device");
  TORCH_CHECK_VALUE(t.scalar_type() == x.scalar_type() || t.scalar_type() == at::kFloat, what, ": parameters must be ",
                    x.scalar_type(), " or torch.float32, got ", t.scalar_type());
}

// A NormSpec: the named tuple (weight, bias, kind, eps).
struct Spec {
  Tensor weight, bias;
  int kind = P3D_NORM_NONE;
  float eps = 0.f;
};
Spec spec_of(PyObject *o, const Tensor &x, const char *what) {
  Spec s;
  if (o == Py_None) return s;
  TORCH_CHECK_VALUE(PyTuple_Check(o) && PyTuple_GET_SIZE(o) == 4, what, " must be a NormSpec");
  PyObject *kind = PyTuple_GET_ITEM(o, 2);
  s.kind = is_word(kind, "rms") ? P3D_NORM_RMS : is_word(kind, "layer") ? P3D_NORM_LAYER : P3D_NORM_NONE;
  TORCH_CHECK_VALUE(s.kind != P3D_NORM_NONE, what, ": kind must be 'rms' or 'layer'");
  const double eps = number(PyTuple_GET_ITEM(o, 3), "eps");
  TORCH_CHECK_VALUE(std::isfinite(eps) && eps >= 0, what, ": eps must be finite and not negative");
  s.eps = (float)eps;
  s.weight = tensor_or_none(PyTuple_GET_ITEM(o, 0), what);
  s.bias = tensor_or_none(PyTuple_GET_ITEM(o, 1), what);
  check_vector(s.weight, x, what);
  check_vector(s.bias, x, what);
  return s;
}

uint32_t threshold_of(PyObject *o) {
  const double p = number(o, "dropout probability");
  TORCH_CHECK_VALUE(p >= 0.0 && p <= 1.0, "dropout probability must lie between 0 and 1");
  return (uint32_t)std::nearbyint(65536.0 * p);   // ties to even, as Python's round
}

// (seed, offset), or an int64 tensor of the two on the input's device.
struct Rng {
  Tensor tensor;
  uint64_t seed = 0, offset = 0;
};
Rng rng_of(PyObject *o, const Tensor &x) {
  Rng r;
  TORCH_CHECK_VALUE(o != Py_None, "dropout needs rng: (seed, offset) or an int64 tensor of the two");
  if (THPVariable_Check(o)) {
    r.tensor = THPVariable_Unpack(o);
    TORCH_CHECK_VALUE(r.tensor.scalar_type() == at::kLong && r.tensor.numel() == 2 && r.tensor.device() == x.device() &&
                          r.tensor.is_contiguous(),
                      "rng must hold (seed, offset): two contiguous int64 on the input's device");
    return r;
  }
  const bool pair = (PyTuple_Check(o) || PyList_Check(o)) && PySequence_Fast_GET_SIZE(o) == 2;
  TORCH_CHECK_VALUE(pair, "rng must be (seed, offset) or an int64 tensor of the two");
  uint64_t *to[2] = {&r.seed, &r.offset};
  for (int i = 0; i < 2; ++i) {
    PyObject *v = PyNumber_Index(PySequence_Fast_GET_ITEM(o, i));
    if (!v) PyErr_Clear();
    TORCH_CHECK_VALUE(v, "rng must be (seed, offset) or an int64 tensor of the two");
    *to[i] = PyLong_AsUnsignedLongLongMask(v);
    Py_DECREF(v);
  }
  return r;
}

const void *ptr(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }
void *out_ptr(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }
void *stream() { return at::cuda::getCurrentCUDAStream().stream(); }

void check_status(int status, const char *what) {
  if (status == P3D_OK) return;
  const std::string text = std::string(what) + ": " + p3d_strerror(status) + ": " + p3d_last_error();
  TORCH_CHECK_VALUE(status != P3D_ERR_INVALID_ARGUMENT && status != P3D_ERR_UNSUPPORTED, text);
  TORCH_CHECK(false, text);
}

// What a backward pass returns cannot be differentiated again: where its own upstream gradients ask for that, the
// results carry an error for whoever tries.
variable_list once(variable_list grads, const variable_list &up) {
  bool asked = false;
  for (const Tensor &t : up) asked |= t.defined() && t.requires_grad();
  if (!asked || !at::GradMode::is_enabled()) return grads;
  for (Tensor &g : grads)
    if (g.defined()) g = g.detach().set_requires_grad(true);
  auto node = std::make_shared<torch::autograd::DelayedError>(
      "trying to differentiate twice a function that can be differentiated once", (int64_t)grads.size());
  return (*node)(std::move(grads));
}

// A tensor that may be absent, as the autograd functions take it: edges exist for those that are there.
using Optional = std::optional<Tensor>;
Optional optional(const Tensor &t) { return t.defined() ? Optional(t) : Optional(); }
Tensor value(const Optional &t) { return t ? *t : Tensor(); }

bool wants_grad(std::initializer_list<const Tensor *> tensors) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor *t : tensors)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

// Forward-mode derivatives are not there: a tangent is refused, whether or not the tensor takes part in reverse mode too, as
// a result without one would read as a zero derivative.
void refuse_tangents(std::initializer_list<const Tensor *> tensors) {
  for (const Tensor *t : tensors)
    TORCH_CHECK_NOT_IMPLEMENTED(!(t->defined() && t->_fw_grad(0).defined()),
                                "forward-mode derivatives of this operator are not implemented");
}

// ------------------------------------------------------------------------------- dropout
Tensor run_dropout(const Tensor &x, uint32_t threshold, const Tensor &rng, uint64_t seed, uint64_t offset) {
  const c10::cuda::CUDAGuard guard(x.device());
  const Tensor in = x.contiguous(), y = at::empty_like(in);
  if (in.numel() == 0) return y;
  const int64_t dim = in.dim() ? in.size(-1) : 1;
  check_status(p3d_dropout(in.data_ptr(), y.data_ptr(), dtype_code(in.scalar_type()), in.numel() / dim, dim, threshold,
                           static_cast<const uint64_t *>(ptr(rng)), seed, offset, stream()),
               "p3d_dropout");
  return y;
}

struct Dropout : torch::autograd::Function<Dropout> {
  static Tensor forward(AutogradContext *ctx, const Tensor &x, const Optional &rng, int64_t threshold, int64_t seed,
                        int64_t offset) {
    ctx->save_for_backward({value(rng)});
    ctx->saved_data["threshold"] = threshold;
    ctx->saved_data["seed"] = seed;
    ctx->saved_data["offset"] = offset;
    return run_dropout(x, (uint32_t)threshold, value(rng), (uint64_t)seed, (uint64_t)offset);
  }
  static variable_list backward(AutogradContext *ctx, variable_list dy) {
    const Tensor rng = ctx->get_saved_variables()[0];
    refuse_tangents({&dy[0]});
    return once({run_dropout(dy[0].detach(), (uint32_t)ctx->saved_data["threshold"].toInt(), rng,
                             (uint64_t)ctx->saved_data["seed"].toInt(), (uint64_t)ctx->saved_data["offset"].toInt()),
                 Tensor(), Tensor(), Tensor(), Tensor()},
                dy);
  }
};

PyObject *py_dropout(PyObject *, PyObject *const *args, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_VALUE(count == 3, "dropout takes x, p, rng");
  const Tensor x = tensor(args[0], "x");
  refuse_tangents({&x});
  check_cuda(x);
  const uint32_t threshold = threshold_of(args[1]);
  const Rng r = rng_of(args[2], x);
  if (wants_grad({&x}))
    return THPVariable_Wrap(Dropout::apply(x, optional(r.tensor), (int64_t)threshold, (int64_t)r.seed, (int64_t)r.offset));
  return THPVariable_Wrap(run_dropout(x, threshold, r.tensor, r.seed, r.offset));
  END_HANDLE_TH_ERRORS
}

// ------------------------------------------------------------------------------- norms and residual
// A call: its description without addresses, and its tensors in the order of their gradients.
enum : int { kX, kH, kGate, kPostW, kPostB, kScale, kNextW, kNextB, kTensors };
struct Call {
  p3d_residual args = {};
  Tensor t[kTensors];
  Tensor rng;
  void address() {
    args.x = ptr(t[kX]);
    args.h = ptr(t[kH]);
    args.gate = ptr(t[kGate]);
    args.post_weight = ptr(t[kPostW]);
    args.post_bias = ptr(t[kPostB]);
    args.scale = ptr(t[kScale]);
    args.next_weight = ptr(t[kNextW]);
    args.next_bias = ptr(t[kNextB]);
    args.rng = static_cast<const uint64_t *>(ptr(rng));
  }
};

// (out, y, stats): out undefined without a block, y without a next norm, stats unless `save`.
struct Results {
  Tensor out, y, stats;
};
Results run_residual(Call &c, bool save) {
  const Tensor &x = c.t[kX];
  const c10::cuda::CUDAGuard guard(x.device());
  Results r;
  if (c.t[kH].defined()) r.out = at::empty_like(x);
  if (c.args.next_kind != P3D_NORM_NONE) r.y = at::empty_like(x);
  if (save) r.stats = at::empty({c.args.rows, 4}, x.options().dtype(at::kFloat));
  if (x.numel() == 0) return r;
  c.address();
  check_status(p3d_residual_fwd(&c.args, out_ptr(r.out), out_ptr(r.y), static_cast<float *>(out_ptr(r.stats)), stream()),
               "p3d_residual_fwd");
  return r;
}

struct Residual : torch::autograd::Function<Residual> {
  static variable_list forward(AutogradContext *ctx, const p3d_residual &args, const Optional &rng, const Optional &x,
                               const Optional &h, const Optional &gate, const Optional &post_w, const Optional &post_b,
                               const Optional &scale, const Optional &next_w, const Optional &next_b) {
    ctx->set_materialize_grads(false);
    Call c;
    c.args = args;
    c.rng = value(rng);
    const Optional *given[kTensors] = {&x, &h, &gate, &post_w, &post_b, &scale, &next_w, &next_b};
    for (int i = 0; i < kTensors; ++i) c.t[i] = value(*given[i]);
    Results r = run_residual(c, true);
    variable_list saved = {c.rng, r.stats};
    saved.insert(saved.end(), c.t, c.t + kTensors);
    ctx->save_for_backward(std::move(saved));
    ctx->saved_data["args"] = std::string(reinterpret_cast<const char *>(&args), sizeof(args));
    variable_list out;
    if (r.out.defined()) out.push_back(r.out);
    if (r.y.defined()) out.push_back(r.y);
    return out;
  }
  static variable_list backward(AutogradContext *ctx, variable_list up) {
    const variable_list saved = ctx->get_saved_variables();
    Call c;
    const std::string &args = ctx->saved_data["args"].toStringRef();
    memcpy(&c.args, args.data(), sizeof(c.args));
    c.rng = saved[0];
    const Tensor stats = saved[1];
    for (int i = 0; i < kTensors; ++i) c.t[i] = saved[2 + i];
    const Tensor &x = c.t[kX];
    const bool block = c.t[kH].defined(), next = c.args.next_kind != P3D_NORM_NONE;
    Tensor dout = block ? up[0] : Tensor(), dy = next ? up[block ? 1 : 0] : Tensor();
    variable_list grads(2 + kTensors);
    if (!dout.defined() && !dy.defined()) return grads;
    refuse_tangents({&dout, &dy});
    const c10::cuda::CUDAGuard guard(x.device());
    Tensor *d = grads.data() + 2;
    size_t edge = c.rng.defined() ? 1 : 0;   // of the next tensor that is there
    for (int i = 0; i < kTensors; ++i)
      if (c.t[i].defined() && ctx->needs_input_grad(edge++))
        d[i] = x.numel() ? at::empty_like(c.t[i]) : at::zeros_like(c.t[i]);
    if (x.numel() == 0) return once(std::move(grads), up);
    if (dout.defined()) dout = dout.detach().contiguous();
    if (dy.defined()) dy = dy.detach().contiguous();
    c.address();
    const size_t need = p3d_residual_bwd_workspace(&c.args);
    const Tensor ws = at::empty({(int64_t)need}, x.options().dtype(at::kByte));
    check_status(p3d_residual_bwd(&c.args, ptr(dout), ptr(dy), static_cast<const float *>(stats.data_ptr()), out_ptr(d[kX]),
                                  out_ptr(d[kH]), out_ptr(d[kGate]), out_ptr(d[kScale]), out_ptr(d[kPostW]),
                                  out_ptr(d[kPostB]), out_ptr(d[kNextW]), out_ptr(d[kNextB]), ws.data_ptr(), need, stream()),
                 "p3d_residual_bwd");
    return once(std::move(grads), up);
  }
};

// The parameters contiguous and of one dtype: where they differ, all in fp32.
void same_params(Call &c) {
  at::ScalarType type = at::ScalarType::Undefined;
  bool differ = false;
  for (int i = kPostW; i <= kNextB; ++i) {
    if (!c.t[i].defined()) continue;
    differ |= type != at::ScalarType::Undefined && c.t[i].scalar_type() != type;
    type = c.t[i].scalar_type();
  }
  for (int i = kPostW; i <= kNextB; ++i)
    if (c.t[i].defined()) c.t[i] = (differ ? c.t[i].to(at::kFloat) : c.t[i]).contiguous();
  c.args.param_dtype = type == at::ScalarType::Undefined ? c.args.dtype : differ ? P3D_F32 : dtype_code(type);
}

PyObject *run_call(Call &c) {
  c.args.dim = (int32_t)c.t[kX].size(-1);
  c.args.rows = c.t[kX].numel() / c.args.dim;
  c.args.dtype = dtype_code(c.t[kX].scalar_type());
  for (const Tensor &t : c.t) refuse_tangents({&t});
  same_params(c);
  const bool block = c.t[kH].defined();
  bool grad = false;
  for (const Tensor &t : c.t) grad |= wants_grad({&t});
  Tensor out, y;
  if (grad) {
    const variable_list r =
        Residual::apply(c.args, optional(c.rng), optional(c.t[kX]), optional(c.t[kH]), optional(c.t[kGate]),
                        optional(c.t[kPostW]), optional(c.t[kPostB]), optional(c.t[kScale]), optional(c.t[kNextW]),
                        optional(c.t[kNextB]));
    size_t i = 0;
    if (block) out = r[i++];
    if (c.args.next_kind != P3D_NORM_NONE) y = r[i];
  } else {
    const Results r = run_residual(c, false);
    out = r.out;
    y = r.y;
  }
  if (!block) return THPVariable_Wrap(y);
  PyObject *pair = PyTuple_New(2);
  if (!pair) throw python_error();
  PyTuple_SET_ITEM(pair, 0, THPVariable_Wrap(out));
  if (y.defined()) {
    PyTuple_SET_ITEM(pair, 1, THPVariable_Wrap(y));
  } else {
    Py_INCREF(Py_None);
    PyTuple_SET_ITEM(pair, 1, Py_None);
  }
  return pair;
}

PyObject *py_norm(PyObject *, PyObject *const *args, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_VALUE(count == 2, "norm takes x, spec");
  const Tensor x = tensor(args[0], "x");
  refuse_tangents({&x});
  check_input(x, "norm");
  TORCH_CHECK_VALUE(args[1] != Py_None, "norm must be given a NormSpec");
  const Spec s = spec_of(args[1], x, "norm");
  Call c;
  c.t[kX] = x.contiguous();
  c.t[kNextW] = s.weight;
  c.t[kNextB] = s.bias;
  c.args.next_kind = s.kind;
  c.args.next_eps = s.eps;
  c.args.scale_value = 1.f;
  return run_call(c);
  END_HANDLE_TH_ERRORS
}

// Sets the gate's mode from its shape against x's.
void set_gate(Call &c, const Tensor &gate, const Tensor &x) {
  TORCH_CHECK_VALUE(gate.device() == x.device() && gate.scalar_type() == x.scalar_type(),
                    "gate must have the dtype and device of x");
  const int64_t n = x.dim(), dim = x.size(-1), rows = x.numel() / dim;
  c.t[kGate] = gate.contiguous();
  if (gate.sizes() == x.sizes()) {
    c.args.gate_mode = P3D_GATE_ELEMENT;
    return;
  }
  if (gate.dim() == n && gate.size(-1) == 1 && gate.sizes().slice(0, n - 1) == x.sizes().slice(0, n - 1)) {
    c.args.gate_mode = P3D_GATE_TOKEN;
    return;
  }
  if (gate.dim() >= 1 && gate.size(-1) == dim && (gate.dim() == 1 || gate.dim() == n)) {
    int64_t vectors = gate.numel() / dim;
    bool fits = vectors == 1;
    if (!fits && gate.dim() == n && n >= 2 && gate.size(0) == x.size(0)) fits = vectors == x.size(0);
    if (fits) {
      c.args.gate_mode = P3D_GATE_SAMPLE;
      c.args.rows_per_sample = std::max<int64_t>(1, rows / std::max<int64_t>(1, vectors));
      return;
    }
  }
  TORCH_CHECK_VALUE(false, "gate must have the shape of x ", x.sizes(), ", one value for each token, or one vector for each "
                    "sample or for all; got ", gate.sizes());
}

PyObject *py_residual_norm(PyObject *, PyObject *const *args, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_VALUE(count == 9, "residual_norm takes x, h, post_norm, gate, gate_activation, scale, next_norm, p, rng");
  const Tensor x = tensor(args[0], "x"), h = tensor(args[1], "h");
  refuse_tangents({&x, &h});
  check_input(x, "residual_norm");
  TORCH_CHECK_VALUE(h.sizes() == x.sizes() && h.scalar_type() == x.scalar_type() && h.device() == x.device(),
                    "h must have the shape, dtype and device of x");
  const Spec post = spec_of(args[2], x, "post_norm"), next = spec_of(args[6], x, "next_norm");
  Call c;
  c.args.gate_act = is_word(args[4], "identity")  ? P3D_ACT_IDENTITY
                    : is_word(args[4], "sigmoid") ? P3D_ACT_SIGMOID
                    : is_word(args[4], "tanh")    ? P3D_ACT_TANH
                                                  : -1;
  TORCH_CHECK_VALUE(c.args.gate_act >= 0, "gate_activation must be 'identity', 'sigmoid' or 'tanh'");
  c.args.scale_value = 1.f;
  if (THPVariable_Check(args[5])) {
    c.t[kScale] = THPVariable_Unpack(args[5]);
    check_vector(c.t[kScale], x, "scale");
  } else if (args[5] != Py_None) {
    c.args.scale_value = (float)number(args[5], "scale");
  }
  const Tensor gate = tensor_or_none(args[3], "gate");
  if (gate.defined()) set_gate(c, gate, x);
  c.args.threshold = threshold_of(args[7]);
  if (c.args.threshold) {
    const Rng r = rng_of(args[8], x);
    c.rng = r.tensor;
    c.args.seed = r.seed;
    c.args.offset = r.offset;
  }
  c.args.post_kind = post.kind;
  c.args.post_eps = post.eps;
  c.args.next_kind = next.kind;
  c.args.next_eps = next.eps;
  c.t[kX] = x.contiguous();
  c.t[kH] = h.contiguous();
  c.t[kPostW] = post.weight;
  c.t[kPostB] = post.bias;
  c.t[kNextW] = next.weight;
  c.t[kNextB] = next.bias;
  return run_call(c);
  END_HANDLE_TH_ERRORS
}

// ------------------------------------------------------------------------------- 8-bit linear layer
p3d_fp8_linear linear_args(const Tensor &x, int64_t n, const Tensor &weight, const Tensor &bias) {
  p3d_fp8_linear a = {};
  a.rows = x.size(0);
  a.k = x.size(1);
  a.n = n;
  a.dtype = dtype_code(x.scalar_type());
  a.weight_dtype = weight.defined() ? dtype_code(weight.scalar_type()) : P3D_F32;
  a.bias_dtype = bias.defined() ? dtype_code(bias.scalar_type()) : P3D_F32;
  return a;
}

// y; *saved: what the backward needs, where the arguments ask for gradients.
Tensor run_linear(const p3d_fp8_linear &a, const Tensor &x, const Tensor &bias, Tensor *saved) {
  const c10::cuda::CUDAGuard guard(x.device());
  const auto bytes = x.options().dtype(at::kByte);
  const Tensor y = at::empty({a.rows, a.n}, x.options());
  if (saved) *saved = at::empty({(int64_t)p3d_fp8_linear_saved(&a)}, bytes);
  const size_t need = p3d_fp8_linear_fwd_workspace(&a);
  const Tensor ws = at::empty({(int64_t)need}, bytes);
  check_status(p3d_fp8_linear_fwd(&a, x.data_ptr(), ptr(bias), y.data_ptr(), saved ? saved->data_ptr() : nullptr,
                                  ws.data_ptr(), need, stream()),
               "p3d_fp8_linear_fwd");
  return y;
}

// Keeps x and the weight in 8 bits only: x with blocks along its rows for dW, the weight transposed for dx (its
// 128 x 128 blocks serve both directions).
struct Linear : torch::autograd::Function<Linear> {
  static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &weight, const Optional &given_bias) {
    const Tensor bias = value(given_bias);
    p3d_fp8_linear a = linear_args(x, weight.size(0), weight, bias);
    a.weight = weight.data_ptr();
    a.need_dx = x.requires_grad();
    a.need_dw = weight.requires_grad();
    Tensor saved;
    const Tensor y = run_linear(a, x, bias, a.need_dx || a.need_dw ? &saved : nullptr);
    ctx->save_for_backward({saved});
    ctx->saved_data["args"] = std::string(reinterpret_cast<const char *>(&a), sizeof(a));
    ctx->saved_data["has_bias"] = bias.defined();
    ctx->saved_data["weight"] = (int64_t)weight.scalar_type();
    ctx->saved_data["bias"] = (int64_t)(bias.defined() ? bias.scalar_type() : at::kFloat);
    return y;
  }
  static variable_list backward(AutogradContext *ctx, variable_list up) {
    p3d_fp8_linear a;
    memcpy(&a, ctx->saved_data["args"].toStringRef().data(), sizeof(a));
    refuse_tangents({&up[0]});
    const Tensor saved = ctx->get_saved_variables()[0], dy = up[0].detach().contiguous();
    const c10::cuda::CUDAGuard guard(dy.device());
    Tensor dx, dw, db;
    // what the forward kept is laid out for the gradients that it was told of: all of those are computed
    if (!a.need_dx && !a.need_dw && !(ctx->saved_data["has_bias"].toBool() && ctx->needs_input_grad(2))) return {dx, dw, db};
    if (a.need_dx) dx = at::empty({a.rows, a.k}, dy.options());
    if (a.need_dw) dw = at::empty({a.n, a.k}, dy.options().dtype((at::ScalarType)ctx->saved_data["weight"].toInt()));
    if (ctx->saved_data["has_bias"].toBool() && ctx->needs_input_grad(2))
      db = at::empty({a.n}, dy.options().dtype((at::ScalarType)ctx->saved_data["bias"].toInt()));
    const size_t need = p3d_fp8_linear_bwd_workspace(&a);
    const Tensor ws = at::empty({(int64_t)need}, dy.options().dtype(at::kByte));
    check_status(p3d_fp8_linear_bwd(&a, dy.data_ptr(), ptr(saved), out_ptr(dx), out_ptr(dw), out_ptr(db), ws.data_ptr(),
                                    need, stream()),
                 "p3d_fp8_linear_bwd");
    return once({dx, dw, db}, up);
  }
};

// x, weight (or None), bias, and where the weight is kept in 8 bits its values, scales, rows and columns.
PyObject *py_fp8_linear(PyObject *, PyObject *const *args, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_VALUE(count == 7, "fp8_linear takes x, weight, bias, values, scales, rows, cols");
  const Tensor x = tensor(args[0], "x");
  Tensor weight = tensor_or_none(args[1], "weight"), bias = tensor_or_none(args[2], "bias");
  const Tensor values = tensor_or_none(args[3], "values"), scales = tensor_or_none(args[4], "scales");
  refuse_tangents({&x, &weight, &bias});
  check_cuda(x);
  TORCH_CHECK_VALUE(x.dim() >= 1, "fp8_linear needs at least one dimension");
  const bool kept = !weight.defined();
  const int64_t n = kept ? PyLong_AsLongLong(args[5]) : weight.dim() == 2 ? weight.size(0) : 0;
  const int64_t k = kept ? PyLong_AsLongLong(args[6]) : weight.dim() == 2 ? weight.size(1) : 0;
  TORCH_CHECK_VALUE(n >= 1 && k >= 1 && x.size(-1) == k, "weight must be [out, ", x.size(-1), "], got [", n, ", ", k, "]");
  if (kept) {   // an Fp8Matrix, whose attributes may have been set since it was made
    TORCH_CHECK_VALUE(values.defined() && values.scalar_type() == at::kFloat8_e4m3fn && values.dim() == 2 &&
                          values.is_contiguous() && values.size(0) == n && values.size(1) >= k && values.size(1) % 16 == 0,
                      "values of a ", n, " x ", k, " Fp8Matrix must be contiguous float8_e4m3fn [rows, pitch], the pitch a "
                      "multiple of 16 and at least the columns");
    TORCH_CHECK_VALUE(scales.defined() && scales.scalar_type() == at::kByte && scales.is_contiguous() &&
                          scales.device() == values.device() && scales.numel() == p3d_fp8_scale_bytes(n, k),
                      "scales of a ", n, " x ", k, " Fp8Matrix must be ", p3d_fp8_scale_bytes(n, k),
                      " contiguous uint8 on the device of its values");
  }
  TORCH_CHECK_VALUE((kept ? values : weight).device() == x.device(), "x and weight must be on the same device");
  TORCH_CHECK_VALUE(kept || dtype_code(weight.scalar_type()) >= 0, "weight must be fp32, fp16 or bf16");
  if (bias.defined()) {
    TORCH_CHECK_VALUE(bias.dim() == 1 && bias.size(0) == n && bias.device() == x.device() &&
                          dtype_code(bias.scalar_type()) >= 0,
                      "bias must be ", n, " fp32, fp16 or bf16 values on the input's device");
    bias = bias.contiguous();
  }
  const bool grad = wants_grad({&x, &weight, &bias});
  TORCH_CHECK_VALUE(!(kept && grad),
                    "an 8-bit weight has no gradients: pass the weight itself, or call under torch.no_grad()");
  if (!kept) weight = weight.contiguous();
  const Tensor rows = (x.dim() == 2 ? x : x.reshape({x.numel() / k, k})).contiguous();
  Tensor y;
  if (rows.size(0) == 0) {
    // zero gradients for the weight and bias, as of an empty sum
    y = grad ? rows.matmul(weight.t().to(x.scalar_type())) : at::empty({0, n}, x.options());
    if (grad && bias.defined()) y = y + bias.to(x.scalar_type());
  } else if (grad) {
    y = Linear::apply(rows, weight, optional(bias));
  } else {
    p3d_fp8_linear a = linear_args(rows, n, weight, bias);
    if (kept) {
      a.weight_values = values.data_ptr();
      a.weight_scales = scales.data_ptr();
      a.weight_pitch = values.size(1);
    } else {
      a.weight = weight.data_ptr();
    }
    y = run_linear(a, rows, bias, nullptr);
  }
  if (x.dim() != 2) {
    std::vector<int64_t> shape = x.sizes().vec();
    shape.back() = n;
    y = y.view(shape);
  }
  return THPVariable_Wrap(y);
  END_HANDLE_TH_ERRORS
}

PyMethodDef g_methods[] = {
    {"dropout", (PyCFunction)(void (*)(void))py_dropout, METH_FASTCALL, "dropout(x, p, rng)"},
    {"norm", (PyCFunction)(void (*)(void))py_norm, METH_FASTCALL, "norm(x, spec)"},
    {"residual_norm", (PyCFunction)(void (*)(void))py_residual_norm, METH_FASTCALL,
     "residual_norm(x, h, post_norm, gate, gate_activation, scale, next_norm, p, rng)"},
    {"fp8_linear", (PyCFunction)(void (*)(void))py_fp8_linear, METH_FASTCALL,
     "fp8_linear(x, weight, bias, values, scales, rows, cols)"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "pack3d_b200_host", nullptr, -1, g_methods, nullptr, nullptr, nullptr,
                        nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject *PyInit_pack3d_b200_host() { return PyModule_Create(&g_module); }
