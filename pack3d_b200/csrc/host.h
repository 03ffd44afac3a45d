// What the files of the host module share: argument checks, autograd helpers, status codes to exceptions.
#pragma once

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

namespace p3d_host {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

constexpr int64_t kMaxDim = 16384;

// ------------------------------------------------------------------------------- arguments
inline int dtype_code(at::ScalarType t) {
  return t == at::kFloat ? P3D_F32 : t == at::kHalf ? P3D_F16 : t == at::kBFloat16 ? P3D_BF16 : -1;
}

inline Tensor tensor_or_none(PyObject *o, const char *what) {
  if (o == Py_None) return Tensor();
  TORCH_CHECK_VALUE(THPVariable_Check(o), what, " must be a tensor");
  return THPVariable_Unpack(o);
}
inline Tensor tensor(PyObject *o, const char *what) {
  TORCH_CHECK_VALUE(THPVariable_Check(o), what, " must be a tensor");
  return THPVariable_Unpack(o);
}
inline double number(PyObject *o, const char *what) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    TORCH_CHECK_VALUE(false, what, " must be a number");
  }
  return v;
}
inline bool is_word(PyObject *o, const char *word) {
  return PyUnicode_Check(o) && PyUnicode_CompareWithASCIIString(o, word) == 0;
}

inline void check_cuda(const Tensor &x) {
  TORCH_CHECK_VALUE(x.is_cuda() && dtype_code(x.scalar_type()) >= 0, "b200 backend requires CUDA fp32/fp16/bf16 tensors");
  TORCH_CHECK_VALUE(at::cuda::getDeviceProperties(x.device().index())->major == 10,
                    "b200 backend targets compute capability 10.x (sm_100a) devices");
}
inline void check_input(const Tensor &x, const char *what) {
  TORCH_CHECK_VALUE(x.dim() >= 1, what, " needs at least one dimension");
  check_cuda(x);
  TORCH_CHECK_VALUE(x.size(-1) >= 1 && x.size(-1) <= kMaxDim, what, ": the last dimension must be 1 to ", kMaxDim, ", got ",
                    x.size(-1));
}
inline void check_vector(const Tensor &t, const Tensor &x, const char *what) {
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
inline Spec spec_of(PyObject *o, const Tensor &x, const char *what) {
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

inline uint32_t threshold_of(PyObject *o) {
  const double p = number(o, "dropout probability");
  TORCH_CHECK_VALUE(p >= 0.0 && p <= 1.0, "dropout probability must lie between 0 and 1");
  return (uint32_t)std::nearbyint(65536.0 * p);   // ties to even, as Python's round
}

// (seed, offset), or an int64 tensor of the two on the input's device.
struct Rng {
  Tensor tensor;
  uint64_t seed = 0, offset = 0;
};
inline Rng rng_of(PyObject *o, const Tensor &x) {
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

inline const void *ptr(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }
inline void *out_ptr(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }
inline void *stream() { return at::cuda::getCurrentCUDAStream().stream(); }

inline void check_status(int status, const char *what) {
  if (status == P3D_OK) return;
  const std::string text = std::string(what) + ": " + p3d_strerror(status) + ": " + p3d_last_error();
  TORCH_CHECK_VALUE(status != P3D_ERR_INVALID_ARGUMENT && status != P3D_ERR_UNSUPPORTED, text);
  TORCH_CHECK(false, text);
}

// What a backward pass returns cannot be differentiated again: where its own upstream gradients ask for that, the
// results carry an error for whoever tries.
inline variable_list once(variable_list grads, const variable_list &up) {
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
inline Optional optional(const Tensor &t) { return t.defined() ? Optional(t) : Optional(); }
inline Tensor value(const Optional &t) { return t ? *t : Tensor(); }

inline bool wants_grad(std::initializer_list<const Tensor *> tensors) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor *t : tensors)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

// Forward-mode derivatives are not there: a tangent is refused, whether or not the tensor takes part in reverse mode too, as
// a result without one would read as a zero derivative.
inline void refuse_tangents(std::initializer_list<const Tensor *> tensors) {
  for (const Tensor *t : tensors)
    TORCH_CHECK_NOT_IMPLEMENTED(!(t->defined() && t->_fw_grad(0).defined()),
                                "forward-mode derivatives of this operator are not implemented");
}

// While a graph of a leaf that was recorded on the default stream lives, its gradient is added up on that stream, which a backward
// pass under capture cannot reach: PyTorch then fails outside of any exception handler. So the forward pass is refused.
inline void refuse_live_graph(std::initializer_list<const Tensor *> tensors) {
  if (c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None) return;
  for (const Tensor *t : tensors) {
    if (!t->defined() || !t->is_leaf() || !t->requires_grad()) continue;
    const auto node = torch::autograd::impl::try_get_grad_accumulator(*t);
    const auto stream = node ? node->stream() : std::nullopt;
    TORCH_CHECK_VALUE(!stream || *stream != c10::cuda::getDefaultCUDAStream(stream->device_index()).unwrap(),
                      "a graph recorded on the default stream still holds this input's gradient: drop its results before "
                      "the capture, or record it on another stream");
  }
}

// host_sequence.cpp
extern PyMethodDef g_sequence_methods[];

}  // namespace p3d_host
