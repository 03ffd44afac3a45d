// The host side of norm_rotate, sequence_attention, the paged cache and paged_attention, as host.cpp for the row operators:
// called with positional arguments by pack3d_b200.sequence and pack3d_b200.cache, whose docstrings describe them.
#include <torch/csrc/DynamicTypes.h>
#include <torch/csrc/autograd/variable.h>

#include "host.h"

namespace p3d_host {
namespace {

// ------------------------------------------------------------------------------- arguments
PyObject *pair_of(const Tensor &a, const Tensor &b) {
  PyObject *pair = PyTuple_New(2);
  if (!pair) throw python_error();
  const Tensor *t[2] = {&a, &b};
  for (int i = 0; i < 2; ++i) {
    PyObject *o = Py_None;
    if (t[i]->defined()) o = THPVariable_Wrap(*t[i]);
    else Py_INCREF(o);
    PyTuple_SET_ITEM(pair, i, o);
  }
  return pair;
}

bool flag(PyObject *o, const char *what) {
  TORCH_CHECK_VALUE(PyBool_Check(o), what, " must be True or False");
  return o == Py_True;
}

// Rows of dim consecutive elements, 16-byte aligned with strides to match: as it is, or a copy. Rows that share memory are
// copied too: a tensor map has no stride of 0.
Tensor rows16(const Tensor &t) {
  const int64_t unit = 16 / t.element_size();
  bool fits = t.size(-1) == 1 || t.stride(-1) == 1;
  for (int64_t i = 0; i + 1 < t.dim(); ++i)
    fits = fits && (t.size(i) <= 1 || (t.stride(i) % unit == 0 && t.stride(i) > 0 && t.stride(i) < 1ll << 38));
  if (fits && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0) return t;
  return t.is_contiguous() ? t.clone(at::MemoryFormat::Contiguous) : t.contiguous();
}
int64_t stride_of(const Tensor &t, int64_t i) { return t.size(i) <= 1 ? 0 : t.stride(i); }

Tensor whole_numbers(PyObject *o, const Tensor &x, int64_t dims, const char *what) {
  const Tensor t = tensor(o, what);
  TORCH_CHECK_VALUE(t.scalar_type() == at::kInt && t.dim() == dims && t.device() == x.device(), what, " must be int32, ", dims,
                    dims == 1 ? " dimension" : " dimensions", ", on the input's device");
  return t.contiguous();
}

void check_16bit(const Tensor &x, const char *what) {
  check_cuda(x);
  TORCH_CHECK_VALUE(x.scalar_type() == at::kHalf || x.scalar_type() == at::kBFloat16, what, " needs fp16 or bf16 tensors, got ",
                    x.scalar_type());
}

void no_gradients(std::initializer_list<const Tensor *> tensors, const char *what) {
  TORCH_CHECK_VALUE(!wants_grad(tensors), what, " has no gradients: detach its inputs, or call under torch.no_grad()");
}

double positive(PyObject *o, const char *what) {
  const double v = number(o, what);
  TORCH_CHECK_VALUE(std::isfinite(v) && v > 0, what, " must be finite and positive");
  return v;
}

// ------------------------------------------------------------------------------- norms with rotation
enum : int { kQ, kK, kQW, kQB, kKW, kKB, kTensors };
struct Rotation {
  p3d_norm_rotate args = {};
  Tensor t[kTensors], positions;
  void address() {
    for (int i = 0; i < 2; ++i) {
      const Tensor &x = t[kQ + i];
      args.x[i] = ptr(x);
      if (x.defined()) {
        args.token_stride[i] = stride_of(x, 0);
        args.head_stride[i] = stride_of(x, 1);
      }
      args.weight[i] = ptr(t[kQW + 2 * i]);
      args.bias[i] = ptr(t[kQB + 2 * i]);
    }
    args.positions = ptr(positions);
  }
};

variable_list run_rotate(Rotation &r) {
  const Tensor &q = r.t[kQ], &k = r.t[kK];
  const c10::cuda::CUDAGuard guard(q.device());
  variable_list y = {at::empty(q.sizes(), q.options())};
  if (k.defined()) y.push_back(at::empty(k.sizes(), k.options()));
  r.address();
  check_status(p3d_norm_rotate_fwd(&r.args, y[0].data_ptr(), k.defined() ? y[1].data_ptr() : nullptr, stream()),
               "p3d_norm_rotate_fwd");
  return y;
}

struct NormRotate : torch::autograd::Function<NormRotate> {
  static variable_list forward(AutogradContext *ctx, const p3d_norm_rotate &args, const Tensor &positions, const Optional &q,
                               const Optional &k, const Optional &qw, const Optional &qb, const Optional &kw,
                               const Optional &kb) {
    ctx->set_materialize_grads(false);
    Rotation r;
    r.args = args;
    r.positions = positions;
    const Optional *given[kTensors] = {&q, &k, &qw, &qb, &kw, &kb};
    for (int i = 0; i < kTensors; ++i) r.t[i] = value(*given[i]);
    variable_list saved = {positions};
    saved.insert(saved.end(), r.t, r.t + kTensors);
    ctx->save_for_backward(std::move(saved));
    ctx->saved_data["args"] = std::string(reinterpret_cast<const char *>(&args), sizeof(args));
    return run_rotate(r);
  }
  static variable_list backward(AutogradContext *ctx, variable_list up) {
    const variable_list saved = ctx->get_saved_variables();
    Rotation r;
    memcpy(&r.args, ctx->saved_data["args"].toStringRef().data(), sizeof(r.args));
    r.positions = saved[0];
    for (int i = 0; i < kTensors; ++i) r.t[i] = saved[1 + i];
    const bool two = r.t[kK].defined();
    variable_list grads(2 + kTensors);
    if (!up[0].defined() && !(two && up[1].defined())) return grads;
    Tensor dy[2];
    for (int i = 0; i < 1 + two; ++i) {
      refuse_tangents({&up[i]});
      dy[i] = up[i].defined() ? up[i].detach().contiguous() : at::zeros(r.t[i].sizes(), r.t[i].options());
    }
    const c10::cuda::CUDAGuard guard(r.t[kQ].device());
    Tensor *d = grads.data() + 2;
    size_t edge = 1;   // positions have the first
    for (int i = 0; i < kTensors; ++i)
      if (r.t[i].defined() && ctx->needs_input_grad(edge++))
        d[i] = r.args.tokens ? at::empty(r.t[i].sizes(), r.t[i].options()) : at::zeros(r.t[i].sizes(), r.t[i].options());
    r.address();
    const size_t need = p3d_norm_rotate_bwd_workspace(&r.args);
    const Tensor ws = at::empty({(int64_t)need}, r.t[kQ].options().dtype(at::kByte));
    const void *dys[2] = {ptr(dy[0]), ptr(dy[1])};
    void *dx[2] = {out_ptr(d[kQ]), out_ptr(d[kK])}, *dw[2] = {out_ptr(d[kQW]), out_ptr(d[kKW])},
         *db[2] = {out_ptr(d[kQB]), out_ptr(d[kKB])};
    check_status(p3d_norm_rotate_bwd(&r.args, dys, dx, dw, db, ws.data_ptr(), need, stream()), "p3d_norm_rotate_bwd");
    return once(std::move(grads), up);
  }
};

// [.., heads, dim] as [tokens, heads, dim] with the dim columns consecutive.
Tensor head_rows(const Tensor &x) {
  const int64_t heads = x.size(-2), dim = x.size(-1), tokens = x.numel() / std::max<int64_t>(1, heads * dim);
  Tensor rows = x.dim() == 3 ? x : x.reshape({tokens, heads, dim});
  return dim == 1 || rows.stride(2) == 1 ? rows : rows.contiguous();
}

PyObject *py_norm_rotate(PyObject *, PyObject *const *args, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_VALUE(count == 7, "norm_rotate takes q, k, positions, q_norm, k_norm, pairs, base");
  const Tensor q = tensor(args[0], "q"), k = tensor_or_none(args[1], "k");
  refuse_tangents({&q, &k});
  check_cuda(q);
  TORCH_CHECK_VALUE(q.dim() >= 3 && q.size(-2) >= 1, "q must have shape [.., tokens, heads, head_dim]");
  const int64_t dim = q.size(-1);
  TORCH_CHECK_VALUE(dim >= 2 && dim <= 256 && dim % 2 == 0, "norm_rotate: the head dim must be even, 2 to 256, got ", dim);
  if (k.defined())
    TORCH_CHECK_VALUE(k.dim() == q.dim() && k.size(-1) == dim && k.size(-2) >= 1 && k.scalar_type() == q.scalar_type() &&
                          k.device() == q.device() && k.sizes().slice(0, k.dim() - 2) == q.sizes().slice(0, q.dim() - 2),
                      "k must have the shape of q up to its heads, and q's dtype and device");
  Tensor positions = tensor(args[2], "positions");
  TORCH_CHECK_VALUE((positions.scalar_type() == at::kInt || positions.scalar_type() == at::kLong) &&
                        positions.device() == q.device() && (positions.dim() == 1 || positions.dim() == 2) &&
                        positions.size(0) == q.size(-3) && (positions.dim() == 1 || (positions.size(1) >= 1 && positions.size(1) <= 3)),
                    "positions must be int32 or int64 [", q.size(-3), "] or [", q.size(-3),
                    ", 1 to 3 axes] on the input's device");
  const Spec qs = spec_of(args[3], q, "q_norm"), ks = k.defined() ? spec_of(args[4], k, "k_norm") : Spec();
  TORCH_CHECK_VALUE(k.defined() || args[4] == Py_None, "k_norm without k");
  Rotation r;
  p3d_norm_rotate &a = r.args;
  a.axes = positions.dim() == 1 ? 1 : (int32_t)positions.size(1);
  int64_t total = 0;
  if (args[5] == Py_None) {
    for (int i = 0; i < a.axes; ++i) a.pairs[i] = (int32_t)(dim / 2 / a.axes + (i < dim / 2 % a.axes ? 1 : 0));
  } else {
    const bool fits = (PyTuple_Check(args[5]) || PyList_Check(args[5])) && PySequence_Fast_GET_SIZE(args[5]) == a.axes;
    TORCH_CHECK_VALUE(fits, "pairs must be a number of rotated pairs for each of ", a.axes, " axes");
    for (int i = 0; i < a.axes; ++i) {
      PyObject *o = PySequence_Fast_GET_ITEM(args[5], i);
      const long long v = PyLong_Check(o) ? PyLong_AsLongLong(o) : -1;
      if (PyErr_Occurred()) PyErr_Clear();
      TORCH_CHECK_VALUE(v >= 0 && v <= dim / 2, "pairs must be whole numbers from 0 to half the head dim");
      a.pairs[i] = (int32_t)v;
      total += v;
    }
    TORCH_CHECK_VALUE(2 * total <= dim, "pairs take ", 2 * total, " of ", dim, " columns");
  }
  a.base = number(args[6], "base");
  TORCH_CHECK_VALUE(std::isfinite(a.base) && a.base >= 1, "base must be at least 1");
  r.t[kQ] = head_rows(q);
  if (k.defined()) r.t[kK] = head_rows(k);
  a.tokens = r.t[kQ].size(0);
  a.position_rows = positions.size(0);
  a.heads[0] = (int32_t)q.size(-2);
  a.heads[1] = k.defined() ? (int32_t)k.size(-2) : 0;
  a.dim = (int32_t)dim;
  a.dtype = dtype_code(q.scalar_type());
  a.position_bytes = positions.scalar_type() == at::kInt ? 4 : 8;
  a.position_stride = positions.stride(0);
  a.axis_stride = positions.dim() == 2 ? positions.stride(1) : 0;
  r.positions = positions;
  const Spec *specs[2] = {&qs, &ks};
  bool grad = wants_grad({&r.t[kQ], &r.t[kK]});
  for (int i = 0; i < 2; ++i) {
    Tensor w = specs[i]->weight, b = specs[i]->bias;
    refuse_tangents({&w, &b});
    if (w.defined() && b.defined() && w.scalar_type() != b.scalar_type()) {
      w = w.to(at::kFloat);
      b = b.to(at::kFloat);
    }
    const Tensor &any = w.defined() ? w : b;
    a.kind[i] = specs[i]->kind;
    a.eps[i] = specs[i]->eps;
    a.param_dtype[i] = any.defined() ? dtype_code(any.scalar_type()) : a.dtype;
    if (w.defined()) r.t[kQW + 2 * i] = w.contiguous();
    if (b.defined()) r.t[kQB + 2 * i] = b.contiguous();
    grad = grad || wants_grad({&w, &b});
  }
  variable_list y;
  if (grad) refuse_live_graph({&q, &k, &qs.weight, &qs.bias, &ks.weight, &ks.bias});
  if (grad)
    y = NormRotate::apply(a, r.positions, optional(r.t[kQ]), optional(r.t[kK]), optional(r.t[kQW]), optional(r.t[kQB]),
                          optional(r.t[kKW]), optional(r.t[kKB]));
  else
    y = run_rotate(r);
  if (q.dim() != 3)
    for (size_t i = 0; i < y.size(); ++i) y[i] = y[i].view(i ? k.sizes() : q.sizes());
  return pair_of(y[0], k.defined() ? y[1] : Tensor());
  END_HANDLE_TH_ERRORS
}

// ------------------------------------------------------------------------------- packed sequences
struct Sequence {
  p3d_sequence args = {};
  Tensor q, k, v, q_offsets, k_offsets;
  void address() {
    args.q = ptr(q), args.k = ptr(k), args.v = ptr(v);
    args.q_offsets = static_cast<const int32_t *>(ptr(q_offsets));
    args.k_offsets = static_cast<const int32_t *>(ptr(k_offsets));
    for (int i = 0; i < 2; ++i) {
      args.q_stride[i] = stride_of(q, i);
      args.k_stride[i] = stride_of(k, i);
      args.v_stride[i] = stride_of(v, i);
    }
  }
};

Tensor run_sequence(Sequence &s, Tensor *lse) {
  const c10::cuda::CUDAGuard guard(s.q.device());
  const Tensor out = at::empty(s.q.sizes(), s.q.options());
  if (lse) *lse = at::empty({s.q.size(1), s.q.size(0)}, s.q.options().dtype(at::kFloat));
  s.address();
  check_status(p3d_sequence_fwd(&s.args, out.data_ptr(), lse ? static_cast<float *>(lse->data_ptr()) : nullptr, stream()),
               "p3d_sequence_fwd");
  return out;
}

struct SequenceAttention : torch::autograd::Function<SequenceAttention> {
  static Tensor forward(AutogradContext *ctx, const p3d_sequence &args, const Tensor &q, const Tensor &k, const Tensor &v,
                        const Tensor &q_offsets, const Tensor &k_offsets) {
    Sequence s = {args, q, k, v, q_offsets, k_offsets};
    Tensor lse;
    const Tensor out = run_sequence(s, &lse);
    ctx->save_for_backward({q, k, v, q_offsets, k_offsets, out, lse});
    ctx->saved_data["args"] = std::string(reinterpret_cast<const char *>(&args), sizeof(args));
    return out;
  }
  static variable_list backward(AutogradContext *ctx, variable_list up) {
    const variable_list saved = ctx->get_saved_variables();
    Sequence s = {{}, saved[0], saved[1], saved[2], saved[3], saved[4]};
    memcpy(&s.args, ctx->saved_data["args"].toStringRef().data(), sizeof(s.args));
    refuse_tangents({&up[0]});
    const c10::cuda::CUDAGuard guard(s.q.device());
    Tensor d[3];
    const Tensor *x[3] = {&s.q, &s.k, &s.v};
    bool any = false;
    for (int i = 0; i < 3; ++i)
      if (ctx->needs_input_grad(i)) {
        d[i] = at::empty(x[i]->sizes(), x[i]->options());
        any = true;
      }
    if (any) {
      const Tensor dout = rows16(up[0].detach().contiguous());
      s.address();
      const size_t need = p3d_sequence_bwd_workspace(&s.args);
      const Tensor ws = at::empty({(int64_t)need}, s.q.options().dtype(at::kByte));
      check_status(p3d_sequence_bwd(&s.args, saved[5].data_ptr(), static_cast<const float *>(saved[6].data_ptr()),
                                    dout.data_ptr(), out_ptr(d[0]), out_ptr(d[1]), out_ptr(d[2]), ws.data_ptr(), need,
                                    stream()),
                   "p3d_sequence_bwd");
    }
    return once({Tensor(), d[0], d[1], d[2], Tensor(), Tensor()}, up);
  }
};

PyObject *py_sequence_attention(PyObject *, PyObject *const *args, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_VALUE(count == 7, "sequence_attention takes q, k, v, q_offsets, k_offsets, causal, scale");
  Sequence s;
  s.q = tensor(args[0], "q"), s.k = tensor(args[1], "k"), s.v = tensor(args[2], "v");
  refuse_tangents({&s.q, &s.k, &s.v});
  check_16bit(s.q, "sequence_attention");
  TORCH_CHECK_VALUE(s.q.dim() == 3 && s.k.dim() == 3 && s.v.sizes() == s.k.sizes(),
                    "q must be [rows, heads, head_dim], k and v [rows, kv_heads, head_dim]");
  const int64_t dim = s.q.size(2);
  TORCH_CHECK_VALUE(s.k.size(2) == dim && dim >= 8 && dim <= 128 && dim % 8 == 0,
                    "q, k and v must have one head dim, a multiple of 8 up to 128, got ", dim, " and ", s.k.size(2));
  TORCH_CHECK_VALUE(s.q.size(1) >= 1 && s.k.size(1) >= 1 && s.q.size(1) % s.k.size(1) == 0,
                    "query heads must be divisible by KV heads, got ", s.q.size(1), " and ", s.k.size(1));
  for (const Tensor *t : {&s.k, &s.v})
    TORCH_CHECK_VALUE(t->scalar_type() == s.q.scalar_type() && t->device() == s.q.device(),
                      "q, k and v must have the same dtype and device");
  s.q_offsets = whole_numbers(args[3], s.q, 1, "q_offsets");
  s.k_offsets = args[4] == Py_None ? s.q_offsets : whole_numbers(args[4], s.q, 1, "k_offsets");
  TORCH_CHECK_VALUE(args[4] != Py_None || s.k.size(0) == s.q.size(0), "keys of other lengths than the queries need k_offsets");
  TORCH_CHECK_VALUE(s.q_offsets.size(0) >= 2 && s.k_offsets.size(0) == s.q_offsets.size(0),
                    "offsets must be [sequences + 1], as many for the keys as for the queries, at least one sequence");
  p3d_sequence &a = s.args;
  a.causal = flag(args[5], "causal");
  a.scale = args[6] == Py_None ? (float)(1.0 / std::sqrt((double)dim)) : (float)positive(args[6], "scale");
  a.q_rows = s.q.size(0), a.k_rows = s.k.size(0);
  a.sequences = (int32_t)(s.q_offsets.size(0) - 1);
  a.heads = (int32_t)s.q.size(1), a.kv_heads = (int32_t)s.k.size(1), a.dim = (int32_t)dim;
  a.dtype = dtype_code(s.q.scalar_type());
  const bool grad = wants_grad({&s.q, &s.k, &s.v});
  if (grad) refuse_live_graph({&s.q, &s.k, &s.v});
  s.q = rows16(s.q), s.k = rows16(s.k), s.v = rows16(s.v);
  if (grad) return THPVariable_Wrap(SequenceAttention::apply(a, s.q, s.k, s.v, s.q_offsets, s.k_offsets));
  return THPVariable_Wrap(run_sequence(s, nullptr));
  END_HANDLE_TH_ERRORS
}

// ------------------------------------------------------------------------------- paged cache
// k, v, k_scales, v_scales, table: the cache's tensors (whose attributes may have been set since it was made) and a page table.
struct Pages {
  p3d_cache c = {};
  Tensor k, v, k_scales, v_scales, table;
};
Pages pages_of(PyObject *const *args) {
  Pages p;
  p.k = tensor(args[0], "k"), p.v = tensor(args[1], "v");
  p.k_scales = tensor_or_none(args[2], "k_scales"), p.v_scales = tensor_or_none(args[3], "v_scales");
  const bool bits8 = p.k.scalar_type() == at::kFloat8_e4m3fn;
  TORCH_CHECK_VALUE(p.k.is_cuda() && (bits8 || dtype_code(p.k.scalar_type()) >= 0),
                    "b200 backend requires CUDA fp32/fp16/bf16 or float8_e4m3fn pages");
  TORCH_CHECK_VALUE(at::cuda::getDeviceProperties(p.k.device().index())->major == 10,
                    "b200 backend targets compute capability 10.x (sm_100a) devices");
  TORCH_CHECK_VALUE(p.k.dim() == 4 && p.v.sizes() == p.k.sizes() && p.v.scalar_type() == p.k.scalar_type() &&
                        p.v.device() == p.k.device() && p.k.is_contiguous() && p.v.is_contiguous(),
                    "pages must be two contiguous tensors [pages, kv_heads, page_size, head_dim] of one dtype and device");
  TORCH_CHECK_VALUE(!p.k.requires_grad() && !p.v.requires_grad(), "pages have no gradients");
  if (bits8)
    for (const Tensor *t : {&p.k_scales, &p.v_scales})
      TORCH_CHECK_VALUE(t->defined() && t->scalar_type() == at::kByte && t->is_contiguous() && t->device() == p.k.device() &&
                            t->sizes() == p.k.sizes().slice(0, 3),
                        "8-bit pages need contiguous uint8 scales [pages, kv_heads, page_size] on their device");
  p.table = whole_numbers(args[4], p.k, 2, "table");
  p3d_cache &c = p.c;
  for (int i = 1; i < 4; ++i) TORCH_CHECK_VALUE(p.k.size(i) >= 1 && p.k.size(i) < (1ll << 30), "pages must not be empty");
  c.k = p.k.data_ptr(), c.v = p.v.data_ptr();
  c.k_scales = bits8 ? static_cast<uint8_t *>(p.k_scales.data_ptr()) : nullptr;
  c.v_scales = bits8 ? static_cast<uint8_t *>(p.v_scales.data_ptr()) : nullptr;
  c.table = static_cast<const int32_t *>(ptr(p.table));
  c.pages = p.k.size(0);
  c.kv_heads = (int32_t)p.k.size(1), c.page_size = (int32_t)p.k.size(2), c.dim = (int32_t)p.k.size(3);
  c.dtype = bits8 ? P3D_E4M3 : dtype_code(p.k.scalar_type());
  TORCH_CHECK_VALUE(p.table.size(0) < (1ll << 30) && p.table.size(1) < (1ll << 30), "page table too large");
  c.sequences = (int32_t)p.table.size(0), c.table_width = (int32_t)p.table.size(1);
  c.table_stride = p.table.size(1);
  return p;
}

Tensor per_sequence(PyObject *o, const Pages &p, int64_t more, const char *what) {
  const Tensor t = whole_numbers(o, p.k, 1, what);
  TORCH_CHECK_VALUE(t.size(0) == p.table.size(0) + more, what, " must hold ", p.table.size(0) + more, " values for a table of ",
                    p.table.size(0), " sequences, got ", t.size(0));
  return t;
}
const int32_t *ints(const Tensor &t) { return static_cast<const int32_t *>(ptr(t)); }

PyObject *py_cache_append(PyObject *, PyObject *const *args, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_VALUE(count == 9, "cache_append takes k, v, k_scales, v_scales, table, new_k, new_v, starts, offsets");
  const Pages p = pages_of(args);
  Tensor nk = tensor(args[5], "k"), nv = tensor(args[6], "v");
  refuse_tangents({&nk, &nv});
  no_gradients({&nk, &nv}, "append");
  TORCH_CHECK_VALUE(nk.dim() == 3 && nv.sizes() == nk.sizes() && nk.size(1) == p.k.size(1) && nk.size(2) == p.k.size(3),
                    "new k and v must be [rows, ", p.k.size(1), ", ", p.k.size(3), "], got ", nk.sizes(), " and ", nv.sizes());
  TORCH_CHECK_VALUE(nv.scalar_type() == nk.scalar_type() && nk.device() == p.k.device() && nv.device() == p.k.device() &&
                        (p.c.dtype == P3D_E4M3 ? dtype_code(nk.scalar_type()) >= 0 : nk.scalar_type() == p.k.scalar_type()),
                    "new k and v must be on the cache's device, of its dtype (fp32, fp16 or bf16 for an 8-bit cache)");
  const Tensor starts = per_sequence(args[7], p, 0, "lengths"), offsets = per_sequence(args[8], p, 1, "offsets");
  const c10::cuda::CUDAGuard guard(p.k.device());
  nk = rows16(nk), nv = rows16(nv);
  const int64_t ks[2] = {stride_of(nk, 0), stride_of(nk, 1)}, vs[2] = {stride_of(nv, 0), stride_of(nv, 1)};
  check_status(p3d_cache_append(&p.c, ptr(nk), ks, ptr(nv), vs, dtype_code(nk.scalar_type()), nk.size(0), ints(starts),
                                ints(offsets), stream()),
               "p3d_cache_append");
  for (const Tensor *t : {&p.k, &p.v, &p.k_scales, &p.v_scales})
    if (t->defined() && !t->is_inference()) torch::autograd::impl::bump_version(*t);
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

PyObject *py_cache_read(PyObject *, PyObject *const *args, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_VALUE(count == 9, "cache_read takes k, v, k_scales, v_scales, table, starts, offsets, rows, dtype");
  const Pages p = pages_of(args);
  const Tensor starts = args[5] == Py_None ? Tensor() : per_sequence(args[5], p, 0, "starts");
  const Tensor offsets = per_sequence(args[6], p, 1, "offsets");
  const long long rows = PyLong_Check(args[7]) ? PyLong_AsLongLong(args[7]) : -1;
  if (PyErr_Occurred()) PyErr_Clear();
  TORCH_CHECK_VALUE(rows >= 0 && rows < (1ll << 31) - 64, "rows must be a whole number, 0 to 2^31 - 65");
  TORCH_CHECK_VALUE(args[8] == Py_None || THPDtype_Check(args[8]), "dtype must be fp32, fp16 or bf16");
  const at::ScalarType type = args[8] == Py_None
                                  ? (p.c.dtype == P3D_E4M3 ? at::kBFloat16 : p.k.scalar_type())
                                  : reinterpret_cast<THPDtype *>(args[8])->scalar_type;
  TORCH_CHECK_VALUE(dtype_code(type) >= 0, "dtype must be fp32, fp16 or bf16");
  const c10::cuda::CUDAGuard guard(p.k.device());
  const Tensor k = at::empty({rows, p.k.size(1), p.k.size(3)}, p.k.options().dtype(type)), v = at::empty_like(k);
  if (p.table.size(0) == 0) {
    k.zero_();
    v.zero_();
  } else {
    check_status(p3d_cache_read(&p.c, ints(starts), ints(offsets), rows, out_ptr(k), out_ptr(v), dtype_code(type), stream()),
                 "p3d_cache_read");
  }
  return pair_of(k, v);
  END_HANDLE_TH_ERRORS
}

PyObject *py_paged_attention(PyObject *, PyObject *const *args, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_VALUE(count == 8, "paged_attention takes k, v, k_scales, v_scales, table, q, lengths, scale");
  const Pages p = pages_of(args);
  Tensor q = tensor(args[5], "q");
  refuse_tangents({&q});
  no_gradients({&q}, "paged_attention");
  check_16bit(q, "paged_attention");
  TORCH_CHECK_VALUE(q.dim() == 3 && q.size(0) == p.table.size(0) && q.size(2) == p.k.size(3) && q.device() == p.k.device(),
                    "q must be [", p.table.size(0), ", heads, ", p.k.size(3), "] on the cache's device, got ", q.sizes());
  TORCH_CHECK_VALUE(p.c.dtype == P3D_E4M3 || q.scalar_type() == p.k.scalar_type(), "q must have the cache's dtype");
  TORCH_CHECK_VALUE(q.size(1) >= 1 && q.size(1) % p.k.size(1) == 0, "query heads must be divisible by KV heads, got ", q.size(1),
                    " and ", p.k.size(1));
  const Tensor lengths = per_sequence(args[6], p, 0, "lengths");
  const float scale = args[7] == Py_None ? (float)(1.0 / std::sqrt((double)q.size(2))) : (float)positive(args[7], "scale");
  const c10::cuda::CUDAGuard guard(p.k.device());
  q = rows16(q);
  const Tensor out = at::empty(q.sizes(), q.options());
  const int64_t strides[2] = {stride_of(q, 0), stride_of(q, 1)};
  const size_t need = p3d_paged_attention_workspace(&p.c, (int)q.size(1));
  const Tensor ws = at::empty({(int64_t)need}, q.options().dtype(at::kByte));
  check_status(p3d_paged_attention(&p.c, ptr(q), strides, dtype_code(q.scalar_type()), (int)q.size(1), ints(lengths), scale,
                                   out_ptr(out), ws.data_ptr(), need, stream()),
               "p3d_paged_attention");
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

#define METHOD(name, doc) {#name, (PyCFunction)(void (*)(void))py_##name, METH_FASTCALL, doc}
}  // namespace

PyMethodDef g_sequence_methods[] = {
    METHOD(norm_rotate, "norm_rotate(q, k, positions, q_norm, k_norm, pairs, base)"),
    METHOD(sequence_attention, "sequence_attention(q, k, v, q_offsets, k_offsets, causal, scale)"),
    METHOD(cache_append, "cache_append(k, v, k_scales, v_scales, table, new_k, new_v, starts, offsets)"),
    METHOD(cache_read, "cache_read(k, v, k_scales, v_scales, table, starts, offsets, rows, dtype)"),
    METHOD(paged_attention, "paged_attention(k, v, k_scales, v_scales, table, q, lengths, scale)"),
    {nullptr, nullptr, 0, nullptr}};
#undef METHOD

}  // namespace p3d_host
