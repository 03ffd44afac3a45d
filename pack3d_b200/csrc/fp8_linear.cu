// A linear layer in 8-bit blocks as one call a direction: quantisers and products of fp8.cu and
// fp8_gemm.cu over one workspace, so that a layer costs its caller two allocations and one call.
//
// forward   y = Q(x) Q(w)^T + bias; keeps x with blocks along its rows and w transposed, both in 8 bits
// backward  dx = Q(dy) Q(w); dw = Q(dy)^T Q(x), blocks along the rows; dbias = the column sums of dy,
//           taken while dy is quantised
#include "common.cuh"
#include "kernels.cuh"

namespace p3d {
namespace {

int64_t pitch_of(int64_t cols) { return (cols + 15) / 16 * 16; }

// Pieces of a buffer, 256 bytes apart at least; with no buffer only the size is counted.
struct Pieces {
  char *base;
  size_t used = 0;
  void *take(size_t bytes) {
    void *at = base ? base + used : nullptr;
    used += (bytes + 255) / 256 * 256;
    return at;
  }
};

struct Matrix {   // [rows, cols] in 8 bits
  int64_t rows, cols, pitch;
  void *values, *scales;
};
Matrix take_matrix(Pieces &p, int64_t rows, int64_t cols) {
  Matrix m{rows, cols, pitch_of(cols), nullptr, nullptr};
  m.values = p.take((size_t)(rows * m.pitch));
  m.scales = p.take((size_t)p3d_fp8_scale_bytes(rows, cols));
  return m;
}

struct Saved {
  Matrix xt, wt;   // [k, rows], [k, n]; empty where their gradient is not wanted
  size_t bytes;
};
Saved saved_of(const p3d_fp8_linear &a, void *buffer) {
  Pieces p{static_cast<char *>(buffer)};
  Saved s = {};
  if (a.need_dw) s.xt = take_matrix(p, a.k, a.rows);
  if (a.need_dx) s.wt = take_matrix(p, a.k, a.n);
  s.bytes = p.used;
  return s;
}

struct Forward {
  Matrix x, w;
  void *sums;
  size_t sum_bytes, bytes;
};
// Few tokens without a gradient of the weight are quantised inside their product.
bool in_product(const p3d_fp8_linear &a) { return !a.need_dw && fp8_tokens_fit(a.rows, a.n, a.k); }
Forward forward_of(const p3d_fp8_linear &a, void *buffer) {
  Pieces p{static_cast<char *>(buffer)};
  Forward f = {};
  if (!in_product(a)) f.x = take_matrix(p, a.rows, a.k);
  if (a.weight) f.w = take_matrix(p, a.n, a.k);
  f.sum_bytes = p3d_fp8_matmul_workspace(a.rows, a.n, a.k);
  f.sums = p.take(f.sum_bytes);
  f.bytes = p.used;
  return f;
}

struct Backward {
  Matrix dy, dyt;
  void *columns, *sums;
  size_t column_bytes, sum_bytes, bytes;
};
Backward backward_of(const p3d_fp8_linear &a, bool bias, void *buffer) {
  Pieces p{static_cast<char *>(buffer)};
  Backward b = {};
  if (a.need_dx) b.dy = take_matrix(p, a.rows, a.n);
  if (a.need_dw) b.dyt = take_matrix(p, a.n, a.rows);
  b.column_bytes = bias ? p3d_fp8_quantize_workspace(a.rows, a.n) : 0;
  b.columns = p.take(b.column_bytes);
  size_t dx = 0, dw = 0;   // one after the other
  if (a.need_dx) dx = p3d_fp8_matmul_workspace(a.rows, a.k, a.n);
  if (a.need_dw) dw = p3d_fp8_matmul_workspace(a.n, a.k, a.rows);
  b.sum_bytes = dx > dw ? dx : dw;
  b.sums = p.take(b.sum_bytes);
  b.bytes = p.used;
  return b;
}

int check(const p3d_fp8_linear *a, const char *what) {
  P3D_CHECK_ARG(a != nullptr, "%s: null arguments", what);
  P3D_CHECK_ARG(a->rows >= 1 && a->k >= 1 && a->n >= 1, "%s: extents must be positive", what);
  // sizes of buffers stay far below 2^63
  const int64_t most = (int64_t)1 << 30;
  if (a->rows > most || a->k > most || a->n > most) return fail(P3D_ERR_UNSUPPORTED, "%s: extents too large", what);
  P3D_CHECK_ARG(dtype_ok(a->dtype) && dtype_ok(a->weight_dtype) && dtype_ok(a->bias_dtype), "%s: unknown dtype", what);
  return P3D_OK;
}

}  // namespace
}  // namespace p3d

using namespace p3d;

extern "C" size_t p3d_fp8_linear_saved(const p3d_fp8_linear *a) {
  return check(a, "p3d_fp8_linear_saved") ? 0 : saved_of(*a, nullptr).bytes;
}
extern "C" size_t p3d_fp8_linear_fwd_workspace(const p3d_fp8_linear *a) {
  return check(a, "p3d_fp8_linear_fwd_workspace") ? 0 : forward_of(*a, nullptr).bytes;
}
extern "C" size_t p3d_fp8_linear_bwd_workspace(const p3d_fp8_linear *a) {
  return check(a, "p3d_fp8_linear_bwd_workspace") ? 0 : backward_of(*a, true, nullptr).bytes;
}

extern "C" int p3d_fp8_linear_fwd(const p3d_fp8_linear *a, const void *x, const void *bias, void *y, void *saved,
                                  void *workspace, size_t workspace_bytes, void *stream) {
  if (int st = check(a, "p3d_fp8_linear_fwd")) return st;
  P3D_CHECK_ARG(x && y && (a->weight || (a->weight_values && a->weight_scales)), "p3d_fp8_linear_fwd: null pointer");
  P3D_CHECK_ARG(!(a->need_dx || a->need_dw) || (a->weight && saved && ((uintptr_t)saved & 255) == 0),
                "p3d_fp8_linear_fwd: gradients need the weight itself and 256-byte aligned room for what they keep");
  const Forward f = forward_of(*a, workspace);
  if (f.bytes && (!workspace || ((uintptr_t)workspace & 255) || workspace_bytes < f.bytes))
    return fail(P3D_ERR_WORKSPACE, "p3d_fp8_linear_fwd: 256-byte aligned workspace of %zu bytes, %zu needed",
                workspace_bytes, f.bytes);
  const Saved s = saved_of(*a, saved);
  const bool tokens = in_product(*a);
  Matrix w = f.w;
  // x's transposed copy makes it a tiles' kernel like the weight's, and one launch does both
  const bool both = a->need_dw && a->weight && a->dtype == a->weight_dtype && a->rows + a->n <= 65000LL * 128;
  if (both) {
    const QuantOperand qx = {x, a->rows, f.x.values, f.x.scales, f.x.pitch, s.xt.values, s.xt.scales, s.xt.pitch};
    const QuantOperand qw = {a->weight, a->n, w.values, w.scales, w.pitch, s.wt.values, s.wt.scales, s.wt.pitch};
    if (int st = launch_quantize_both(qx, qw, a->k, a->dtype, static_cast<cudaStream_t>(stream))) return st;
  } else if (!tokens) {
    if (int st = p3d_fp8_quantize(x, a->dtype, a->rows, a->k, 0, f.x.values, f.x.pitch, f.x.scales, s.xt.values, s.xt.pitch,
                                  s.xt.scales, nullptr, 0, nullptr, 0, stream))
      return st;
  }
  if (a->weight) {
    if (!both)
      if (int st = p3d_fp8_quantize(a->weight, a->weight_dtype, a->n, a->k, 1, w.values, w.pitch, w.scales, s.wt.values,
                                    s.wt.pitch, s.wt.scales, nullptr, 0, nullptr, 0, stream))
        return st;
  } else {
    w = Matrix{a->n, a->k, a->weight_pitch, const_cast<void *>(a->weight_values), const_cast<void *>(a->weight_scales)};
  }
  if (tokens)
    return launch_fp8_tokens(x, a->dtype, w.values, w.pitch, w.scales, a->rows, a->n, a->k, bias, a->bias_dtype, y, a->dtype,
                             static_cast<cudaStream_t>(stream));
  return p3d_fp8_matmul(f.x.values, f.x.pitch, f.x.scales, w.values, w.pitch, w.scales, a->rows, a->n, a->k, bias,
                        a->bias_dtype, y, a->dtype, f.sums, f.sum_bytes, stream);
}

extern "C" int p3d_fp8_linear_bwd(const p3d_fp8_linear *a, const void *dy, const void *saved, void *dx, void *dw,
                                  void *dbias, void *workspace, size_t workspace_bytes, void *stream) {
  if (int st = check(a, "p3d_fp8_linear_bwd")) return st;
  P3D_CHECK_ARG(dy && (dx != nullptr) == (a->need_dx != 0) && (dw != nullptr) == (a->need_dw != 0) && (dx || dw || dbias),
                "p3d_fp8_linear_bwd: gradients must be those that the forward kept for");
  P3D_CHECK_ARG(!(dx || dw) || saved, "p3d_fp8_linear_bwd: nothing kept");
  const Backward b = backward_of(*a, dbias != nullptr, workspace);
  if (!workspace || ((uintptr_t)workspace & 255) || workspace_bytes < b.bytes)
    return fail(P3D_ERR_WORKSPACE, "p3d_fp8_linear_bwd: 256-byte aligned workspace of %zu bytes, %zu needed",
                workspace_bytes, b.bytes);
  const Saved s = saved_of(*a, const_cast<void *>(saved));
  if (int st = p3d_fp8_quantize(dy, a->dtype, a->rows, a->n, 0, b.dy.values, b.dy.pitch, b.dy.scales, b.dyt.values,
                                b.dyt.pitch, b.dyt.scales, dbias, a->bias_dtype, b.columns, b.column_bytes, stream))
    return st;
  if (dx)
    if (int st = p3d_fp8_matmul(b.dy.values, b.dy.pitch, b.dy.scales, s.wt.values, s.wt.pitch, s.wt.scales, a->rows, a->k,
                                a->n, nullptr, 0, dx, a->dtype, b.sums, b.sum_bytes, stream))
      return st;
  if (dw)
    return p3d_fp8_matmul(b.dyt.values, b.dyt.pitch, b.dyt.scales, s.xt.values, s.xt.pitch, s.xt.scales, a->n, a->k,
                          a->rows, nullptr, 0, dw, a->weight_dtype, b.sums, b.sum_bytes, stream);
  return P3D_OK;
}
