// Attention over packed sequences, a warp to a row: each lane holds four columns and the dot products are warp sums.
#include <math.h>

#include <algorithm>

#include "kernels.cuh"
#include "seq_tc.cuh"

namespace p3d {
namespace {

constexpr int kWarps = 8;

template <typename T> __device__ __forceinline__ void load4(const T *row, int lane, int dim, float (&v)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = lane * 4 + i < dim ? to_f32<T>(row[lane * 4 + i]) : 0.f;
}
template <typename T> __device__ __forceinline__ void store4(T *row, int lane, int dim, const float (&v)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (lane * 4 + i < dim) row[lane * 4 + i] = from_f32<T>(v[i]);
}
__device__ __forceinline__ float dot4(const float (&a)[4], const float (&b)[4]) {
  return warp_sum(a[0] * b[0] + a[1] * b[1] + a[2] * b[2] + a[3] * b[3]);
}

template <typename T>
__global__ void dq_kernel(const __grid_constant__ p3d_sequence a, const T *out, const float *lse, const T *dout, T *dq) {
  const int64_t item = (int64_t)blockIdx.x * kWarps + threadIdx.x / 32;
  const int lane = threadIdx.x & 31, h = (int)(item % a.heads), t = (int)(item / a.heads);
  if (t >= a.q_rows) return;
  const int b = cache::sequence_of(a.q_offsets, a.sequences, (int)a.q_rows, t), g = h / (a.heads / a.kv_heads);
  const seq::Range r = seq::range_of(a, b);
  const int n = t - r.q0 < r.nq ? seq::seen_by(r, t - r.q0, a.causal) : 0;
  const int64_t row = ((int64_t)t * a.heads + h) * a.dim;
  float q[4], o[4], d[4], k[4], v[4], sum[4] = {0.f, 0.f, 0.f, 0.f};
  load4(static_cast<const T *>(a.q) + t * a.q_stride[0] + h * a.q_stride[1], lane, a.dim, q);
  load4(out + row, lane, a.dim, o);
  load4(dout + row, lane, a.dim, d);
  const float delta = dot4(o, d), l = lse[h * a.q_rows + t];
  for (int j = 0; j < n; ++j) {
    load4(static_cast<const T *>(a.k) + (int64_t)(r.k0 + j) * a.k_stride[0] + g * a.k_stride[1], lane, a.dim, k);
    load4(static_cast<const T *>(a.v) + (int64_t)(r.k0 + j) * a.v_stride[0] + g * a.v_stride[1], lane, a.dim, v);
    const float ds = expf(dot4(q, k) * a.scale - l) * (dot4(d, v) - delta) * a.scale;
#pragma unroll
    for (int i = 0; i < 4; ++i) sum[i] += ds * k[i];
  }
  store4(dq + row, lane, a.dim, sum);
}

template <typename T>
__global__ void dkv_kernel(const __grid_constant__ p3d_sequence a, const T *out, const float *lse, const T *dout, T *dk, T *dv) {
  const int64_t item = (int64_t)blockIdx.x * kWarps + threadIdx.x / 32;
  const int lane = threadIdx.x & 31, g = (int)(item % a.kv_heads), t = (int)(item / a.kv_heads), group = a.heads / a.kv_heads;
  if (t >= a.k_rows) return;
  const int b = cache::sequence_of(a.k_offsets, a.sequences, (int)a.k_rows, t);
  const seq::Range r = seq::range_of(a, b);
  const int j = t - r.k0;
  const int i0 = j >= r.nk ? r.nq : a.causal ? max(0, j + r.nq - r.nk) : 0;   // the first row that sees key j
  float q[4], o[4], d[4], k[4], v[4], sk[4] = {0.f, 0.f, 0.f, 0.f}, sv[4] = {0.f, 0.f, 0.f, 0.f};
  load4(static_cast<const T *>(a.k) + t * a.k_stride[0] + g * a.k_stride[1], lane, a.dim, k);
  load4(static_cast<const T *>(a.v) + t * a.v_stride[0] + g * a.v_stride[1], lane, a.dim, v);
  for (int h = g * group; h < (g + 1) * group; ++h)
    for (int i = i0; i < r.nq; ++i) {
      const int64_t row = ((int64_t)(r.q0 + i) * a.heads + h) * a.dim;
      load4(static_cast<const T *>(a.q) + (int64_t)(r.q0 + i) * a.q_stride[0] + h * a.q_stride[1], lane, a.dim, q);
      load4(out + row, lane, a.dim, o);
      load4(dout + row, lane, a.dim, d);
      const float p = expf(dot4(q, k) * a.scale - lse[h * a.q_rows + r.q0 + i]);
      const float ds = p * (dot4(d, v) - dot4(o, d)) * a.scale;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        sk[c] += ds * q[c];
        sv[c] += p * d[c];
      }
    }
  const int64_t row = ((int64_t)t * a.kv_heads + g) * a.dim;
  if (dk) store4(dk + row, lane, a.dim, sk);
  if (dv) store4(dv + row, lane, a.dim, sv);
}

int blocks_of(int64_t warps) { return (int)((warps + kWarps - 1) / kWarps); }
bool aligned(const void *q) { return (uintptr_t)q % 16 == 0; }

}  // namespace

namespace seq {

int check(const p3d_sequence *a, const char *what) {
  P3D_CHECK_ARG(a != nullptr, "%s: null arguments", what);
  P3D_CHECK_ARG(a->dtype == P3D_F16 || a->dtype == P3D_BF16, "%s: f16 or bf16 tensors only", what);
  P3D_CHECK_ARG(a->dim >= 8 && a->dim <= 128 && a->dim % 8 == 0, "%s: head dim must be a multiple of 8 up to 128, got %d", what,
                a->dim);
  P3D_CHECK_ARG(a->heads >= 1 && a->kv_heads >= 1 && a->heads % a->kv_heads == 0 && a->heads <= 65535,
                "%s: query heads must be a multiple of the key heads", what);
  P3D_CHECK_ARG(a->sequences >= 0 && a->q_rows >= 0 && a->k_rows >= 0, "%s: counts must not be negative", what);
  if (a->q_rows >= (1ll << 30) || a->k_rows >= (1ll << 30) || a->sequences >= (1 << 24))
    return fail(P3D_ERR_UNSUPPORTED, "%s: at most 2^30 - 1 rows and 2^24 - 1 sequences", what);
  P3D_CHECK_ARG(isfinite(a->scale) && a->scale > 0, "%s: scale must be finite and positive", what);
  P3D_CHECK_ARG(a->sequences >= 1 || (a->q_rows == 0 && a->k_rows == 0), "%s: rows without a sequence", what);
  P3D_CHECK_ARG(a->sequences == 0 || (a->q_offsets && a->k_offsets), "%s: null offsets", what);
  P3D_CHECK_ARG((a->q || !a->q_rows) && (!a->k_rows || (a->k && a->v)), "%s: null input", what);
  bool fits = aligned(a->q) && aligned(a->k) && aligned(a->v);
  for (int i = 0; i < 2; ++i) fits = fits && a->q_stride[i] % 8 == 0 && a->k_stride[i] % 8 == 0 && a->v_stride[i] % 8 == 0;
  P3D_CHECK_ARG(fits, "%s: rows must be 16-byte aligned", what);
  // as a tensor map takes them
  auto steps = [&](const int64_t (&stride)[2], int64_t rows, int heads) {
    return (rows <= 1 || (stride[0] > 0 && stride[0] < 1ll << 38)) && (heads <= 1 || (stride[1] > 0 && stride[1] < 1ll << 38));
  };
  P3D_CHECK_ARG(steps(a->q_stride, a->q_rows, a->heads) && steps(a->k_stride, a->k_rows, a->kv_heads) &&
                    steps(a->v_stride, a->k_rows, a->kv_heads),
                "%s: strides must be positive and below 2^38", what);
  return P3D_OK;
}

}  // namespace seq

int take_sequence_errors(unsigned *flags) { return seq::take_errors_fwd(flags); }

}  // namespace p3d

using namespace p3d;

extern "C" {

int p3d_sequence_fwd(const p3d_sequence *a, void *out, float *lse, void *stream) {
  if (int st = seq::check(a, "p3d_sequence_fwd")) return st;
  if (a->q_rows == 0) return P3D_OK;
  P3D_CHECK_ARG(out && aligned(out), "p3d_sequence_fwd: the output must be given and 16-byte aligned");
  return seq::launch_fwd(*a, out, lse, (cudaStream_t)stream);
}

size_t p3d_sequence_bwd_workspace(const p3d_sequence *a) {
  return 0;
}

int p3d_sequence_bwd(const p3d_sequence *a, const void *out, const float *lse, const void *dout, void *dq, void *dk, void *dv,
                     void *workspace, size_t workspace_bytes, void *stream) {
  if (int st = seq::check(a, "p3d_sequence_bwd")) return st;
  const cudaStream_t s = (cudaStream_t)stream;
  P3D_CHECK_ARG(!a->q_rows || (out && lse && dout && aligned(out) && aligned(dout)),
                "p3d_sequence_bwd: out, lse and dout must be given and 16-byte aligned");
  auto go = [&](auto type) {
    using T = decltype(type);
    if (dq && a->q_rows)
      dq_kernel<T><<<blocks_of(a->q_rows * a->heads), kWarps * 32, 0, s>>>(*a, (const T *)out, lse, (const T *)dout, (T *)dq);
    if ((dk || dv) && a->k_rows)
      dkv_kernel<T><<<blocks_of(a->k_rows * a->kv_heads), kWarps * 32, 0, s>>>(*a, (const T *)out, lse, (const T *)dout,
                                                                               (T *)dk, (T *)dv);
  };
  a->dtype == P3D_F16 ? go(__half()) : go(__nv_bfloat16());
  P3D_LAUNCH_CHECK();
  return P3D_OK;
}

}  // extern "C"
