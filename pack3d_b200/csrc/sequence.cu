// p3d_sequence: the checks of arguments and the entry points; the kernels are in seq_fwd.cu and seq_bwd.cu.
#include <math.h>

#include "kernels.cuh"
#include "seq_tc.cuh"

namespace p3d {
namespace {

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

int take_sequence_errors(unsigned *flags) {
  if (int st = seq::take_errors_fwd(flags)) return st;
  return seq::take_errors_bwd(flags);
}

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
  size_t bytes = 0;
  if (seq::check(a, "p3d_sequence_bwd") != P3D_OK || seq::bwd_workspace(*a, &bytes) != P3D_OK) return 0;
  return bytes;
}

int p3d_sequence_bwd(const p3d_sequence *a, const void *out, const float *lse, const void *dout, void *dq, void *dk, void *dv,
                     void *workspace, size_t workspace_bytes, void *stream) {
  if (int st = seq::check(a, "p3d_sequence_bwd")) return st;
  P3D_CHECK_ARG(!a->q_rows || (out && lse && dout && aligned(out) && aligned(dout)),
                "p3d_sequence_bwd: out, lse and dout must be given and 16-byte aligned");
  P3D_CHECK_ARG(aligned(dq) && aligned(dk) && aligned(dv), "p3d_sequence_bwd: gradients must be 16-byte aligned");
  if (a->sequences == 0) return P3D_OK;
  return seq::launch_bwd(*a, out, lse, dout, dq, dk, dv, workspace, workspace_bytes, (cudaStream_t)stream);
}

}  // extern "C"
