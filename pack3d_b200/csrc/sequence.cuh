// Packed sequences: arguments and index arithmetic shared by the forward and backward kernels of p3d_sequence.
#pragma once

#include "cache.cuh"

namespace p3d {
namespace seq {

// One sequence's rows in the packed tensors.
struct Range {
  int q0, nq, k0, nk;
};
__device__ __forceinline__ Range range_of(const p3d_sequence &a, int b) {
  Range r;
  r.q0 = cache::offset_at(a.q_offsets, b, (int)a.q_rows);
  r.nq = max(cache::offset_at(a.q_offsets, b + 1, (int)a.q_rows) - r.q0, 0);
  r.k0 = cache::offset_at(a.k_offsets, b, (int)a.k_rows);
  r.nk = max(cache::offset_at(a.k_offsets, b + 1, (int)a.k_rows) - r.k0, 0);
  return r;
}
// Keys that row i of a sequence sees: those below this number.
__device__ __forceinline__ int seen_by(const Range &r, int i, bool causal) {
  return causal ? min(r.nk, max(0, i + 1 + r.nk - r.nq)) : r.nk;
}

int check(const p3d_sequence *a, const char *what);   // sequence.cu

}  // namespace seq
}  // namespace p3d
