// Packed sequences: arguments and index arithmetic shared by the forward and backward kernels of p3d_sequence.
#pragma once

#include "cache.cuh"

namespace p3d {
namespace seq {

// One sequence's rows in the packed tensors.
struct Range {
  int q0, nq, k0, nk;
};
// Keys that row i of a sequence sees: those below this number.
__device__ __forceinline__ int seen_by(const Range &r, int i, bool causal) {
  return causal ? min(r.nk, max(0, i + 1 + r.nk - r.nq)) : r.nk;
}

int check(const p3d_sequence *a, const char *what);   // sequence.cu

}  // namespace seq
}  // namespace p3d
