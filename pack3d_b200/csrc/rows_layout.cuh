// How the row kernels of the norms lay a row over threads.  Plain C++ where no CUDA compiler reads it, so that the
// rules can be checked over all widths without a GPU.
#pragma once

#include <algorithm>

#include <stdint.h>

#include "pack3d_b200.h"

#ifdef __CUDACC__
#define P3D_ROWS_FN __device__ __forceinline__
#else
#define P3D_ROWS_FN inline
#endif

namespace p3d {
namespace rows {

constexpr int kUnit = 8;   // columns of a unit; a thread owns up to three (NU)
constexpr int kMaxGroups = 8;

// Threads that work on a row (or on a warp's rows), lanes a row, units of eight columns a thread, rows or warps of
// rows a CTA works on at once, and CTAs a row.
//   Forward: up to 384 columns a warp holds several rows, on 8 or 16 lanes with one or three units each, so that
//   sums take three or four steps for all of them and the bookkeeping is shared; wider rows take two
//   units a thread and up to 256 threads.  (524288 x 192 bf16 with dropout: one row a warp 388 us,
//   four rows 223 us; 166 us since with leaner bookkeeping and the gate folded into the parameters.)
//   Backward: a row a warp at least and one unit, whose column sums fill the registers already.  At most 512
//   threads a row, 256 in 32 bits, where two stages of five arrays of 4096 columns would not fit
//   beside the parameters.
struct Shape {
  int row_threads, lanes, units, groups, members;
  int columns() const { return (lanes < 32 ? lanes : row_threads) * kUnit * units; }   // of a CTA
  int rows_at_once() const { return 32 / lanes; }
};
inline Shape shape_of(int dim, int dtype, bool backward) {
  Shape s;
  s.members = 1;
  s.lanes = backward || dim > 384 ? 32 : dim > 192 ? 16 : 8;
  s.units = backward || dim <= 64 ? 1 : s.lanes == 32 ? 2 : 3;
  s.row_threads = 32;
  if (s.lanes == 32) {
    const int threads = (dim + kUnit * s.units - 1) / (kUnit * s.units), most = backward && dtype != P3D_F32 ? 512 : 256;
    while (threads > s.members * most) s.members *= 2;
    const int mine = (threads + s.members - 1) / s.members;
    s.row_threads = (mine + 31) / 32 * 32;
    // rounded up to whole warps, fewer CTAs may hold the row: every CTA that there is has columns of it (at 8200 columns in
    // 32 bits seven of 160 threads, not eight)
    s.members = (threads + s.row_threads - 1) / s.row_threads;
  }
  s.groups = std::min(kMaxGroups, std::max(1, 256 / s.row_threads));
  return s;
}

// An unaligned batch of `n` rows from `row` on is copied with the up to 15 bytes before and after it that complete 16-byte
// pieces.  Batches whose pieces may pass the tensor's ends are not copied but read in place: those with one of the
// edge_rows first or last rows, which is one row at each end, and more where a row is shorter than 15 bytes.
inline int edge_rows(int64_t row_bytes) { return (int)((15 + row_bytes - 1) / row_bytes); }
P3D_ROWS_FN bool in_place(int row, int n, int rows, int edge) { return row < edge || row + n > rows - edge; }
// Bytes of the pieces that hold `bytes` bytes from `shift` after a 16-byte boundary on.
P3D_ROWS_FN uint32_t piece_bytes(uint32_t shift, uint32_t bytes) { return (shift + bytes + 15u) & ~15u; }

// Where a warp is in its group's ring: the stages are filled in turn, at most all but one ahead of the batch in use.
// A batch that does not arrive in time is the last one waited for: the warp goes through its remaining batches on the
// stage where it stopped, so that barriers stay matched, and neither loads nor stores.
struct RingState {
  int stage = 0, phase = 0;   // of the next batch to use
  int fill = 0;               // stage of the next batch to load
  bool ok = true;             // all batches so far have arrived

  P3D_ROWS_FN void step(int stages) {
    if (++stage == stages) {
      stage = 0;
      phase ^= 1;
    }
  }
  P3D_ROWS_FN int load(int stages) {   // the stage to load the next batch into
    const int s = fill;
    fill = fill + 1 == stages ? 0 : fill + 1;
    return s;
  }
  // The next batch's stage; arrived(stage, phase) waits for it.
  template <typename F>
  P3D_ROWS_FN int use(int stages, F &&arrived) {
    const int s = stage;
    if (ok) ok = arrived(s, phase);
    if (ok) step(stages);
    return s;
  }
  // Waits once more for what is on its way, before the shared memory is given up.
  template <typename F>
  P3D_ROWS_FN void drain(int stages, F &&arrived) {
    while (stage != fill) {
      arrived(stage, phase);
      step(stages);
    }
  }
};

}  // namespace rows
}  // namespace p3d
