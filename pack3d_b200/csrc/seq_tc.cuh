// What the tensor-core kernels of p3d_sequence share: operand tiles of 128 rows, where a CTA's rows are, bounded waits.
#pragma once

#include <type_traits>

#include "sequence.cuh"
#include "sm100.cuh"
#include "tma_host.cuh"

namespace p3d {
namespace seq {

using namespace sm100;

constexpr int kTile = 128;                       // rows of an operand tile
constexpr uint32_t kBox = kTile * 128;           // bytes of one TMA box: 128 rows of 64 columns, SWIZZLE_128B
constexpr uint64_t kWaitNs = 2000000000ull;      // every wait is bounded: 2 s

// Columns of a head rounded up to whole boxes; a box's columns past dim are zero-filled by the copy.
constexpr int padded(int dim) { return dim <= 64 ? 64 : 128; }

// A tile as the products read it. K-major: 16 columns (32 bytes of each row) a step, four steps a box.
__device__ __forceinline__ uint64_t desc_rows(uint32_t tile) { return desc_sw128(tile, 1024); }
__device__ __forceinline__ uint32_t step_rows(int k) { return ((k / 4) * kBox + (k % 4) * 32) >> 4; }
// MN-major (the rows are summed over): 64-column atoms a box apart, groups of eight rows 1024 bytes apart; 16 rows a step.
__device__ __forceinline__ uint64_t desc_cols(uint32_t tile) {
  uint64_t d = desc_sw128(tile, 1024);
  d &= ~((uint64_t)0x3FFFu << 16);
  return d | (uint64_t)(kBox >> 4) << 16;
}
__device__ __forceinline__ uint32_t step_cols(int k) { return (uint32_t)(k * 16 * 128) >> 4; }

// Which sequence a slot belongs to, and which of its groups of `rows` rows: a sequence b that begins at row o_b has the slots from
// o_b / rows + b on, one more than it can need; the rows behind the last sequence are sequence `sequences`. All lanes of a warp
// take part and search 32 ways at a time.
struct Slot {
  int sequence, group;
};
__device__ __forceinline__ Slot find_slot(const int32_t *offsets, int sequences, int total, int rows, int slot) {
  int lo = 0, n = sequences + 1;   // the answer is one of lo .. lo + n - 1; the one at lo qualifies
  const int lane = threadIdx.x & 31;
  while (n > 1) {
    const int step = (n + 31) / 32, at = lane * step;
    const bool in = at < n && (lane == 0 || cache::offset_at(offsets, lo + at, total) / rows + lo + at <= slot);
    const int last = 31 - __clz(__ballot_sync(0xffffffffu, in));
    lo += last * step;
    n = min(step, n - last * step);
  }
  return {lo, slot - (cache::offset_at(offsets, lo, total) / rows + lo)};
}
// Its rows; those of the last, empty one see no keys.
__device__ __forceinline__ Range slot_range(const p3d_sequence &a, int b) {
  if (b < a.sequences) return range_of(a, b);
  Range r = {};
  r.q0 = cache::offset_at(a.q_offsets, b, (int)a.q_rows);
  r.nq = (int)a.q_rows - r.q0;
  r.k0 = cache::offset_at(a.k_offsets, b, (int)a.k_rows);
  return r;
}
inline int64_t slots_of(int64_t rows, int sequences, int per_slot) { return rows / per_slot + sequences + 1; }

// A warp leaves a wait together, whatever its lanes saw.
__device__ __forceinline__ bool wait_warp(uint32_t bar, uint32_t parity, unsigned *errors, unsigned role) {
  const bool all = __all_sync(0xffffffffu, mbar_wait(bar, parity, errors, kWaitNs, role));
  if (all) tc_fence_after();
  return all;
}

// Work beyond a CTA's own: a CTA that is about to be done takes over one that the grid has not launched yet (cluster launch control), so
// that long and short pieces even out as they would by separate launches, without setting a CTA up for each. The answer, 16 bytes,
// arrives at `slot` and completes on the barrier (which expects them); after a -1 nothing may be asked any more.
__device__ __forceinline__ void ask_for_work(uint32_t slot, uint32_t bar) {
  mbar_expect_tx(bar, 16);
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(slot), "r"(bar)
               : "memory");
}
__device__ __forceinline__ int work_given(uint32_t slot) {
  int index;
  asm volatile(
      "{\n\t.reg .b128 answer;\n\t.reg .pred given;\n\t"
      "ld.shared.b128 answer, [%1];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 given, answer;\n\t"
      "mov.s32 %0, -1;\n\t"
      "@given clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %0, answer;\n\t}"
      : "=r"(index)
      : "r"(slot)
      : "memory");
  return index;
}

template <typename T> __device__ __forceinline__ uint32_t pack(float a, float b) {
  return std::is_same<T, __half>::value ? pack_f16(a, b) : pack_bf16(a, b);
}

// The larger, NaN if either is: a NaN score makes its row's maximum NaN, and with it all that the row gives.
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// Elements of a tile that are not finite become 0 (a warp; `bytes` of it). A product with a weight of 0 would make them NaN in rows
// that do not see them. Returns whether there were any. Bits: the exponent is all ones where adding one to its last place
// carries into the sign's place.
template <typename T>
__device__ __forceinline__ bool clear_not_finite(uint8_t *tile, int bytes) {
  constexpr uint32_t one = std::is_same<T, __half>::value ? 0x04000400u : 0x00800080u;
  const int lane = threadIdx.x & 31;
  bool found = false;
  for (int i = lane; i < bytes / 16; i += 32 * 4) {
    uint4 w[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) w[u] = reinterpret_cast<const uint4 *>(tile)[i + 32 * u];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const uint32_t m[4] = {(w[u].x & 0x7fff7fffu) + one, (w[u].y & 0x7fff7fffu) + one, (w[u].z & 0x7fff7fffu) + one,
                             (w[u].w & 0x7fff7fffu) + one};
      if ((m[0] | m[1] | m[2] | m[3]) & 0x80008000u) {
        found = true;
        auto keep = [](uint32_t v, uint32_t odd) {
          return v & ((odd & 0x8000u ? 0u : 0xffffu) | (odd & 0x80000000u ? 0u : 0xffff0000u));
        };
        reinterpret_cast<uint4 *>(tile)[i + 32 * u] = make_uint4(keep(w[u].x, m[0]), keep(w[u].y, m[1]), keep(w[u].z, m[2]), keep(w[u].w, m[3]));
      }
    }
  }
  return __any_sync(0xffffffffu, found);
}

// The tensor map of [rows, heads, dim] with strides in elements: boxes of 64 columns of 128 rows of one head.
inline int encode_heads(CUtensorMap *map, int dtype, const void *p, int dim, int heads, int64_t rows, const int64_t stride[2]) {
  const uint64_t dims[3] = {(uint64_t)dim, (uint64_t)heads, (uint64_t)rows};
  // a stride that nothing steps over may be anything; the map wants one that is not zero
  const uint64_t strides[2] = {2 * (uint64_t)(heads > 1 ? stride[1] : dim), 2 * (uint64_t)(rows > 1 ? stride[0] : dim)};
  const uint32_t box[3] = {64, 1, kTile};
  return encode_operand_sw128(map, dtype, p, 3, dims, strides, box);
}

int take_errors_fwd(unsigned *flags);   // seq_fwd.cu
int launch_fwd(const p3d_sequence &a, void *out, float *lse, cudaStream_t s);
int take_errors_bwd(unsigned *flags);   // seq_bwd.cu
int bwd_workspace(const p3d_sequence &a, size_t *bytes);
int launch_bwd(const p3d_sequence &a, const void *out, const float *lse, const void *dout, void *dq, void *dk, void *dv,
               void *workspace, size_t workspace_bytes, cudaStream_t s);

}  // namespace seq
}  // namespace p3d
