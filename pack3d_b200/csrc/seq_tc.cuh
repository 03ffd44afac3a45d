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

template <typename T> __device__ __forceinline__ uint32_t pack(float a, float b) {
  return std::is_same<T, __half>::value ? pack_f16(a, b) : pack_bf16(a, b);
}

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

// Which sequence a slot belongs to, its rows, and which of its groups of 2^shift rows the slot is: a sequence b that begins at row o_b
// has the slots from o_b / 2^shift + b on, one more than it can need; the rows behind the last sequence are sequence
// `sequences`, without rows on the other side. By queries, or by keys. All lanes of a warp take part and search 32 ways at a
// time; the last round brings both sides' offsets, so that up to 30 sequences cost one memory latency.
struct Place {
  Range r;
  int group;
};
template <bool kByKeys>
__device__ __forceinline__ Place place_of(const p3d_sequence &a, int shift, int slot) {
  const int32_t *const mine = kByKeys ? a.k_offsets : a.q_offsets, *const other = kByKeys ? a.q_offsets : a.k_offsets;
  const int total = (int)(kByKeys ? a.k_rows : a.q_rows), other_total = (int)(kByKeys ? a.q_rows : a.k_rows);
  int lo = 0, n = a.sequences + 1;   // the answer is one of lo .. lo + n - 1; the one at lo qualifies
  const int lane = threadIdx.x & 31;
  while (n > 31) {
    const int step = (n + 31) / 32, at = lane * step;
    const bool in = at < n && (lane == 0 || (cache::offset_at(mine, lo + at, total) >> shift) + lo + at <= slot);
    const int last = 31 - __clz(__ballot_sync(0xffffffffu, in));
    lo += last * step;
    n = min(step, n - last * step);
  }
  const int at = min(lo + lane, a.sequences);
  const int m = cache::offset_at(mine, at, total), o = cache::offset_at(other, at, other_total);
  const bool in = lane < n && (lane == 0 || (m >> shift) + lo + lane <= slot);
  const int last = 31 - __clz(__ballot_sync(0xffffffffu, in)), b = lo + last;
  const int m0 = __shfl_sync(0xffffffffu, m, last), m1 = b < a.sequences ? __shfl_sync(0xffffffffu, m, last + 1) : total;
  const int o0 = __shfl_sync(0xffffffffu, o, last), o1 = b < a.sequences ? __shfl_sync(0xffffffffu, o, last + 1) : o0;
  const int mn = max(m1 - m0, 0), on = max(o1 - o0, 0);
  return {kByKeys ? Range{o0, on, m0, mn} : Range{m0, mn, o0, on}, slot - ((m0 >> shift) + b)};
}

// The same in another order, for causal masks: by d, falling, the d-th tile of a sequence from the side that has the least work
// (queries: its first, keys: its last). Six sequences of 1,400 to 4,000, 16 heads of 128 over 4: forward 317 us in the packed order,
// 268 in this one, the keys' gradients 480 and 433, as the last CTAs to run have short tiles. As many tiles lie before d + 1 as sum up over sequences to max(0, tiles - d - 1), so a
// warp finds d by halving, with four sequences a lane; where there are more of them, or an SM for each tile (the search costs 0.7 us), the
// packed order serves.
inline int falling(const p3d_sequence &a, int64_t grid, int sms) { return a.causal && a.sequences <= 127 && grid > sms; }
template <bool kByKeys>
__device__ __forceinline__ Place place_falling(const p3d_sequence &a, int shift, int rank) {
  const int32_t *const mine = kByKeys ? a.k_offsets : a.q_offsets, *const other = kByKeys ? a.q_offsets : a.k_offsets;
  const int total = (int)(kByKeys ? a.k_rows : a.q_rows), other_total = (int)(kByKeys ? a.q_rows : a.k_rows);
  const int lane = threadIdx.x & 31, rounds = a.sequences / 32 + 1;   // rows behind the last sequence are one more, without keys
  int m0[4], m1[4], o0[4], o1[4], tiles[4], most = 0;
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    m0[u] = m1[u] = o0[u] = o1[u] = 0;
    const int b = u * 32 + lane;
    if (u < rounds && b <= a.sequences) {
      const int next = min(b + 1, a.sequences);
      m0[u] = cache::offset_at(mine, b, total), m1[u] = b < a.sequences ? cache::offset_at(mine, next, total) : total;
      o0[u] = cache::offset_at(other, b, other_total), o1[u] = b < a.sequences ? cache::offset_at(other, next, other_total) : o0[u];
    }
  }
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    m1[u] = max(m1[u] - m0[u], 0), o1[u] = max(o1[u] - o0[u], 0);   // lengths
    tiles[u] = (m1[u] + (1 << shift) - 1) >> shift;
    most = max(most, tiles[u]);
  }
  const auto before = [&](int d) {   // tiles that are the d-th or a later one
    int n = 0;
#pragma unroll
    for (int u = 0; u < 4; ++u) n += max(tiles[u] - d, 0);
    return (int)__reduce_add_sync(0xffffffffu, n);
  };
  int lo = 0, hi = (int)__reduce_max_sync(0xffffffffu, most);
  if (before(0) <= rank) return {Range{0, 0, 0, 0}, -1};
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    (before(mid) > rank ? lo : hi) = mid;
  }
  int left = rank - before(lo + 1);
  Place place = {Range{0, 0, 0, 0}, -1};
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const bool in = tiles[u] > lo;
    const unsigned all = __ballot_sync(0xffffffffu, in);
    if (left >= 0 && left < __popc(all)) {
      const int from = __ffs(__ballot_sync(0xffffffffu, in && __popc(all & ((1u << lane) - 1)) == left)) - 1;
      const int a0 = __shfl_sync(0xffffffffu, m0[u], from), an = __shfl_sync(0xffffffffu, m1[u], from);
      const int b0 = __shfl_sync(0xffffffffu, o0[u], from), bn = __shfl_sync(0xffffffffu, o1[u], from);
      const int n = __shfl_sync(0xffffffffu, tiles[u], from);
      place = {kByKeys ? Range{b0, bn, a0, an} : Range{a0, an, b0, bn}, kByKeys ? n - 1 - lo : lo};
    }
    left -= __popc(all);
  }
  return place;
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

// Masked weights and values that are not finite.  A masked weight is 0, but 0 times an infinity or NaN is NaN: a product over a whole tile
// would pass on what a row does not see. So in tiles that some row does not see whole, such values are set to 0 before the product reads
// them (clear_not_finite), and added again to the rows that see them once the sum is there (add_not_finite): an infinity whose weight is
// positive makes the sum that infinity, two that meet make it NaN (a value whose key has a score of -inf counts by its sign). Each such
// value is looked at once for 32 rows, so the work is bounded by what is read anyway, whatever the values are.
// * Forward: the softmax warps look through the values of those tiles before they hand over their weights.
// * dQ: a key that is not finite makes the scores of its column not finite, also of the rows that do not see it: the softmax warps have them.
//   A query that sees the key has no score gradient there (its score is -inf: 0 times the infinity) or nowhere: NaN.
// * dK, dV: a query or a gradient row that is not finite has an lse or a delta that is not. A key that such a query sees gets NaN from its
//   weight; a gradient row's value is added to dV.
// * Backward, rows of a tile behind the end of its sequence (another sequence's, or memory that nobody filled): cleared by the copying warp,
//   which has the tile land on a barrier of its own (clear_rows). In the forward pass they are among what the softmax warps look at.
template <int kBoxes>
__device__ __forceinline__ void clear_rows(uint8_t *tile, int first) {
  for (int i = threadIdx.x & 31; i < (kTile - first) * 8; i += 32)
#pragma unroll
    for (int b = 0; b < kBoxes; ++b) *reinterpret_cast<uint4 *>(tile + b * kBox + first * 128 + i * 16) = make_uint4(0, 0, 0, 0);
  fence_proxy_async_smem();
  __syncwarp();
}
// `kRows` rows of each box from `tile` on (shared memory, by a warp): infinities and NaN become 0. Where there are any, *flag becomes `value`, and
// it does before they go: another warp that finds them cleared finds the flag. All finite, it costs a load and four additions of zeros
// for 16 bytes.
template <typename T, int kBoxes, int kRows>
__device__ __forceinline__ void clear_not_finite(uint8_t *tile, volatile int *flag, int value) {
  constexpr int kEach = kRows * 128 / 512;   // loads of a lane in a box
  constexpr uint32_t kExp = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
  uint4 w[kBoxes * kEach];
  uint32_t sum = 0;
  auto add = [&](uint32_t v) {   // v * 0 + sum, each half: 0, or NaN for ever
    if constexpr (std::is_same<T, __half>::value) asm("fma.rn.f16x2 %0, %1, %2, %0;" : "+r"(sum) : "r"(v), "r"(0u));
    else asm("fma.rn.bf16x2 %0, %1, %2, %0;" : "+r"(sum) : "r"(v), "r"(0u));
  };
#pragma unroll
  for (int i = 0; i < kBoxes * kEach; ++i)
    w[i] = *reinterpret_cast<const uint4 *>(tile + i / kEach * kBox + i % kEach * 512 + (threadIdx.x & 31) * 16);
  const int set = *flag;
#pragma unroll
  for (int i = 0; i < kBoxes * kEach; ++i) add(w[i].x), add(w[i].y), add(w[i].z), add(w[i].w);
  if (!__any_sync(0xffffffffu, (sum & 0x7fff7fffu) != 0)) {
    if (set == value) fence_proxy_async_smem();   // what another warp has written, for this one's product
    return;
  }
  if ((threadIdx.x & 31) == 0) *flag = value;
  __threadfence_block();
  __syncwarp();
  auto clean = [&](uint32_t &v) {
    if ((v & kExp) == kExp) v &= 0xffff0000u;
    if ((v & kExp << 16) == kExp << 16) v &= 0xffffu;
  };
#pragma unroll
  for (int i = 0; i < kBoxes * kEach; ++i) {
    clean(w[i].x), clean(w[i].y), clean(w[i].z), clean(w[i].w);
    *reinterpret_cast<uint4 *>(tile + i / kEach * kBox + i % kEach * 512 + (threadIdx.x & 31) * 16) = w[i];
  }
  fence_proxy_async_smem();
}
__device__ __forceinline__ bool not_finite(float v) { return (__float_as_uint(v) & 0x7f800000u) == 0x7f800000u; }

// Four columns of a row for each lane.
template <typename T>
__device__ __forceinline__ void load4(const T *row, int dim, float (&v)[4]) {
  const int c = (threadIdx.x & 31) * 4;
  if (c < dim) {   // dim is a multiple of 8, rows are 16-byte aligned
    const uint2 w = *reinterpret_cast<const uint2 *>(row + c);
    const float2 a = unpack2<T>(w.x), b = unpack2<T>(w.y);
    v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y;
  } else {
    v[0] = v[1] = v[2] = v[3] = 0.f;
  }
}

// Adds what is not finite in the rows from j on of `rows` (`stride` elements apart), from column lo up to hi, to a warp's rows of out that see
// them. These see the more of them the further down they are, so one pass serves all. `at` (a row's place in out, -1 for none, which come
// last) and `seen` (it sees the rows below) are of a lane's row. `as_nan`: whatever is not finite counts as NaN.
template <typename T>
__device__ __noinline__ void add_not_finite(const T *rows, int64_t stride, int j, int lo, int hi, bool as_nan, int64_t at, int seen, T *out) {
  const int c = (threadIdx.x & 31) * 4;
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
  for (int from = 0; from < 32; ++from) {
    const int64_t to = __shfl_sync(0xffffffffu, at, from);
    const int upto = __shfl_sync(0xffffffffu, seen, from);
    if (to < 0) break;
    for (; j < upto; ++j) {
      float v[4];
      load4(rows + j * stride, c < lo ? 0 : hi, v);
#pragma unroll
      for (int i = 0; i < 4; ++i) sum[i] += not_finite(v[i]) ? as_nan ? NAN : v[i] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (sum[i] != 0.f) out[to + c + i] = from_f32<T>(to_f32<T>(out[to + c + i]) + sum[i]);
  }
}

// A warp's 32 rows (a row a lane, 64 columns of 16 bits as 32 words) to memory by way of shared memory, whole lines at a time: `stage` is
// the warp's own 4 KB. Lane i's row is at `row` elements from `out` where it is not negative; columns from `dim` on are left out.
template <typename T>
__device__ __forceinline__ void store_rows(uint8_t *stage, const uint32_t (&w)[32], T *out, int64_t row, int col, int dim) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    *reinterpret_cast<uint4 *>(stage + lane * 128 + ((i ^ (lane & 7)) * 16)) = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
  __syncwarp();
  const int chunk = lane & 7;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = i * 4 + lane / 8;
    const int64_t to = __shfl_sync(0xffffffffu, row, r);
    const uint4 v = *reinterpret_cast<const uint4 *>(stage + r * 128 + ((chunk ^ (r & 7)) * 16));
    if (to >= 0 && col + chunk * 8 < dim) *reinterpret_cast<uint4 *>(out + to + col + chunk * 8) = v;
  }
  __syncwarp();
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
