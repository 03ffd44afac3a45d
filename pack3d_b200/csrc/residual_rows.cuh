// Row kernels of the norms around a block (norm, gate, dropout, residual scale, residual, next norm) and
// of their backward; instantiated for each type in residual_{f32,f16,bf16}.cu.
//
// One pass over the data in each direction, bound by HBM: forward 4 (x, h, out, y) and backward 6 (x, h,
// dout, dy, dx, dh) values an element, plus the gate's.  A row is held by 8 or 16 lanes of a warp with up to 24
// columns each (forward, up to 384 columns) to 512 threads of each of up to eight CTAs of a cluster, with 16 columns
// a thread in the forward and eight in the backward (rows_layout.cuh), so the row statistics cost shuffles
// and no second read.  Row groups of a CTA work independently: each has a ring of row batches in shared
// memory that bulk copies fill ahead of it, so the bytes in flight do not depend on how many
// warps fit beside the column sums' registers.  A warp waits for a batch for 2 s at most: if that runs out it
// records an error bit (p3d_device_errors), stores and loads nothing more, makes the sums that it has part in NaN, and waits
// once more for the copies on their way before it ends.
//
// The backward makes out = x + s d again from x and h instead of reading the stored out: the same
// bytes, and the normalised row keeps its 32 bits (the stored one is rounded to 16).  Every
// thread keeps the column sums of its eight columns over all rows of its CTA in registers; they
// are joined over the CTA's row groups in shared memory, written once per CTA and summed over the
// CTAs by a second small kernel, all in a fixed order.  With K the gradient of s (u act) where it was kept (times
// the gate, where that changes from row to row), the block's gradients all come from the sums of K h~ and K: dw = s sum K
// h~, db = s sum K, ds = w sum K h~ + b sum K and, for a sample's gate, s act' times that.  So two sums a
// column are kept instead of four, what does not change from row to row (s, w, b, a sample's gate) is
// multiplied once, and a sample's gate is activated once (364 -> 284 us at 524288 x 192, 120 -> 97 us at 8192 x
// 4096).
//
// Measured on B200 (bf16): 524288 x 192 layer norm, sample gate and dropout, forward 166 us, backward 305 us (287 before
// dropped values were kept out of its sums when they are infinite and waits that run out ended a warp's
// stores); 8192 x 4096 RMS norm, token gate, 55 and 99 us; norm by itself 16384 x 4096 51 and 79 us.  Forward at 4.9 to
// 5.2, backward at 4.0 to 5.1 TB/s: both are bound by issue before HBM, the backward because its column sums leave
// room for 512 threads an SM only.
//
// What a call does not have (a norm, a bias, a gate) is a neutral value in the same formula.  Only what
// costs registers or many instructions is a variant of its own: whether there is a block at all,
// a gate, dropout, and centring (layer norm or a bias).
#pragma once

#include <algorithm>

#include "common.cuh"
#include "kernels.cuh"
#include "philox.cuh"
#include "rows_layout.cuh"
#include "sm100.cuh"

namespace p3d {
namespace rows {

using sm100::add2;
using sm100::fma2;
using sm100::mul2;

constexpr int kMaxCluster = 8;
constexpr int kMaxStages = 4;
constexpr uint64_t kWaitNs = 2000000000ull;

static __device__ unsigned g_row_errors = 0;

enum : int { kX = 0, kH = 1, kGate = 2, kDout = 3, kDy = 4, kArrays = 5 };
enum : int { kPostW = 0, kScale = 1, kNextW = 2, kPostB = 3, kNextB = 4, kParams = 5 };
// Vectors that a variant keeps in shared memory, and the place of each.
__host__ __device__ constexpr int param_count(bool block, bool center) {
  return block ? (center ? 5 : 3) : (center ? 2 : 1);
}
__host__ __device__ constexpr int param_slot(bool block, int k) { return block ? k : k == kNextW ? 0 : 1; }
enum : int { kGateAny = -1 };   // a variant that reads the gate's mode from its arguments

struct Args {
  p3d_residual p;
  const void *in[kArrays];   // streamed rows; null: not read
  const void *params[kParams];   // null: the neutral value
  void *out, *y;
  float *stats;              // [rows][4]; the backward streams them too
  void *dx, *dh, *dgate;
  float *partials;  // [kSums - 1][CTA slots][dim], then the sample gate's [samples][slices][dim]
  int row_threads, groups, members;
  int batch_rows, stages;
  int edge_rows;             // unaligned: rows at either end whose batches are read in place
  uint32_t stage_bytes;      // of all arrays' batches and the statistics
  uint32_t slots[kArrays], stats_at;   // where each lies in a stage
  int slot_count;            // arrays
  int segments, slices, segment_rows;   // the rows are `segments` runs, each cut into slices
  bool gate_folded;          // forward: the segments are samples, whose gate is multiplied into the parameters
};

__device__ __forceinline__ float nan() { return __uint_as_float(0x7fffffffu); }
__device__ __forceinline__ float2 splat(float v) { return make_float2(v, v); }
__device__ __forceinline__ float2 sub2(float2 a, float2 b) { return fma2(b, splat(-1.f), a); }

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// ------------------------------------------------------------------------ a thread's columns of a row
// Aligned: units of eight consecutive columns that move in 16-byte pieces, a thread's second unit
// row_threads units after its first.  Threads past the row's end read its last unit and neither
// add to a sum nor store.  Otherwise (odd dim, or a pointer off 16 bytes) a warp has a run of columns and a lane
// every 32nd of them, so that the lanes stay on consecutive elements at offsets known to the compiler;
// columns past the end read as zero.
struct Place {
  int group, t, warps, warp, lane;
  int rank, first;         // CTA of the cluster, its first column
  int threads, dim, end;   // threads of the row here; columns in all; columns from `first` on
  int sub;                 // which of the warp's rows, where it holds several
  int base, count;         // unaligned: the thread's first column from `first` on, and how many it has
  bool live[3];            // aligned: whether the unit is inside the row
  int at[3];               // aligned: the unit's first column from `first` on, inside the row

  __device__ __forceinline__ void barrier() const {   // of the row group
    if (warps > 1) asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(warps * 32) : "memory");
    else __syncwarp();
  }
  // Column j of the thread (from `first` on).
  template <bool ALIGNED, int LANES>
  __device__ __forceinline__ int col(int j) const {
    return ALIGNED ? (t + j / kUnit * threads) * kUnit + j % kUnit : base + j * LANES;
  }
};

// LANES: threads of a row where a warp holds several rows, else 32.
template <int LANES, bool ALIGNED, int NU>
__device__ __forceinline__ Place place_of(const Args &a) {
  Place q;
  // group, warp and rank are the same in a whole warp; a shuffle tells the compiler, which then keeps what
  // follows from them in uniform registers
  q.group = __shfl_sync(0xffffffffu, (int)threadIdx.x / a.row_threads, 0);
  q.lane = threadIdx.x % 32;
  q.rank = 0;
  q.sub = 0;
  if constexpr (LANES < 32) {
    q.threads = LANES;
    q.t = q.lane % LANES;
    q.sub = q.lane / LANES;
    q.warps = 1;
    q.warp = 0;
  } else {
    q.threads = a.row_threads;
    q.t = threadIdx.x - q.group * a.row_threads;
    q.warps = a.row_threads / 32;
    q.warp = __shfl_sync(0xffffffffu, q.t / 32, 0);
    if (a.members > 1) {
      asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(q.rank));
      q.rank = __shfl_sync(0xffffffffu, q.rank, 0);
    }
  }
  q.dim = a.p.dim;
  q.first = q.rank * q.threads * kUnit * NU;
  q.end = q.dim - q.first;
  q.base = LANES < 32 ? q.t : q.warp * 32 * kUnit * NU + q.lane;
  q.count = ALIGNED ? 0 : min(kUnit * NU, max(0, (q.end - q.base + LANES - 1) / LANES));
#pragma unroll
  for (int n = 0; n < NU; ++n) {
    const int c = (q.t + n * q.threads) * kUnit;
    q.live[n] = c < q.end;
    q.at[n] = min(c, q.end - kUnit);
  }
  return q;
}

template <typename T>
__device__ __forceinline__ float2 pair_of(const T *v) {
  if constexpr (sizeof(T) == 2) return unpack2<T>(*reinterpret_cast<const uint32_t *>(v));
  else return make_float2(v[0], v[1]);
}

// `row`: the row's column `first`.
template <typename T, bool ALIGNED, int NU, int LANES>
__device__ __forceinline__ void load_cols(float2 (&f)[4 * NU], const T *row, const Place &q) {
  if constexpr (ALIGNED) {
#pragma unroll
    for (int n = 0; n < NU; ++n) {
      alignas(16) T v[kUnit];
      constexpr int pieces = sizeof(v) / 16;
      uint4 raw[pieces];
#pragma unroll
      for (int i = 0; i < pieces; ++i) raw[i] = reinterpret_cast<const uint4 *>(row + q.at[n])[i];
      memcpy(v, raw, sizeof(v));
#pragma unroll
      for (int i = 0; i < 4; ++i) f[4 * n + i] = pair_of<T>(v + 2 * i);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4 * NU; ++i) {
      const T *at = row + q.base + 2 * i * LANES;
      f[i].x = 2 * i < q.count ? to_f32<T>(at[0]) : 0.f;
      f[i].y = 2 * i + 1 < q.count ? to_f32<T>(at[LANES]) : 0.f;
    }
  }
}

template <typename T, bool ALIGNED, int NU, int LANES>
__device__ __forceinline__ void store_cols(T *row, const float2 (&f)[4 * NU], const Place &q, bool valid = true) {
  if constexpr (ALIGNED) {
#pragma unroll
    for (int n = 0; n < NU; ++n) {
      if (!(valid && q.live[n])) continue;
      const float2 *v = f + 4 * n;
      if constexpr (sizeof(T) == 4) {
        reinterpret_cast<float4 *>(row + q.at[n])[0] = make_float4(v[0].x, v[0].y, v[1].x, v[1].y);
        reinterpret_cast<float4 *>(row + q.at[n])[1] = make_float4(v[2].x, v[2].y, v[3].x, v[3].y);
      } else {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (std::is_same<T, __nv_bfloat16>::value) w[i] = sm100::pack_bf16(v[i].x, v[i].y);
          else w[i] = sm100::pack_f16(v[i].x, v[i].y);
        }
        *reinterpret_cast<uint4 *>(row + q.at[n]) = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4 * NU; ++i) {
      T *at = row + q.base + 2 * i * LANES;
      if (valid && 2 * i < q.count) at[0] = from_f32<T>(f[i].x);
      if (valid && 2 * i + 1 < q.count) at[LANES] = from_f32<T>(f[i].y);
    }
  }
}

// What the thread adds to a sum over the row, from its columns' v: nothing for units past the end
// (unaligned columns there hold zeros already).
template <bool ALIGNED, int NU>
__device__ __forceinline__ float total(const Place &q, const float2 (&v)[NU]) {
  float s = 0.f;
#pragma unroll
  for (int n = 0; n < NU; ++n) s += ALIGNED && !q.live[n] ? 0.f : v[n].x + v[n].y;
  return s;
}

struct Exchange {
  alignas(16) float slots[2][4][16];   // [2][values][warps of the CTA]
  float peers[2][kMaxCluster][4];      // [2][CTA of the cluster][values]
};

// Sums of N values over a row's lanes, in every one of them.  Over a whole warp two values share their way down:
// lanes 16 to 31 take over the second in the first step, so that later steps move one value; a lane
// of each kind then hands its total out.
template <int LANES>
__device__ __forceinline__ float lane_sum(float v) {
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
template <int LANES, int N>
__device__ __forceinline__ void lane_sums(int lane, float (&v)[N]) {
  if constexpr (LANES == 32 && N >= 2) {
    const bool high = lane & 16;
    const float keep = high ? v[1] : v[0], give = high ? v[0] : v[1];
    const float s = lane_sum<16>(keep + __shfl_xor_sync(0xffffffffu, give, 16));
    v[0] = __shfl_sync(0xffffffffu, s, 0);
    v[1] = __shfl_sync(0xffffffffu, s, 16);
    if constexpr (N > 2) v[2] = lane_sum<32>(v[2]);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = lane_sum<LANES>(v[i]);
  }
}

// N values of every thread summed over the row, the same total in every thread, always added in the
// same order.  The shared slots alternate between calls (`at`): a thread two calls ahead has passed the
// barrier of the call between, so nobody still reads the slots it writes.
template <int LANES>
struct RowSum {
  Exchange *x;
  int members;
  int at = 0;
  bool ok = true;   // otherwise the warp's rows did not arrive, and it makes the row's sums NaN for all who share them

  // Sums of N values over the row's warps (up to sixteen): each half of a warp adds up one value's slots, both
  // halves the same one where there is one.
  template <int N>
  __device__ __forceinline__ void over_warps(const Place &q, float (&v)[N]) const {
    const int w = q.lane & 15, from = q.group * q.warps + w;
    const bool mine = w < q.warps;
    if constexpr (N == 1) {
      v[0] = lane_sum<16>(mine ? x->slots[at][0][from] : 0.f);
    } else {
      const float s = lane_sum<16>(mine ? x->slots[at][q.lane >> 4][from] : 0.f);
      v[0] = __shfl_sync(0xffffffffu, s, 0);
      v[1] = __shfl_sync(0xffffffffu, s, 16);
      if constexpr (N > 2) v[2] = lane_sum<16>(mine ? x->slots[at][2][from] : 0.f);
    }
  }

  template <int N>
  __device__ __forceinline__ void operator()(const Place &q, float (&v)[N]) {
    lane_sums<LANES>(q.lane, v);
    if (LANES == 32 && q.warps > 1) {
      if (q.lane == 0) {
#pragma unroll
        for (int i = 0; i < N; ++i) x->slots[at][i][q.group * q.warps + q.warp] = ok ? v[i] : nan();
      }
      q.barrier();
      over_warps(q, v);
      if (members > 1) over_cluster(q, v);
      at ^= 1;
    }
  }

  // Mean and sum of squares about it: each warp takes its own mean and the squares about that, and the
  // warps' pairs are joined (n (mean_w - mean)^2 each), so one barrier serves both and nothing cancels
  // where the mean is large.
  template <bool ALIGNED, int NU>
  __device__ __forceinline__ float2 moments(const Place &q, const float2 (&z)[4 * NU], float inv_dim) {
    float2 s[NU], d2[NU];
    float count = 0.f;   // columns of the warp, where the row has several
    if (LANES < 32 || q.warps == 1) {
    } else if constexpr (ALIGNED) {
#pragma unroll
      for (int n = 0; n < NU; ++n)
        count += (float)(kUnit * __popc(__ballot_sync(0xffffffffu, q.live[n])));
    } else {
      count = (float)max(0, min(32 * kUnit * NU, q.end - q.warp * 32 * kUnit * NU));
    }
#pragma unroll
    for (int n = 0; n < NU; ++n) s[n] = add2(add2(z[4 * n], z[4 * n + 1]), add2(z[4 * n + 2], z[4 * n + 3]));
    float mean = lane_sum<LANES>(total<ALIGNED, NU>(q, s));
    mean = LANES < 32 || q.warps == 1 ? mean * inv_dim : count > 0.f ? mean / count : 0.f;
#pragma unroll
    for (int n = 0; n < NU; ++n) {
      d2[n] = splat(0.f);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float2 d = sub2(z[4 * n + i], splat(mean));
        if constexpr (!ALIGNED) {
          if (8 * n + 2 * i >= q.count) d.x = 0.f;
          if (8 * n + 2 * i + 1 >= q.count) d.y = 0.f;
        }
        d2[n] = fma2(d, d, d2[n]);
      }
    }
    float m2 = lane_sum<LANES>(total<ALIGNED, NU>(q, d2));
    if (LANES < 32 || q.warps == 1) return make_float2(mean, m2);
    if (q.lane == 0) {
      const int w = q.group * q.warps + q.warp;
      x->slots[at][0][w] = count;
      x->slots[at][1][w] = ok ? mean : nan();
      x->slots[at][2][w] = m2;
    }
    q.barrier();
    const bool mine = q.lane < q.warps;
    const int w = q.group * q.warps + q.lane;
    const float n_w = mine ? x->slots[at][0][w] : 0.f, mean_w = mine ? x->slots[at][1][w] : 0.f;
    float two[2] = {n_w, n_w * mean_w};
    lane_sums<32>(q.lane, two);
    mean = two[1] / two[0];
    const float off = mean_w - mean;
    m2 = warp_sum(fmaf(n_w * off, off, mine ? x->slots[at][2][w] : 0.f));
    if (members > 1) {
      float v[2] = {two[0], two[0] * mean};
      over_cluster(q, v);
      const float all = v[1] / v[0], d = mean - all;
      at ^= 1;
      float u[1] = {fmaf(two[0] * d, d, m2)};
      over_cluster(q, u);
      mean = all;
      m2 = u[0];
    }
    at ^= 1;
    return make_float2(mean, m2);
  }

  template <int N>
  __device__ __forceinline__ void over_cluster(const Place &q, float (&v)[N]) {
    if (q.warp == 0 && q.lane < members) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const uint32_t mine = sm100::smem_u32(&x->peers[at][q.rank][i]);
        uint32_t theirs;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(theirs) : "r"(mine), "r"(q.lane));
        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(theirs), "f"(v[i]) : "memory");
      }
    }
    __syncwarp();
    cluster_sync();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[i] = 0.f;
      for (int c = 0; c < members; ++c) v[i] += x->peers[at][c][i];
    }
  }
};

// ------------------------------------------------------------------------ the ring of row batches
// The batches of a row group, in order: R = batch_rows rows from `row` on, groups * R rows apart within the CTA's slice
// of a segment, which ends at `end`.
struct Batches {
  int seg, row, end;
  int first, size, seg_step, stride;   // of the group in a slice: first row, rows of the slice from there; steps

  __device__ __forceinline__ void enter(const Args &a) {   // segment seg
    row = seg * a.segment_rows + first;
    end = row + size;
  }
  __device__ __forceinline__ bool valid(const Args &a) const { return seg < a.segments; }
  __device__ __forceinline__ void next(const Args &a) {
    row += stride;
    if (row >= end) {
      seg += seg_step;
      if (valid(a)) enter(a);
    }
  }
  __device__ __forceinline__ int count(const Args &a) const { return min(a.batch_rows, end - row); }
};

__device__ __forceinline__ Batches batches_of(const Args &a, int group, int cta, int ctas) {
  Batches k;
  const int slice = cta % a.slices;
  const int row0 = (int)((int64_t)a.segment_rows * slice / a.slices);
  const int row1 = (int)((int64_t)a.segment_rows * (slice + 1) / a.slices);
  k.first = row0 + group * a.batch_rows;
  k.size = row1 - k.first;
  k.seg_step = ctas / a.slices;
  k.stride = a.groups * a.batch_rows;
  k.seg = k.size > 0 ? cta / a.slices : a.segments;   // no batch for this group in any segment
  k.row = k.end = 0;
  if (k.valid(a)) k.enter(a);
  return k;
}

// Bytes from the last 16-byte boundary to column `first` of `row`.
template <typename T>
__device__ __forceinline__ uint32_t shift_of(const Args &a, const Place &q, int array, int row) {
  const uint32_t base = (uint32_t)reinterpret_cast<uintptr_t>(a.in[array]);
  return (base + ((uint32_t)row * (uint32_t)q.dim + (uint32_t)q.first) * (uint32_t)sizeof(T)) & 15u;
}

// Shared memory: exchange slots, keep bits and the rings' barriers; then, dynamic, the parameters and each
// group's ring.
struct Shared {
  Exchange exchange;
  uint64_t bars[kMaxGroups * kMaxStages];
  RoundKeys keys;
  uint8_t keep[3 * 256];
};

// Issued by one elected lane of a converged warp.
__device__ __forceinline__ void elect_expect_tx(uint32_t bar, uint32_t bytes) {
  asm volatile(
      "{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
      "@e mbarrier.arrive.expect_tx.release.cta.shared::cta.b64 _, [%0], %1;\n\t}" ::"r"(bar),
      "r"(bytes)
      : "memory");
}
__device__ __forceinline__ void elect_bulk_load(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar) {
  asm volatile(
      "{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
      "@e cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n\t}" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(src)), "r"(bytes), "r"(bar)
      : "memory");
}

template <typename T, bool ALIGNED, int NU, bool STATS>
struct Ring {
  uint32_t bars;             // the group's
  char *data;                // the group's stages
  RingState state;
  Batches ahead;             // the next batch to load

  // Called by the group's first warp, all of it.
  __device__ __forceinline__ void issue(const Args &a, const Place &q) {
    if (!state.ok || !ahead.valid(a)) return;
    const int n = ahead.count(a), row = ahead.row, stage = state.load(a.stages);
    const uint32_t to = sm100::smem_u32(data) + (uint32_t)stage * a.stage_bytes, b = bars + 8u * stage;
    const int cols = min(q.threads * kUnit * NU, q.end);
    const uint32_t bytes = (uint32_t)(((n - 1) * q.dim + cols) * (int)sizeof(T));
    const int64_t off = ((int64_t)row * q.dim + q.first) * (int64_t)sizeof(T);
    if constexpr (ALIGNED) {
      elect_expect_tx(b, (STATS ? 16u * n : 0u) + bytes * a.slot_count);
#pragma unroll
      for (int i = 0; i < kArrays; ++i)
        if (a.in[i]) elect_bulk_load(to + a.slots[i], static_cast<const char *>(a.in[i]) + off, bytes, b);
    } else {
      const bool copied = !in_place(row, n, (int)a.p.rows, a.edge_rows);
      uint32_t all = STATS ? 16u * n : 0u;
      if (copied) {
#pragma unroll 1
        for (int i = 0; i < kArrays; ++i)
          if (a.in[i]) all += piece_bytes(shift_of<T>(a, q, i, row), bytes);
      }
      elect_expect_tx(b, all);
      if (copied) {
#pragma unroll 1
        for (int i = 0; i < kArrays; ++i)
          if (a.in[i]) {
            const uint32_t shift = shift_of<T>(a, q, i, row);
            elect_bulk_load(to + a.slots[i], static_cast<const char *>(a.in[i]) + off - shift,
                            piece_bytes(shift, bytes), b);
          }
      }
    }
    if (STATS) elect_bulk_load(to + a.stats_at, a.stats + 4 * (int64_t)row, 16u * n, b);
    ahead.next(a);
  }
  // Waits for the next batch and returns where its stage lies; state.ok says whether it is there, the same in the whole
  // warp.
  __device__ __forceinline__ char *wait(const Args &a) {
    const int stage = state.use(a.stages, [&](int s, int phase) {
      return __all_sync(0xffffffffu, sm100::mbar_wait(bars + 8u * s, phase, &g_row_errors, kWaitNs, sm100::kErrProducer));
    });
    return data + (uint32_t)stage * a.stage_bytes;
  }
  // At the kernel's end: after a batch that did not arrive, the warp that issued waits for its copies.
  __device__ __forceinline__ void finish(const Args &a, const Place &q) {
    if (state.ok || q.warp != 0) return;
    state.drain(a.stages, [&](int s, int phase) {
      sm100::mbar_wait(bars + 8u * s, phase, &g_row_errors, kWaitNs, sm100::kErrTeardown);
    });
  }
  // Row i of the batch of `n` rows at `row`, from the CTA's first column on.
  __device__ __forceinline__ const T *row_ptr(const Args &a, const Place &q, const char *at, int array, int row, int n,
                                              int i) const {
    const char *slot = at + a.slots[array];
    if constexpr (!ALIGNED) {
      slot += shift_of<T>(a, q, array, row);
      if (in_place(row, n, (int)a.p.rows, a.edge_rows))
        slot = static_cast<const char *>(a.in[array]) + ((int64_t)row * q.dim + q.first) * (int64_t)sizeof(T);
    }
    return reinterpret_cast<const T *>(slot) + i * q.dim;
  }
  __device__ __forceinline__ float4 stats(const Args &a, const char *at, int i) const {
    return reinterpret_cast<const float4 *>(at + a.stats_at)[i];
  }
};

template <typename T, bool ALIGNED, int NU, bool STATS>
__device__ __forceinline__ Ring<T, ALIGNED, NU, STATS> start_ring(const Args &a, const Place &q, Shared *s, char *data,
                                                                  int cta, int ctas) {
  Ring<T, ALIGNED, NU, STATS> r;
  r.bars = sm100::smem_u32(s->bars + q.group * kMaxStages);
  r.data = data + (size_t)q.group * a.stages * a.stage_bytes;
  r.ahead = batches_of(a, q.group, cta, ctas);
  if (threadIdx.x < kMaxGroups * kMaxStages) sm100::mbar_init(sm100::smem_u32(s->bars + threadIdx.x), 1);
  sm100::fence_mbar_init();
  __syncthreads();
  if (a.members > 1) cluster_sync();
  if (q.warp == 0) {
#pragma unroll 1
    for (int i = 0; i < a.stages - 1; ++i) r.issue(a, q);
  }
  return r;
}

// ------------------------------------------------------------------------ pieces of the formula
// 16-bit types take the sigmoid's exponential from the fast unit, whose error grows with |g|: two ulp near zero, 2 + 1.2
// |g| of them elsewhere (2^-19 of the value at 20), against the 2^-9 and 2^-12 of their results.
template <typename T>
__device__ __forceinline__ float activate(float g, int act) {
  if (act == P3D_ACT_SIGMOID) return __fdividef(1.f, 1.f + (sizeof(T) == 2 ? __expf(-g) : expf(-g)));
  if (act == P3D_ACT_TANH) return tanhf(g);
  return g;
}
// Over a thread's columns, the kind chosen once: a choice for each element would put every kind's code between the
// others'.
template <typename T, int N>
__device__ __forceinline__ void activate_all(float2 (&g)[N], int act) {
  if (act == P3D_ACT_SIGMOID) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      g[i] = make_float2(activate<T>(g[i].x, P3D_ACT_SIGMOID), activate<T>(g[i].y, P3D_ACT_SIGMOID));
  } else if (act == P3D_ACT_TANH) {
#pragma unroll 1
    for (int i = 0; i < N; ++i) {
      // one copy of the code; the array stays in registers
      float2 v = g[0];
#pragma unroll
      for (int j = 0; j + 1 < N; ++j) g[j] = g[j + 1];
      v.x = tanhf(v.x);
      v.y = tanhf(v.y);
      g[N - 1] = v;
    }
  }
}
// The parameters' columns of each thread in fp32, in shared memory: two 16-byte pieces a unit, all threads' first
// pieces and then their second ones, so that a warp reads consecutive banks.  (In registers they would take
// eight a vector and thread beside the column sums.)  What is not given is its neutral value;
// `factor`, the dropout's scale, multiplies the post norm's weight and bias; FOLD (the forward): so do the residual's
// scale, which then has no place of its own, and a sample's gate.
template <typename P, typename T, bool ALIGNED, bool BLOCK, bool CENTER, bool FOLD, int NU, int LANES>
__device__ __forceinline__ void stage_params_of(float4 *params, const Args &a, const Place &q, float factor, const T *gate) {
  float2 fold[4 * NU];
#pragma unroll
  for (int i = 0; i < 4 * NU; ++i) fold[i] = splat(factor);
  if constexpr (FOLD) {
    if (a.params[kScale]) load_cols<P, ALIGNED, NU, LANES>(fold, static_cast<const P *>(a.params[kScale]) + q.first, q);
    const float mul = a.params[kScale] ? factor : factor * a.p.scale_value;
#pragma unroll
    for (int i = 0; i < 4 * NU; ++i) fold[i] = a.params[kScale] ? mul2(fold[i], splat(mul)) : splat(mul);
    if (gate) {
      float2 g[4 * NU];
      load_cols<T, ALIGNED, NU, LANES>(g, gate + q.first, q);
      activate_all<T>(g, a.p.gate_act);
#pragma unroll
      for (int i = 0; i < 4 * NU; ++i) fold[i] = mul2(fold[i], g[i]);
    }
  }
#pragma unroll
  for (int k = 0; k < kParams; ++k) {
    if (!BLOCK && k != kNextW && k != kNextB) continue;
    if (!CENTER && (k == kPostB || k == kNextB)) continue;
    if (FOLD && k == kScale) continue;
    float2 f[4 * NU];
    if (a.params[k]) {   // all of a vector's loads at once
      load_cols<P, ALIGNED, NU, LANES>(f, static_cast<const P *>(a.params[k]) + q.first, q);
    } else {
      const float fill = k == kScale ? a.p.scale_value : k == kPostB || k == kNextB ? 0.f : 1.f;
#pragma unroll
      for (int i = 0; i < 4 * NU; ++i) f[i] = splat(fill);
    }
    if (k == kPostW || k == kPostB) {
#pragma unroll
      for (int i = 0; i < 4 * NU; ++i) f[i] = mul2(f[i], fold[i]);
    }
#pragma unroll
    for (int n = 0; n < NU; ++n) {
      const float2 *v = f + 4 * n;
      float4 *to = params + 2 * (param_slot(BLOCK, k) * NU + n) * q.threads + q.t;
      to[0] = make_float4(v[0].x, v[0].y, v[1].x, v[1].y);
      to[q.threads] = make_float4(v[2].x, v[2].y, v[3].x, v[3].y);
    }
  }
}
template <typename T, bool ALIGNED, bool BLOCK, bool CENTER, bool FOLD, int NU, int LANES>
__device__ __forceinline__ void stage_params(float4 *params, const Args &a, const Place &q, float factor,
                                             const T *gate = nullptr) {
  if (q.group == 0) {
    if (sizeof(T) == 4 || a.p.param_dtype != P3D_F32)
      stage_params_of<T, T, ALIGNED, BLOCK, CENTER, FOLD, NU, LANES>(params, a, q, factor, gate);
    else
      stage_params_of<float, T, ALIGNED, BLOCK, CENTER, FOLD, NU, LANES>(params, a, q, factor, gate);
  }
  if (a.groups > 1) __syncthreads();   // otherwise every thread reads what it wrote
}
template <int NU>   // k: the vector's place
__device__ __forceinline__ void param(float2 (&f)[4 * NU], const float4 *params, int k, const Place &q) {
#pragma unroll
  for (int n = 0; n < NU; ++n) {
    const float4 *from = params + 2 * (k * NU + n) * q.threads + q.t;
    const float4 x = from[0], y = from[q.threads];
    f[4 * n] = make_float2(x.x, x.y);
    f[4 * n + 1] = make_float2(x.z, x.w);
    f[4 * n + 2] = make_float2(y.x, y.y);
    f[4 * n + 3] = make_float2(y.z, y.w);
  }
}

// act'(gate) from act(gate)
__device__ __forceinline__ float slope(float a, int act) {
  return act == P3D_ACT_IDENTITY ? 1.f : act == P3D_ACT_SIGMOID ? a * (1.f - a) : fmaf(-a, a, 1.f);
}
// d act'(gate) from act(gate) over a thread's columns
template <int N>
__device__ __forceinline__ void times_slope(float2 (&d)[N], const float2 (&a)[N], int act) {
  if (act == P3D_ACT_IDENTITY) return;
#pragma unroll
  for (int i = 0; i < N; ++i)
    d[i] = mul2(d[i], act == P3D_ACT_SIGMOID ? mul2(a[i], sub2(splat(1.f), a[i]))
                                             : fma2(mul2(a[i], splat(-1.f)), a[i], splat(1.f)));
}

// Keep decisions of the thread's columns of a row: aligned, its units' random words; unaligned threads own a column
// of each of many blocks, so the lanes of a row (of a warp's run of columns) make a block's decisions
// each and pass them through shared memory as bits.
template <bool ALIGNED, int NU, int LANES>
struct RowKeep {
  uint32_t w[ALIGNED ? 4 * NU : 1];

  __device__ __forceinline__ void draw(const Args &a, const Place &q, const Keep &keep, const RoundKeys &key, int64_t row,
                                       uint8_t *shared) {
    const uint64_t row_block = (uint64_t)row * (uint32_t)((a.p.dim + 7) / 8) + (uint32_t)(q.first / 8);
    if constexpr (ALIGNED) {
#pragma unroll
      for (int n = 0; n < NU; ++n) keep.words(key, row_block + q.at[n] / 8, w + 4 * n);
    } else {
      const int lane = LANES < 32 ? q.t : q.lane, run = q.base - lane;   // the run's first column
      shared += (LANES < 32 ? q.sub : q.warp) * LANES * NU;
      __syncwarp();   // the row before is done with the bits
#pragma unroll
      for (int n = 0; n < NU; ++n) {
        const int b = lane + n * LANES;
        if (run + 8 * b < q.end) shared[b] = (uint8_t)keep.bits(key, row_block + run / 8 + b);
      }
      __syncwarp();
      w[0] = 0;
#pragma unroll
      for (int j = 0; j < kUnit * NU; ++j) {
        const int c = lane + j * LANES;
        if (j < q.count) w[0] |= ((uint32_t)(shared[c >> 3] >> (c & 7)) & 1u) << j;
      }
    }
  }
  // v with what is dropped of columns 2 i and 2 i + 1 set to zero
  __device__ __forceinline__ float2 operator()(const Keep &keep, int i, float2 v) const {
    const bool lo = ALIGNED ? keep.low(w[ALIGNED ? i : 0]) : (w[0] >> (2 * i) & 1u);
    const bool hi = ALIGNED ? keep.high(w[ALIGNED ? i : 0]) : (w[0] >> (2 * i + 1) & 1u);
    return make_float2(lo ? v.x : 0.f, hi ? v.y : 0.f);
  }
};

// (mean, 1/deviation) of a row
template <bool ALIGNED, bool CENTER, int NU, int LANES>
__device__ __forceinline__ float2 row_stats(RowSum<LANES> &sum, const Place &q, const float2 (&z)[4 * NU], int kind, float eps,
                                            float inv_dim) {
  if (CENTER && kind == P3D_NORM_LAYER) {
    const float2 m = sum.template moments<ALIGNED, NU>(q, z, inv_dim);
    return make_float2(m.x, rsqrtf(fmaf(m.y, inv_dim, eps)));
  }
  float2 s[NU];
#pragma unroll
  for (int n = 0; n < NU; ++n) {
    s[n] = mul2(z[4 * n], z[4 * n]);
#pragma unroll
    for (int i = 1; i < 4; ++i) s[n] = fma2(z[4 * n + i], z[4 * n + i], s[n]);
  }
  float v[1] = {total<ALIGNED, NU>(q, s)};
  sum(q, v);
  return make_float2(0.f, rsqrtf(fmaf(v[0], inv_dim, eps)));
}

// ------------------------------------------------------------------------ forward
// WHOLE: both norms are there.  CENTER: a layer norm or a bias somewhere.
template <typename T, bool ALIGNED, int LANES, int NU, bool BLOCK, bool WHOLE, bool DROP, bool CENTER>
__global__ void __launch_bounds__(256, NU == 1 ? 4 : 2) fwd_kernel(const __grid_constant__ Args a) {
  const p3d_residual &p = a.p;
  extern __shared__ __align__(128) char s_data[];
  __shared__ Shared s;
  constexpr int kRows = 32 / LANES;   // of a warp at once
  const Place q = place_of<LANES, ALIGNED, NU>(a);
  RowSum<LANES> sum{&s.exchange, a.members};
  const int cta = blockIdx.x / a.members, ctas = gridDim.x / a.members;
  float4 *const params = reinterpret_cast<float4 *>(s_data);
  if constexpr (DROP) s.keys.set(philox_key(p.rng, p.seed, p.offset));
  auto ring = start_ring<T, ALIGNED, NU, false>(
      a, q, &s, s_data + (size_t)2 * param_count(BLOCK, CENTER) * NU * q.threads * sizeof(float4), cta, ctas);
  const Keep keep(p.threshold);
  const float drop_scale = DROP ? keep_scale(p.threshold) : 1.f, inv_dim = 1.f / (float)q.dim;
  const bool folded = BLOCK && a.gate_folded;   // the segments are samples, whose gate the parameters hold
  const int gate_mode = folded ? P3D_GATE_NONE : p.gate_mode;
  const bool post_norm = WHOLE || p.post_kind != P3D_NORM_NONE, next_norm = WHOLE || p.next_kind != P3D_NORM_NONE;
  const Batches first_batch = batches_of(a, q.group, cta, ctas);
#pragma unroll 1
  for (int seg = cta / a.slices; seg < a.segments; seg += first_batch.seg_step) {
    if (a.groups > 1 && seg != cta / a.slices) __syncthreads();   // the groups are done with the sample before
    stage_params<T, ALIGNED, BLOCK, CENTER, BLOCK, NU, LANES>(
        params, a, q, drop_scale, folded ? static_cast<const T *>(p.gate) + (int64_t)seg * q.dim : nullptr);
    Batches k = first_batch;
    k.seg = seg;
#pragma unroll 1
    for (k.enter(a); k.row < k.end; k.row += k.stride) {
      const char *at = ring.wait(a);
      const bool ok = sum.ok = ring.state.ok;
      const int n = k.count(a), row0 = k.row;
      bool refilled = false;
      auto refill = [&] {   // every thread of the group has left the batch before
        if (!refilled && q.warp == 0) ring.issue(a, q);
        refilled = true;
      };
#pragma unroll 1
      for (int i0 = 0; i0 < n; i0 += kRows) {
        // past the batch's end a lane group goes over its last row again, without storing
        const bool valid = ok && (LANES == 32 || i0 + q.sub < n);
        const int i = LANES == 32 ? i0 : min(i0 + q.sub, n - 1);
        const int64_t row = row0 + i, base = row * q.dim + q.first;
        float2 z[4 * NU], w[4 * NU], b[4 * NU];
        float2 post = make_float2(0.f, 1.f), next = make_float2(0.f, 1.f);
        if constexpr (BLOCK) {
          float2 u[4 * NU], g[4 * NU];
          load_cols<T, ALIGNED, NU, LANES>(u, ring.row_ptr(a, q, at, kH, row0, n, i), q);
          if (gate_mode == P3D_GATE_ELEMENT) load_cols<T, ALIGNED, NU, LANES>(g, ring.row_ptr(a, q, at, kGate, row0, n, i), q);
          if (gate_mode == P3D_GATE_SAMPLE)
            load_cols<T, ALIGNED, NU, LANES>(
                g, static_cast<const T *>(p.gate) + (int64_t)((int)row / (int)p.rows_per_sample) * q.dim + q.first, q);
          float token = 1.f;
          if (gate_mode == P3D_GATE_TOKEN) token = activate<T>(to_f32<T>(static_cast<const T *>(p.gate)[row]), p.gate_act);
          if (post_norm) {
            post = row_stats<ALIGNED, CENTER, NU>(sum, q, u, p.post_kind, p.post_eps, inv_dim);
            refill();
          }
          // without a post norm u itself: mean 0, 1/deviation 1
          param<NU>(w, params, param_slot(BLOCK, kPostW), q);
          if constexpr (CENTER) param<NU>(b, params, param_slot(BLOCK, kPostB), q);
#pragma unroll
          for (int j = 0; j < 4 * NU; ++j) {
            if constexpr (CENTER) u[j] = fma2(mul2(sub2(u[j], splat(post.x)), splat(post.y)), w[j], b[j]);
            else u[j] = mul2(mul2(u[j], splat(post.y)), w[j]);
          }
          if (gate_mode == P3D_GATE_TOKEN) {
#pragma unroll
            for (int j = 0; j < 4 * NU; ++j) u[j] = mul2(u[j], splat(token));
          } else if (gate_mode != P3D_GATE_NONE) {
            activate_all<T>(g, p.gate_act);
#pragma unroll
            for (int j = 0; j < 4 * NU; ++j) u[j] = mul2(u[j], g[j]);
          }
          if constexpr (DROP) {
            RowKeep<ALIGNED, NU, LANES> kept;
            kept.draw(a, q, keep, s.keys, row, s.keep + q.group * a.row_threads * NU);
#pragma unroll
            for (int j = 0; j < 4 * NU; ++j) u[j] = kept(keep, j, u[j]);
          }
          load_cols<T, ALIGNED, NU, LANES>(z, ring.row_ptr(a, q, at, kX, row0, n, i), q);
#pragma unroll
          for (int j = 0; j < 4 * NU; ++j) {
            z[j] = add2(u[j], z[j]);
            if constexpr (!ALIGNED) {
              if (2 * j >= q.count) z[j].x = 0.f;
              if (2 * j + 1 >= q.count) z[j].y = 0.f;
            }
          }
          store_cols<T, ALIGNED, NU, LANES>(static_cast<T *>(a.out) + base, z, q, valid);
        } else {
          load_cols<T, ALIGNED, NU, LANES>(z, ring.row_ptr(a, q, at, kX, row0, n, i), q);
        }
        if (next_norm) {
          next = row_stats<ALIGNED, CENTER, NU>(sum, q, z, p.next_kind, p.next_eps, inv_dim);
          refill();
          param<NU>(w, params, param_slot(BLOCK, kNextW), q);
          if constexpr (CENTER) param<NU>(b, params, param_slot(BLOCK, kNextB), q);
#pragma unroll
          for (int j = 0; j < 4 * NU; ++j) {
            if constexpr (CENTER) z[j] = fma2(mul2(sub2(z[j], splat(next.x)), splat(next.y)), w[j], b[j]);
            else z[j] = mul2(mul2(z[j], splat(next.y)), w[j]);
          }
          store_cols<T, ALIGNED, NU, LANES>(static_cast<T *>(a.y) + base, z, q, valid);
        }
        if (a.stats && q.t == 0 && q.rank == 0 && valid)
          reinterpret_cast<float4 *>(a.stats)[row] = make_float4(post.x, post.y, next.x, next.y);
      }
      if (!refilled) {
        q.barrier();
        refill();
      }
    }
  }
  ring.finish(a, q);
}

// ------------------------------------------------------------------------ backward
constexpr int kSums = 6;  // written: dscale, dpost_weight, dpost_bias, dnext_weight, dnext_bias, dgate

// The thread's sums added over the CTA's row groups (in group order), complete in the first group; they start again at 0.
__device__ __forceinline__ void join_groups(float2 (&acc)[4], float *smem, const Args &a, const Place &q) {
  if (a.groups > 1) {
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      smem[(q.group * kUnit + 2 * j) * a.row_threads + q.t] = acc[j].x;
      smem[(q.group * kUnit + 2 * j + 1) * a.row_threads + q.t] = acc[j].y;
    }
    __syncthreads();
    if (q.group == 0) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        for (int g = 1; g < a.groups; ++g)
          acc[j] = add2(acc[j], make_float2(smem[(g * kUnit + 2 * j) * a.row_threads + q.t],
                                            smem[(g * kUnit + 2 * j + 1) * a.row_threads + q.t]));
    }
  }
}
// The thread's columns of a row of sums in global memory.
template <bool ALIGNED>
__device__ __forceinline__ void get_sums(float2 (&v)[4], const float *src, const Place &q) {
  if constexpr (ALIGNED) {
    const float4 *from = reinterpret_cast<const float4 *>(src + q.first + q.at[0]);
    const float4 x = from[0], y = from[1];
    v[0] = make_float2(x.x, x.y);
    v[1] = make_float2(x.z, x.w);
    v[2] = make_float2(y.x, y.y);
    v[3] = make_float2(y.z, y.w);
  } else {
    float f[kUnit];
#pragma unroll
    for (int j = 0; j < kUnit; ++j) {
      const int c = q.col<ALIGNED, 32>(j);
      f[j] = c < q.end ? src[q.first + c] : 0.f;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = make_float2(f[2 * j], f[2 * j + 1]);
  }
}
template <bool ALIGNED>
__device__ __forceinline__ void put_sums(const float2 (&v)[4], float *dst, const Place &q) {
  if constexpr (ALIGNED) {
    float4 *to = reinterpret_cast<float4 *>(dst + q.first + q.at[0]);
    if (q.live[0]) {
      to[0] = make_float4(v[0].x, v[0].y, v[1].x, v[1].y);
      to[1] = make_float4(v[2].x, v[2].y, v[3].x, v[3].y);
    }
  } else {
#pragma unroll
    for (int j = 0; j < kUnit; ++j) {
      const int c = q.col<ALIGNED, 32>(j);
      if (c < q.end) dst[q.first + c] = j & 1 ? v[j / 2].y : v[j / 2].x;
    }
  }
}

// WHOLE: both norms, both upstream gradients and both gradients of tensors are there.
template <typename T, bool ALIGNED, bool BLOCK, bool WHOLE, int GATE, bool DROP, bool CENTER>
__global__ void __launch_bounds__(512, BLOCK ? 1 : 2) bwd_kernel(const __grid_constant__ Args a) {
  constexpr bool kSampled = BLOCK && (GATE == kGateAny || GATE == P3D_GATE_SAMPLE);
  constexpr bool kTokens = BLOCK && GATE == P3D_GATE_TOKEN;
  constexpr bool kElements = BLOCK && (GATE == kGateAny || GATE == P3D_GATE_ELEMENT);   // act and v = d / act a column
  const p3d_residual &p = a.p;
  extern __shared__ __align__(128) char s_data[];
  __shared__ Shared s;
  const Place q = place_of<32, ALIGNED, 1>(a);
  RowSum<32> sum{&s.exchange, a.members};
  const int cta = blockIdx.x / a.members, ctas = gridDim.x / a.members;
  float4 *const params = reinterpret_cast<float4 *>(s_data);
  if constexpr (DROP) s.keys.set(philox_key(p.rng, p.seed, p.offset));
  auto ring = start_ring<T, ALIGNED, 1, true>(
      a, q, &s, s_data + (size_t)2 * param_count(BLOCK, CENTER) * a.row_threads * sizeof(float4), cta, ctas);
  float *joins = reinterpret_cast<float *>(ring.data + (size_t)(a.groups - q.group) * a.stages * a.stage_bytes);
  // the dropout's scale is folded into the post norm's weight and bias, and into their gradients' sums at the end
  const Keep keep(p.threshold);
  const float drop_scale = DROP ? keep_scale(p.threshold) : 1.f;
  stage_params<T, ALIGNED, BLOCK, CENTER, false, 1, 32>(params, a, q, drop_scale);
  const float inv_dim = 1.f / (float)q.dim;
  const int gate_mode = GATE == kGateAny ? p.gate_mode : GATE;
  const bool next_sums = WHOLE || a.in[kDy], has_dout = WHOLE || a.in[kDout];
  const bool post_norm = WHOLE || p.post_kind != P3D_NORM_NONE, token = (kTokens || kElements) && gate_mode == P3D_GATE_TOKEN;
  const bool want_dx = WHOLE || a.dx, want_dh = WHOLE || a.dh;
  // means of the normalised rows' gradients: nothing to take off where there is no norm, no mean in an RMS norm
  const float next_mean = p.next_kind == P3D_NORM_LAYER ? -inv_dim : 0.f;
  const float post_mean = p.post_kind == P3D_NORM_LAYER ? -inv_dim : 0.f, post_dot = post_norm ? -inv_dim : 0.f;
  // K: the gradient of d = s (u act) where it was kept, and a gate's part of it that changes from row to row
  float2 a_kh[4] = {}, a_k[4] = {}, a_nw[4] = {}, a_nb[4] = {};   // sums of K h~, K, dy z~, dy
  float *const mine = a.partials + (int64_t)cta * q.dim;
  const int64_t one_sum = (int64_t)ctas * q.dim;
  const Batches first_batch = batches_of(a, q.group, cta, ctas);
  // sums over rows that did not all arrive are NaN
  auto mark = [&](float2 (&v)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = ring.state.ok ? v[j] : splat(nan());
  };
#pragma unroll 1
  for (int seg = cta / a.slices; seg < a.segments; seg += first_batch.seg_step) {
    const T *const sample = static_cast<const T *>(p.gate) + (int64_t)seg * q.dim + q.first;
    // d of a row is h~ e_w + e_b, times a gate that changes from row to row
    float2 e_w[4], e_b[4];
    if constexpr (BLOCK) {
      float2 f[4];
      param<1>(e_w, params, param_slot(BLOCK, kPostW), q);
      if constexpr (CENTER) param<1>(e_b, params, param_slot(BLOCK, kPostB), q);
      param<1>(f, params, param_slot(BLOCK, kScale), q);
      if (kSampled && gate_mode == P3D_GATE_SAMPLE) {
        float2 g[4];
        load_cols<T, ALIGNED, 1, 32>(g, sample, q);
        activate_all<T>(g, p.gate_act);
#pragma unroll
        for (int j = 0; j < 4; ++j) f[j] = mul2(f[j], g[j]);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        e_w[j] = mul2(e_w[j], f[j]);
        if constexpr (CENTER) e_b[j] = mul2(e_b[j], f[j]);
      }
    }
    Batches k = first_batch;
    k.seg = seg;
#pragma unroll 1
    for (k.enter(a); k.row < k.end; k.row += k.stride) {
      const char *at = ring.wait(a);
      const bool ok = sum.ok = ring.state.ok;
      const int n = k.count(a), row0 = k.row;
      bool refilled = false;
      auto refill = [&] {
        if (!refilled && q.warp == 0) ring.issue(a, q);
        refilled = true;
      };
#pragma unroll 1
      for (int i = 0; i < n; ++i) {
        const int64_t row = row0 + i, base = row * q.dim + q.first;
        const float4 st = ring.stats(a, at, i);   // mean, 1/deviation of h, then of out
        float2 w[4], v[4], hn[4], act[4], zn[4], G[4];
        float gate = 1.f;   // the token's
        RowKeep<ALIGNED, 1, 32> kept;
        if constexpr (BLOCK) {
          load_cols<T, ALIGNED, 1, 32>(hn, ring.row_ptr(a, q, at, kH, row0, n, i), q);
          if constexpr (DROP) kept.draw(a, q, keep, s.keys, row, s.keep + q.group * a.row_threads);
          if (token) gate = activate<T>(to_f32<T>(static_cast<const T *>(p.gate)[row]), p.gate_act);
          if constexpr (kElements) {
            if (gate_mode == P3D_GATE_ELEMENT) {
              load_cols<T, ALIGNED, 1, 32>(act, ring.row_ptr(a, q, at, kGate, row0, n, i), q);
              activate_all<T>(act, p.gate_act);
            } else {
#pragma unroll
              for (int j = 0; j < 4; ++j) act[j] = splat(gate);
            }
            if constexpr (DROP) {   // an infinite gate too: 0 * inf would reach out, made again, and the sums
#pragma unroll
              for (int j = 0; j < 4; ++j) act[j] = kept(keep, j, act[j]);
            }
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if constexpr (CENTER) hn[j] = sub2(hn[j], splat(st.x));
            hn[j] = mul2(hn[j], splat(st.y));      // h itself without a post norm: mean 0, 1/deviation 1
            v[j] = CENTER ? fma2(hn[j], e_w[j], e_b[j]) : mul2(hn[j], e_w[j]);
            if constexpr (DROP) v[j] = kept(keep, j, v[j]);
          }
        }
        if (has_dout) load_cols<T, ALIGNED, 1, 32>(G, ring.row_ptr(a, q, at, kDout, row0, n, i), q);
        else
#pragma unroll
          for (int j = 0; j < 4; ++j) G[j] = splat(0.f);
        if (next_sums) {
          float2 gy[4], s0[1], s1[1];
          load_cols<T, ALIGNED, 1, 32>(zn, ring.row_ptr(a, q, at, kX, row0, n, i), q);
          load_cols<T, ALIGNED, 1, 32>(gy, ring.row_ptr(a, q, at, kDy, row0, n, i), q);
          if constexpr (BLOCK) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              zn[j] = kElements ? fma2(v[j], act[j], zn[j]) : kTokens ? fma2(v[j], splat(gate), zn[j]) : add2(v[j], zn[j]);
          }
          param<1>(w, params, param_slot(BLOCK, kNextW), q);
          s0[0] = s1[0] = splat(0.f);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if constexpr (CENTER) zn[j] = sub2(zn[j], splat(st.z));
            zn[j] = mul2(zn[j], splat(st.w));
            a_nw[j] = fma2(gy[j], zn[j], a_nw[j]);
            if constexpr (CENTER) a_nb[j] = add2(a_nb[j], gy[j]);
            gy[j] = mul2(gy[j], w[j]);
            s1[0] = fma2(gy[j], zn[j], s1[0]);
            if constexpr (CENTER) s0[0] = add2(s0[0], gy[j]);
          }
          float m0 = 0.f, m1;
          if constexpr (CENTER) {
            float v[2] = {total<ALIGNED, 1>(q, s1), total<ALIGNED, 1>(q, s0)};
            sum(q, v);
            m1 = v[0] * -inv_dim;
            m0 = v[1] * next_mean;
          } else {
            float v[1] = {total<ALIGNED, 1>(q, s1)};
            sum(q, v);
            m1 = v[0] * -inv_dim;
          }
          refill();
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            float2 t = fma2(zn[j], splat(m1), gy[j]);
            if constexpr (CENTER) t = add2(t, splat(m0));
            G[j] = fma2(t, splat(st.w), G[j]);
            if constexpr (!ALIGNED) {   // no column: nothing for the sums below
              if (2 * j >= q.count) G[j].x = 0.f;
              if (2 * j + 1 >= q.count) G[j].y = 0.f;
            }
          }
        }
        if (want_dx) store_cols<T, ALIGNED, 1, 32>(static_cast<T *>(a.dx) + base, G, q, ok);
        if constexpr (BLOCK) {
          float2 s0[1], s1[1], s2[1];
          s0[0] = s1[0] = s2[0] = splat(0.f);
          if constexpr (kElements) {   // zn is free: the gate's gradient
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              zn[j] = mul2(G[j], v[j]);
              G[j] = mul2(G[j], act[j]);
            }
            times_slope(zn, act, p.gate_act);
            if (gate_mode == P3D_GATE_ELEMENT && a.dgate)
              store_cols<T, ALIGNED, 1, 32>(static_cast<T *>(a.dgate) + base, zn, q, ok);
          }
          // G becomes K e_w (a token's gate left out until the end)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if constexpr (DROP) G[j] = kept(keep, j, G[j]);
            const float2 K = kTokens ? mul2(G[j], splat(gate)) : G[j];
            // what is dropped adds nothing, an infinite h~ included
            if constexpr (DROP) a_kh[j] = fma2(K, kept(keep, j, hn[j]), a_kh[j]);
            else a_kh[j] = fma2(K, hn[j], a_kh[j]);
            if constexpr (CENTER) a_k[j] = add2(a_k[j], K);
            if constexpr (GATE == kGateAny) s2[0] = add2(s2[0], zn[j]);
            if constexpr (kTokens && CENTER) s2[0] = fma2(G[j], e_b[j], s2[0]);
            G[j] = mul2(G[j], e_w[j]);
            s1[0] = fma2(G[j], hn[j], s1[0]);
            if constexpr (CENTER) s0[0] = add2(s0[0], G[j]);
          }
          float m0 = 0.f, m1 = 0.f;
          if (post_norm || token) {
            float dgate = 0.f;   // the token's: the sum of G v is that of G e_w h~ and of G e_b
            if constexpr (CENTER && (GATE == kGateAny || kTokens)) {
              float v[3] = {total<ALIGNED, 1>(q, s1), total<ALIGNED, 1>(q, s0), total<ALIGNED, 1>(q, s2)};
              sum(q, v);
              m1 = v[0] * post_dot;
              m0 = v[1] * post_mean;
              dgate = kTokens ? (v[0] + v[2]) * slope(gate, p.gate_act) : v[2];
            } else if constexpr (GATE == kGateAny) {
              float v[2] = {total<ALIGNED, 1>(q, s1), total<ALIGNED, 1>(q, s2)};
              sum(q, v);
              m1 = v[0] * post_dot;
              dgate = v[1];
            } else if constexpr (CENTER) {
              float v[2] = {total<ALIGNED, 1>(q, s1), total<ALIGNED, 1>(q, s0)};
              sum(q, v);
              m1 = v[0] * post_dot;
              m0 = v[1] * post_mean;
            } else {
              float v[1] = {total<ALIGNED, 1>(q, s1)};
              sum(q, v);
              m1 = v[0] * post_dot;
              if constexpr (kTokens) dgate = v[0] * slope(gate, p.gate_act);
            }
            if (token && a.dgate && q.t == 0 && q.rank == 0 && ok) static_cast<T *>(a.dgate)[row] = from_f32<T>(dgate);
            refill();
          }
          if (want_dh) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              if (post_norm) {   // otherwise h, which may be infinite, has no part in its gradient
                G[j] = fma2(hn[j], splat(m1), G[j]);
                if constexpr (CENTER) G[j] = add2(G[j], splat(m0));
              }
              G[j] = mul2(G[j], splat(kTokens ? st.y * gate : st.y));
            }
            store_cols<T, ALIGNED, 1, 32>(static_cast<T *>(a.dh) + base, G, q, ok);
          }
        }
      }
      if (!refilled) {
        q.barrier();
        refill();
      }
    }
    // The block's gradients from the two sums: with A = w sum K h~ + b sum K (the sum of K u), dscale = A, dw = s sum
    // K h~, db = s sum K.  A sample's gate is not in K: dgate = s A act', and the others times act.
    if constexpr (BLOCK) {
      // what the CTA's samples before have summed up to, on its way while the groups are joined
      float2 was[3][4] = {};
      if (kSampled && seg != cta / a.slices && q.group == 0) {
#pragma unroll
        for (int i = 0; i < (CENTER ? 3 : 2); ++i) get_sums<ALIGNED>(was[i], mine + i * one_sum, q);
      }
      mark(a_kh);
      join_groups(a_kh, joins, a, q);
      if constexpr (CENTER) {
        mark(a_k);
        join_groups(a_k, joins, a, q);
      }
      if (q.group == 0) {
        const bool sampled = kSampled && gate_mode == P3D_GATE_SAMPLE;
        float2 w[4], f[4], A[4];
        param<1>(w, params, param_slot(BLOCK, kPostW), q);
        param<1>(f, params, param_slot(BLOCK, kScale), q);
#pragma unroll
        for (int j = 0; j < 4; ++j) A[j] = mul2(w[j], a_kh[j]);
        if constexpr (CENTER) {
          param<1>(w, params, param_slot(BLOCK, kPostB), q);
#pragma unroll
          for (int j = 0; j < 4; ++j) A[j] = fma2(w[j], a_k[j], A[j]);
        }
        if (sampled) {
          float2 g[4], dgate[4];
          load_cols<T, ALIGNED, 1, 32>(g, sample, q);
          activate_all<T>(g, p.gate_act);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            dgate[j] = mul2(f[j], A[j]);
            A[j] = mul2(A[j], g[j]);
            f[j] = mul2(f[j], g[j]);
          }
          times_slope(dgate, g, p.gate_act);
          if (a.dgate)
            put_sums<ALIGNED>(dgate, a.partials + (kSums - 1) * one_sum + ((int64_t)seg * a.slices + cta % a.slices) * q.dim,
                              q);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          f[j] = mul2(f[j], splat(drop_scale));
          A[j] = add2(was[0][j], A[j]);
          a_kh[j] = fma2(a_kh[j], f[j], was[1][j]);
          if constexpr (CENTER) a_k[j] = fma2(a_k[j], f[j], was[2][j]);
        }
        // the slots of sums that a variant does not have are not read either
        put_sums<ALIGNED>(A, mine, q);
        put_sums<ALIGNED>(a_kh, mine + one_sum, q);
        if constexpr (CENTER) put_sums<ALIGNED>(a_k, mine + 2 * one_sum, q);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) a_kh[j] = a_k[j] = splat(0.f);
    }
  }
  mark(a_nw);
  join_groups(a_nw, joins, a, q);
  if (q.group == 0) put_sums<ALIGNED>(a_nw, mine + 3 * one_sum, q);
  if constexpr (CENTER) {
    mark(a_nb);
    join_groups(a_nb, joins, a, q);
    if (q.group == 0) put_sums<ALIGNED>(a_nb, mine + 4 * one_sum, q);
  }
  ring.finish(a, q);
}

// ------------------------------------------------------------------------ launches
template <typename K>
int launch(K kernel, const Args &a, int64_t ctas, size_t smem, size_t (&seen)[kMaxDevices], cudaStream_t stream) {
  // always the same amount: calls of several threads then cannot lower each other's
  if (int st = smem_optin(kernel, std::max<size_t>(smem, 224 * 1024), seen)) return st;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(ctas * a.members));
  cfg.blockDim = dim3((unsigned)(a.row_threads * a.groups));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)a.members;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = a.members > 1 ? 1 : 0;
  P3D_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, a));
  return P3D_OK;
}

template <typename T, bool ALIGNED, int LANES, int NU, bool BLOCK, bool WHOLE, bool DROP, bool CENTER>
int fwd(const Args &a, int64_t ctas, size_t smem, cudaStream_t s) {
  static size_t seen[kMaxDevices] = {};
  return launch(fwd_kernel<T, ALIGNED, LANES, NU, BLOCK, WHOLE, DROP, CENTER>, a, ctas, smem, seen, s);
}
template <typename T, bool ALIGNED, bool BLOCK, bool WHOLE, int GATE, bool DROP, bool CENTER>
int bwd(const Args &a, int64_t ctas, size_t smem, cudaStream_t s) {
  static size_t seen[kMaxDevices] = {};
  return launch(bwd_kernel<T, ALIGNED, BLOCK, WHOLE, GATE, DROP, CENTER>, a, ctas, smem, seen, s);
}

// Calls f with `b` as a constant.
template <typename F>
int with(bool b, F &&f) {
  return b ? f(std::true_type{}) : f(std::false_type{});
}
// Calls f with the gate's mode as a constant.
template <typename F>
int with_gate(int mode, F &&f) {
  switch (mode) {
    case P3D_GATE_NONE: return f(std::integral_constant<int, P3D_GATE_NONE>{});
    case P3D_GATE_ELEMENT: return f(std::integral_constant<int, P3D_GATE_ELEMENT>{});
    case P3D_GATE_SAMPLE: return f(std::integral_constant<int, P3D_GATE_SAMPLE>{});
    default: return f(std::integral_constant<int, P3D_GATE_TOKEN>{});
  }
}

// Calls that have no block, or a block between two norms (in the backward with all gradients), have
// variants of their own; the other aligned ones share one that centres.
inline bool whole_fwd(const Args &a) {
  return !a.p.h || (a.p.post_kind != P3D_NORM_NONE && a.p.next_kind != P3D_NORM_NONE);
}
inline bool whole_bwd(const Args &a) {
  return !a.p.h || (a.p.post_kind != P3D_NORM_NONE && a.in[kDy] && a.in[kDout] && a.dx && a.dh);
}

// Aligned rows between two norms, the usual block, get variants of their own for dropout, centring and (in the
// backward) the gate: each
// saves registers or instructions of a kernel that is bound by both.  Other calls share variants that read
// what they have from the arguments.
template <typename T, int LANES, int NU>
int fwd_of(const Args &a, bool aligned, bool center, int64_t ctas, size_t smem, cudaStream_t s) {
  return with(center, [&](auto ce) {
    constexpr bool C = decltype(ce)::value;
    if (!a.p.h)
      return aligned ? fwd<T, true, LANES, NU, false, false, false, C>(a, ctas, smem, s)
                     : fwd<T, false, LANES, NU, false, false, false, C>(a, ctas, smem, s);
    if (aligned && !whole_fwd(a)) return fwd<T, true, LANES, NU, true, false, true, true>(a, ctas, smem, s);
    return with(a.p.threshold != 0, [&](auto dr) {
      constexpr bool D = decltype(dr)::value;
      return aligned ? fwd<T, true, LANES, NU, true, true, D, C>(a, ctas, smem, s)
                     : fwd<T, false, LANES, NU, true, false, D, C>(a, ctas, smem, s);
    });
  });
}
// lanes, units: of the forward's layout, as shape_of chooses them.
template <typename T>
int run_fwd(const Args &a, bool aligned, bool center, int lanes, int units, int64_t ctas, size_t smem, cudaStream_t s) {
  if (lanes == 8 && units == 1) return fwd_of<T, 8, 1>(a, aligned, center, ctas, smem, s);
  if (lanes == 8) return fwd_of<T, 8, 3>(a, aligned, center, ctas, smem, s);
  if (lanes == 16) return fwd_of<T, 16, 3>(a, aligned, center, ctas, smem, s);
  return fwd_of<T, 32, 2>(a, aligned, center, ctas, smem, s);
}

template <typename T>
int run_bwd(const Args &a, bool aligned, bool center, int64_t ctas, size_t smem, cudaStream_t s) {
  const bool whole = aligned && whole_bwd(a);
  return with(center, [&](auto ce) {
    constexpr bool C = decltype(ce)::value;
    if (!a.p.h)
      return aligned ? bwd<T, true, false, false, P3D_GATE_NONE, false, C>(a, ctas, smem, s)
                     : bwd<T, false, false, false, P3D_GATE_NONE, false, C>(a, ctas, smem, s);
    if (!whole) {
      if (aligned) return bwd<T, true, true, false, kGateAny, true, true>(a, ctas, smem, s);
      return with(a.p.gate_mode != P3D_GATE_NONE, [&](auto ga) {
        return with(a.p.threshold != 0, [&](auto dr) {
          return bwd<T, false, true, false, decltype(ga)::value ? kGateAny : P3D_GATE_NONE, decltype(dr)::value, C>(
              a, ctas, smem, s);
        });
      });
    }
    return with_gate(a.p.gate_mode, [&](auto ga) {
      return with(a.p.threshold != 0, [&](auto dr) {
        return bwd<T, true, true, true, decltype(ga)::value, decltype(dr)::value, C>(a, ctas, smem, s);
      });
    });
  });
}

template <typename T>
int take_errors(unsigned *flags) {
  unsigned v = 0, zero = 0;
  P3D_CUDA_TRY(cudaMemcpyFromSymbol(&v, g_row_errors, sizeof(v)));
  P3D_CUDA_TRY(cudaMemcpyToSymbol(g_row_errors, &zero, sizeof(zero)));
  *flags |= v;
  return P3D_OK;
}

#define P3D_ROW_KERNELS(T)                                                                        \
  template int run_fwd<T>(const Args &, bool, bool, int, int, int64_t, size_t, cudaStream_t);      \
  template int run_bwd<T>(const Args &, bool, bool, int64_t, size_t, cudaStream_t);               \
  template int take_errors<T>(unsigned *);

}  // namespace rows
}  // namespace p3d
