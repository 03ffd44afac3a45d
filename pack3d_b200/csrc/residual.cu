// The feed-forward half of a block around its matrix products: dropout, and the norms before and
// after a block fused with its gate, dropout, residual scale and residual, with their backward.
//
// One pass over the data in each direction.  A row of `dim` columns is held in registers, eight
// columns a thread, by 32 to 512 threads (up to four CTAs of a cluster for dim > 4096), so the
// row statistics cost shuffles and no second read.  Bound by HBM: forward 4 (x, h, out, y) and
// backward 6 (x, h, dout, dy, dx, dh) values an element, plus the gate's.
//
// The backward makes out = x + s d again from x and h instead of reading the stored out: the same
// bytes, and the normalised row keeps its 32 bits (the stored one is rounded to 16).  Every
// thread keeps the column sums of its eight columns over all rows of its CTA in registers; they
// are joined over the CTA's row groups in shared memory, written once per CTA and summed over the
// CTAs by a second small kernel, all in a fixed order.
#include <algorithm>

#include "common.cuh"
#include "kernels.cuh"
#include "philox.cuh"

namespace p3d {
namespace {

constexpr int kUnit = 8;             // columns a thread owns
constexpr int kMaxRowThreads = 512;  // threads a row of one CTA
constexpr int kMaxDim = 16384;       // kUnit * kMaxRowThreads * 4 CTAs
constexpr int kSums = 6;             // dscale, dpost_weight, dpost_bias, dnext_weight, dnext_bias, dgate

// ------------------------------------------------------------------------ eight columns of a row
// Aligned: the thread's columns are consecutive and move in 16-byte pieces.  Otherwise (odd dim, or a
// pointer off 16 bytes) column j of the thread is `stride` columns after column j - 1, so that
// the lanes of a warp stay on consecutive elements.
template <typename T, bool ALIGNED>
struct Cols {
  T v[kUnit];
  __device__ __forceinline__ void load(const T *row, int col, int stride, int dim) {
    if constexpr (ALIGNED) {
      if (col < dim) {
        constexpr int n = sizeof(T) * kUnit / 16;
        uint4 raw[n];
#pragma unroll
        for (int i = 0; i < n; ++i) raw[i] = reinterpret_cast<const uint4 *>(row + col)[i];
        memcpy(v, raw, sizeof(v));
        return;
      }
#pragma unroll
      for (int j = 0; j < kUnit; ++j) v[j] = from_f32<T>(0.f);
    } else {
#pragma unroll
      for (int j = 0; j < kUnit; ++j) v[j] = col + j * stride < dim ? row[col + j * stride] : from_f32<T>(0.f);
    }
  }
  __device__ __forceinline__ void store(T *row, int col, int stride, int dim) const {
    if constexpr (ALIGNED) {
      if (col < dim) {
        constexpr int n = sizeof(T) * kUnit / 16;
        uint4 raw[n];
        memcpy(raw, v, sizeof(v));
#pragma unroll
        for (int i = 0; i < n; ++i) reinterpret_cast<uint4 *>(row + col)[i] = raw[i];
      }
    } else {
#pragma unroll
      for (int j = 0; j < kUnit; ++j)
        if (col + j * stride < dim) row[col + j * stride] = v[j];
    }
  }
  __device__ __forceinline__ float operator[](int j) const { return to_f32<T>(v[j]); }
  __device__ __forceinline__ void set(int j, float f) { v[j] = from_f32<T>(f); }
  __device__ __forceinline__ void fill(float f) {
#pragma unroll
    for (int j = 0; j < kUnit; ++j) v[j] = from_f32<T>(f);
  }
};

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Sums over the threads of one row.  A row group is `warps` warps of the CTA (group g of them),
// or all threads of all CTAs of the cluster.  Every thread gets the same total, added in the same
// order.  The shared slots alternate between calls: a thread two calls ahead has passed the
// barrier of the call between, so nobody still reads the slots it writes.
constexpr int kMaxCluster = 4;
template <bool CLUSTER>
struct RowSum {
  float (*slots)[16][4];     // [2][warps of the CTA][values]
  float (*peers)[kMaxCluster][4];  // [2][cta][values]
  int warps, group, warp, lane;
  int at = 0;

  template <int N>
  __device__ __forceinline__ void operator()(float (&v)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = warp_sum(v[i]);
    if (warps == 1 && !CLUSTER) return;
    if (warps > 1) {
      if (lane == 0) {
#pragma unroll
        for (int i = 0; i < N; ++i) slots[at][group * warps + warp][i] = v[i];
      }
      group_barrier();
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = warp_sum(lane < warps ? slots[at][group * warps + lane][i] : 0.f);
    }
    if constexpr (CLUSTER) {
      const uint32_t n = cluster_size(), me = cluster_rank();
      if (warp == 0 && lane < n) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const uint32_t mine = static_cast<uint32_t>(__cvta_generic_to_shared(&peers[at][me][i]));
          uint32_t theirs;
          asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(theirs) : "r"(mine), "r"(lane));
          asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(theirs), "f"(v[i]) : "memory");
        }
      }
      __syncwarp();
      cluster_sync();
#pragma unroll
      for (int i = 0; i < N; ++i) {
        v[i] = 0.f;
        for (uint32_t c = 0; c < n; ++c) v[i] += peers[at][c][i];
      }
    }
    at ^= 1;
  }
  __device__ __forceinline__ void group_barrier() const {
    asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(warps * 32) : "memory");
  }
};

// ------------------------------------------------------------------------ shared pieces
struct Args {
  p3d_residual p;
  void *out, *y;
  float *stats;
  const void *dout, *dy;
  void *dx, *dh, *dgate;
  float *partials;   // [sums 0..4 used][CTA slots][dim], then the sample gate's [samples][slices][dim]
  int row_threads, groups;
  int64_t segments, slices;  // the rows are `segments` runs (samples, or one), each cut into slices
  int64_t segment_rows;
};

__device__ __forceinline__ float activate(float g, int act) {
  if (act == P3D_ACT_SIGMOID) return 1.f / (1.f + expf(-g));
  if (act == P3D_ACT_TANH) return tanhf(g);
  return g;
}
// act'(gate) from act(gate)
__device__ __forceinline__ float slope(float a, int act) {
  if (act == P3D_ACT_SIGMOID) return a * (1.f - a);
  if (act == P3D_ACT_TANH) return 1.f - a * a;
  return 1.f;
}

// Keep bits of the thread's eight columns of a row.  Unaligned threads own a column of each of eight
// blocks: the row's threads make one block's bits each and pass them through shared memory.
template <bool ALIGNED, typename Sum>
__device__ __forceinline__ uint32_t row_keep(const p3d_residual &p, PhiloxKey key, int64_t row, int col, int stride,
                                             int first, int t, uint8_t *shared, const Sum &sum) {
  const uint64_t row_block = (uint64_t)row * (uint64_t)((p.dim + 7) / 8);
  if constexpr (ALIGNED) return col < p.dim ? keep_bits(key, row_block + col / 8, p.threshold) : 0u;
  else {
    if (sum.warps > 1) sum.group_barrier(); else __syncwarp();   // the row before is done with the bits
    if (first + t * 8 < p.dim) shared[t] = (uint8_t)keep_bits(key, row_block + first / 8 + t, p.threshold);
    if (sum.warps > 1) sum.group_barrier(); else __syncwarp();
    uint32_t bits = 0;
#pragma unroll
    for (int j = 0; j < kUnit; ++j) {
      const int local = col - first + j * stride;
      if (col + j * stride < p.dim) bits |= ((uint32_t)(shared[local >> 3] >> (local & 7)) & 1u) << j;
    }
    return bits;
  }
}

// Mean and 1/deviation of the row z.  Layer norm takes the mean first and then the squares about it
// (both from registers): one pass of sums and squares would cancel where the mean is large.
template <bool ALIGNED, typename Sum>
__device__ __forceinline__ float2 row_stats(const float (&z)[kUnit], int kind, float eps, int col, int stride, int dim,
                                            Sum &sum) {
  float mean = 0.f;
  if (kind == P3D_NORM_LAYER) {
    float s[1] = {0.f};
#pragma unroll
    for (int j = 0; j < kUnit; ++j) s[0] += z[j];
    sum(s);
    mean = s[0] / (float)dim;
  }
  float q[1] = {0.f};
#pragma unroll
  for (int j = 0; j < kUnit; ++j) {
    const float d = z[j] - mean;
    if (col + (ALIGNED ? 0 : j * stride) < dim) q[0] = fmaf(d, d, q[0]);
  }
  sum(q);
  return make_float2(mean, 1.f / sqrtf(q[0] / (float)dim + eps));
}

#define P3D_ROW_SETUP()                                                                                     \
  __shared__ float s_slots[2][16][4];                                                                       \
  __shared__ float s_peers[2][kMaxCluster][4];                                                              \
  __shared__ uint8_t s_keep[kMaxRowThreads];                                                                \
  const int group = threadIdx.x / a.row_threads, t = threadIdx.x % a.row_threads;                           \
  RowSum<CLUSTER> sum{s_slots, s_peers, a.row_threads / 32, group, t / 32, t % 32};                          \
  const int rank = CLUSTER ? (int)cluster_rank() : 0, members = CLUSTER ? (int)cluster_size() : 1;          \
  const int first = rank * a.row_threads * kUnit, dim = p.dim;                                              \
  const int col = ALIGNED ? first + t * kUnit : first + t, stride = ALIGNED ? 1 : a.row_threads;            \
  const PhiloxKey key = philox_key(p.threshold ? p.rng : nullptr, p.seed, p.offset);                        \
  const float drop_scale = p.threshold ? keep_scale(p.threshold) : 1.f;

// ------------------------------------------------------------------------ forward
template <typename T, typename P, bool ALIGNED, bool CLUSTER>
__global__ void __launch_bounds__(512) residual_fwd_kernel(const __grid_constant__ Args a) {
  const p3d_residual &p = a.p;
  P3D_ROW_SETUP();
  using C = Cols<T, ALIGNED>;
  Cols<P, ALIGNED> pw, pb, sc, nw, nb;
  pw.load(static_cast<const P *>(p.post_weight), p.post_weight ? col : dim, stride, dim);
  pb.load(static_cast<const P *>(p.post_bias), p.post_bias ? col : dim, stride, dim);
  nw.load(static_cast<const P *>(p.next_weight), p.next_weight ? col : dim, stride, dim);
  nb.load(static_cast<const P *>(p.next_bias), p.next_bias ? col : dim, stride, dim);
  if (!p.post_weight) pw.fill(1.f);
  if (!p.next_weight) nw.fill(1.f);
  if (p.scale) sc.load(static_cast<const P *>(p.scale), col, stride, dim);
  const int64_t step = (int64_t)(gridDim.x / members) * a.groups;
  for (int64_t row = (int64_t)(blockIdx.x / members) * a.groups + group; row < p.rows; row += step) {
    const int64_t base = row * dim;
    C in;
    float z[kUnit];
    in.load(static_cast<const T *>(p.x) + base, col, stride, dim);
#pragma unroll
    for (int j = 0; j < kUnit; ++j) z[j] = in[j];
    float2 post = make_float2(0.f, 1.f), next = make_float2(0.f, 1.f);
    if (p.h) {
      C hin, gin;
      float u[kUnit];
      hin.load(static_cast<const T *>(p.h) + base, col, stride, dim);
      float token = 1.f;
      if (p.gate_mode == P3D_GATE_ELEMENT) gin.load(static_cast<const T *>(p.gate) + base, col, stride, dim);
      if (p.gate_mode == P3D_GATE_SAMPLE)
        gin.load(static_cast<const T *>(p.gate) + row / p.rows_per_sample * dim, col, stride, dim);
      if (p.gate_mode == P3D_GATE_TOKEN) token = activate(to_f32<T>(static_cast<const T *>(p.gate)[row]), p.gate_act);
#pragma unroll
      for (int j = 0; j < kUnit; ++j) u[j] = hin[j];
      if (p.post_kind != P3D_NORM_NONE) {
        post = row_stats<ALIGNED>(u, p.post_kind, p.post_eps, col, stride, dim, sum);
#pragma unroll
        for (int j = 0; j < kUnit; ++j) u[j] = fmaf((u[j] - post.x) * post.y, pw[j], pb[j]);
      }
      if (p.gate_mode == P3D_GATE_ELEMENT || p.gate_mode == P3D_GATE_SAMPLE) {
#pragma unroll
        for (int j = 0; j < kUnit; ++j) u[j] *= activate(gin[j], p.gate_act);
      } else if (p.gate_mode == P3D_GATE_TOKEN) {
#pragma unroll
        for (int j = 0; j < kUnit; ++j) u[j] *= token;
      }
      if (p.threshold) {
        const uint32_t keep = row_keep<ALIGNED>(p, key, row, col, stride, first, t, s_keep + group * a.row_threads, sum);
#pragma unroll
        for (int j = 0; j < kUnit; ++j) u[j] = (keep >> j & 1u) ? u[j] * drop_scale : 0.f;
      }
      C o;
#pragma unroll
      for (int j = 0; j < kUnit; ++j) {
        z[j] = fmaf(p.scale ? sc[j] : p.scale_value, u[j], z[j]);
        if (col + (ALIGNED ? 0 : j * stride) >= dim) z[j] = 0.f;
        o.set(j, z[j]);
      }
      o.store(static_cast<T *>(a.out) + base, col, stride, dim);
    }
    if (p.next_kind != P3D_NORM_NONE) {
      next = row_stats<ALIGNED>(z, p.next_kind, p.next_eps, col, stride, dim, sum);
      C o;
#pragma unroll
      for (int j = 0; j < kUnit; ++j) o.set(j, fmaf((z[j] - next.x) * next.y, nw[j], nb[j]));
      o.store(static_cast<T *>(a.y) + base, col, stride, dim);
    }
    if (a.stats && t == 0 && rank == 0)
      reinterpret_cast<float4 *>(a.stats)[row] = make_float4(post.x, post.y, next.x, next.y);
  }
}

// ------------------------------------------------------------------------ backward
// Adds the thread's eight sums over the CTA's row groups (in group order) and writes them to dst.
template <bool ALIGNED>
__device__ __forceinline__ void join_groups(float (&acc)[kUnit], float *smem, float *dst, const Args &a, int group,
                                            int t, int col, int stride) {
  if (a.groups > 1) {
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kUnit; ++j) smem[(group * kUnit + j) * a.row_threads + t] = acc[j];
    __syncthreads();
    if (group == 0) {
#pragma unroll
      for (int j = 0; j < kUnit; ++j)
        for (int g = 1; g < a.groups; ++g) acc[j] += smem[(g * kUnit + j) * a.row_threads + t];
    }
  }
  if (group == 0) {
#pragma unroll
    for (int j = 0; j < kUnit; ++j) {
      const int c = ALIGNED ? col + j : col + j * stride;
      if (c < a.p.dim) dst[c] = acc[j];
    }
  }
#pragma unroll
  for (int j = 0; j < kUnit; ++j) acc[j] = 0.f;
}

template <typename T, typename P, bool ALIGNED, bool CLUSTER>
__global__ void __launch_bounds__(512) residual_bwd_kernel(const __grid_constant__ Args a) {
  const p3d_residual &p = a.p;
  P3D_ROW_SETUP();
  extern __shared__ float s_join[];  // [groups][8][row_threads] when a CTA has several groups
  using C = Cols<T, ALIGNED>;
  Cols<P, ALIGNED> pw, pb, sc, nw;
  pw.load(static_cast<const P *>(p.post_weight), p.post_weight ? col : dim, stride, dim);
  pb.load(static_cast<const P *>(p.post_bias), p.post_bias ? col : dim, stride, dim);
  nw.load(static_cast<const P *>(p.next_weight), p.next_weight ? col : dim, stride, dim);
  if (!p.post_weight) pw.fill(1.f);
  if (!p.next_weight) nw.fill(1.f);
  if (p.scale) sc.load(static_cast<const P *>(p.scale), col, stride, dim);
  const float inv_dim = 1.f / (float)dim;
  float acc[kSums][kUnit] = {};
  // CTA b takes slice b % slices of the segments b / slices, b / slices + CTAs / slices, ...
  const int64_t cta = blockIdx.x / members, ctas = gridDim.x / members;
  const int64_t slice = cta % a.slices;
  const int64_t row0 = a.segment_rows * slice / a.slices, row1 = a.segment_rows * (slice + 1) / a.slices;
  for (int64_t seg = cta / a.slices; seg < a.segments; seg += ctas / a.slices) {
    C gin;
    if (p.gate_mode == P3D_GATE_SAMPLE) gin.load(static_cast<const T *>(p.gate) + seg * dim, col, stride, dim);
    for (int64_t local = row0 + group; local < row1; local += a.groups) {
      const int64_t row = seg * a.segment_rows + local, base = row * dim;
      const float4 st = reinterpret_cast<const float4 *>(a.stats)[row];
      C in, hin, go, gy;
      in.load(static_cast<const T *>(p.x) + base, p.next_kind != P3D_NORM_NONE && a.dy ? col : dim, stride, dim);
      hin.load(static_cast<const T *>(p.h) + base, p.h ? col : dim, stride, dim);
      go.load(static_cast<const T *>(a.dout) + base, a.dout ? col : dim, stride, dim);
      gy.load(static_cast<const T *>(a.dy) + base, a.dy ? col : dim, stride, dim);
      if (p.gate_mode == P3D_GATE_ELEMENT) gin.load(static_cast<const T *>(p.gate) + base, col, stride, dim);
      float token = 1.f;
      if (p.gate_mode == P3D_GATE_TOKEN) token = activate(to_f32<T>(static_cast<const T *>(p.gate)[row]), p.gate_act);
      uint32_t keep = 0xffu;
      if (p.threshold)
        keep = row_keep<ALIGNED>(p, key, row, col, stride, first, t, s_keep + group * a.row_threads, sum);
      float hn[kUnit], d[kUnit], G[kUnit];
      if (p.h) {
#pragma unroll
        for (int j = 0; j < kUnit; ++j) {
          hn[j] = (hin[j] - st.x) * st.y;
          const float u = p.post_kind != P3D_NORM_NONE ? fmaf(hn[j], pw[j], pb[j]) : hin[j];
          const float act = p.gate_mode == P3D_GATE_NONE    ? 1.f
                            : p.gate_mode == P3D_GATE_TOKEN ? token
                                                            : activate(gin[j], p.gate_act);
          d[j] = (keep >> j & 1u) ? u * act * drop_scale : 0.f;
        }
      }
#pragma unroll
      for (int j = 0; j < kUnit; ++j) G[j] = go[j];
      if (a.dy && p.next_kind != P3D_NORM_NONE) {
        float s[2] = {0.f, 0.f};
#pragma unroll
        for (int j = 0; j < kUnit; ++j) {
          const float z = p.h ? fmaf(p.scale ? sc[j] : p.scale_value, d[j], in[j]) : in[j];
          const float zn = (z - st.z) * st.w, g = gy[j] * nw[j];
          s[0] += g;
          s[1] = fmaf(g, zn, s[1]);
          acc[3][j] = fmaf(gy[j], zn, acc[3][j]);
          acc[4][j] += gy[j];
        }
        sum(s);
        const float m0 = p.next_kind == P3D_NORM_LAYER ? s[0] * inv_dim : 0.f, m1 = s[1] * inv_dim;
#pragma unroll
        for (int j = 0; j < kUnit; ++j) {
          const float z = p.h ? fmaf(p.scale ? sc[j] : p.scale_value, d[j], in[j]) : in[j];
          G[j] += st.w * (gy[j] * nw[j] - m0 - (z - st.z) * st.w * m1);
          if (col + (ALIGNED ? 0 : j * stride) >= dim) G[j] = 0.f;   // no column: nothing for the sums below
        }
      }
      if (a.dx) {
        C o;
#pragma unroll
        for (int j = 0; j < kUnit; ++j) o.set(j, G[j]);
        o.store(static_cast<T *>(a.dx) + base, col, stride, dim);
      }
      if (p.h) {
        float s[3] = {0.f, 0.f, 0.f}, du[kUnit];
        C o;
#pragma unroll
        for (int j = 0; j < kUnit; ++j) {
          const bool kept = keep >> j & 1u;
          const float u = p.post_kind != P3D_NORM_NONE ? fmaf(hn[j], pw[j], pb[j]) : hin[j];
          const float act = p.gate_mode == P3D_GATE_NONE    ? 1.f
                            : p.gate_mode == P3D_GATE_TOKEN ? token
                                                            : activate(gin[j], p.gate_act);
          acc[0][j] = fmaf(G[j], d[j], acc[0][j]);
          const float dv = kept ? G[j] * (p.scale ? sc[j] : p.scale_value) * drop_scale : 0.f;
          const float dg = kept ? dv * u * slope(act, p.gate_act) : 0.f;
          du[j] = dv * act;
          const float g = du[j] * pw[j];
          s[0] += g;
          s[1] = fmaf(g, hn[j], s[1]);
          s[2] += dg;
          o.set(j, dg);
          acc[1][j] = fmaf(du[j], hn[j], acc[1][j]);
          acc[2][j] += du[j];
          acc[5][j] += dg;
        }
        if (p.gate_mode == P3D_GATE_ELEMENT && a.dgate) o.store(static_cast<T *>(a.dgate) + base, col, stride, dim);
        const bool token_gate = p.gate_mode == P3D_GATE_TOKEN && a.dgate;
        if (p.post_kind != P3D_NORM_NONE || token_gate) sum(s);
        if (token_gate && t == 0 && rank == 0) static_cast<T *>(a.dgate)[row] = from_f32<T>(s[2]);
        if (a.dh) {
          const float m0 = p.post_kind == P3D_NORM_LAYER ? s[0] * inv_dim : 0.f, m1 = s[1] * inv_dim;
#pragma unroll
          for (int j = 0; j < kUnit; ++j)
            o.set(j, p.post_kind == P3D_NORM_NONE ? du[j] : st.y * (du[j] * pw[j] - m0 - hn[j] * m1));
          o.store(static_cast<T *>(a.dh) + base, col, stride, dim);
        }
      }
    }
    if (p.gate_mode == P3D_GATE_SAMPLE && a.dgate)
      join_groups<ALIGNED>(acc[5], s_join, a.partials + ((int64_t)(kSums - 1) * ctas + seg * a.slices + slice) * dim, a,
                           group, t, col, stride);
  }
#pragma unroll
  for (int q = 0; q < kSums - 1; ++q)
    join_groups<ALIGNED>(acc[q], s_join, a.partials + (q * ctas + cta) * dim, a, group, t, col, stride);
}

// out[row, c] = sum over k of in[row, k, c], k in order within each of eight interleaved runs, the runs
// in order.  One CTA sums 32 columns of one row.
struct Joins {
  const float *in;
  void *out[kSums - 1];
};
template <typename P>
__global__ void __launch_bounds__(256) join_kernel(const float *in, P *single, Joins several, int64_t k_count, int dim) {
  __shared__ float s[8][33];
  P *out = single ? single + (int64_t)blockIdx.y * dim : static_cast<P *>(several.out[blockIdx.y]);
  if (out == nullptr) return;
  const int c = blockIdx.x * 32 + threadIdx.x;
  const float *src = in + (int64_t)blockIdx.y * k_count * dim;
  float v = 0.f;
  if (c < dim)
    for (int64_t k = threadIdx.y; k < k_count; k += 8) v += src[k * dim + c];
  s[threadIdx.y][threadIdx.x] = v;
  __syncthreads();
  if (threadIdx.y == 0 && c < dim) {
    for (int i = 1; i < 8; ++i) v += s[i][threadIdx.x];
    out[c] = from_f32<P>(v);
  }
}

// ------------------------------------------------------------------------ dropout
// dim a multiple of 8 and 16-byte pointers: block b is elements [8b, 8b + 8) of the whole tensor.
template <typename T>
__global__ void __launch_bounds__(256) dropout_kernel(const T *x, T *y, int64_t blocks, uint32_t threshold,
                                                      const uint64_t *rng, uint64_t seed, uint64_t offset) {
  const PhiloxKey key = philox_key(rng, seed, offset);
  const float scale = keep_scale(threshold);
  const int64_t step = (int64_t)gridDim.x * blockDim.x;
  for (int64_t b = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; b < blocks; b += step) {
    Cols<T, true> c;
    c.load(x + b * 8, 0, 1, 8);
    const uint32_t keep = keep_bits(key, (uint64_t)b, threshold);
#pragma unroll
    for (int j = 0; j < 8; ++j) c.set(j, (keep >> j & 1u) ? c[j] * scale : 0.f);
    c.store(y + b * 8, 0, 1, 8);
  }
}

// Any dim: eight consecutive elements of the whole tensor a thread; they lie in one block of a row or
// in a few, and a new block's bits are made where the row or the block changes.
template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(256) dropout_any_kernel(const T *x, T *y, int64_t total, int64_t dim,
                                                          uint32_t threshold, const uint64_t *rng, uint64_t seed,
                                                          uint64_t offset) {
  const PhiloxKey key = philox_key(rng, seed, offset);
  const float scale = keep_scale(threshold);
  const int64_t row_blocks = (dim + 7) / 8, step = (int64_t)gridDim.x * blockDim.x;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i * 8 < total; i += step) {
    const int64_t e = i * 8;
    const bool whole = ALIGNED && e + 8 <= total;
    Cols<T, true> c;
    if (whole) c.load(x + e, 0, 1, 8);
    else
#pragma unroll
      for (int j = 0; j < 8; ++j) c.v[j] = e + j < total ? x[e + j] : from_f32<T>(0.f);
    int64_t row = e / dim, col = e - row * dim;
    uint32_t keep = keep_bits(key, (uint64_t)(row * row_blocks + col / 8), threshold);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (j > 0) {
        if (++col == dim) {
          col = 0;
          ++row;
        }
        if ((col & 7) == 0) keep = keep_bits(key, (uint64_t)(row * row_blocks + col / 8), threshold);
      }
      c.set(j, (keep >> (col & 7) & 1u) ? c[j] * scale : 0.f);
    }
    if (whole) c.store(y + e, 0, 1, 8);
    else
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (e + j < total) y[e + j] = c.v[j];
  }
}

// ------------------------------------------------------------------------ host side
bool aligned16(const void *ptr) { return (reinterpret_cast<uintptr_t>(ptr) & 15u) == 0; }

// Threads a row, rows a CTA at once and CTAs a row.
struct Shape {
  int row_threads, groups, members;
};
Shape shape_of(int dim) {
  const int units = (dim + kUnit - 1) / kUnit;
  Shape s;
  s.members = units <= kMaxRowThreads ? 1 : units <= 2 * kMaxRowThreads ? 2 : 4;
  const int mine = (units + s.members - 1) / s.members;
  s.row_threads = (mine + 31) / 32 * 32;
  s.groups = std::max(1, 256 / s.row_threads);
  return s;
}

struct Split {
  int64_t segments, slices, segment_rows, ctas;
};
// Rows are cut over about as many CTAs as the GPU holds at once; with a gate for each sample a CTA stays
// within a sample at a time, so that the sample's gradient is summed in registers.
Split split_of(const p3d_residual &p, const Shape &s, int sms) {
  Split c;
  c.segments = p.gate_mode == P3D_GATE_SAMPLE ? p.rows / p.rows_per_sample : 1;
  c.segment_rows = p.rows / std::max<int64_t>(c.segments, 1);
  const int per_sm = std::max(1, 512 / (s.row_threads * s.groups));
  const int64_t room = std::max<int64_t>(1, (int64_t)sms * per_sm / s.members);
  const int64_t useful = std::max<int64_t>(1, (c.segment_rows + s.groups - 1) / s.groups);
  c.slices = std::min(useful, std::max<int64_t>(1, room / std::max<int64_t>(c.segments, 1)));
  c.ctas = c.slices * std::min(c.segments, std::max<int64_t>(1, room / c.slices));
  return c;
}

int check_args(const p3d_residual *p, const char *what) {
  P3D_CHECK_ARG(p != nullptr, "%s: null arguments", what);
  P3D_CHECK_ARG(dtype_ok(p->dtype), "%s: unknown dtype %d", what, p->dtype);
  P3D_CHECK_ARG(p->param_dtype == p->dtype || p->param_dtype == P3D_F32,
                "%s: parameters must be of the tensors' dtype or fp32", what);
  P3D_CHECK_ARG(p->rows >= 0 && p->rows < (int64_t)1 << 40, "%s: bad row count", what);
  P3D_CHECK_ARG(p->dim >= 1, "%s: dim must be positive", what);
  if (p->dim > kMaxDim) return fail(P3D_ERR_UNSUPPORTED, "%s: dim %d above %d", what, p->dim, kMaxDim);
  P3D_CHECK_ARG(p->post_kind >= P3D_NORM_NONE && p->post_kind <= P3D_NORM_LAYER && p->next_kind >= P3D_NORM_NONE &&
                    p->next_kind <= P3D_NORM_LAYER,
                "%s: unknown norm", what);
  P3D_CHECK_ARG(p->gate_mode >= P3D_GATE_NONE && p->gate_mode <= P3D_GATE_TOKEN && p->gate_act >= P3D_ACT_IDENTITY &&
                    p->gate_act <= P3D_ACT_TANH,
                "%s: unknown gate", what);
  P3D_CHECK_ARG(p->threshold <= 65536u, "%s: dropout threshold above 65536", what);
  P3D_CHECK_ARG(p->post_eps >= 0.f && p->next_eps >= 0.f, "%s: negative eps", what);
  P3D_CHECK_ARG(p->h || (p->post_kind == P3D_NORM_NONE && p->gate_mode == P3D_GATE_NONE && !p->scale && !p->threshold),
                "%s: a post norm, gate, scale or dropout needs h", what);
  P3D_CHECK_ARG(p->h || p->next_kind != P3D_NORM_NONE, "%s: nothing to compute", what);
  P3D_CHECK_ARG((p->gate != nullptr) == (p->gate_mode != P3D_GATE_NONE), "%s: gate and its mode disagree", what);
  P3D_CHECK_ARG(p->gate_mode != P3D_GATE_SAMPLE || (p->rows_per_sample >= 1 && p->rows % p->rows_per_sample == 0),
                "%s: rows must be whole samples", what);
  return P3D_OK;
}

bool all_aligned(const p3d_residual &p, std::initializer_list<const void *> more) {
  if (p.dim % kUnit) return false;
  for (const void *q : {p.x, p.h, p.gate_mode == P3D_GATE_TOKEN ? nullptr : p.gate, p.post_weight, p.post_bias, p.scale,
                        p.next_weight, p.next_bias})
    if (!aligned16(q)) return false;
  for (const void *q : more)
    if (!aligned16(q)) return false;
  return true;
}

template <typename K>
int launch_rows(K kernel, const Args &a, int64_t ctas, int members, size_t smem, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(ctas * members));
  cfg.blockDim = dim3((unsigned)(a.row_threads * a.groups));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)members;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = members > 1 ? 1 : 0;
  P3D_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, a));
  return P3D_OK;
}

template <typename T, typename P>
int run_fwd(const Args &a, bool aligned, int64_t ctas, int members, cudaStream_t s) {
  if (members > 1)
    return aligned ? launch_rows(residual_fwd_kernel<T, P, true, true>, a, ctas, members, 0, s)
                   : launch_rows(residual_fwd_kernel<T, P, false, true>, a, ctas, members, 0, s);
  return aligned ? launch_rows(residual_fwd_kernel<T, P, true, false>, a, ctas, 1, 0, s)
                 : launch_rows(residual_fwd_kernel<T, P, false, false>, a, ctas, 1, 0, s);
}

template <typename T, typename P>
int run_bwd(const Args &a, const Split &c, bool aligned, int members, void *const (&sums)[kSums - 1], cudaStream_t s) {
  const size_t smem = a.groups > 1 ? (size_t)a.groups * kUnit * a.row_threads * sizeof(float) : 0;
  int st;
  if (members > 1)
    st = aligned ? launch_rows(residual_bwd_kernel<T, P, true, true>, a, c.ctas, members, smem, s)
                 : launch_rows(residual_bwd_kernel<T, P, false, true>, a, c.ctas, members, smem, s);
  else
    st = aligned ? launch_rows(residual_bwd_kernel<T, P, true, false>, a, c.ctas, 1, smem, s)
                 : launch_rows(residual_bwd_kernel<T, P, false, false>, a, c.ctas, 1, smem, s);
  if (st != P3D_OK) return st;
  const dim3 block(32, 8);
  const unsigned tiles = (unsigned)((a.p.dim + 31) / 32);
  Joins j{};
  bool any = false;
  for (int q = 0; q < kSums - 1; ++q) any |= (j.out[q] = sums[q]) != nullptr;
  if (any) {
    join_kernel<P><<<dim3(tiles, kSums - 1), block, 0, s>>>(a.partials, nullptr, j, c.ctas, a.p.dim);
    P3D_LAUNCH_CHECK();
  }
  if (a.p.gate_mode == P3D_GATE_SAMPLE && a.dgate) {
    const float *part = a.partials + (int64_t)(kSums - 1) * c.ctas * a.p.dim;
    for (int64_t first = 0; first < c.segments; first += 65535) {   // the grid's y limit
      const unsigned n = (unsigned)std::min<int64_t>(65535, c.segments - first);
      join_kernel<T><<<dim3(tiles, n), block, 0, s>>>(part + first * c.slices * a.p.dim,
                                                      static_cast<T *>(a.dgate) + first * a.p.dim, j, c.slices,
                                                      a.p.dim);
      P3D_LAUNCH_CHECK();
    }
  }
  return P3D_OK;
}

template <typename F>
int by_type(const p3d_residual &p, F &&f) {
  if (p.dtype == P3D_F32) return f(float{}, float{});
  if (p.dtype == P3D_F16) return p.param_dtype == P3D_F32 ? f(__half{}, float{}) : f(__half{}, __half{});
  return p.param_dtype == P3D_F32 ? f(__nv_bfloat16{}, float{}) : f(__nv_bfloat16{}, __nv_bfloat16{});
}

size_t partial_floats(const p3d_residual &p, const Split &c) {
  size_t n = (size_t)(kSums - 1) * c.ctas * p.dim;
  if (p.gate_mode == P3D_GATE_SAMPLE) n += (size_t)c.segments * c.slices * p.dim;
  return n;
}

}  // namespace

int launch_column_join(const float *partials, void *out, int dtype, int64_t count, int dim, cudaStream_t s) {
  const dim3 grid((unsigned)((dim + 31) / 32)), block(32, 8);
  const Joins none = {};
  if (dtype == P3D_F32) join_kernel<float><<<grid, block, 0, s>>>(partials, static_cast<float *>(out), none, count, dim);
  else if (dtype == P3D_F16)
    join_kernel<__half><<<grid, block, 0, s>>>(partials, static_cast<__half *>(out), none, count, dim);
  else
    join_kernel<__nv_bfloat16><<<grid, block, 0, s>>>(partials, static_cast<__nv_bfloat16 *>(out), none, count, dim);
  P3D_LAUNCH_CHECK();
  return P3D_OK;
}

}  // namespace p3d

using namespace p3d;

extern "C" int p3d_dropout(const void *x, void *y, int dtype, int64_t rows, int64_t dim, uint32_t threshold,
                           const uint64_t *rng, uint64_t seed, uint64_t offset, void *stream) {
  P3D_CHECK_ARG(dtype_ok(dtype), "p3d_dropout: unknown dtype %d", dtype);
  P3D_CHECK_ARG(rows >= 0 && dim >= 0 && (dim == 0 || rows <= ((int64_t)1 << 44) / dim), "p3d_dropout: bad extents");
  P3D_CHECK_ARG(threshold <= 65536u, "p3d_dropout: threshold above 65536");
  if (rows == 0 || dim == 0) return P3D_OK;
  P3D_CHECK_ARG(x && y, "p3d_dropout: null pointer");
  DeviceInfo info;
  if (int st = device_info(&info)) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool aligned = aligned16(x) && aligned16(y);
  const int64_t total = rows * dim, blocks = (total + 7) / 8;
  const unsigned grid = (unsigned)std::min<int64_t>((blocks + 255) / 256, (int64_t)info.sm_count * 8);
  p3d_residual kind = {};
  kind.dtype = kind.param_dtype = dtype;
  return by_type(kind, [&](auto t, auto) {
    using T = decltype(t);
    const T *in = static_cast<const T *>(x);
    T *out = static_cast<T *>(y);
    if (aligned && dim % 8 == 0)
      dropout_kernel<T><<<grid, 256, 0, s>>>(in, out, blocks, threshold, rng, seed, offset);
    else if (aligned)
      dropout_any_kernel<T, true><<<grid, 256, 0, s>>>(in, out, total, dim, threshold, rng, seed, offset);
    else
      dropout_any_kernel<T, false><<<grid, 256, 0, s>>>(in, out, total, dim, threshold, rng, seed, offset);
    P3D_LAUNCH_CHECK();
    return (int)P3D_OK;
  });
}

extern "C" int p3d_residual_fwd(const p3d_residual *args, void *out, void *y, float *stats, void *stream) {
  if (int st = check_args(args, "p3d_residual_fwd")) return st;
  const p3d_residual &p = *args;
  if (p.rows == 0) return P3D_OK;
  P3D_CHECK_ARG(p.x && (!p.h || out) && (p.next_kind == P3D_NORM_NONE || y), "p3d_residual_fwd: null pointer");
  P3D_CHECK_ARG(aligned16(stats), "p3d_residual_fwd: stats must be 16-byte aligned");
  DeviceInfo info;
  if (int st = device_info(&info)) return st;
  const Shape s = shape_of(p.dim);
  Args a = {};
  a.p = p;
  a.out = out;
  a.y = y;
  a.stats = stats;
  a.row_threads = s.row_threads;
  a.groups = s.groups;
  const int64_t most = std::max<int64_t>(1, (int64_t)info.sm_count * (1024 / (s.row_threads * s.groups)) / s.members);
  const int64_t ctas = std::min<int64_t>((p.rows + s.groups - 1) / s.groups, most);
  const bool aligned = all_aligned(p, {out, y});
  return by_type(p, [&](auto t, auto w) {
    return run_fwd<decltype(t), decltype(w)>(a, aligned, ctas, s.members, static_cast<cudaStream_t>(stream));
  });
}

extern "C" size_t p3d_residual_bwd_workspace(const p3d_residual *args) {
  DeviceInfo info;
  if (check_args(args, "p3d_residual_bwd_workspace") || args->rows == 0 || device_info(&info)) return 0;
  return partial_floats(*args, split_of(*args, shape_of(args->dim), info.sm_count)) * sizeof(float);
}

extern "C" int p3d_residual_bwd(const p3d_residual *args, const void *dout, const void *dy, const float *stats,
                                void *dx, void *dh, void *dgate, void *dscale, void *dpost_weight, void *dpost_bias,
                                void *dnext_weight, void *dnext_bias, void *workspace, size_t workspace_bytes,
                                void *stream) {
  if (int st = check_args(args, "p3d_residual_bwd")) return st;
  const p3d_residual &p = *args;
  P3D_CHECK_ARG(p.rows >= 1, "p3d_residual_bwd: no rows");
  P3D_CHECK_ARG(p.x && stats && aligned16(stats), "p3d_residual_bwd: x and 16-byte aligned stats required");
  P3D_CHECK_ARG(!dy || p.next_kind != P3D_NORM_NONE, "p3d_residual_bwd: dy without a next norm");
  P3D_CHECK_ARG(p.h || !(dh || dgate || dscale || dpost_weight || dpost_bias),
                "p3d_residual_bwd: gradients of a block that is not there");
  DeviceInfo info;
  if (int st = device_info(&info)) return st;
  const Shape s = shape_of(p.dim);
  const Split c = split_of(p, s, info.sm_count);
  const size_t need = partial_floats(p, c) * sizeof(float);
  if (workspace_bytes < need || !workspace)
    return fail(P3D_ERR_WORKSPACE, "p3d_residual_bwd: workspace of %zu bytes, %zu needed", workspace_bytes, need);
  Args a = {};
  a.p = p;
  a.dout = dout;
  a.dy = dy;
  a.stats = const_cast<float *>(stats);
  a.dx = dx;
  a.dh = dh;
  a.dgate = dgate;
  a.partials = static_cast<float *>(workspace);
  a.row_threads = s.row_threads;
  a.groups = s.groups;
  a.segments = c.segments;
  a.slices = c.slices;
  a.segment_rows = c.segment_rows;
  const bool aligned =
      all_aligned(p, {dout, dy, dx, dh, p.gate_mode == P3D_GATE_ELEMENT ? (const void *)dgate : nullptr});
  void *const sums[kSums - 1] = {dscale, dpost_weight, dpost_bias, dnext_weight, dnext_bias};
  return by_type(p, [&](auto t, auto w) {
    return run_bwd<decltype(t), decltype(w)>(a, c, aligned, s.members, sums, static_cast<cudaStream_t>(stream));
  });
}
