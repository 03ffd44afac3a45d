// The feed-forward half of a block around its matrix products: dropout, the column sums that end the
// backward of the norms, and the C entry points.  The row kernels themselves are in residual_rows.cuh.
#include <algorithm>
#include <initializer_list>

#include "common.cuh"
#include "kernels.cuh"
#include "philox.cuh"
#include "residual_rows.cuh"

namespace p3d {

namespace rows {   // instantiated in residual_{f32,f16,bf16}.cu
extern template int run_fwd<float>(const Args &, bool, bool, int, int, int64_t, size_t, cudaStream_t);
extern template int run_fwd<__half>(const Args &, bool, bool, int, int, int64_t, size_t, cudaStream_t);
extern template int run_fwd<__nv_bfloat16>(const Args &, bool, bool, int, int, int64_t, size_t, cudaStream_t);
extern template int run_bwd<float>(const Args &, bool, bool, int64_t, size_t, cudaStream_t);
extern template int run_bwd<__half>(const Args &, bool, bool, int64_t, size_t, cudaStream_t);
extern template int run_bwd<__nv_bfloat16>(const Args &, bool, bool, int64_t, size_t, cudaStream_t);
extern template int take_errors<float>(unsigned *);
extern template int take_errors<__half>(unsigned *);
extern template int take_errors<__nv_bfloat16>(unsigned *);
}  // namespace rows

namespace {

using rows::Args;
using rows::kSums;
using rows::kUnit;
using rows::Shape;
using rows::shape_of;

constexpr int kMaxDim = 16384;   // 512 threads of four CTAs in 16 bits, 256 of eight in 32
constexpr int kFoldRows = 8;
constexpr int64_t kMaxRows = ((int64_t)1 << 31) - 1024;

// out[row, c] = sum over k of in[row, k, c], k in order within each of 32 interleaved runs, the runs in order.  One CTA
// sums 32 columns of one row.
constexpr int kRuns = 32;
struct Joins {
  void *out[kSums - 1];
};
template <typename P>
__global__ void __launch_bounds__(32 * kRuns) join_kernel(const float *in, P *single, Joins several, int64_t k_count, int dim) {
  __shared__ float s[kRuns][33];
  P *out = single ? single + (int64_t)blockIdx.y * dim : static_cast<P *>(several.out[blockIdx.y]);
  if (out == nullptr) return;
  const int c = blockIdx.x * 32 + threadIdx.x;
  const float *src = in + (int64_t)blockIdx.y * k_count * dim;
  float v = 0.f;
  if (c < dim)
    for (int64_t k = threadIdx.y; k < k_count; k += kRuns) v += src[k * dim + c];
  s[threadIdx.y][threadIdx.x] = v;
  __syncthreads();
  if (threadIdx.y == 0 && c < dim) {
#pragma unroll
    for (int i = 1; i < kRuns; ++i) v += s[i][threadIdx.x];
    out[c] = from_f32<P>(v);
  }
}

// ------------------------------------------------------------------------ dropout
template <typename T>
struct Eight {
  T v[8];
  __device__ __forceinline__ void load(const T *from) {
    constexpr int n = sizeof(T) * 8 / 16;
    uint4 raw[n];
#pragma unroll
    for (int i = 0; i < n; ++i) raw[i] = reinterpret_cast<const uint4 *>(from)[i];
    memcpy(v, raw, sizeof(v));
  }
  __device__ __forceinline__ void store(T *to) const {
    constexpr int n = sizeof(T) * 8 / 16;
    uint4 raw[n];
    memcpy(raw, v, sizeof(v));
#pragma unroll
    for (int i = 0; i < n; ++i) reinterpret_cast<uint4 *>(to)[i] = raw[i];
  }
  __device__ __forceinline__ float operator[](int j) const { return to_f32<T>(v[j]); }
  __device__ __forceinline__ void set(int j, float f) { v[j] = from_f32<T>(f); }
};

// dim a multiple of 8 and 16-byte pointers: block b is elements [8b, 8b + 8) of the whole tensor.  Bound by issue as
// much as by HBM (about a hundred instructions a block, forty of them the rounds): the round keys come from
// shared memory, and two blocks at a time hide the rounds' latency.  Measured at 262144 x 384 bf16: 74 us
// (5.4 TB/s read and written); one block at a time on six CTAs an SM 82 us, on eight (which
// spill) 88 us, and with the keys added up each time 87 us.
template <typename T>
__global__ void __launch_bounds__(256, 4) dropout_kernel(const T *x, T *y, int64_t blocks, uint32_t threshold,
                                                      const uint64_t *rng, uint64_t seed, uint64_t offset) {
  __shared__ RoundKeys keys;
  keys.set(philox_key(rng, seed, offset));
  __syncthreads();
  const Keep keep(threshold);
  const float scale = keep_scale(threshold);
  const int64_t step = (int64_t)gridDim.x * blockDim.x;
  auto one = [&](int64_t b, Eight<T> &c) {
    uint32_t w[4];
    keep.words(keys, (uint64_t)b, w);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      c.set(j, (j & 1 ? keep.high(w[j / 2]) : keep.low(w[j / 2])) ? c[j] * scale : 0.f);
  };
  int64_t b = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  for (; b + step < blocks; b += 2 * step) {
    Eight<T> p, q;
    p.load(x + b * 8);
    q.load(x + (b + step) * 8);
    one(b, p);
    one(b + step, q);
    p.store(y + b * 8);
    q.store(y + (b + step) * 8);
  }
  if (b < blocks) {
    Eight<T> p;
    p.load(x + b * 8);
    one(b, p);
    p.store(y + b * 8);
  }
}

// Any dim: eight consecutive elements of the whole tensor a thread; they lie in one block of a row or
// in a few, and a new block's bits are made where the row or the block changes.
template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(256) dropout_any_kernel(const T *x, T *y, int64_t total, int64_t dim,
                                                          uint32_t threshold, const uint64_t *rng, uint64_t seed,
                                                          uint64_t offset) {
  const PhiloxKey key = philox_key(rng, seed, offset);
  const Keep keep(threshold);
  const float scale = keep_scale(threshold);
  const int64_t row_blocks = (dim + 7) / 8, step = (int64_t)gridDim.x * blockDim.x;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i * 8 < total; i += step) {
    const int64_t e = i * 8;
    const bool whole = ALIGNED && e + 8 <= total;
    Eight<T> c;
    if (whole) c.load(x + e);
    else
#pragma unroll
      for (int j = 0; j < 8; ++j) c.v[j] = e + j < total ? x[e + j] : from_f32<T>(0.f);
    int64_t row = e / dim, col = e - row * dim;
    uint32_t bits = keep.bits(key, (uint64_t)(row * row_blocks + col / 8));
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (j > 0) {
        if (++col == dim) {
          col = 0;
          ++row;
        }
        if ((col & 7) == 0) bits = keep.bits(key, (uint64_t)(row * row_blocks + col / 8));
      }
      c.set(j, (bits >> (col & 7) & 1u) ? c[j] * scale : 0.f);
    }
    if (whole) c.store(y + e);
    else
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (e + j < total) y[e + j] = c.v[j];
  }
}

// ------------------------------------------------------------------------ host side
bool aligned16(const void *ptr) { return (reinterpret_cast<uintptr_t>(ptr) & 15u) == 0; }

// Whether a call needs a mean or a bias.
bool centred(const p3d_residual &p) {
  return p.post_kind == P3D_NORM_LAYER || p.next_kind == P3D_NORM_LAYER || p.post_bias || p.next_bias;
}

constexpr size_t kSharedPerSm = 228 * 1024, kSharedReserve = 4096;   // reserve: static, and what the driver keeps of a CTA

// Dynamic shared memory without the rings, and what a stage of one row (or turn of the warps) takes.
struct Room {
  size_t fixed, stage;
};
Room room_of(const Shape &s, int dim, int dtype, size_t arrays, size_t params, bool aligned, bool backward) {
  const size_t columns = (size_t)s.columns(), row = std::min((size_t)dim, columns) * (size_t)dtype_size(dtype);
  Room r;
  r.fixed = params * columns * sizeof(float) + (backward && s.groups > 1 ? s.groups * columns * sizeof(float) : 0);
  r.stage = s.groups * (s.rows_at_once() * (arrays * row + 16) + (aligned ? 0 : arrays * 32));
  return r;
}

// CTAs that an SM's registers hold: 64 registers a thread in the forward's narrowest form and in the backward of a norm
// by itself, else 128.
int per_sm_of(const p3d_residual &p, const Shape &s, bool backward) {
  const int threads = (backward ? p.h == nullptr : s.units == 1) ? 1024 : 512;
  return std::max(1, threads / (s.row_threads * s.groups));
}

// The row groups of a CTA: of 256 threads' worth and its halves the number that keeps most threads on an SM, as
// far as that can be told from the call's description (all streams there, rows unaligned).
Shape shape_for(const p3d_residual &p, bool backward) {
  Shape best = shape_of(p.dim, p.dtype, backward);
  const size_t arrays = (p.h ? 2 : 1) * (backward ? 2 : 1) + (p.gate_mode == P3D_GATE_ELEMENT ? 1 : 0);
  const size_t params = rows::param_count(p.h != nullptr, centred(p));
  int most = 0;
  for (Shape s = best; s.groups >= 1; s.groups /= 2) {
    const Room r = room_of(s, p.dim, p.dtype, arrays, params, false, backward);
    const int fit = (int)std::max<size_t>(1, kSharedPerSm / (r.fixed + 2 * r.stage + kSharedReserve));
    const int threads = std::min(fit, per_sm_of(p, s, backward)) * s.row_threads * s.groups;
    if (threads > most) {
      most = threads;
      best = s;
    }
  }
  return best;
}

// How the rows are cut over the CTAs: contiguous slices of the whole or, by_sample, of every sample that has a gate of its
// own: always in the backward, so that the sample's gradient is summed in registers, and in the forward
// where the gate is folded into the parameters.  per_sm: CTAs an SM is meant to hold.
struct Split {
  int64_t segments, slices, segment_rows, ctas;
};
Split split_of(const p3d_residual &p, const Shape &s, int sms, int per_sm, bool by_sample) {
  Split c;
  c.segments = by_sample && p.gate_mode == P3D_GATE_SAMPLE ? p.rows / p.rows_per_sample : 1;
  c.segment_rows = p.rows / std::max<int64_t>(c.segments, 1);
  const int64_t room = std::max<int64_t>(1, (int64_t)sms * per_sm / s.members);
  const int64_t step = (int64_t)s.groups * s.rows_at_once();
  const int64_t useful = std::max<int64_t>(1, (c.segment_rows + step - 1) / step);
  c.slices = std::min(useful, std::max<int64_t>(1, room / std::max<int64_t>(c.segments, 1)));
  c.ctas = c.slices * std::min(c.segments, std::max<int64_t>(1, room / c.slices));
  return c;
}

// Shared memory of a CTA: the parameters in fp32, the joins of the column sums, and the rings: batches of about
// 2 KB an array (one row where rows are longer or shared by a cluster), as many stages as the CTA's
// share holds, at least two.  Fills in the layout and returns the bytes; *per_sm comes in as the CTAs an SM's
// registers hold and goes out as what its shared memory holds too.
size_t lay_out(Args &a, const Shape &s, bool aligned, bool center, bool backward, int *per_sm) {
  a.row_threads = s.row_threads;
  a.groups = s.groups;
  a.members = s.members;
  a.slot_count = 0;
  for (int i = 0; i < rows::kArrays; ++i) a.slot_count += a.in[i] ? 1 : 0;
  const size_t arrays = (size_t)std::max(1, a.slot_count), at_once = (size_t)s.rows_at_once();
  const size_t row = (size_t)std::min(a.p.dim, s.columns()) * (size_t)dtype_size(a.p.dtype);
  const Room r = room_of(s, a.p.dim, a.p.dtype, arrays, rows::param_count(a.p.h != nullptr, center), aligned, backward);
  while (*per_sm > 1 && kSharedPerSm / *per_sm < r.fixed + 2 * r.stage + kSharedReserve) --*per_sm;
  const size_t share = kSharedPerSm / *per_sm - r.fixed - kSharedReserve;
  size_t turns = 1;   // rows (or turns of a warp's rows) a batch
  if (s.members == 1) turns = std::max<size_t>(1, std::min({8 / at_once, 2048 / (at_once * row), share / (2 * r.stage)}));
  a.batch_rows = (int)(turns * at_once);
  a.edge_rows = rows::edge_rows((int64_t)a.p.dim * dtype_size(a.p.dtype));
  const size_t batch = row * a.batch_rows;
  const uint32_t slot = (uint32_t)(aligned ? batch : (batch + 15) / 16 * 16 + 16);
  a.stats_at = 0;
  for (int i = 0; i < rows::kArrays; ++i)
    if (a.in[i]) {
      a.slots[i] = a.stats_at;
      a.stats_at += slot;
    }
  a.stage_bytes = a.stats_at + 16u * (uint32_t)a.batch_rows;
  a.stages = (int)std::max<size_t>(2, std::min<size_t>(rows::kMaxStages, share / (s.groups * (size_t)a.stage_bytes)));
  return (size_t)s.groups * a.stages * a.stage_bytes + r.fixed;
}

// What the layout goes by, without the tensors that only the call itself has.
void set_params(Args &a, const p3d_residual &p) {
  a.p = p;
  a.params[rows::kPostW] = p.post_weight;
  a.params[rows::kPostB] = p.post_bias;
  a.params[rows::kScale] = p.scale;
  a.params[rows::kNextW] = p.next_weight;
  a.params[rows::kNextB] = p.next_bias;
}

int check_args(const p3d_residual *p, const char *what) {
  P3D_CHECK_ARG(p != nullptr, "%s: null arguments", what);
  P3D_CHECK_ARG(dtype_ok(p->dtype), "%s: unknown dtype %d", what, p->dtype);
  P3D_CHECK_ARG(p->param_dtype == p->dtype || p->param_dtype == P3D_F32,
                "%s: parameters must be of the tensors' dtype or fp32", what);
  P3D_CHECK_ARG(p->rows >= 0, "%s: bad row count", what);
  // the kernels step through the rows in 32 bits, by up to kMaxGroups batches of eight
  if (p->rows > kMaxRows) return fail(P3D_ERR_UNSUPPORTED, "%s: more than %lld rows", what, (long long)kMaxRows);
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

template <typename F>
int by_type(int dtype, F &&f) {
  if (dtype == P3D_F32) return f(float{});
  if (dtype == P3D_F16) return f(__half{});
  return f(__nv_bfloat16{});
}

size_t partial_floats(const p3d_residual &p, const Split &c) {
  size_t n = (size_t)(kSums - 1) * c.ctas * p.dim;
  if (p.gate_mode == P3D_GATE_SAMPLE) n += (size_t)c.segments * c.slices * p.dim;
  return n;
}

}  // namespace

int take_row_errors(unsigned *flags) {
  if (int st = rows::take_errors<float>(flags)) return st;
  if (int st = rows::take_errors<__half>(flags)) return st;
  return rows::take_errors<__nv_bfloat16>(flags);
}

int launch_column_join(const float *partials, void *out, int dtype, int64_t count, int dim, cudaStream_t s) {
  const dim3 grid((unsigned)((dim + 31) / 32)), block(32, kRuns);
  by_type(dtype, [&](auto t) {
    using T = decltype(t);
    join_kernel<T><<<grid, block, 0, s>>>(partials, static_cast<T *>(out), Joins{}, count, dim);
    return 0;
  });
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
  const unsigned grid = (unsigned)std::min<int64_t>((blocks + 255) / 256, (int64_t)info.sm_count * 4);
  return by_type(dtype, [&](auto t) {
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
  const Shape s = shape_for(p, false);
  Args a = {};
  set_params(a, p);
  a.in[rows::kX] = p.x;
  a.in[rows::kH] = p.h;
  a.in[rows::kGate] = p.gate_mode == P3D_GATE_ELEMENT ? p.gate : nullptr;
  a.out = out;
  a.y = y;
  a.stats = stats;
  const bool aligned = all_aligned(p, {out, y});
  const bool center = centred(p) || (aligned && !rows::whole_fwd(a));
  int per_sm = per_sm_of(p, s, false);
  const size_t smem = lay_out(a, s, aligned, center, false, &per_sm);
  Split c = split_of(p, s, info.sm_count, per_sm, false);
  if (p.gate_mode == P3D_GATE_SAMPLE) {
    // A CTA that has at least kFoldRows turns of a sample's rows sets that sample's parameters up (524288 x 192, two
    // samples: 166 us, read and activated for each row 185 us), where cutting the rows by sample leaves the longest
    // CTA at most a sixth more of them (16 % more, 512 samples of 1024 x 192: 190 us against 208; 48 % more, 200 of
    // 64 x 4096: 320 against about 260).
    const Split by_sample = split_of(p, s, info.sm_count, per_sm, true);
    const int64_t at_once = by_sample.ctas / by_sample.slices, turns = (by_sample.segments + at_once - 1) / at_once;
    const int64_t rows = (by_sample.segment_rows + by_sample.slices - 1) / by_sample.slices;
    a.gate_folded = rows >= (int64_t)kFoldRows * s.groups * s.rows_at_once() && turns * rows * c.ctas <= p.rows + p.rows / 6;
    if (a.gate_folded) c = by_sample;
  }
  a.segments = (int)c.segments;
  a.slices = (int)c.slices;
  a.segment_rows = (int)c.segment_rows;
  return by_type(p.dtype, [&](auto t) {
    return rows::run_fwd<decltype(t)>(a, aligned, center, s.lanes, s.units, c.ctas, smem, static_cast<cudaStream_t>(stream));
  });
}

extern "C" size_t p3d_residual_bwd_workspace(const p3d_residual *args) {
  DeviceInfo info;
  if (check_args(args, "p3d_residual_bwd_workspace") || args->rows == 0 || device_info(&info)) return 0;
  const Shape s = shape_for(*args, true);
  return partial_floats(*args, split_of(*args, s, info.sm_count, per_sm_of(*args, s, true), true)) * sizeof(float);
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
  const Shape s = shape_for(p, true);
  int per_sm = per_sm_of(p, s, true);
  const Split c = split_of(p, s, info.sm_count, per_sm, true);   // as the workspace was sized
  const size_t need = partial_floats(p, c) * sizeof(float);
  if (workspace_bytes < need || !workspace)
    return fail(P3D_ERR_WORKSPACE, "p3d_residual_bwd: workspace of %zu bytes, %zu needed", workspace_bytes, need);
  Args a = {};
  set_params(a, p);
  a.in[rows::kX] = dy ? p.x : nullptr;
  a.in[rows::kH] = p.h;
  a.in[rows::kGate] = p.gate_mode == P3D_GATE_ELEMENT ? p.gate : nullptr;
  a.in[rows::kDout] = dout;
  a.in[rows::kDy] = dy;
  a.stats = const_cast<float *>(stats);
  a.dx = dx;
  a.dh = dh;
  a.dgate = dgate;
  a.partials = static_cast<float *>(workspace);
  a.segments = (int)c.segments;
  a.slices = (int)c.slices;
  a.segment_rows = (int)c.segment_rows;
  const bool aligned =
      all_aligned(p, {dout, dy, dx, dh, workspace, p.gate_mode == P3D_GATE_ELEMENT ? (const void *)dgate : nullptr});
  const bool center = centred(p) || dpost_bias || dnext_bias || (aligned && !rows::whole_bwd(a));
  const size_t smem = lay_out(a, s, aligned, center, true, &per_sm);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (int status = by_type(p.dtype, [&](auto t) {
        return rows::run_bwd<decltype(t)>(a, aligned, center, c.ctas, smem, st);
      }))
    return status;
  // the column sums over the CTAs
  const dim3 block(32, kRuns);
  const unsigned tiles = (unsigned)((p.dim + 31) / 32);
  const Joins j = {{dscale, dpost_weight, dpost_bias, dnext_weight, dnext_bias}};
  if (dscale || dpost_weight || dpost_bias || dnext_weight || dnext_bias) {
    by_type(p.param_dtype, [&](auto w) {
      join_kernel<decltype(w)><<<dim3(tiles, kSums - 1), block, 0, st>>>(a.partials, nullptr, j, c.ctas, p.dim);
      return 0;
    });
    P3D_LAUNCH_CHECK();
  }
  if (p.gate_mode == P3D_GATE_SAMPLE && dgate) {
    const float *part = a.partials + (int64_t)(kSums - 1) * c.ctas * p.dim;
    for (int64_t first = 0; first < c.segments; first += 65535) {   // the grid's y limit
      const unsigned n = (unsigned)std::min<int64_t>(65535, c.segments - first);
      by_type(p.dtype, [&](auto t) {
        using T = decltype(t);
        join_kernel<T><<<dim3(tiles, n), block, 0, st>>>(part + first * c.slices * p.dim,
                                                         static_cast<T *>(dgate) + first * p.dim, j, c.slices, p.dim);
        return 0;
      });
      P3D_LAUNCH_CHECK();
    }
  }
  return P3D_OK;
}
