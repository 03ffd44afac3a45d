// Norms of queries and keys for each head with the rotation of their positions, one pass in each direction:
//
//     y = R(pos) u,   u = N(x) * w + b,   pair i of an axis:  (u_a cos - u_b sin, u_a sin + u_b cos),  angle pos * base^(-i / pairs)
//     up = R(-pos) dy,  dw = sum up * N(x),  db = sum up,  g = up * w,  dx = r (g - N mean(g N) [- mean(g)])
//
// Angles: the frequency of each pair is a whole number f of 2^-64 turns, and pos * f modulo 2^64 is the angle's fraction of a
// turn without any rounding, at any position (an fp32 angle is off by 2^-24 of itself: 0.006 radians at position 100,000). Its
// top 32 bits go to sine and cosine: for 16-bit tensors from the special-function unit (2^-21 absolute, against half a
// step of 2^-11 at best), for fp32 sincospif.
//
// Bound by HBM: forward reads x and writes y, backward reads x and dy and writes dx; nothing is saved between them but x, as
// N(x) costs less to make again than to read. Layout: a row (token, head) of D columns is S = D / 8 lanes (up to a power of two), 16
// bytes each; 32 / S rows a pass, U passes of loads in flight. A lane keeps the same four pairs for all rows, so a token's
// angles are computed once for its rows, and each of the 32 / S lane groups computes a share of the four and hands it round by
// shuffles.
#include <math.h>

#include <algorithm>

#include "common.cuh"
#include "sm100.cuh"

namespace p3d {
namespace {

constexpr int kWarps = 8;
constexpr int kMaxPairs = 128;

struct RotateParams {
  const void *x0, *x1, *dy0, *dy1;
  void *y0, *y1;   // dx in the backward
  const void *w0, *w1, *b0, *b1;
  float *partial;  // [4][blocks][dim]: dweight 0, 1, dbias 0, 1
  const void *pos;
  int64_t ts0, ts1, hs0, hs1, ps, as;
  uint32_t items, chunks, tokens, position_rows;
  int h0, h1, kind0, kind1, pd0, pd1, dim, pos4;
  float eps0, eps1;
  int end0, end1, end2;   // pairs up to the end of each axis
  uint64_t turns[kMaxPairs];
};

// Eight columns of a row in fp32; those past `n` are zero.
template <typename T, bool kVec>
__device__ __forceinline__ void load8(const T *p, int n, float2 (&v)[4]) {
  if constexpr (kVec) {
    if (n <= 0) {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = make_float2(0.f, 0.f);
    } else if constexpr (sizeof(T) == 2) {
      const uint4 raw = __ldcs(reinterpret_cast<const uint4 *>(p));
      v[0] = unpack2<T>(raw.x), v[1] = unpack2<T>(raw.y), v[2] = unpack2<T>(raw.z), v[3] = unpack2<T>(raw.w);
    } else {
      const float4 a = __ldcs(reinterpret_cast<const float4 *>(p)), b = __ldcs(reinterpret_cast<const float4 *>(p) + 1);
      v[0] = make_float2(a.x, a.y), v[1] = make_float2(a.z, a.w);
      v[2] = make_float2(b.x, b.y), v[3] = make_float2(b.z, b.w);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      v[i] = make_float2(2 * i < n ? to_f32<T>(p[2 * i]) : 0.f, 2 * i + 1 < n ? to_f32<T>(p[2 * i + 1]) : 0.f);
  }
}

template <typename T> __device__ __forceinline__ uint32_t pack2(float2 v);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float2 v) { return sm100::pack_bf16(v.x, v.y); }
template <> __device__ __forceinline__ uint32_t pack2<__half>(float2 v) { return sm100::pack_f16(v.x, v.y); }
template <> __device__ __forceinline__ uint32_t pack2<float>(float2) { return 0; }

template <typename T, bool kVec>
__device__ __forceinline__ void store8(T *p, int n, const float2 (&v)[4]) {
  if constexpr (kVec) {
    if (n <= 0) return;
    if constexpr (sizeof(T) == 2) {
      *reinterpret_cast<uint4 *>(p) = make_uint4(pack2<T>(v[0]), pack2<T>(v[1]), pack2<T>(v[2]), pack2<T>(v[3]));
    } else {
      reinterpret_cast<float4 *>(p)[0] = make_float4(v[0].x, v[0].y, v[1].x, v[1].y);
      reinterpret_cast<float4 *>(p)[1] = make_float4(v[2].x, v[2].y, v[3].x, v[3].y);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (2 * i < n) p[2 * i] = from_f32<T>(v[i].x);
      if (2 * i + 1 < n) p[2 * i + 1] = from_f32<T>(v[i].y);
    }
  }
}

template <int S>
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
  for (int o = S / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// A lane's eight columns of a parameter (`missing` where there is none).
__device__ __forceinline__ void load_param(const void *p, int dtype, int c, int n, float missing, float2 (&v)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[i].x = p && 2 * i < n ? load_any(p, dtype, c + 2 * i) : missing;
    v[i].y = p && 2 * i + 1 < n ? load_any(p, dtype, c + 2 * i + 1) : missing;
  }
}

// What a lane knows of its four pairs: its share of the frequencies and the axes they belong to.
template <int S>
struct Phases {
  static constexpr int R = 32 / S, kGroups = R < 4 ? R : 4, kMine = 4 / kGroups;
  uint64_t turn[kMine];
  int axis[kMine];
  float2 cs[4], sn[4];   // (cos, cos) and (-sin, sin) of each pair
  __device__ __forceinline__ void init(const RotateParams &p, int lane) {
    const int chunk = lane % S, group = lane / S % kGroups;
#pragma unroll
    for (int m = 0; m < kMine; ++m) {
      const int pair = chunk * 4 + m * kGroups + group;
      turn[m] = pair < p.end2 ? p.turns[pair] : 0;
      axis[m] = pair < p.end0 || pair >= p.end2 ? 0 : pair < p.end1 ? 1 : 2;
    }
  }
  template <typename T>
  __device__ __forceinline__ void at(const RotateParams &p, uint32_t token, int lane) {
    const uint32_t row = p.position_rows == p.tokens ? token : token % p.position_rows;
    float c[kMine], s[kMine];
#pragma unroll
    for (int m = 0; m < kMine; ++m) {
      const int64_t where = (int64_t)row * p.ps + axis[m] * p.as;
      const int64_t pos = p.pos4 ? static_cast<const int32_t *>(p.pos)[where] : static_cast<const int64_t *>(p.pos)[where];
      const int32_t part = (int32_t)(((uint64_t)pos * turn[m]) >> 32);   // 2^-32 turns, -0.5 .. 0.5
      const float half_turns = (float)part * 4.656612873077393e-10f;     // 2^-31
      if constexpr (sizeof(T) == 2)
        __sincosf(half_turns * 3.14159265f, &s[m], &c[m]);
      else
        sincospif(half_turns, &s[m], &c[m]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int from = (i % kGroups) * S + lane % S;
      const float ci = __shfl_sync(0xffffffffu, c[i / kGroups], from);
      const float si = __shfl_sync(0xffffffffu, s[i / kGroups], from);
      cs[i] = make_float2(ci, ci);
      sn[i] = make_float2(-si, si);
    }
  }
  // R(pos), or R(-pos) for kBack, of the four pairs
  template <bool kBack>
  __device__ __forceinline__ void turn4(float2 (&v)[4]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 swapped = kBack ? make_float2(-v[i].y, -v[i].x) : make_float2(v[i].y, v[i].x);
      v[i] = sm100::fma2(swapped, sn[i], sm100::mul2(v[i], cs[i]));
    }
  }
};

// N(x) in place; returns 1 / deviation (1 without a norm).
template <int S>
__device__ __forceinline__ float normalise(float2 (&v)[4], int n, int kind, float eps, float inv_dim) {
  if (kind == P3D_NORM_NONE) return 1.f;
  if (kind == P3D_NORM_LAYER) {
    const float2 t = sm100::add2(sm100::add2(v[0], v[1]), sm100::add2(v[2], v[3]));
    const float mean = row_sum<S>(t.x + t.y) * inv_dim;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i].x = 2 * i < n ? v[i].x - mean : 0.f;
      v[i].y = 2 * i + 1 < n ? v[i].y - mean : 0.f;
    }
  }
  float2 q = sm100::mul2(v[0], v[0]);
#pragma unroll
  for (int i = 1; i < 4; ++i) q = sm100::fma2(v[i], v[i], q);
  const float r = rsqrtf(row_sum<S>(q.x + q.y) * inv_dim + eps);
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = sm100::mul2(v[i], make_float2(r, r));
  return r;
}

// A row: its input, its place in the contiguous output, its norm.
struct Row {
  int64_t in, out;
  bool second;
};
__device__ __forceinline__ Row row_at(const RotateParams &p, uint32_t token, int h) {
  Row r;
  r.second = h >= p.h0;
  const int head = r.second ? h - p.h0 : h;
  r.in = (int64_t)token * (r.second ? p.ts1 : p.ts0) + head * (r.second ? p.hs1 : p.hs0);
  r.out = ((int64_t)token * (r.second ? p.h1 : p.h0) + head) * p.dim;
  return r;
}

template <typename T, int S, int U, bool kVec>
__global__ void __launch_bounds__(kWarps * 32) norm_rotate_kernel(const __grid_constant__ RotateParams p) {
  constexpr int R = 32 / S;
  const int lane = threadIdx.x & 31, c = lane % S * 8, n = p.dim - c, rows = p.h0 + p.h1;
  const float inv_dim = 1.f / p.dim;
  Phases<S> ph;
  ph.init(p, lane);
  float2 w[2][4], b[2][4];
  load_param(p.w0, p.pd0, c, n, 1.f, w[0]);
  load_param(p.w1, p.pd1, c, n, 1.f, w[1]);
  load_param(p.b0, p.pd0, c, n, 0.f, b[0]);
  load_param(p.b1, p.pd1, c, n, 0.f, b[1]);
  const uint32_t stride = gridDim.x * kWarps;
  for (uint32_t item = blockIdx.x * kWarps + threadIdx.x / 32; item < p.items; item += stride) {
    const uint32_t token = p.chunks == 1 ? item : item / p.chunks;
    const int first = (int)(item - token * p.chunks) * U * R + lane / S;
    float2 v[U][4];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = first + u * R;
      const Row r = row_at(p, token, h);
      load8<T, kVec>(static_cast<const T *>(r.second ? p.x1 : p.x0) + r.in + c, h < rows ? n : 0, v[u]);
    }
    ph.template at<T>(p, token, lane);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = first + u * R;
      const Row r = row_at(p, token, h);
      normalise<S>(v[u], n, r.second ? p.kind1 : p.kind0, r.second ? p.eps1 : p.eps0, inv_dim);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        v[u][i] = r.second ? sm100::fma2(v[u][i], w[1][i], b[1][i]) : sm100::fma2(v[u][i], w[0][i], b[0][i]);
      ph.template turn4<false>(v[u]);
      store8<T, kVec>(static_cast<T *>(r.second ? p.y1 : p.y0) + r.out + c, h < rows ? n : 0, v[u]);
    }
  }
}

template <typename T, int S, int U, bool kVec, bool kParams>
__global__ void __launch_bounds__(kWarps * 32) norm_rotate_bwd_kernel(const __grid_constant__ RotateParams p) {
  constexpr int R = 32 / S;
  const int lane = threadIdx.x & 31, c = lane % S * 8, n = p.dim - c, rows = p.h0 + p.h1;
  const float inv_dim = 1.f / p.dim;
  Phases<S> ph;
  ph.init(p, lane);
  float2 w[2][4], sum[4][4];   // sums: dweight 0, 1, dbias 0, 1
  load_param(p.w0, p.pd0, c, n, 1.f, w[0]);
  load_param(p.w1, p.pd1, c, n, 1.f, w[1]);
#pragma unroll
  for (int i = 0; i < 16; ++i) sum[i / 4][i % 4] = make_float2(0.f, 0.f);
  const uint32_t stride = gridDim.x * kWarps;
  for (uint32_t item = blockIdx.x * kWarps + threadIdx.x / 32; item < p.items; item += stride) {
    const uint32_t token = p.chunks == 1 ? item : item / p.chunks;
    const int first = (int)(item - token * p.chunks) * U * R + lane / S;
    float2 v[U][4], g[U][4];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = first + u * R;
      const Row r = row_at(p, token, h);
      load8<T, kVec>(static_cast<const T *>(r.second ? p.x1 : p.x0) + r.in + c, h < rows ? n : 0, v[u]);
      load8<T, kVec>(static_cast<const T *>(r.second ? p.dy1 : p.dy0) + r.out + c, h < rows ? n : 0, g[u]);
    }
    ph.template at<T>(p, token, lane);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = first + u * R;
      const Row r = row_at(p, token, h);
      const int kind = r.second ? p.kind1 : p.kind0;
      const float dev = normalise<S>(v[u], n, kind, r.second ? p.eps1 : p.eps0, inv_dim);
      ph.template turn4<true>(g[u]);
      if constexpr (kParams) {
        // rows past the last are zeros in g: an eps of 0 would make their norm NaN
        if (h < rows) {
          if (r.second) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              sum[1][i] = sm100::fma2(g[u][i], v[u][i], sum[1][i]);
              sum[3][i] = sm100::add2(g[u][i], sum[3][i]);
            }
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              sum[0][i] = sm100::fma2(g[u][i], v[u][i], sum[0][i]);
              sum[2][i] = sm100::add2(g[u][i], sum[2][i]);
            }
          }
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) g[u][i] = sm100::mul2(g[u][i], r.second ? w[1][i] : w[0][i]);
      if (kind != P3D_NORM_NONE) {
        float2 t = sm100::mul2(g[u][0], v[u][0]);
#pragma unroll
        for (int i = 1; i < 4; ++i) t = sm100::fma2(g[u][i], v[u][i], t);
        const float gn = -row_sum<S>(t.x + t.y) * inv_dim;
        float mean = 0.f;
        if (kind == P3D_NORM_LAYER) {
          t = sm100::add2(sm100::add2(g[u][0], g[u][1]), sm100::add2(g[u][2], g[u][3]));
          mean = -row_sum<S>(t.x + t.y) * inv_dim;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          g[u][i] = sm100::fma2(v[u][i], make_float2(gn, gn), sm100::add2(g[u][i], make_float2(mean, mean)));
          g[u][i] = sm100::mul2(g[u][i], make_float2(dev, dev));
        }
      }
      T *const dx = static_cast<T *>(r.second ? p.y1 : p.y0);
      if (dx) store8<T, kVec>(dx + r.out + c, h < rows ? n : 0, g[u]);
    }
  }
  if constexpr (kParams) {
    // the rows of a warp, then the warps of the block, each in a fixed order
    __shared__ float2 joined[kWarps][S][4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int o = S; o < 32; o <<= 1) {
          sum[k][i].x += __shfl_xor_sync(0xffffffffu, sum[k][i].x, o);
          sum[k][i].y += __shfl_xor_sync(0xffffffffu, sum[k][i].y, o);
        }
      __syncthreads();
      if (lane < S) {
#pragma unroll
        for (int i = 0; i < 4; ++i) joined[threadIdx.x / 32][lane][i] = sum[k][i];
      }
      __syncthreads();
      for (int col = threadIdx.x; col < p.dim; col += kWarps * 32) {
        float total = 0.f;
        for (int q = 0; q < kWarps; ++q) total += reinterpret_cast<const float *>(joined[q])[col];
        p.partial[((int64_t)k * gridDim.x + blockIdx.x) * p.dim + col] = total;
      }
    }
  }
}

// Column sums of the blocks' partial sums: blockIdx.y says which of the four.
struct JoinParams {
  void *out[4];
  int dtype[4];
};
__global__ void __launch_bounds__(1024) rotate_join_kernel(const float *partial, int blocks, int dim, const JoinParams j) {
  __shared__ float s[32][33];
  const int k = blockIdx.y, col = blockIdx.x * 32 + threadIdx.x % 32;
  void *const out = k == 0 ? j.out[0] : k == 1 ? j.out[1] : k == 2 ? j.out[2] : j.out[3];
  const int dtype = k == 0 ? j.dtype[0] : k == 1 ? j.dtype[1] : k == 2 ? j.dtype[2] : j.dtype[3];
  if (!out) return;
  float v = 0.f;
  if (col < dim)
    for (int i = threadIdx.x / 32; i < blocks; i += 32) v += partial[((int64_t)k * blocks + i) * dim + col];
  s[threadIdx.x / 32][threadIdx.x % 32] = v;
  __syncthreads();
  if (threadIdx.x >= 32 || col >= dim) return;
  float total = 0.f;
  for (int i = 0; i < 32; ++i) total += s[i][threadIdx.x];
  store_any(out, dtype, col, total);
}

// ------------------------------------------------------------------------------- host
struct Plan {
  RotateParams p;
  int lanes, passes, vec;
  int warps;   // that one wave of the device holds
};

int plan(const p3d_norm_rotate *a, Plan *out) {
  P3D_CHECK_ARG(a != nullptr, "p3d_norm_rotate: null arguments");
  P3D_CHECK_ARG(dtype_ok(a->dtype), "p3d_norm_rotate: unknown dtype %d", a->dtype);
  P3D_CHECK_ARG(a->dim >= 2 && a->dim <= 256 && a->dim % 2 == 0, "p3d_norm_rotate: head dim must be even, 2 to 256, got %d",
                a->dim);
  P3D_CHECK_ARG(a->heads[0] >= 1 && a->heads[1] >= 0, "p3d_norm_rotate: heads must be positive");
  P3D_CHECK_ARG(a->tokens >= 0 && a->position_rows >= (a->tokens ? 1 : 0), "p3d_norm_rotate: token count must not be negative");
  if (a->tokens >= (1ll << 31) || (int64_t)a->tokens * (a->heads[0] + (int64_t)a->heads[1]) >= (1ll << 31))
    return fail(P3D_ERR_UNSUPPORTED, "p3d_norm_rotate: at most 2^31 - 1 rows (tokens x heads)");
  P3D_CHECK_ARG(a->axes >= 1 && a->axes <= 3, "p3d_norm_rotate: 1 to 3 position axes");
  P3D_CHECK_ARG(a->position_bytes == 4 || a->position_bytes == 8, "p3d_norm_rotate: positions must be int32 or int64");
  P3D_CHECK_ARG(isfinite(a->base) && a->base >= 1.0, "p3d_norm_rotate: base must be at least 1");
  int total = 0;
  for (int i = 0; i < a->axes; ++i) {
    P3D_CHECK_ARG(a->pairs[i] >= 0 && a->pairs[i] <= kMaxPairs, "p3d_norm_rotate: pairs must not be negative");
    total += a->pairs[i];
  }
  P3D_CHECK_ARG(2 * total <= a->dim, "p3d_norm_rotate: the axes' pairs take more than the head dim's columns");
  for (int i = 0; i < 2; ++i) {
    P3D_CHECK_ARG(a->kind[i] >= P3D_NORM_NONE && a->kind[i] <= P3D_NORM_LAYER, "p3d_norm_rotate: unknown norm kind");
    P3D_CHECK_ARG(isfinite(a->eps[i]) && a->eps[i] >= 0, "p3d_norm_rotate: eps must be finite and not negative");
    P3D_CHECK_ARG(a->param_dtype[i] == a->dtype || a->param_dtype[i] == P3D_F32,
                  "p3d_norm_rotate: parameters must be of the tensors' dtype or fp32");
  }
  P3D_CHECK_ARG(a->tokens == 0 || (a->x[0] && (a->x[1] || !a->heads[1]) && a->positions), "p3d_norm_rotate: null input");
  RotateParams &p = out->p;
  p = {};
  p.x0 = a->x[0], p.x1 = a->x[1];
  const bool n0 = a->kind[0] != P3D_NORM_NONE, n1 = a->kind[1] != P3D_NORM_NONE;
  p.w0 = n0 ? a->weight[0] : nullptr, p.b0 = n0 ? a->bias[0] : nullptr;
  p.w1 = n1 ? a->weight[1] : nullptr, p.b1 = n1 ? a->bias[1] : nullptr;
  p.pos = a->positions;
  p.ts0 = a->token_stride[0], p.ts1 = a->token_stride[1], p.hs0 = a->head_stride[0], p.hs1 = a->head_stride[1];
  p.ps = a->position_stride, p.as = a->axis_stride;
  p.tokens = (uint32_t)a->tokens;
  p.position_rows = (uint32_t)std::min(a->position_rows, a->tokens);
  p.h0 = a->heads[0], p.h1 = a->heads[1], p.kind0 = a->kind[0], p.kind1 = a->kind[1];
  p.pd0 = a->param_dtype[0], p.pd1 = a->param_dtype[1], p.eps0 = a->eps[0], p.eps1 = a->eps[1];
  p.dim = a->dim, p.pos4 = a->position_bytes == 4;
  p.end0 = a->pairs[0];
  p.end1 = p.end0 + (a->axes > 1 ? a->pairs[1] : 0);
  p.end2 = p.end1 + (a->axes > 2 ? a->pairs[2] : 0);
  // frequencies in 2^-64 turns; those of the last base and pairs are still there
  struct Memo {
    double base = 0;
    int pairs[3] = {-1, -1, -1};
    uint64_t turns[kMaxPairs];
  };
  static thread_local Memo memo;
  const int pairs[3] = {p.end0, p.end1 - p.end0, p.end2 - p.end1};
  if (memo.base != a->base || !std::equal(pairs, pairs + 3, memo.pairs)) {
    int at = 0;
    for (int axis = 0; axis < 3; ++axis)
      for (int i = 0; i < pairs[axis]; ++i)
        memo.turns[at++] = (uint64_t)llroundl(ldexpl((long double)pow(a->base, -(double)i / pairs[axis]) / 6.283185307179586476925287L, 64) );
    memo.base = a->base;
    std::copy(pairs, pairs + 3, memo.pairs);
  }
  std::copy(memo.turns, memo.turns + p.end2, p.turns);
  int lanes = 1;
  while (lanes * 8 < a->dim) lanes *= 2;
  out->lanes = lanes;
  out->passes = (p.h0 + p.h1 + 32 / lanes - 1) / (32 / lanes);
  const int unit = 16 / dtype_size(a->dtype);
  auto fits = [&](const void *x, int64_t ts, int64_t hs) { return (uintptr_t)x % 16 == 0 && ts % unit == 0 && hs % unit == 0; };
  out->vec = a->dim % 8 == 0 && fits(p.x0, p.ts0, p.hs0) && (!p.h1 || fits(p.x1, p.ts1, p.hs1));
  DeviceInfo info;
  if (int st = device_info(&info)) return st;
  out->warps = info.sm_count * 32;
  return P3D_OK;
}

// Passes of a warp's item: as many loads in flight as the row's heads give, but not so many that the device's warps lack items.
int set_items(Plan *pl, int most) {
  int u = 1;
  while (u < most && u < pl->passes && (int64_t)pl->p.tokens * ((pl->passes + 2 * u - 1) / (2 * u)) >= pl->warps) u *= 2;
  pl->p.chunks = (pl->passes + u - 1) / u;
  pl->p.items = pl->p.tokens * pl->p.chunks;
  return u;
}

template <typename T, int S, int U, bool kVec>
int launch_u(const Plan &pl, bool backward, bool params, int blocks, cudaStream_t s) {
  if (!backward)
    norm_rotate_kernel<T, S, U, kVec><<<blocks, kWarps * 32, 0, s>>>(pl.p);
  else if (params)
    norm_rotate_bwd_kernel<T, S, U, kVec, true><<<blocks, kWarps * 32, 0, s>>>(pl.p);
  else
    norm_rotate_bwd_kernel<T, S, U, kVec, false><<<blocks, kWarps * 32, 0, s>>>(pl.p);
  P3D_LAUNCH_CHECK();
  return P3D_OK;
}

template <typename T, int S>
int launch_s(const Plan &pl, int u, bool backward, bool params, int blocks, cudaStream_t s) {
  if (!pl.vec) return launch_u<T, S, 1, false>(pl, backward, params, blocks, s);
  switch (u) {
    case 1: return launch_u<T, S, 1, true>(pl, backward, params, blocks, s);
    case 2: return launch_u<T, S, 2, true>(pl, backward, params, blocks, s);
    default: return launch_u<T, S, 4, true>(pl, backward, params, blocks, s);
  }
}

template <typename T>
int launch_t(const Plan &pl, int u, bool backward, bool params, int blocks, cudaStream_t s) {
  switch (pl.lanes) {
    case 1: return launch_s<T, 1>(pl, u, backward, params, blocks, s);
    case 2: return launch_s<T, 2>(pl, u, backward, params, blocks, s);
    case 4: return launch_s<T, 4>(pl, u, backward, params, blocks, s);
    case 8: return launch_s<T, 8>(pl, u, backward, params, blocks, s);
    case 16: return launch_s<T, 16>(pl, u, backward, params, blocks, s);
    default: return launch_s<T, 32>(pl, u, backward, params, blocks, s);
  }
}

int launch(const Plan &pl, int dtype, int u, bool backward, bool params, int blocks, cudaStream_t s) {
  switch (dtype) {
    case P3D_F16: return launch_t<__half>(pl, u, backward, params, blocks, s);
    case P3D_BF16: return launch_t<__nv_bfloat16>(pl, u, backward, params, blocks, s);
    default: return launch_t<float>(pl, u, backward, params, blocks, s);
  }
}

// Blocks of the backward: what one wave holds, as each leaves a row of partial sums.
int backward_blocks(const Plan &pl) {
  return (int)std::min<int64_t>((pl.p.items + kWarps - 1) / kWarps, std::max(1, pl.warps / 32 * 2));
}

}  // namespace
}  // namespace p3d

using namespace p3d;

extern "C" {

int p3d_norm_rotate_fwd(const p3d_norm_rotate *args, void *y0, void *y1, void *stream) {
  Plan pl;
  if (int st = plan(args, &pl)) return st;
  if (args->tokens == 0) return P3D_OK;
  P3D_CHECK_ARG(y0 && (y1 || !args->heads[1]), "p3d_norm_rotate_fwd: null output");
  pl.vec = pl.vec && (uintptr_t)y0 % 16 == 0 && (uintptr_t)y1 % 16 == 0;
  pl.p.y0 = y0, pl.p.y1 = y1;
  const int u = set_items(&pl, pl.vec ? 4 : 1);
  const int64_t blocks = std::min<int64_t>((pl.p.items + kWarps - 1) / kWarps, pl.warps / 32 * 6);
  return launch(pl, args->dtype, u, false, false, (int)blocks, (cudaStream_t)stream);
}

size_t p3d_norm_rotate_bwd_workspace(const p3d_norm_rotate *args) {
  Plan pl;
  if (plan(args, &pl) != P3D_OK || args->tokens == 0) return 0;
  set_items(&pl, 1);
  return sizeof(float) * 4 * (size_t)backward_blocks(pl) * pl.p.dim;
}

int p3d_norm_rotate_bwd(const p3d_norm_rotate *args, const void *const dy[2], void *const dx[2], void *const dweight[2],
                        void *const dbias[2], void *workspace, size_t workspace_bytes, void *stream) {
  Plan pl;
  if (int st = plan(args, &pl)) return st;
  if (args->tokens == 0) return P3D_OK;
  P3D_CHECK_ARG(dy && dx && dweight && dbias && dy[0] && (dy[1] || !args->heads[1]), "p3d_norm_rotate_bwd: null gradient");
  const bool params = dweight[0] || dweight[1] || dbias[0] || dbias[1];
  for (int i = 0; i < 2; ++i)
    P3D_CHECK_ARG(args->kind[i] != P3D_NORM_NONE || (!dweight[i] && !dbias[i]),
                  "p3d_norm_rotate_bwd: parameters' gradients without a norm");
  auto aligned = [](const void *q) { return (uintptr_t)q % 16 == 0; };
  pl.vec = pl.vec && aligned(dy[0]) && aligned(dy[1]) && aligned(dx[0]) && aligned(dx[1]);
  pl.p.dy0 = dy[0], pl.p.dy1 = dy[1], pl.p.y0 = dx[0], pl.p.y1 = dx[1];
  // two passes in flight: four take the registers of the parameters' sums
  const int u = set_items(&pl, pl.vec ? 2 : 1);
  const int blocks = backward_blocks(pl);
  pl.p.partial = static_cast<float *>(workspace);
  if (params && (!workspace || workspace_bytes < sizeof(float) * 4 * (size_t)blocks * pl.p.dim))
    return fail(P3D_ERR_WORKSPACE, "p3d_norm_rotate_bwd: workspace of %zu bytes needed",
                sizeof(float) * 4 * (size_t)blocks * pl.p.dim);
  if (int st = launch(pl, args->dtype, u, true, params, blocks, (cudaStream_t)stream)) return st;
  if (!params) return P3D_OK;
  JoinParams j = {{dweight[0], dweight[1], dbias[0], dbias[1]},
                  {args->param_dtype[0], args->param_dtype[1], args->param_dtype[0], args->param_dtype[1]}};
  rotate_join_kernel<<<dim3((pl.p.dim + 31) / 32, 4), 1024, 0, (cudaStream_t)stream>>>(pl.p.partial, blocks, pl.p.dim, j);
  P3D_LAUNCH_CHECK();
  return P3D_OK;
}

}  // extern "C"
