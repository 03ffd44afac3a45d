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
// bytes each; 32 / S rows a pass, U passes an item, an item a warp. A warp has the same heads of one token after another, so that a
// lane's parameters and places are fixed, and the rows of two items ahead are in flight while one is worked on. A lane holds the
// same four pairs of every row, and each of the 32 / S lane groups computes a share of their angles and hands it round by
// shuffles.
//
// Measured, bf16: 16,384 tokens of 32 + 8 heads of 128, forward 70 us (4.8 TB/s), backward 110 (4.6); 262,144 tokens of 4 + 4 heads of
// 48 on three axes, 91 (4.4) and 145 (4.2), where two lanes of eight are idle. Issue slots are 60 % used at 30 and 23 % occupancy: the
// registers of the rows ahead and of the sums are what more warps would need. At those dims the forward spills nothing up to 64 columns and 32
// bytes of two passes of 128, the backward 12; above 128 columns 124 and up to 196 (not measured).
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "sm100.cuh"

namespace p3d {
namespace {

constexpr int kWarps = 4, kAhead = 2;
constexpr int kMaxPairs = 128;

struct RotateParams {
  const void *x0, *x1, *dy0, *dy1;
  void *y0, *y1;   // dx in the backward
  const void *w0, *w1, *b0, *b1;
  float *partial;  // [4][blocks][dim]: dweight 0, 1, dbias 0, 1
  const void *pos;
  int64_t ts0, ts1, hs0, hs1, ps, as;
  uint32_t tokens, position_rows, chunks;   // chunks: items of a token; the grid's warps are a multiple of it
  int h0, h1, kind0, kind1, pd0, pd1, dim, pos4;
  float eps0, eps1;
  int end0, end1, end2;   // pairs up to the end of each axis
  uint64_t turns[kMaxPairs];
};

// Eight columns of a row as they lie in memory; those past `n` are zero.
template <typename T> struct Raw {
  uint32_t w[2 * sizeof(T)];
};
template <typename T, bool kVec>
__device__ __forceinline__ void load8(Raw<T> &r, const T *p, int n) {
  constexpr int kWords = 2 * sizeof(T);
  if constexpr (kVec) {
#pragma unroll
    for (int i = 0; i < kWords; i += 4) {
      uint4 v = make_uint4(0, 0, 0, 0);
      if (n > 0) v = __ldcs(reinterpret_cast<const uint4 *>(p) + i / 4);
      r.w[i] = v.x, r.w[i + 1] = v.y, r.w[i + 2] = v.z, r.w[i + 3] = v.w;
    }
  } else {
    alignas(16) T v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? p[i] : from_f32<T>(0.f);
    memcpy(r.w, v, sizeof(r.w));
  }
}
template <typename T>
__device__ __forceinline__ void unpack8(const Raw<T> &r, float2 (&v)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 2) v[i] = unpack2<T>(r.w[i]);
    else v[i] = make_float2(__uint_as_float(r.w[2 * i]), __uint_as_float(r.w[2 * i + 1]));
  }
}

template <typename T> __device__ __forceinline__ uint32_t pack2(float2 v);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float2 v) { return sm100::pack_bf16(v.x, v.y); }
template <> __device__ __forceinline__ uint32_t pack2<__half>(float2 v) { return sm100::pack_f16(v.x, v.y); }

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
  int64_t axis[kMine];   // where the axis lies in a token's positions
  __device__ __forceinline__ void init(const RotateParams &p, int lane) {
    const int chunk = lane % S, group = lane / S % kGroups;
#pragma unroll
    for (int m = 0; m < kMine; ++m) {
      const int pair = chunk * 4 + m * kGroups + group;
      turn[m] = pair < p.end2 ? p.turns[pair] : 0;
      axis[m] = p.as * (pair < p.end0 || pair >= p.end2 ? 0 : pair < p.end1 ? 1 : 2);
    }
  }
  struct Position {
    int64_t at[kMine];
  };
  __device__ __forceinline__ Position load(const RotateParams &p, uint32_t token) const {
    Position r;
    const uint32_t row = p.position_rows == p.tokens ? token : token % p.position_rows;
#pragma unroll
    for (int m = 0; m < kMine; ++m) {
      const int64_t where = (int64_t)row * p.ps + axis[m];
      r.at[m] = token >= p.tokens ? 0 : p.pos4 ? static_cast<const int32_t *>(p.pos)[where] : static_cast<const int64_t *>(p.pos)[where];
    }
    return r;
  }
  struct Angles {
    float c[4], s[4];
    // R(pos), or R(-pos) for kBack, of the four pairs, of which only the first `turned` turn: columns past them stand alone, whatever is
    // beside them
    template <bool kBack>
    __device__ __forceinline__ void turn4(int turned, float2 (&v)[4]) const {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float a = v[i].x, b = v[i].y, t = kBack ? -s[i] : s[i];
        if (i < turned) v[i] = make_float2(fmaf(-b, t, a * c[i]), fmaf(a, t, b * c[i]));
      }
    }
  };
  template <typename T>
  __device__ __forceinline__ Angles angles(const Position &at, int lane) const {
    float mc[kMine], ms[kMine];
#pragma unroll
    for (int m = 0; m < kMine; ++m) {
      const int32_t part = (int32_t)(((uint64_t)at.at[m] * turn[m]) >> 32);   // 2^-32 turns, -0.5 .. 0.5
      if constexpr (sizeof(T) == 2) __sincosf((float)part * 1.4629180792671596e-9f, &ms[m], &mc[m]);   // 2 pi 2^-32
      else sincospif((float)part * 4.656612873077393e-10f, &ms[m], &mc[m]);                            // 2^-31
    }
    Angles r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int from = (i % kGroups) * S + lane % S;
      r.c[i] = __shfl_sync(0xffffffffu, mc[i / kGroups], from);
      r.s[i] = __shfl_sync(0xffffffffu, ms[i / kGroups], from);
    }
    return r;
  }
};

// N(x) in place; returns 1 / deviation (1 without a norm).  Kinds may differ within a warp: all lanes take part in the sums.
template <int S>
__device__ __forceinline__ float normalise(float2 (&v)[4], int n, int kind, float eps, float inv_dim, bool any_layer) {
  if (any_layer) {
    const float2 t = sm100::add2(sm100::add2(v[0], v[1]), sm100::add2(v[2], v[3]));
    const float mean = row_sum<S>(t.x + t.y) * inv_dim;
    if (kind == P3D_NORM_LAYER) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[i].x = 2 * i < n ? v[i].x - mean : 0.f;
        v[i].y = 2 * i + 1 < n ? v[i].y - mean : 0.f;
      }
    }
  }
  float2 q = sm100::mul2(v[0], v[0]);
#pragma unroll
  for (int i = 1; i < 4; ++i) q = sm100::fma2(v[i], v[i], q);
  const float sum = row_sum<S>(q.x + q.y);
  const float r = kind == P3D_NORM_NONE ? 1.f : rsqrtf(fmaf(sum, inv_dim, eps));
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = sm100::mul2(v[i], make_float2(r, r));
  return r;
}

// A lane's row of every token that its warp visits: addresses at the warp's first token and steps to the next one.
struct Row {
  bool on, second;
  int64_t in, in_step, out, out_step;   // elements
};
__device__ __forceinline__ Row row_of(const RotateParams &p, int h, uint32_t token, uint32_t tokens_step, int c) {
  Row r;
  r.second = h >= p.h0;
  r.on = h < p.h0 + p.h1 && c < p.dim;
  const int head = r.second ? h - p.h0 : h, heads = r.second ? p.h1 : p.h0;
  const int64_t ts = r.second ? p.ts1 : p.ts0;
  r.in = (int64_t)token * ts + head * (r.second ? p.hs1 : p.hs0) + c;
  r.in_step = (int64_t)tokens_step * ts;
  r.out = ((int64_t)token * heads + head) * p.dim + c;
  r.out_step = (int64_t)tokens_step * heads * p.dim;
  return r;
}

template <typename T, int S, int U, bool kVec, bool kBias>
__global__ void __launch_bounds__(kWarps * 32, sizeof(T) == 2 && kVec && !kBias ? 5 : 3)
    norm_rotate_kernel(const __grid_constant__ RotateParams p) {
  constexpr int R = 32 / S;
  const int lane = threadIdx.x & 31, c = lane % S * 8, n = p.dim - c;
  const uint32_t warp = blockIdx.x * kWarps + threadIdx.x / 32, step = gridDim.x * kWarps / p.chunks;
  const uint32_t token0 = warp / p.chunks;
  const float inv_dim = 1.f / p.dim;
  const bool any_layer = p.kind0 == P3D_NORM_LAYER || p.kind1 == P3D_NORM_LAYER;
  const int turned = p.end2 - lane % S * 4;
  Phases<S> ph;
  ph.init(p, lane);
  Row row[U];
  const T *in[U];
  T *out[U];
  float2 w[U][4], b[U][4];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    row[u] = row_of(p, ((int)(warp - token0 * p.chunks) * U + u) * R + lane / S, token0, step, c);
    in[u] = static_cast<const T *>(row[u].second ? p.x1 : p.x0) + row[u].in;
    out[u] = static_cast<T *>(row[u].second ? p.y1 : p.y0) + row[u].out;
    load_param(row[u].second ? p.w1 : p.w0, row[u].second ? p.pd1 : p.pd0, c, n, 1.f, w[u]);
    if constexpr (kBias) load_param(row[u].second ? p.b1 : p.b0, row[u].second ? p.pd1 : p.pd0, c, n, 0.f, b[u]);
  }
  Raw<T> ahead[kAhead][U];
  typename Phases<S>::Position position[kAhead];
  auto fetch = [&](Raw<T> (&r)[U], typename Phases<S>::Position &at, uint32_t token) {
    at = ph.load(p, token);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      load8<T, kVec>(r[u], in[u], row[u].on && token < p.tokens ? n : 0);
      in[u] += row[u].in_step;
    }
  };
  // tokens are below 2^31 and steps far smaller: no token number wraps
#pragma unroll
  for (int k = 0; k < kAhead; ++k) fetch(ahead[k], position[k], token0 + k * step);
  for (uint32_t token = token0; token < p.tokens; token += step) {
    Raw<T> now[U];
#pragma unroll
    for (int u = 0; u < U; ++u) now[u] = ahead[0][u];
    const typename Phases<S>::Angles turn = ph.template angles<T>(position[0], lane);
#pragma unroll
    for (int k = 0; k + 1 < kAhead; ++k) {
#pragma unroll
      for (int u = 0; u < U; ++u) ahead[k][u] = ahead[k + 1][u];
      position[k] = position[k + 1];
    }
    fetch(ahead[kAhead - 1], position[kAhead - 1], token + kAhead * step);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float2 v[4];
      unpack8(now[u], v);
      normalise<S>(v, n, row[u].second ? p.kind1 : p.kind0, row[u].second ? p.eps1 : p.eps0, inv_dim, any_layer);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (kBias) v[i] = sm100::fma2(v[i], w[u][i], b[u][i]);
        else v[i] = sm100::mul2(v[i], w[u][i]);
      }
      turn.template turn4<false>(turned, v);
      store8<T, kVec>(out[u], row[u].on ? n : 0, v);
      out[u] += row[u].out_step;
    }
  }
}

// kAll: every pair of columns turns. A kernel of its own, as the choice costs a tenth here (registers; nothing in the forward). Without it the
// parameters' sums are made whether or not anybody wants them.
template <typename T, int S, bool kVec, bool kParams, bool kAll>
__global__ void __launch_bounds__(kWarps * 32, sizeof(T) == 2 && kVec ? 4 : 3)
    norm_rotate_bwd_kernel(const __grid_constant__ RotateParams p) {
  constexpr int R = 32 / S;
  const int lane = threadIdx.x & 31, c = lane % S * 8, n = p.dim - c;
  const uint32_t warp = blockIdx.x * kWarps + threadIdx.x / 32, step = gridDim.x * kWarps / p.chunks;
  const uint32_t token0 = warp / p.chunks;
  const float inv_dim = 1.f / p.dim;
  const bool any_layer = p.kind0 == P3D_NORM_LAYER || p.kind1 == P3D_NORM_LAYER;
  Phases<S> ph;
  ph.init(p, lane);
  const Row row = row_of(p, (int)(warp - token0 * p.chunks) * R + lane / S, token0, step, c);
  const T *in = static_cast<const T *>(row.second ? p.x1 : p.x0) + row.in;
  const T *up = static_cast<const T *>(row.second ? p.dy1 : p.dy0) + row.out;
  T *out = static_cast<T *>(row.second ? p.y1 : p.y0);
  const bool write = out && row.on;
  out += row.out;
  const int kind = row.second ? p.kind1 : p.kind0;
  const float eps = row.second ? p.eps1 : p.eps0;
  float2 w[4], sum_w[4], sum_b[4];
  load_param(row.second ? p.w1 : p.w0, row.second ? p.pd1 : p.pd0, c, n, 1.f, w);
#pragma unroll
  for (int i = 0; i < 4; ++i) sum_w[i] = sum_b[i] = make_float2(0.f, 0.f);
  // two tokens at a time: one row's sums over its lanes wait on one another, two rows' do not
  Raw<T> ahead_x[2], ahead_g[2];
  typename Phases<S>::Position position[2];
  auto fetch = [&](int k, uint32_t token) {
    position[k] = ph.load(p, token);
    const int m = row.on && token < p.tokens ? n : 0;
    load8<T, kVec>(ahead_x[k], in, m);
    load8<T, kVec>(ahead_g[k], up, m);
    in += row.in_step;
    up += row.out_step;
  };
  fetch(0, token0);
  fetch(1, token0 + step);
  for (uint32_t token = token0; token < p.tokens; token += 2 * step) {
    float2 v[2][4], g[2][4];
    float dev[2], gn[2], mean[2];
    typename Phases<S>::Angles turn[2];
    const bool there[2] = {true, token + step < p.tokens};
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      unpack8(ahead_x[k], v[k]);
      unpack8(ahead_g[k], g[k]);
      turn[k] = ph.template angles<T>(position[k], lane);
    }
    fetch(0, token + 2 * step);
    fetch(1, token + 3 * step);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      // zeros stand for a token that is not there: its norm has to be finite
      dev[k] = normalise<S>(v[k], n, kind, there[k] ? eps : 1.f, inv_dim, any_layer);
      turn[k].template turn4<true>(kAll ? 4 : p.end2 - lane % S * 4, g[k]);
    }
    if constexpr (kParams) {
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          sum_w[i] = sm100::fma2(g[k][i], v[k][i], sum_w[i]);
          sum_b[i] = sm100::add2(g[k][i], sum_b[i]);
        }
    }
    // the norm of a lane group without a row (zeros, an eps of 0) is NaN and goes nowhere; kinds may differ within a warp, the
    // sums are over a row's lanes, so all lanes take part in them
#pragma unroll
    for (int k = 0; k < 2; ++k) {
#pragma unroll
      for (int i = 0; i < 4; ++i) g[k][i] = sm100::mul2(g[k][i], w[i]);
      float2 t = sm100::mul2(g[k][0], v[k][0]);
#pragma unroll
      for (int i = 1; i < 4; ++i) t = sm100::fma2(g[k][i], v[k][i], t);
      gn[k] = -row_sum<S>(t.x + t.y) * inv_dim;
      mean[k] = 0.f;
      if (any_layer) {
        t = sm100::add2(sm100::add2(g[k][0], g[k][1]), sm100::add2(g[k][2], g[k][3]));
        mean[k] = -row_sum<S>(t.x + t.y) * inv_dim;
      }
      if (kind != P3D_NORM_LAYER) mean[k] = 0.f;
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (kind != P3D_NORM_NONE) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          g[k][i] = sm100::fma2(v[k][i], make_float2(gn[k], gn[k]), sm100::add2(g[k][i], make_float2(mean[k], mean[k])));
          g[k][i] = sm100::mul2(g[k][i], make_float2(dev[k], dev[k]));
        }
      }
      store8<T, kVec>(out, write && there[k] ? n : 0, g[k]);
      out += row.out_step;
    }
  }
  if (kParams && (kAll || p.partial)) {
    // the rows of a warp (each of the first or the second input), then the warps of the block, each in a fixed order
    __shared__ float2 joined[kWarps][S][4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float2 v = k < 2 ? sum_w[i] : sum_b[i];
        if (!row.on || row.second != (k % 2 == 1)) v = make_float2(0.f, 0.f);
#pragma unroll
        for (int o = S; o < 32; o <<= 1) {
          v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
          v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
        }
        if (lane < S) joined[threadIdx.x / 32][lane][i] = v;
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
  if (col < dim) {
    const float *from = partial + (int64_t)k * blocks * dim + col;
#pragma unroll 8
    for (int i = threadIdx.x / 32; i < blocks; i += 32) v += from[(int64_t)i * dim];
  }
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
  int lanes, passes, vec, sms;
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
  out->sms = info.sm_count;
  return P3D_OK;
}

// Blocks so that `per_sm` fill the device or each warp has one item, with the warps a multiple of a token's items.
int set_items(Plan *pl, int u, int per_sm) {
  RotateParams &p = pl->p;
  p.chunks = (uint32_t)(pl->passes + u - 1) / u;
  uint32_t unit = p.chunks, warps = kWarps;   // blocks that make whole tokens
  while (unit % 2 == 0 && warps > 1) unit /= 2, warps /= 2;
  const int64_t most = std::max<int64_t>((int64_t)pl->sms * per_sm / unit, 1);
  const int64_t need = ((int64_t)p.tokens * p.chunks + (int64_t)unit * kWarps - 1) / ((int64_t)unit * kWarps);
  return (int)(std::min(most, need) * unit);
}

// Two passes an item, where a warp's first item leaves work for the others.
int passes_of(const Plan &pl) { return pl.vec && pl.passes >= 2 && (int64_t)pl.p.tokens * pl.passes >= 8ll * pl.sms ? 2 : 1; }

template <typename T, int S>
int launch_s(Plan pl, bool backward, bool params, int blocks, int u, cudaStream_t s) {
  const RotateParams &p = pl.p;
  const bool bias = p.b0 || p.b1;
  auto fwd = [&](auto vec, auto passes, auto with_bias) {
    norm_rotate_kernel<T, S, decltype(passes)::value, decltype(vec)::value, decltype(with_bias)::value><<<blocks, kWarps * 32, 0, s>>>(p);
  };
  auto bwd = [&](auto vec, auto with_params, auto all) {
    norm_rotate_bwd_kernel<T, S, decltype(vec)::value, decltype(with_params)::value, decltype(all)::value><<<blocks, kWarps * 32, 0, s>>>(p);
  };
  using One = std::integral_constant<int, 1>;
  using Two = std::integral_constant<int, 2>;
  using Yes = std::true_type;
  using No = std::false_type;
  if (backward) {
    if (2 * p.end2 != p.dim) pl.vec ? bwd(Yes(), Yes(), No()) : bwd(No(), Yes(), No());
    else if (pl.vec) params ? bwd(Yes(), Yes(), Yes()) : bwd(Yes(), No(), Yes());
    else params ? bwd(No(), Yes(), Yes()) : bwd(No(), No(), Yes());
  } else if (!pl.vec) {
    fwd(No(), One(), Yes());
  } else if (u == 2) {
    bias ? fwd(Yes(), Two(), Yes()) : fwd(Yes(), Two(), No());
  } else {
    bias ? fwd(Yes(), One(), Yes()) : fwd(Yes(), One(), No());
  }
  P3D_LAUNCH_CHECK();
  return P3D_OK;
}

template <typename T>
int launch_t(const Plan &pl, bool backward, bool params, int blocks, int u, cudaStream_t s) {
  switch (pl.lanes) {
    case 1: return launch_s<T, 1>(pl, backward, params, blocks, u, s);
    case 2: return launch_s<T, 2>(pl, backward, params, blocks, u, s);
    case 4: return launch_s<T, 4>(pl, backward, params, blocks, u, s);
    case 8: return launch_s<T, 8>(pl, backward, params, blocks, u, s);
    case 16: return launch_s<T, 16>(pl, backward, params, blocks, u, s);
    default: return launch_s<T, 32>(pl, backward, params, blocks, u, s);
  }
}

int launch(const Plan &pl, int dtype, bool backward, bool params, int blocks, int u, cudaStream_t s) {
  switch (dtype) {
    case P3D_F16: return launch_t<__half>(pl, backward, params, blocks, u, s);
    case P3D_BF16: return launch_t<__nv_bfloat16>(pl, backward, params, blocks, u, s);
    default: return launch_t<float>(pl, backward, params, blocks, u, s);
  }
}

// Blocks an SM, by the kernels' registers.
constexpr int kPerSmForward = 5, kPerSmBackward = 4;

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
  const int u = passes_of(pl), blocks = set_items(&pl, u, kPerSmForward);
  return launch(pl, args->dtype, false, false, blocks, u, (cudaStream_t)stream);
}

size_t p3d_norm_rotate_bwd_workspace(const p3d_norm_rotate *args) {
  Plan pl;
  if (plan(args, &pl) != P3D_OK || args->tokens == 0) return 0;
  return sizeof(float) * 4 * (size_t)set_items(&pl, 1, kPerSmBackward) * pl.p.dim;
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
  const int blocks = set_items(&pl, 1, kPerSmBackward);
  pl.p.partial = params ? static_cast<float *>(workspace) : nullptr;
  if (params && (!workspace || workspace_bytes < sizeof(float) * 4 * (size_t)blocks * pl.p.dim))
    return fail(P3D_ERR_WORKSPACE, "p3d_norm_rotate_bwd: workspace of %zu bytes needed",
                sizeof(float) * 4 * (size_t)blocks * pl.p.dim);
  if (int st = launch(pl, args->dtype, true, params, blocks, 1, (cudaStream_t)stream)) return st;
  if (!params) return P3D_OK;
  JoinParams j = {{dweight[0], dweight[1], dbias[0], dbias[1]},
                  {args->param_dtype[0], args->param_dtype[1], args->param_dtype[0], args->param_dtype[1]}};
  rotate_join_kernel<<<dim3((pl.p.dim + 31) / 32, 4), 1024, 0, (cudaStream_t)stream>>>(pl.p.partial, blocks, pl.p.dim, j);
  P3D_LAUNCH_CHECK();
  return P3D_OK;
}

}  // extern "C"
