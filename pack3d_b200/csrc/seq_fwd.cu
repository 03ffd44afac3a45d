// Attention over packed sequences, forward, on the tensor cores:  S = Q K^T,  P = 2^(S c - m),  O = P V,  out = O / sum P.
//
// A CTA has two tiles of 128 query rows that read the same keys: one place in a sequence for two heads of a group (where groups are
// even: equal work and masks), else two neighbouring places of one head. Keys and values come in tiles of 128 through a
// ring; S and O of both tiles are in tensor memory, P is written over its S. Two groups of four softmax warps (a row a thread)
// take a tile each, two warps issue the products, one the copies.
//
// What bounds it: at dim 128 a tile of 128 x 128 costs the tensor pipe 1024 cycles and, at 16 exponentials a clock, the
// special-function units as many, so a quarter of the exponentials go to the FMA pipe as polynomials; at dim 64 and below
// the exponentials are the bound. What counts is that neither waits for the other: the softmax goes by 64 keys, and each tile has two
// buffers of S (64 columns; P of 16 bits goes over its own S), so that S of the next 64 keys is made while the softmax works on
// these (one buffer of 128 columns, S waiting for the product that reads P: 350 us for the figure below). S of 64 keys costs a
// third more of the pipe than half of 128, as its operands come from shared memory.
// O is rescaled only where a row's maximum has grown by more than 2^8 (weights up to 2^8 cost no precision), after the product before
// has completed.
//
// Masks: key j counts for row i where j < seen(i); tiles of keys that some row does not see whole ("border" tiles, the last ones) are masked
// by columns. A masked weight is 0, but 0 times an infinity or NaN of a value that the row does not see is NaN. So in border tiles the copying
// warp, which has nothing else to do by then, sets values that are not finite to 0 before the product, and the epilogue adds them back
// for the rows that see them.
#include <math.h>

#include <algorithm>

#include "seq_tc.cuh"

namespace p3d {
namespace seq {
namespace {

__device__ unsigned g_seq_fwd_errors = 0;

constexpr int kMmaWarp = 8, kCopyWarp = 10, kThreads = 352;   // a warp of products for each tile
constexpr int kKeys = 64;                    // of one softmax step
constexpr uint32_t kColS = 0, kColO = 256;   // tensor memory: S of tile t at 128 t and 128 t + 64, O at 256 + 128 t
constexpr float kSlack = 8.f;                // the maximum may lag by 2^8
constexpr int kPoly = 2;                     // exponentials of eight that are polynomials

template <int DP>
struct Layout {
  static constexpr uint32_t kTileBytes = DP / 64 * kBox;
  static constexpr int kStages = DP == 128 ? 5 : 8;
  static constexpr size_t kBytes = 1024 + (2 + kStages) * (size_t)kTileBytes;
};

// Every wait on a barrier that completes more than once is by someone who has seen the completion before, and whose own next step the
// one after needs. Border tiles, at most kBorders of them (the rows of a CTA see the same keys but for 255), are cleared ahead
// of that order: each has a barrier of its own.
constexpr int kBorders = 3;
enum { kQFull, kSFull, kPFull = kSFull + 4, kODone = kPFull + 2, kClean = kODone + 2, kDrain = kClean + kBorders, kFull = kDrain + 2 };
template <int DP> constexpr int bars() { return kFull + 2 * Layout<DP>::kStages; }

struct Params {
  p3d_sequence a;
  void *out;
  float *lse;
  int units;       // of heads: pairs, or single ones
  int two_heads;   // a CTA's tiles are two heads
  int steps;       // of 16 columns
  uint32_t idesc_o;
  float sc;        // scale * log2(e)
};

// What a CTA does: rows i0 (+ 128 for the second tile where the tiles are of one head) of sequence `r`.
struct Work {
  Range r;
  int row[2], head[2], kv;
  int units[2];    // 64 keys that each tile sees any of
  int border;      // the first tile of keys that some row does not see whole
};
__device__ __forceinline__ Work work_of(const Params &p) {
  const int slot = (int)(gridDim.x / p.units - 1 - blockIdx.x / p.units), unit = blockIdx.x % p.units;   // the longest first
  const int per_slot = p.two_heads ? kTile : 2 * kTile;
  const Slot s = find_slot(p.a.q_offsets, p.a.sequences, (int)p.a.q_rows, per_slot, slot);
  Work w;
  w.r = slot_range(p.a, s.sequence);
  const int group = p.a.heads / p.a.kv_heads;
  w.border = 1 << 30;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    w.head[t] = p.two_heads ? 2 * unit + t : unit;
    w.row[t] = s.group * per_slot + (p.two_heads ? 0 : t * kTile);
    w.units[t] = 0;
    if (s.group >= 0 && w.row[t] < w.r.nq) {
      w.units[t] = (seen_by(w.r, min(w.row[t] + kTile, w.r.nq) - 1, p.a.causal) + kKeys - 1) / kKeys;
      if (w.units[t]) w.border = min(w.border, seen_by(w.r, w.row[t], p.a.causal) / kTile);
    }
  }
  w.kv = w.head[0] / group;
  return w;
}

// P = 2^(s sc + shift) of a row's 64 scores, rounded to T and written over them; returns the row's sum.  kPoly of every eight pairs are
// polynomials (scores are not NaN there: the row's maximum, and with it shift, would be).
template <typename T, int kPoly>
__device__ __forceinline__ float weights(const float (&s)[kKeys], float sc, float shift, uint32_t t_s) {
  const float2 sc2 = make_float2(sc, sc), shift2 = make_float2(shift, shift);
  float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
  for (int i = 0; i < kKeys; i += 32) {
    uint32_t pk[16];
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      const float2 x = fma2(make_float2(s[i + 2 * k], s[i + 2 * k + 1]), sc2, shift2);
      float2 e;
      if ((k * kPoly & 7) + kPoly > 7) {
        e = exp2_poly2(x);
      } else {
        e.x = ex2_approx(x.x);
        e.y = ex2_approx(x.y);
      }
      sum[k & 1] = add2(sum[k & 1], e);
      pk[k] = pack<T>(e.x, e.y);
    }
    tmem_st16(t_s + i / 2, pk);
  }
  const float2 both = add2(sum[0], sum[1]);
  return both.x + both.y;
}

template <typename T, int DP>
__global__ void __launch_bounds__(kThreads, 1)
    sequence_fwd_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                        const __grid_constant__ CUtensorMap tv, const __grid_constant__ Params p) {
  using L = Layout<DP>;
  constexpr int NS = L::kStages;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bar_mem[bars<DP>()];
  __shared__ uint32_t tmem_holder;
  __shared__ int not_finite;   // border tiles hold values that are not
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Work w = work_of(p);
  const int units = max(w.units[0], w.units[1]), chunks = (units + 1) / 2;   // chunks: tiles of keys
  if (chunks == 0) {
    // rows that see no key, or none at all
    if (threadIdx.x < 256) {
      const int t = threadIdx.x / 128, row = w.row[t] + threadIdx.x % 128;
      if (w.row[t] >= 0 && row < w.r.nq) {
        const int64_t at = (int64_t)(w.r.q0 + row) * p.a.heads + w.head[t];
        uint4 *out = reinterpret_cast<uint4 *>(static_cast<T *>(p.out) + at * p.a.dim);
        for (int i = 0; i < p.a.dim / 8; ++i) out[i] = make_uint4(0, 0, 0, 0);
        if (p.lse) p.lse[(int64_t)w.head[t] * p.a.q_rows + w.r.q0 + row] = -INFINITY;
      }
    }
    return;
  }
  const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
  uint8_t *const smem = smem_raw + (base - raw);
  const uint32_t ring = base + 2 * L::kTileBytes;
  auto bar = [&](int i) { return smem_u32(&bar_mem[i]); };
  auto full = [&](int s) { return bar(kFull + s); };
  auto empty = [&](int s) { return bar(kFull + NS + s); };
  if (threadIdx.x == 0) {
    not_finite = 0;
    for (int i = 0; i < bars<DP>(); ++i)
      mbar_init(bar(i), i == kPFull || i == kPFull + 1 ? 4 : i >= kFull + NS ? 2 : 1);   // a stage is empty when both tiles are done with it
    fence_mbar_init();
  }
  if (warp == kMmaWarp) {
    tmem_alloc(smem_u32(&tmem_holder), 512);
    tmem_relinquish();
  }
  if (warp == kCopyWarp && lane == 0) {
    prefetch_tmap(&tq);
    prefetch_tmap(&tk);
    prefetch_tmap(&tv);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_holder;

  if (warp == kCopyWarp) {
    // ------------------------------------------------------------------ copies; items K0, V0, K1, V1, ..
    bool ok = true;
    int issued = 0;
    if (lane == 0) {
      mbar_expect_tx(bar(kQFull), 2 * L::kTileBytes);
#pragma unroll
      for (int t = 0; t < 2; ++t)
        for (int c = 0; c < DP / 64; ++c)
          tma_load_3d(base + t * L::kTileBytes + c * kBox, &tq, bar(kQFull), 64 * c, w.head[t], w.r.q0 + w.row[t]);
      for (int i = 0; i < 2 * chunks; ++i) {
        const int s = i % NS;
        if (i >= NS && !mbar_wait(empty(s), (i / NS - 1) & 1, &g_seq_fwd_errors, kWaitNs, kErrProducer)) {
          ok = false;
          break;
        }
        mbar_expect_tx(full(s), L::kTileBytes);
        for (int c = 0; c < DP / 64; ++c)
          tma_load_3d(ring + s * L::kTileBytes + c * kBox, i % 2 ? &tv : &tk, full(s), 64 * c, w.kv, w.r.k0 + i / 2 * kTile);
        issued = i + 1;
      }
    }
    ok = __all_sync(0xffffffffu, ok);
    // values of the border tiles that are not finite
    for (int c = min(w.border, chunks); ok && c < chunks; ++c) {
      const int i = 2 * c + 1, s = i % NS;
      ok = __all_sync(0xffffffffu, mbar_wait(full(s), (i / NS) & 1, &g_seq_fwd_errors, kWaitNs, kErrProducer));
      if (!ok) break;
      if (clear_not_finite<T>(smem + (2 + s) * L::kTileBytes, L::kTileBytes)) {
        fence_proxy_async_smem();
        if (lane == 0) not_finite = 1;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(kClean + c - w.border));
    }
    // no copy in flight into memory that is about to be given up
    if (lane == 0) {
      mbar_wait(bar(kQFull), 0, &g_seq_fwd_errors, kWaitNs, kErrTeardown);
      for (int i = max(0, issued - NS); i < issued; ++i)
        mbar_wait(full(i % NS), (i / NS) & 1, &g_seq_fwd_errors, kWaitNs, kErrTeardown);
    }
  } else if (warp >= kMmaWarp) {
    // ------------------------------------------------------------------ products, of one tile
    // The whole warp runs this, with the same operands in every lane; one elected lane issues (30 cycles a product instead of 75). The
    // pipe takes four products ahead and a wait costs 70 cycles even where there is nothing to wait for: with one warp for both
    // tiles the pipe ran dry at each of them.
    const int t = warp - kMmaWarp, mine = t ? w.units[1] : w.units[0];
    const uint32_t idesc_s = idesc_f16(128, kKeys, std::is_same<T, __nv_bfloat16>::value, false);
    const uint64_t desc_q = desc_rows(base + t * L::kTileBytes), desc_k = desc_rows(ring), desc_v = desc_cols(ring);
    const uint32_t t_s = tmem + kColS + 128 * t, t_o = tmem + kColO + 128 * t;
    int n_s = 0, n_o = 0, landed = 0;
    auto wait = [&](uint32_t b, uint32_t parity) { return wait_warp(b, parity, &g_seq_fwd_errors, kErrMma); };
    // item i is there (and, for values of a border tile, cleared); items are waited for in order, once
    auto wait_item = [&](int i) {
      while (landed <= i) {
        const int c = landed / 2;
        if (!wait(full(landed % NS), (landed / NS) & 1)) return false;
        if (landed % 2 && c >= w.border && !wait(bar(kClean + c - w.border), 0)) return false;
        ++landed;
      }
      return true;
    };
    auto issue_s = [&](int u) {
      const uint64_t k = desc_k + (((uint32_t)(u / 2 * 2 % NS) * L::kTileBytes + (u & 1) * kKeys * 128) >> 4);
#pragma unroll
      for (int j = 0; j < DP / 16; ++j)
        if (j < p.steps) mma_ss_warp(t_s + 64 * (u & 1), desc_q + step_rows(j), k + step_rows(j), idesc_s, j > 0);
      mma_commit_warp(bar(kSFull + 2 * t + (u & 1)));
      ++n_s;
    };
    auto issue_o = [&](int u) {
      const uint64_t v = desc_v + ((uint32_t)((u / 2 * 2 + 1) % NS) * L::kTileBytes >> 4) + step_cols((u & 1) * (kKeys / 16));
#pragma unroll
      for (int j = 0; j < kKeys / 16; ++j)
        mma_ts_warp(t_o, t_s + 64 * (u & 1) + 8 * j, v + step_cols(j), p.idesc_o, u > 0 || j > 0);
      mma_commit_warp(bar(kODone + t));
      ++n_o;
    };
    bool ok = wait(bar(kQFull), 0) && wait_item(0);
    if (ok && mine) issue_s(0);
    for (int u = 0; ok && u < units; ++u) {
      if (u > 0) {
        // O(u - 1) is there, and with it S(u - 1): their keys and values may go. By a plain arrival: a commit after another one's
        // waits until the pipe has run dry. A tile that is done, or has no rows, arrives for what has landed.
        ok = u - 1 < mine ? wait(bar(kODone + t), (u - 1) & 1) : wait_item((u - 1) / 2 * 2 + 1);
        if (!ok) break;
        if ((u & 1) == 0 && lane == 0) {
          mbar_arrive(empty((u - 2) % NS));
          mbar_arrive(empty((u - 1) % NS));
        }
      }
      if (u + 1 < mine) {   // into the buffer that held P(u - 1)
        ok = wait_item((u + 1) / 2 * 2);
        if (!ok) break;
        issue_s(u + 1);
      }
      if (u < mine) {
        ok = wait_item(u / 2 * 2 + 1) && wait(bar(kPFull + t), u & 1);
        if (ok) issue_o(u);
      }
    }
    // every product completed and every commit arrived before tensor memory and barriers are given up
    mma_commit_warp(bar(kDrain + t));
    auto drained = [&](uint32_t b, int times) {
      if (times > 0) mbar_wait(b, (times - 1) & 1, &g_seq_fwd_errors, kWaitNs, kErrTeardown);
    };
    drained(bar(kDrain + t), 1);
    drained(bar(kSFull + 2 * t), (n_s + 1) / 2);
    drained(bar(kSFull + 2 * t + 1), n_s / 2);
    drained(bar(kODone + t), n_o);
  } else {
    // ------------------------------------------------------------------ softmax, a row a thread
    const int t = warp / 4, mine = t ? w.units[1] : w.units[0], head = t ? w.head[1] : w.head[0];
    const int row = (t ? w.row[1] : w.row[0]) + (warp % 4) * 32 + lane;
    const int seen = row < w.r.nq ? seen_by(w.r, row, p.a.causal) : 0;
    const uint32_t lanes = (uint32_t)((warp % 4) * 32) << 16;
    const uint32_t t_s = tmem + kColS + 128 * t + lanes, t_o = tmem + kColO + 128 * t + lanes;
    const float sc = p.sc;
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    for (int u = 0; u < mine; ++u) {
      const uint32_t t_u = t_s + 64 * (u & 1);
      ok = wait_warp(bar(kSFull + 2 * t + (u & 1)), (u >> 1) & 1, &g_seq_fwd_errors, kErrSoftmax);
      if (!ok) break;
      float s[kKeys];
#pragma unroll
      for (int i = 0; i < kKeys; i += 32) tmem_ld32(t_u + i, reinterpret_cast<uint32_t *>(s) + i);
      tmem_wait_ld();
      const int limit = seen - u * kKeys;
      const bool masked = __any_sync(0xffffffffu, limit < kKeys);
      if (masked) {
#pragma unroll
        for (int i = 0; i < kKeys; ++i) s[i] = i < limit ? s[i] : -INFINITY;
      }
      float top[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) top[i] = max_nan(s[2 * i], s[2 * i + 1]);
#pragma unroll
      for (int i = 16; i < kKeys; i += 16)
#pragma unroll
        for (int k = 0; k < 8; ++k) top[k] = max3_nan(top[k], s[i + 2 * k], s[i + 2 * k + 1]);
#pragma unroll
      for (int k = 0; k < 4; ++k) top[k] = max_nan(top[k], top[k + 4]);
      const float now = max3_nan(m, max_nan(top[0], top[1]), max_nan(top[2], top[3]));
      // a row that has seen nothing yet has an empty O: its first maximum rescales nothing
      const bool moves = !((now - m) * sc <= kSlack) && !(now == -INFINITY), rescale = __any_sync(0xffffffffu, moves) && u > 0;
      const float down = moves ? (m == -INFINITY ? 0.f : ex2_approx((m - now) * sc)) : 1.f;
      if (moves) m = now;
      l *= down;
      const float shift = m == -INFINITY ? 0.f : -m * sc;
      // a border's masked scores have weight 0, which the polynomial does not give
      l += masked ? weights<T, 0>(s, sc, shift, t_u) : weights<T, kPoly>(s, sc, shift, t_u);
      // O rests once the product before has completed (waited for at every step, so that the parity is exact)
      if (u > 0) {
        ok = wait_warp(bar(kODone + t), (u - 1) & 1, &g_seq_fwd_errors, kErrSoftmax);
        if (!ok) break;
      }
      if (rescale) {
#pragma unroll
        for (int i = 0; i < DP; i += 32) {
          if (i < p.a.dim) {
            uint32_t o[32];
            tmem_ld32(t_o + i, o);
            tmem_wait_ld();
#pragma unroll
            for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * down);
            tmem_st16(t_o + i, o);
            tmem_st16(t_o + i + 16, o + 16);
          }
        }
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(kPFull + t));
    }
    if (ok && mine) ok = wait_warp(bar(kODone + t), (mine - 1) & 1, &g_seq_fwd_errors, kErrSoftmax);
    if (ok && (mine + 1) / 2 > w.border)   // for what the copying warp says of the values
      ok = wait_warp(bar(kClean + (mine + 1) / 2 - 1 - w.border), 0, &g_seq_fwd_errors, kErrSoftmax);
    if (ok) {
      const float inv = seen > 0 ? 1.f / l : 0.f;
      const int64_t at = (int64_t)(w.r.q0 + row) * p.a.heads + head;
      T *out = static_cast<T *>(p.out) + at * p.a.dim;
      const bool add_back = not_finite != 0;
#pragma unroll
      for (int i = 0; i < DP; i += 32) {
        if (i >= p.a.dim) continue;
        uint32_t o[32];
        if (mine) {
          tmem_ld32(t_o + i, o);
          tmem_wait_ld();
        }
#pragma unroll
        for (int k = 0; k < 32; ++k) o[k] = seen > 0 ? __float_as_uint(__uint_as_float(o[k]) * inv) : 0u;
        if (add_back && seen > 0) {
          for (int j = w.border * kTile; j < seen; ++j) {
            const T *v = static_cast<const T *>(p.a.v) + (int64_t)(w.r.k0 + j) * p.a.v_stride[0] + w.kv * p.a.v_stride[1];
#pragma unroll
            for (int k = 0; k < 32; ++k) {
              const float x = i + k < p.a.dim ? to_f32<T>(v[i + k]) : 0.f;
              if (!isfinite(x)) o[k] = __float_as_uint(__uint_as_float(o[k]) + x);
            }
          }
        }
        if (row < w.r.nq) {
#pragma unroll
          for (int k = 0; k < 32; k += 8)
            if (i + k < p.a.dim)
              *reinterpret_cast<uint4 *>(out + i + k) =
                  make_uint4(pack<T>(__uint_as_float(o[k]), __uint_as_float(o[k + 1])),
                             pack<T>(__uint_as_float(o[k + 2]), __uint_as_float(o[k + 3])),
                             pack<T>(__uint_as_float(o[k + 4]), __uint_as_float(o[k + 5])),
                             pack<T>(__uint_as_float(o[k + 6]), __uint_as_float(o[k + 7])));
        }
      }
      if (p.lse && row < w.r.nq)
        p.lse[(int64_t)head * p.a.q_rows + w.r.q0 + row] = seen > 0 ? (m * sc + log2f(l)) * 0.6931471805599453f : -INFINITY;
    }
    tmem_wait_st();
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

__global__ void fill_kernel(float *p, int64_t n, float v) {
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) p[i] = v;
}

template <typename T, int DP>
int launch_t(const Params &p, int64_t grid, const CUtensorMap &tq, const CUtensorMap &tk, const CUtensorMap &tv, cudaStream_t s) {
  static size_t seen[kMaxDevices] = {};
  if (int st = smem_optin(sequence_fwd_kernel<T, DP>, Layout<DP>::kBytes, seen)) return st;
  sequence_fwd_kernel<T, DP><<<(unsigned)grid, kThreads, Layout<DP>::kBytes, s>>>(tq, tk, tv, p);
  P3D_LAUNCH_CHECK();
  return P3D_OK;
}

}  // namespace

int launch_fwd(const p3d_sequence &a, void *out, float *lse, cudaStream_t s) {
  if (a.k_rows == 0) {
    P3D_CUDA_TRY(cudaMemsetAsync(out, 0, (size_t)a.q_rows * a.heads * a.dim * 2, s));
    if (lse) fill_kernel<<<256, 256, 0, s>>>(lse, a.q_rows * a.heads, -INFINITY);
    P3D_LAUNCH_CHECK();
    return P3D_OK;
  }
  Params p = {};
  p.a = a;
  p.out = out;
  p.lse = lse;
  p.two_heads = a.heads / a.kv_heads % 2 == 0;
  p.units = p.two_heads ? a.heads / 2 : a.heads;
  p.steps = (a.dim + 15) / 16;
  p.idesc_o = idesc_f16(128, p.steps * 16, a.dtype == P3D_BF16, true);
  p.sc = a.scale * 1.4426950408889634f;
  const int64_t grid = slots_of(a.q_rows, a.sequences, p.two_heads ? kTile : 2 * kTile) * p.units;
  if (grid > 0x7fffffff) return fail(P3D_ERR_UNSUPPORTED, "p3d_sequence_fwd: too many tiles");
  CUtensorMap tq, tk, tv;
  if (int st = encode_heads(&tq, a.dtype, a.q, a.dim, a.heads, a.q_rows, a.q_stride)) return st;
  if (int st = encode_heads(&tk, a.dtype, a.k, a.dim, a.kv_heads, a.k_rows, a.k_stride)) return st;
  if (int st = encode_heads(&tv, a.dtype, a.v, a.dim, a.kv_heads, a.k_rows, a.v_stride)) return st;
  if (a.dtype == P3D_BF16)
    return padded(a.dim) == 64 ? launch_t<__nv_bfloat16, 64>(p, grid, tq, tk, tv, s) : launch_t<__nv_bfloat16, 128>(p, grid, tq, tk, tv, s);
  return padded(a.dim) == 64 ? launch_t<__half, 64>(p, grid, tq, tk, tv, s) : launch_t<__half, 128>(p, grid, tq, tk, tv, s);
}

int take_errors_fwd(unsigned *flags) {
  unsigned v = 0, zero = 0;
  P3D_CUDA_TRY(cudaMemcpyFromSymbol(&v, g_seq_fwd_errors, sizeof(v)));
  P3D_CUDA_TRY(cudaMemcpyToSymbol(g_seq_fwd_errors, &zero, sizeof(zero)));
  *flags |= v;
  return P3D_OK;
}

}  // namespace seq
}  // namespace p3d
