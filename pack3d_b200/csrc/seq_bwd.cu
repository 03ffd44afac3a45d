// Attention over packed sequences, backward, on the tensor cores, from lse and delta_i = dout_i . out_i:
//
//     P = 2^(S c - lse),  dS = scale P (dO V^T - delta),  dQ = dS K,  dK = dS^T Q,  dV = P^T dO
//
// In f16 neither P nor dS fits as it is: both get small as keys get many, while the sums over them do not (4,096 keys and a dO of 1e-4: dQ and
// dK off by a tenth), and a large dO overflows dS. So P is held 2^10 times as large for dV, and dS by the power of two that brings the
// largest that it can be, scale |dO_i| max |V_j| + |scale delta_i|, to 2^11 .. 2^12: of a query in dQ, of the whole tile's queries and keys in
// dK, of its own sequence in any case. Sums are brought back in fp32. The norms come from the kernel that makes delta.
//
// Where a query sees a single key, P is 1 and dS is 0; dP - delta, two sums of the same products, would leave the rounding of their orders:
// scale and delta are 0 there (in dK: where a sequence has one key. Among more keys, whose gradients are sums over many queries, that
// rounding is as small as any).
//
// Two kernels, so that each gradient is a sum in one fixed order without atomics: dQ by tiles of queries, dK and dV by tiles of keys.
// They make S and dP both, seven products of which five are the mathematics' own (a tile of 128 x 128 is 512 cycles a product).
//
// dQ: a CTA has 128 queries of a head; S in two buffers, dP and dQ fill the tensor memory (512 columns). dS (16-bit) goes over S. The
//   pipe makes S and dP of the next keys while the softmax warps, in two groups of 64 columns, work on these.
// dK, dV: a CTA has 128 keys of a KV head and goes over the queries that see them of all heads of its group: S^T = K Q^T and
//   dP^T = V dO^T (keys on the lanes), P^T over S^T, dS^T over dP^T, both read from tensor memory by dV += P^T dO and dK += dS^T Q.
//   Where there are few key tiles, a group's heads are shared among several CTAs, whose sums in fp32 are added by a last kernel.
//
// Measured, bf16, 16 heads of 128 over 4, six causal documents, 16,384 tokens: dQ 345 us, dK and dV 447, the sums delta 28 (they read
// 134 MB); looking for what is not finite at the mask's border is 9 us of dK and dV and 2 of dQ, f16's norms and powers of two 3.6 of 69
// for 41 pieces of 5,003 tokens. The tensor pipe is active half of the time; a tile costs 2,900 (three products, 1,536) and 4,500 cycles (four, 2,048). In
// between stand the waits of eight softmax warps for products, each of which takes 900 cycles from its issue to where it is seen.
#include <math.h>

#include <algorithm>

#include "seq_tc.cuh"

namespace p3d {
namespace seq {
namespace {

__device__ unsigned g_seq_bwd_errors = 0;

constexpr int kMmaWarp = 8, kCopyWarp = 10, kThreads = 352, kSoftmaxWarps = 8;   // two warps of products

struct Params {
  p3d_sequence a;
  const float2 *stats;     // [heads][q_rows]: -lse * log2(e), -scale * delta
  const float *dout_norm;  // [heads][q_rows], f16 only
  const float *v_norm;     // [kv_heads][k_rows], f16 only
  const void *dout;        // contiguous
  void *dq, *dk, *dv;
  float *part;             // [2][parts][k_rows * kv_heads * dim] where parts > 1
  int parts;
  int falling;             // the order of key tiles
  int steps;               // of 16 columns
  uint32_t idesc_out;
  float sc;                // scale * log2(e)
};

// 2^(s sc + minus) of 64 scores; minus(k): of columns 2 k, 2 k + 1. All on the special-function units: a pair is 16 cycles there, and
// as many on the FMA pipe as polynomials, which has the products' other arithmetic to do.
template <typename F>
__device__ __forceinline__ void weights(float (&s)[64], float2 sc, F minus) {
#pragma unroll
  for (int k = 0; k < 32; ++k) {
    const float2 x = fma2(make_float2(s[2 * k], s[2 * k + 1]), sc, minus(k));
    s[2 * k] = ex2_approx(x.x), s[2 * k + 1] = ex2_approx(x.y);
  }
}

template <int N>
__device__ __forceinline__ void load_columns(uint32_t t, float *v) {
#pragma unroll
  for (int i = 0; i < N; i += 32) tmem_ld32(t + i, reinterpret_cast<uint32_t *>(v) + i);
}

template <typename T> constexpr bool kScaled = std::is_same<T, __half>::value;   // P and dS are
constexpr int kWeightUp = 10;
__device__ __forceinline__ float two_to(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }
// The power of two that brings `most` (not negative) to 2^11 .. 2^12, as far as 2^+-100.
__device__ __forceinline__ int exponent_for(float most) {
  return min(max(138 - (int)(__float_as_uint(most) >> 23 & 255u), -100), 100);
}
__device__ __forceinline__ float finite_or_0(float v) { return not_finite(v) ? 0.f : v; }
__device__ __forceinline__ float warp_most(float v) {   // of values that are not negative
  return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(v)));
}

// 64 columns of an accumulator, times `factor` (f16), in 16 bits (zeros unless `write`).
template <typename T>
__device__ __forceinline__ void pack_columns(uint32_t t, bool write, float factor, uint32_t (&packed)[32]) {
#pragma unroll
  for (int h = 0; h < 64; h += 32) {
    uint32_t o[32];
    tmem_ld32(t + h, o);
    tmem_wait_ld();
#pragma unroll
    for (int k = 0; k < 32; k += 2) {
      float2 v = make_float2(__uint_as_float(o[k]), __uint_as_float(o[k + 1]));
      if constexpr (kScaled<T>) v = mul2(v, make_float2(factor, factor));
      packed[(h + k) / 2] = pack<T>(write ? v.x : 0.f, write ? v.y : 0.f);
    }
  }
}

// The same for dV from gradient rows of the queries [first, i) of `heads` heads: a warp's keys see the fewer of them the further down they
// are. `at` (-1 for none) and `from` (it sees the rows from there on) are of a lane's key.
template <typename T, typename Out>
__device__ __noinline__ void add_gradients_not_finite(const T *dout, int64_t stride, int heads, int dim, int first, int i, int64_t at, int from,
                                                       Out *out) {
  const int c = (threadIdx.x & 31) * 4;
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
  for (int key = 31; key >= 0; --key) {
    const int64_t to = __shfl_sync(0xffffffffu, at, key);
    const int down = max(first, __shfl_sync(0xffffffffu, from, key));
    if (to < 0) continue;
    while (i > down) {
      --i;
      for (int h = 0; h < heads; ++h) {
        float v[4];
        load4(dout + i * stride + h * dim, dim, v);
#pragma unroll
        for (int k = 0; k < 4; ++k) sum[k] += not_finite(v[k]) ? v[k] : 0.f;
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (sum[k] != 0.f) out[to + c + k] = from_f32<Out>(to_f32<Out>(out[to + c + k]) + sum[k]);
  }
}

// ------------------------------------------------------------------------------- dQ
template <int DP>
struct LayoutQ {
  static constexpr uint32_t kTileBytes = DP / 64 * kBox;
  static constexpr int kK = 3, kV = 2;   // stages
  static constexpr size_t kBytes = 1024 + (2 + kK + kV) * (size_t)kTileBytes;   // O's way out is over the queries
};
// Parity waits: each waiter of a barrier that completes many times has seen every completion before, and the one after its own needs a
// step of the waiter: so dS and dQ have a barrier for each of the two buffers (with one, those of the next keys could be there while the wait for
// these begins, as S and dP of those are made ahead of it).
enum { kQFull, kSFull, kDPFull = kSFull + 2, kDPFree, kDSFull, kDQDone = kDSFull + 2, kDone = kDQDone + 2, kLanded, kDrainQ, kKFull = kDrainQ + 2,
       kKEmpty = kKFull + 3, kVFull = kKEmpty + 3, kVEmpty = kVFull + 2, kBarsQ = kVEmpty + 2 };

template <typename T, int DP>
__global__ void __launch_bounds__(kThreads, 1)
    sequence_dq_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tdo,
                       const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                       const __grid_constant__ Params p) {
  using L = LayoutQ<DP>;
  constexpr uint32_t TB = L::kTileBytes;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bar_mem[kBarsQ];
  __shared__ uint32_t tmem_holder;
  __shared__ int odd_keys;   // keys have been cleared
  __shared__ float most_v[kSoftmaxWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int slot = blockIdx.x / p.a.heads, head = blockIdx.x % p.a.heads;
  const int kv = head / (p.a.heads / p.a.kv_heads);
  // the longest of each sequence first (over all sequences costs each of these short CTAs a microsecond, 348 us for 334)
  const Place at = place_of<false>(p.a, 7, (int)(gridDim.x / p.a.heads) - 1 - slot);
  const Range r = at.r;
  const int row0 = at.group * kTile;
  if (at.group < 0 || row0 >= r.nq) return;
  const int chunks = (seen_by(r, min(row0 + kTile, r.nq) - 1, p.a.causal) + kTile - 1) / kTile;
  if (chunks == 0) {
    const int row = row0 + threadIdx.x;
    if (threadIdx.x < kTile && row < r.nq) {
      uint4 *to = reinterpret_cast<uint4 *>(static_cast<T *>(p.dq) + ((int64_t)(r.q0 + row) * p.a.heads + head) * p.a.dim);
      for (int i = 0; i < p.a.dim / 8; ++i) to[i] = make_uint4(0, 0, 0, 0);
    }
    return;
  }
  const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
  const uint32_t k_ring = base + 2 * TB, v_ring = k_ring + L::kK * TB;
  auto bar = [&](int i) { return smem_u32(&bar_mem[i]); };
  if (threadIdx.x == 0) {
    for (int i = 0; i < kBarsQ; ++i) mbar_init(bar(i), i >= kDPFree && i < kDQDone ? kSoftmaxWarps : 1);
    fence_mbar_init();
    odd_keys = 0;
  }
  if (warp == kMmaWarp) {
    tmem_alloc(smem_u32(&tmem_holder), 512);
    tmem_relinquish();
  }
  if (warp == kCopyWarp && lane == 0) {
    prefetch_tmap(&tq);
    prefetch_tmap(&tdo);
    prefetch_tmap(&tk);
    prefetch_tmap(&tv);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_holder, t_dp = tmem + 256, t_dq = tmem + 384;   // S at 0 and 128

  if (warp == kCopyWarp) {
    int n_k = 0, n_v = 0;
    if (lane == 0) {
      auto tile = [&](uint32_t dst, const CUtensorMap *map, uint32_t full, int h, int row) {
        mbar_expect_tx(full, TB);
        for (int c = 0; c < DP / 64; ++c) tma_load_3d(dst + c * kBox, map, full, 64 * c, h, row);
      };
      mbar_expect_tx(bar(kQFull), 2 * TB);
      for (int c = 0; c < DP / 64; ++c) {
        tma_load_3d(base + c * kBox, &tq, bar(kQFull), 64 * c, head, r.q0 + row0);
        tma_load_3d(base + TB + c * kBox, &tdo, bar(kQFull), 64 * c, head, r.q0 + row0);
      }
      for (int c = 0; c < chunks; ++c) {
        int s = c % L::kK;
        if (c >= L::kK && !mbar_wait(bar(kKEmpty + s), (c / L::kK - 1) & 1, &g_seq_bwd_errors, kWaitNs, kErrProducer)) break;
        // the last keys, where their tile goes past the sequence's end, land on a barrier of their own
        tile(k_ring + s * TB, &tk, bar((c + 1) * kTile > r.nk ? kLanded : kKFull + s), kv, r.k0 + c * kTile);
        n_k = c + 1;
        s = c % L::kV;
        if (c >= L::kV && !mbar_wait(bar(kVEmpty + s), (c / L::kV - 1) & 1, &g_seq_bwd_errors, kWaitNs, kErrProducer)) break;
        tile(v_ring + s * TB, &tv, bar(kVFull + s), kv, r.k0 + c * kTile);
        n_v = c + 1;
      }
    }
    n_k = __shfl_sync(0xffffffffu, n_k, 0);
    if (n_k == chunks && chunks * kTile > r.nk) {
      const int s = (chunks - 1) % L::kK;
      if (wait_warp(bar(kLanded), 0, &g_seq_bwd_errors, kErrProducer)) {
        clear_rows<DP / 64>(smem_raw + (k_ring - raw) + s * TB, r.nk - (chunks - 1) * kTile);
        if (lane == 0) mbar_arrive(bar(kKFull + s));
      }
    }
    if (lane == 0) {
      mbar_wait(bar(kQFull), 0, &g_seq_bwd_errors, kWaitNs, kErrTeardown);
      for (int i = max(0, n_k - L::kK); i < n_k; ++i)
        mbar_wait(bar(kKFull + i % L::kK), (i / L::kK) & 1, &g_seq_bwd_errors, kWaitNs, kErrTeardown);
      for (int i = max(0, n_v - L::kV); i < n_v; ++i)
        mbar_wait(bar(kVFull + i % L::kV), (i / L::kV) & 1, &g_seq_bwd_errors, kWaitNs, kErrTeardown);
    }
  } else if (warp >= kMmaWarp) {
    // Products, warp-wide as in the forward kernel, by two warps that need not wait for one another's: S of the keys ahead, dP and dQ.
    const uint32_t idesc_s = idesc_f16(128, 128, std::is_same<T, __nv_bfloat16>::value, false);
    auto wait = [&](int b, uint32_t parity) { return wait_warp(bar(b), parity, &g_seq_bwd_errors, kErrMma); };
    auto drained = [&](int b, int times) {
      if (times > 0) mbar_wait(bar(b), (times - 1) & 1, &g_seq_bwd_errors, kWaitNs, kErrTeardown);
    };
    bool ok = wait(kQFull, 0);
    if (warp == kMmaWarp) {
      const uint64_t d_q = desc_rows(base), d_k = desc_rows(k_ring);
      int n = 0;
      for (int c = 0; ok && c < chunks; ++c) {
        if (c >= 2) {
          // The buffer held dS(c - 2), and its dQ was the last that its keys were for. They go by a plain arrival: a commit after
          // another one's waits until the pipe has run dry.
          ok = wait(kDQDone + (c & 1), ((c - 2) >> 1) & 1);
          if (!ok) break;
          if (lane == 0) mbar_arrive(bar(kKEmpty + (c - 2) % L::kK));
        }
        ok = wait(kKFull + c % L::kK, (c / L::kK) & 1);
        if (!ok) break;
        const uint64_t k = d_k + ((uint32_t)(c % L::kK) * TB >> 4);
#pragma unroll
        for (int j = 0; j < DP / 16; ++j)
          if (j < p.steps) mma_ss_warp(tmem + 128 * (c & 1), d_q + step_rows(j), k + step_rows(j), idesc_s, j > 0);
        mma_commit_warp(bar(kSFull + (c & 1)));
        ++n;
      }
      mma_commit_warp(bar(kDrainQ));
      drained(kDrainQ, 1);
      drained(kSFull, (n + 1) / 2);
      drained(kSFull + 1, n / 2);
    } else {
      const uint64_t d_do = desc_rows(base + TB), d_v = desc_rows(v_ring), d_kc = desc_cols(k_ring);
      int n_dp = 0, n_dq = 0;
      bool done = false;
      auto issue_dp = [&](int c) {
        const uint64_t v = d_v + ((uint32_t)(c % L::kV) * TB >> 4);
#pragma unroll
        for (int j = 0; j < DP / 16; ++j)
          if (j < p.steps) mma_ss_warp(t_dp, d_do + step_rows(j), v + step_rows(j), idesc_s, j > 0);
        mma_commit_warp(bar(kDPFull));
        ++n_dp;
      };
      ok = ok && wait(kVFull, 0);
      if (ok) issue_dp(0);
      for (int c = 0; ok && c < chunks; ++c) {
        if (c + 1 < chunks) {
          ok = wait(kVFull + (c + 1) % L::kV, ((c + 1) / L::kV) & 1) && wait(kDPFree, c & 1);
          if (!ok) break;
          issue_dp(c + 1);
        }
        ok = wait(kDSFull + (c & 1), (c >> 1) & 1);
        if (!ok) break;
        const uint64_t k = d_kc + ((uint32_t)(c % L::kK) * TB >> 4);
#pragma unroll
        for (int j = 0; j < kTile / 16; ++j)   // each softmax group's dS lies over its own half of S
          mma_ts_warp(t_dq, tmem + 128 * (c & 1) + j / 4 * 64 + j % 4 * 8, k + step_cols(j), p.idesc_out, c > 0 || j > 0);
        mma_commit_warp(bar(kDQDone + (c & 1)));
        ++n_dq;
      }
      if (ok) {
        mma_commit_warp(bar(kDone));
        done = true;
      }
      mma_commit_warp(bar(kDrainQ + 1));
      drained(kDrainQ + 1, 1);
      drained(kDPFull, n_dp);
      drained(kDQDone, (n_dq + 1) / 2);
      drained(kDQDone + 1, n_dq / 2);
      drained(kDone, done);
    }
  } else {
    const int half = warp / 4, row = row0 + (warp % 4) * 32 + lane;
    const bool there = row < r.nq;
    const int seen = there ? seen_by(r, row, p.a.causal) : 0;
    const float2 stat = there ? p.stats[(int64_t)head * p.a.q_rows + r.q0 + row] : make_float2(0.f, 0.f);
    int up = 0;   // dS is 2^up times as large
    if constexpr (kScaled<T>) {
      // while the first tiles are on their way; all eight warps come by here, before any wait that could end early
      const float own = there ? p.dout_norm[(int64_t)head * p.a.q_rows + r.q0 + row] : 0.f, *const norm = p.v_norm + kv * p.a.k_rows + r.k0;
      float v = 0.f;
#pragma unroll 4
      for (int j = threadIdx.x; j < min(chunks * kTile, r.nk); j += kSoftmaxWarps * 32) v = fmaxf(v, finite_or_0(norm[j]));
      most_v[warp] = warp_most(v);
      asm volatile("bar.sync 1, %0;" ::"n"(kSoftmaxWarps * 32) : "memory");
#pragma unroll
      for (int i = 0; i < kSoftmaxWarps; ++i) v = fmaxf(v, most_v[i]);
      up = exponent_for(fmaf(own, p.a.scale * v, fabsf(stat.y)));
    }
    const float one = seen == 1 ? 0.f : p.a.scale * two_to(up), less = seen == 1 ? 0.f : stat.y * two_to(up);
    const float2 sc = make_float2(p.sc, p.sc), shift = make_float2(stat.x, stat.x), minus = make_float2(less, less), scale = make_float2(one, one);
    const uint32_t lanes = (uint32_t)((warp % 4) * 32) << 16;
    bool ok = true;
    for (int c = 0; c < chunks; ++c) {
      const uint32_t t_s = tmem + 128 * (c & 1) + 64 * half + lanes;
      ok = wait_warp(bar(kSFull + (c & 1)), (c >> 1) & 1, &g_seq_bwd_errors, kErrSoftmax);
      if (!ok) break;
      float s[64];
      load_columns<64>(t_s, s);
      tmem_wait_ld();
      const int limit = seen - c * kTile - half * 64;
      const bool masked = __any_sync(0xffffffffu, limit < 64);
      if (masked && __any_sync(0xffffffffu, there && limit < 64)) {
        // Scores that are not finite where some row of the sequence does not see the key (rows behind its end count for nothing: what is
        // cleared has to lie among the keys that add_not_finite goes over): these 64 keys are cleared. Every warp that needs it does
        // so, by now S has been made of them and dQ waits for all warps; what one has cleared another leaves as it is.
        float2 odd = make_float2(0.f, 0.f);
#pragma unroll
        for (int i = 0; i < 32; ++i) odd = fma2(make_float2(s[2 * i], s[2 * i + 1]), make_float2(0.f, 0.f), odd);
        if (__any_sync(0xffffffffu, odd.x != odd.x || odd.y != odd.y)) {
#pragma unroll 1
          for (int i = 0; i < 4; ++i)
            clear_not_finite<T, DP / 64, 16>(smem_raw + (k_ring - raw) + c % L::kK * TB + half * 8192 + i * 2048, &odd_keys, 1);
        }
      }
      weights(s, sc, [&](int) { return shift; });
      ok = wait_warp(bar(kDPFull), c & 1, &g_seq_bwd_errors, kErrSoftmax);
      if (!ok) break;
      float d[64];
      load_columns<64>(t_dp + 64 * half + lanes, d);
      tmem_wait_ld();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(bar(kDPFree));
        if (warp == 0) mbar_arrive(bar(kVEmpty + c % L::kV));   // dP is complete: its values may go
      }
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        const float2 v = mul2(make_float2(s[2 * i], s[2 * i + 1]), fma2(make_float2(d[2 * i], d[2 * i + 1]), scale, minus));
        s[2 * i] = v.x, s[2 * i + 1] = v.y;
      }
      if (masked) {
#pragma unroll
        for (int i = 0; i < 64; ++i) s[i] = i < limit ? s[i] : 0.f;
      }
#pragma unroll
      for (int i = 0; i < 32; i += 16) {
        uint32_t pk[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) pk[k] = pack<T>(s[2 * (i + k)], s[2 * (i + k) + 1]);
        tmem_st16(t_s + i, pk);
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(kDSFull + (c & 1)));
    }
    if (ok) ok = wait_warp(bar(kDone), 0, &g_seq_bwd_errors, kErrSoftmax);
    if (ok) {
      // dQ, by way of the queries' memory: every product has been made
      uint8_t *const stage = smem_raw + (base - raw) + warp * 4096;
      const int64_t to = there ? ((int64_t)(r.q0 + row) * p.a.heads + head) * p.a.dim : -1;
      T *const dq = static_cast<T *>(p.dq);
      if (DP == 128 || half == 0) {
        const int col = DP == 128 ? half * 64 : 0;
        uint32_t packed[32];
        pack_columns<T>(t_dq + lanes + col, seen > 0, two_to(-up), packed);
        store_rows(stage, packed, dq, to, col, p.a.dim);
        // written before an arrival that the last product waited for
        if (*const_cast<volatile int *>(&odd_keys))
          add_not_finite(static_cast<const T *>(p.a.k) + (int64_t)r.k0 * p.a.k_stride[0] + kv * p.a.k_stride[1], p.a.k_stride[0],
                         seen_by(r, row0, p.a.causal) / kTile * kTile, col, min(col + 64, p.a.dim), true, to, seen, dq);
      }
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

// ------------------------------------------------------------------------------- dK, dV
template <int DP>
struct LayoutKV {
  static constexpr uint32_t kTileBytes = DP / 64 * kBox;
  static constexpr int kStages = DP == 128 ? 2 : 4;
  static constexpr uint32_t kStageBytes = 2 * kTileBytes;   // Q, dO
  static constexpr size_t kBytes = 1024 + 2 * kTileBytes + kStages * (size_t)(kStageBytes + kTile * sizeof(float2));
};
enum { kKVFull, kSTFull, kDPTFull, kPFull, kDSTFull, kDVDone, kDKDone, kAllDone, kLandedKV, kDrainKV, kFullKV = kDrainKV + 2 };
template <int DP> constexpr int bars_kv() { return kFullKV + 2 * LayoutKV<DP>::kStages; }

template <typename T, int DP>
__global__ void __launch_bounds__(kThreads, 1)
    sequence_dkv_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tdo,
                        const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                        const __grid_constant__ Params p) {
  using L = LayoutKV<DP>;
  constexpr uint32_t TB = L::kTileBytes;
  constexpr int NS = L::kStages;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bar_mem[bars_kv<DP>()];
  __shared__ uint32_t tmem_holder;
  __shared__ int odd_queries[NS];   // a stage has a query whose lse or delta is not finite
  __shared__ float most[3][kThreads / 32];   // of the queries' |dO| and |scale delta|, the keys' |V|
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // keys at a sequence's start are seen by the most queries
  const int per_slot = p.a.kv_heads * p.parts, slot = blockIdx.x / per_slot, kv = blockIdx.x % per_slot / p.parts,
            part = blockIdx.x % p.parts;
  const Place at = p.falling ? place_falling<true>(p.a, 7, slot) : place_of<true>(p.a, 7, slot);
  const Range r = at.r;
  const int key0 = at.group * kTile;
  if (at.group < 0 || key0 >= r.nk) return;
  const int group = p.a.heads / p.a.kv_heads, head0 = kv * group + group * part / p.parts,
            heads = kv * group + group * (part + 1) / p.parts - head0;
  // query i sees key j where i >= j - (nk - nq)
  const int shift = r.nk - r.nq, first = p.a.causal ? max(0, key0 - shift) : 0;
  const int tiles = first < r.nq ? (r.nq - first + kTile - 1) / kTile : 0, steps = tiles * heads;
  const int key = key0 + (warp % 4) * 32 + lane;   // of a softmax thread
  const bool there = key < r.nk;
  const int64_t out_row = ((int64_t)(r.k0 + key) * p.a.kv_heads + kv) * p.a.dim;
  const int64_t part_size = p.a.k_rows * p.a.kv_heads * p.a.dim;
  float *const wide_k = p.parts > 1 ? p.part + part * part_size : nullptr;
  float *const wide_v = p.parts > 1 ? p.part + (p.parts + part) * part_size : nullptr;
  if (steps == 0) {
    if (warp < 4 && there)
      for (int i = 0; i < p.a.dim; i += 8) {
        if (wide_k) {
          for (int k = 0; k < 8; k += 4) {
            *reinterpret_cast<float4 *>(wide_k + out_row + i + k) = make_float4(0.f, 0.f, 0.f, 0.f);
            *reinterpret_cast<float4 *>(wide_v + out_row + i + k) = make_float4(0.f, 0.f, 0.f, 0.f);
          }
        } else {
          if (p.dk) *reinterpret_cast<uint4 *>(static_cast<T *>(p.dk) + out_row + i) = make_uint4(0, 0, 0, 0);
          if (p.dv) *reinterpret_cast<uint4 *>(static_cast<T *>(p.dv) + out_row + i) = make_uint4(0, 0, 0, 0);
        }
      }
    return;
  }
  // of the queries of every head: the first ones' norms are asked for before the set-up
  const int64_t stat0 = (int64_t)head0 * p.a.q_rows + r.q0;
  float early_n = 0.f, early_y = 0.f, early_v = 0.f;
  if constexpr (kScaled<T>) {
    const int i = first + threadIdx.x;
    if (i < r.nq) early_n = p.dout_norm[stat0 + i], early_y = p.stats[stat0 + i].y;
    if (threadIdx.x < min(kTile, r.nk - key0)) early_v = p.v_norm[kv * p.a.k_rows + r.k0 + key0 + threadIdx.x];
  }
  const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
  uint8_t *const smem = smem_raw + (base - raw);
  const uint32_t ring = base + 2 * TB;
  float *const stats = reinterpret_cast<float *>(smem + 2 * TB + NS * L::kStageBytes);   // [stage][2][128]: both of 128 queries
  auto bar = [&](int i) { return smem_u32(&bar_mem[i]); };
  auto full = [&](int s) { return bar(kFullKV + s); };
  auto empty = [&](int s) { return bar(kFullKV + NS + s); };
  if (threadIdx.x == 0) {
    // all is complete, a stage is empty: when both warps of products say so
    for (int i = 0; i < bars_kv<DP>(); ++i)
      mbar_init(bar(i), i == kPFull || i == kDSTFull ? kSoftmaxWarps : i == kAllDone || i >= kFullKV + NS ? 2 : 1);
    fence_mbar_init();
  }
  if (warp == kMmaWarp) {
    tmem_alloc(smem_u32(&tmem_holder), 512);
    tmem_relinquish();
  }
  if (warp == kCopyWarp && lane == 0) {
    prefetch_tmap(&tq);
    prefetch_tmap(&tdo);
    prefetch_tmap(&tk);
    prefetch_tmap(&tv);
  }
  if constexpr (kScaled<T>) {
    float n = finite_or_0(early_n), y = finite_or_0(fabsf(early_y));
    for (int h = 0; h < heads; ++h) {
      const int64_t to = stat0 + h * p.a.q_rows;
#pragma unroll 4
      for (int i = first + threadIdx.x + (h ? 0 : kThreads); i < r.nq; i += kThreads) {
        n = fmaxf(n, finite_or_0(p.dout_norm[to + i]));
        y = fmaxf(y, finite_or_0(fabsf(p.stats[to + i].y)));
      }
    }
    most[0][warp] = warp_most(n), most[1][warp] = warp_most(y), most[2][warp] = warp_most(finite_or_0(early_v));
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_holder, t_dp = tmem + 128, t_dk = tmem + 256, t_dv = tmem + 384;
  auto exponent = [&] {   // dS is that power of two times as large (by a warp)
    if constexpr (kScaled<T>) {
      const int i = min(lane, kThreads / 32 - 1);
      const float n = warp_most(most[0][i]), y = warp_most(most[1][i]), v = warp_most(most[2][i]);
      return exponent_for(fmaf(n, p.a.scale * v, y));
    } else {
      return 0;
    }
  };
  constexpr int kUp = kScaled<T> ? kWeightUp : 0;   // and P

  if (warp == kCopyWarp) {
    bool ok = true;
    int issued = 0, cleared = 0;
    if (lane == 0) {
      mbar_expect_tx(bar(kKVFull), 2 * TB);
      for (int c = 0; c < DP / 64; ++c) {
        tma_load_3d(base + c * kBox, &tk, bar(kKVFull), 64 * c, kv, r.k0 + key0);
        tma_load_3d(base + TB + c * kBox, &tv, bar(kKVFull), 64 * c, kv, r.k0 + key0);
      }
    }
    __syncwarp();
    const float times = two_to(exponent() - kUp);
    for (int n = 0, head = head0, i0 = first; n < steps; ++n) {
      const int s = n % NS;
      float2 v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int i = i0 + lane + 32 * u;
        v[u] = i < r.nq ? p.stats[(int64_t)head * p.a.q_rows + r.q0 + i] : make_float2(0.f, 0.f);
      }
      if (n >= NS) ok = __all_sync(0xffffffffu, mbar_wait(empty(s), (n / NS - 1) & 1, &g_seq_bwd_errors, kWaitNs, kErrProducer));
      if (!ok) break;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        stats[s * 256 + lane + 32 * u] = v[u].x + kUp;
        stats[s * 256 + 128 + lane + 32 * u] = r.nk == 1 ? 0.f : v[u].y * times;
      }
      const bool odd = __any_sync(0xffffffffu, not_finite(v[0].x + v[0].y) || not_finite(v[1].x + v[1].y) || not_finite(v[2].x + v[2].y) ||
                                                 not_finite(v[3].x + v[3].y));
      if (lane == 0) odd_queries[s] = odd;
      __syncwarp();
      // a head's last queries, where their tile goes past the sequence's end, land on a barrier of their own
      const bool past = i0 + kTile > r.nq;
      if (lane == 0) {
        const uint32_t on = past ? bar(kLandedKV) : full(s);
        mbar_expect_tx(on, 2 * TB);
        for (int c = 0; c < DP / 64; ++c) {
          tma_load_3d(ring + s * L::kStageBytes + c * kBox, &tq, on, 64 * c, head, r.q0 + i0);
          tma_load_3d(ring + s * L::kStageBytes + TB + c * kBox, &tdo, on, 64 * c, head, r.q0 + i0);
        }
      }
      issued = n + 1;
      if (past) {
        ok = wait_warp(bar(kLandedKV), cleared++ & 1, &g_seq_bwd_errors, kErrProducer);
        if (!ok) break;
        uint8_t *const tile = smem + 2 * TB + s * L::kStageBytes;
        clear_rows<DP / 64>(tile, r.nq - i0);
        clear_rows<DP / 64>(tile + TB, r.nq - i0);
        if (lane == 0) mbar_arrive(full(s));
      }
      i0 += kTile;
      if (i0 >= r.nq) i0 = first, ++head;
    }
    if (lane == 0) {
      mbar_wait(bar(kKVFull), 0, &g_seq_bwd_errors, kWaitNs, kErrTeardown);
      for (int i = max(0, issued - NS); i < issued; ++i)
        mbar_wait(full(i % NS), (i / NS) & 1, &g_seq_bwd_errors, kWaitNs, kErrTeardown);
    }
  } else if (warp >= kMmaWarp) {
    // Products, warp-wide as in the forward kernel: two chains that meet only in the softmax, a warp each, so that each fills the other's
    // waits: dV(i), then S(i + 1) over the P that it read; dK(i), then dP(i + 1) over the dS that it read.
    const bool second = warp != kMmaWarp;
    const uint32_t idesc_s = idesc_f16(128, 128, std::is_same<T, __nv_bfloat16>::value, false);
    const uint32_t t_in = second ? t_dp : tmem, t_out = second ? t_dk : t_dv;
    const uint64_t d_a = desc_rows(second ? base + TB : base);                        // V, K
    const uint64_t d_b = desc_rows(second ? ring + TB : ring), d_c = desc_cols(second ? ring : ring + TB);   // dO, Q; then Q, dO
    const int in_full = second ? kDPTFull : kSTFull, weights_full = second ? kDSTFull : kPFull, out_done = second ? kDKDone : kDVDone;
    int n_in = 0, n_out = 0;
    bool done = false;
    auto wait = [&](uint32_t b, uint32_t parity) { return wait_warp(b, parity, &g_seq_bwd_errors, kErrMma); };
    auto stage = [&](int i) { return (uint32_t)(i % NS) * L::kStageBytes >> 4; };
    auto issue_in = [&](int i) {
#pragma unroll
      for (int j = 0; j < DP / 16; ++j)
        if (j < p.steps) mma_ss_warp(t_in, d_a + step_rows(j), d_b + stage(i) + step_rows(j), idesc_s, j > 0);
      mma_commit_warp(bar(in_full));
      ++n_in;
    };
    bool ok = wait(bar(kKVFull), 0) && wait(full(0), 0);
    if (ok) issue_in(0);
    for (int i = 0; ok && i < steps; ++i) {
      ok = wait(bar(weights_full), i & 1);
      if (!ok) break;
#pragma unroll
      for (int j = 0; j < kTile / 16; ++j)
        mma_ts_warp(t_out, t_in + j / 4 * 64 + j % 4 * 8, d_c + stage(i) + step_cols(j), p.idesc_out, i > 0 || j > 0);
      mma_commit_warp(bar(out_done));
      ++n_out;
      if (i + 1 < steps) {
        ok = wait(full((i + 1) % NS), ((i + 1) / NS) & 1) && wait(bar(out_done), i & 1);
        if (!ok) break;
        if (lane == 0) mbar_arrive(empty(i % NS));   // a plain arrival: a second commit would wait until the pipe has run dry
        issue_in(i + 1);
      }
    }
    if (ok) {
      mma_commit_warp(bar(kAllDone));
      done = true;
    }
    mma_commit_warp(bar(kDrainKV + second));
    auto drained = [&](uint32_t b, int times) {
      if (times > 0) mbar_wait(b, (times - 1) & 1, &g_seq_bwd_errors, kWaitNs, kErrTeardown);
    };
    drained(bar(kDrainKV + second), 1);
    drained(bar(in_full), n_in);
    drained(bar(out_done), n_out);
    drained(bar(kAllDone), done);
  } else {
    const int half = warp / 4;
    const uint32_t lanes = (uint32_t)((warp % 4) * 32) << 16, t_s = tmem + 64 * half + lanes, t_d = t_dp + 64 * half + lanes;
    const float one = r.nk == 1 ? 0.f : p.a.scale * two_to(exponent() - kUp);
    const float2 sc = make_float2(p.sc, p.sc), scale = make_float2(one, one);
    const int from = p.a.causal ? key - shift : 0;   // the first query that sees this key
    const int all_from = p.a.causal ? min(key0 + kTile, r.nk) - 1 - shift : 0;   // and that sees all of the tile's
    bool ok = true, cleared = false;
    for (int i = 0, row = first; i < steps; ++i, row = row + kTile < r.nq ? row + kTile : first) {
      const int i0 = row + half * 64, lo = from - i0, hi = r.nq - i0;
      const bool masked = __any_sync(0xffffffffu, lo > 0 || hi < 64);
      const float4 *st = reinterpret_cast<const float4 *>(stats + i % NS * 256 + half * 64);   // of four queries each
      ok = wait_warp(full(i % NS), (i / NS) & 1, &g_seq_bwd_errors, kErrSoftmax) &&
           wait_warp(bar(kSTFull), i & 1, &g_seq_bwd_errors, kErrSoftmax);
      if (!ok) break;
      if (row < all_from && *const_cast<volatile int *>(&odd_queries[i % NS])) {
        // Queries that some key is not seen by, one of them not finite: cleared, by each warp 16 rows, once S and dP have been made of
        // them; dK and dV wait for all warps.
        ok = wait_warp(bar(kDPTFull), i & 1, &g_seq_bwd_errors, kErrSoftmax);
        if (!ok) break;
        uint8_t *const tile = smem + 2 * TB + i % NS * L::kStageBytes + warp * 2048;
        clear_not_finite<T, DP / 64, 16>(tile, &odd_queries[i % NS], 1);
        clear_not_finite<T, DP / 64, 16>(tile + TB, &odd_queries[i % NS], 1);
        cleared = true;
      }
      float s[64];
      load_columns<64>(t_s, s);
      tmem_wait_ld();
      weights(s, sc, [&](int k) {
        const float4 q = st[k / 2];
        return k % 2 ? make_float2(q.z, q.w) : make_float2(q.x, q.y);
      });
      if (masked) {
#pragma unroll
        for (int k = 0; k < 64; ++k) s[k] = k >= lo && k < hi ? s[k] : 0.f;
      }
#pragma unroll
      for (int k = 0; k < 32; k += 16) {
        uint32_t pk[16];
#pragma unroll
        for (int u = 0; u < 16; ++u) pk[u] = pack<T>(s[2 * (k + u)], s[2 * (k + u) + 1]);
        tmem_st16(t_s + k, pk);
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(kPFull));
      ok = wait_warp(bar(kDPTFull), i & 1, &g_seq_bwd_errors, kErrSoftmax);
      if (!ok) break;
      float d[64];
      load_columns<64>(t_d, d);
      tmem_wait_ld();
#pragma unroll
      for (int k = 0; k < 32; ++k) {
        const float4 q = st[32 + k / 2];
        const float2 minus = k % 2 ? make_float2(q.z, q.w) : make_float2(q.x, q.y);
        const float2 v = mul2(make_float2(s[2 * k], s[2 * k + 1]), fma2(make_float2(d[2 * k], d[2 * k + 1]), scale, minus));
        s[2 * k] = v.x, s[2 * k + 1] = v.y;
      }
      if (masked) {
#pragma unroll
        for (int k = 0; k < 64; ++k) s[k] = k >= lo && k < hi ? s[k] : 0.f;
      }
#pragma unroll
      for (int k = 0; k < 32; k += 16) {
        uint32_t pk[16];
#pragma unroll
        for (int u = 0; u < 16; ++u) pk[u] = pack<T>(s[2 * (k + u)], s[2 * (k + u) + 1]);
        tmem_st16(t_d + k, pk);
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(kDSTFull));
    }
    if (ok) ok = wait_warp(bar(kAllDone), 0, &g_seq_bwd_errors, kErrSoftmax);
    if (ok) {
      // a half of the warps writes dK, the other dV; in 16 bits by way of the keys' memory: every product has been made
      uint8_t *const stage = smem + warp * 4096;
      T *const narrow = half ? static_cast<T *>(p.dv) : static_cast<T *>(p.dk);
      float *const wide = half ? wide_v : wide_k;
      const uint32_t t_out = (half ? t_dv : t_dk) + lanes;
      const float back = two_to(half ? -kUp : -exponent());
#pragma unroll
      for (int i = 0; i < DP; i += 64) {
        uint32_t packed[32];
        if (!wide) {
          pack_columns<T>(t_out + i, true, back, packed);
          if (narrow) store_rows(stage, packed, narrow, there ? out_row : -1, i, p.a.dim);
        } else {
#pragma unroll
          for (int h = 0; h < 64; h += 32) {
            uint32_t o[32];
            tmem_ld32(t_out + i + h, o);
            tmem_wait_ld();
#pragma unroll
            for (int k = 0; k < 32; k += 4) {
              if (there && i + h + k < p.a.dim)
                *reinterpret_cast<float4 *>(wide + out_row + i + h + k) =
                    make_float4(__uint_as_float(o[k]) * back, __uint_as_float(o[k + 1]) * back, __uint_as_float(o[k + 2]) * back,
                                __uint_as_float(o[k + 3]) * back);
            }
          }
        }
      }
      __syncwarp();
      if (cleared && half && (narrow || wide)) {   // all in the heads' first tiles
        const T *const d = static_cast<const T *>(p.dout) + ((int64_t)r.q0 * p.a.heads + head0) * p.a.dim;
        const int64_t to = there ? out_row : -1;
        if (wide) add_gradients_not_finite(d, (int64_t)p.a.heads * p.a.dim, heads, p.a.dim, first, min(first + kTile, r.nq), to, from, wide);
        else add_gradients_not_finite(d, (int64_t)p.a.heads * p.a.dim, heads, p.a.dim, first, min(first + kTile, r.nq), to, from, narrow);
      }
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

// Eight columns of a row as pairs; a lane past the row's end has zeros.
template <typename T>
__device__ __forceinline__ void load8(const T *from, bool there, float2 (&v)[4]) {
  const uint4 w = there ? __ldcs(reinterpret_cast<const uint4 *>(from)) : make_uint4(0, 0, 0, 0);
  v[0] = unpack2<T>(w.x), v[1] = unpack2<T>(w.y), v[2] = unpack2<T>(w.z), v[3] = unpack2<T>(w.w);
}
// -lse * log2(e) and -scale * delta of every row, in f16 its |dO| and each value's norm too: a row is `lanes` lanes of 16 bytes.
template <typename T>
__global__ void __launch_bounds__(256) stats_kernel(const T *out, const float *lse, const __grid_constant__ Params p, float2 *stats,
                                                    float *dout_norm, float *v_norm, int lanes) {
  const T *const dout = static_cast<const T *>(p.dout);
  const int lane = threadIdx.x & 31, per_warp = 32 / lanes, col = lane % lanes * 8, dim = p.a.dim;
  const int64_t row_first = ((int64_t)blockIdx.x * 8 + threadIdx.x / 32) * per_warp, stride = (int64_t)gridDim.x * 8 * per_warp;
  const int64_t q_rows = p.a.q_rows * p.a.heads, v_rows = kScaled<T> ? p.a.k_rows * p.a.kv_heads : 0;
  // whole warps take part in the sums: rows past the last are zeros
  for (int64_t row0 = row_first; row0 < max(q_rows, v_rows); row0 += stride) {
    const int64_t row = row0 + lane / lanes;
    const bool there = row < q_rows, value = row < v_rows;
    float2 a[4], b[4], v[4];
    load8(out + row * dim + col, there && col < dim, a);
    load8(dout + row * dim + col, there && col < dim, b);
    const int64_t key = row / p.a.kv_heads, kv = row - key * p.a.kv_heads;
    if constexpr (kScaled<T>)
      load8(static_cast<const T *>(p.a.v) + key * p.a.v_stride[0] + kv * p.a.v_stride[1] + col, value && col < dim, v);
    float sum = 0.f, square = 0.f, square_v = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      sum = fmaf(a[i].x, b[i].x, fmaf(a[i].y, b[i].y, sum));
      if constexpr (kScaled<T>) {
        square = fmaf(b[i].x, b[i].x, fmaf(b[i].y, b[i].y, square));
        square_v = fmaf(v[i].x, v[i].x, fmaf(v[i].y, v[i].y, square_v));
      }
    }
    for (int o = lanes / 2; o > 0; o >>= 1) {
      sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if constexpr (kScaled<T>) {
        square += __shfl_xor_sync(0xffffffffu, square, o);
        square_v += __shfl_xor_sync(0xffffffffu, square_v, o);
      }
    }
    if (lane % lanes) continue;
    if (there) {
      const int64_t t = row / p.a.heads, to = (row - t * p.a.heads) * p.a.q_rows + t;
      stats[to] = make_float2(lse[to] * -1.4426950408889634f, sum * -p.a.scale);
      if constexpr (kScaled<T>) dout_norm[to] = sqrtf(square);
    }
    if constexpr (kScaled<T>)
      if (value) v_norm[kv * p.a.k_rows + key] = sqrtf(square_v);
  }
}

// dk and dv from the sums of the parts, added in order.
template <typename T>
__global__ void __launch_bounds__(256) join_parts_kernel(const float *part, int parts, int64_t size, T *dk, T *dv) {
  T *const out = blockIdx.y ? dv : dk;
  if (!out) return;
  for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4; i < size; i += (int64_t)gridDim.x * 1024) {
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int q = 0; q < parts; ++q) {
      const float4 v = *reinterpret_cast<const float4 *>(part + ((int64_t)blockIdx.y * parts + q) * size + i);
      sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
    }
    *reinterpret_cast<uint2 *>(out + i) = make_uint2(pack<T>(sum.x, sum.y), pack<T>(sum.z, sum.w));
  }
}

// CTAs that share a group's heads: enough that the key tiles fill the device's SMs twice over, as far as heads go.
int parts_of(const p3d_sequence &a, int sms) {
  const int64_t tiles = ((a.k_rows + kTile - 1) / kTile) * a.kv_heads;
  return (int)std::max<int64_t>(1, std::min<int64_t>(a.heads / a.kv_heads, 2 * sms / std::max<int64_t>(tiles, 1)));
}

template <typename T, int DP>
int launch_t(const Params &p, const void *out, const float *lse, float2 *stats, cudaStream_t s) {
  const p3d_sequence &a = p.a;
  CUtensorMap tq, tdo, tk, tv;
  if (a.q_rows && a.k_rows) {
    const int64_t rows = std::max(a.q_rows * a.heads, kScaled<T> ? a.k_rows * a.kv_heads : 0);
    int lanes = 1;
    while (lanes * 8 < a.dim) lanes *= 2;
    const int64_t blocks = std::min<int64_t>((rows * lanes + 255) / 256, 148 * 16);
    stats_kernel<T><<<(unsigned)blocks, 256, 0, s>>>((const T *)out, lse, p, stats, const_cast<float *>(p.dout_norm),
                                                        const_cast<float *>(p.v_norm), lanes);
    P3D_LAUNCH_CHECK();
    const int64_t dense[2] = {(int64_t)a.heads * a.dim, a.dim};
    if (int st = encode_heads(&tq, a.dtype, a.q, a.dim, a.heads, a.q_rows, a.q_stride)) return st;
    if (int st = encode_heads(&tdo, a.dtype, p.dout, a.dim, a.heads, a.q_rows, dense)) return st;
    if (int st = encode_heads(&tk, a.dtype, a.k, a.dim, a.kv_heads, a.k_rows, a.k_stride)) return st;
    if (int st = encode_heads(&tv, a.dtype, a.v, a.dim, a.kv_heads, a.k_rows, a.v_stride)) return st;
  }
  if (p.dq && a.q_rows) {
    if (a.k_rows == 0) {
      P3D_CUDA_TRY(cudaMemsetAsync(p.dq, 0, (size_t)a.q_rows * a.heads * a.dim * 2, s));
    } else {
      const int64_t grid = slots_of(a.q_rows, a.sequences, kTile) * a.heads;
      if (grid > 0x7fffffff) return fail(P3D_ERR_UNSUPPORTED, "p3d_sequence_bwd: too many tiles");
      static size_t seen[kMaxDevices] = {};
      if (int st = smem_optin(sequence_dq_kernel<T, DP>, LayoutQ<DP>::kBytes, seen)) return st;
      sequence_dq_kernel<T, DP><<<(unsigned)grid, kThreads, LayoutQ<DP>::kBytes, s>>>(tq, tdo, tk, tv, p);
      P3D_LAUNCH_CHECK();
    }
  }
  if ((p.dk || p.dv) && a.k_rows) {
    if (a.q_rows == 0) {
      const size_t bytes = (size_t)a.k_rows * a.kv_heads * a.dim * 2;
      if (p.dk) P3D_CUDA_TRY(cudaMemsetAsync(p.dk, 0, bytes, s));
      if (p.dv) P3D_CUDA_TRY(cudaMemsetAsync(p.dv, 0, bytes, s));
      return P3D_OK;
    }
    const int64_t grid = slots_of(a.k_rows, a.sequences, kTile) * a.kv_heads * p.parts;
    if (grid > 0x7fffffff) return fail(P3D_ERR_UNSUPPORTED, "p3d_sequence_bwd: too many tiles");
    static size_t seen[kMaxDevices] = {};
    if (int st = smem_optin(sequence_dkv_kernel<T, DP>, LayoutKV<DP>::kBytes, seen)) return st;
    sequence_dkv_kernel<T, DP><<<(unsigned)grid, kThreads, LayoutKV<DP>::kBytes, s>>>(tq, tdo, tk, tv, p);
    P3D_LAUNCH_CHECK();
    if (p.parts > 1) {
      const int64_t size = a.k_rows * a.kv_heads * a.dim;
      join_parts_kernel<T><<<dim3((unsigned)std::min<int64_t>((size + 1023) / 1024, 148 * 8), 2), 256, 0, s>>>(
          p.part, p.parts, size, (T *)p.dk, (T *)p.dv);
      P3D_LAUNCH_CHECK();
    }
  }
  return P3D_OK;
}

size_t whole(size_t bytes) { return (bytes + 255) / 256 * 256; }
size_t stats_bytes(const p3d_sequence &a) { return whole((size_t)a.q_rows * a.heads * sizeof(float2)); }
size_t norm_bytes(const p3d_sequence &a) {   // of dO, then of V
  return a.dtype == P3D_F16 ? whole(((size_t)a.q_rows * a.heads + (size_t)a.k_rows * a.kv_heads) * sizeof(float)) : 0;
}

}  // namespace

int bwd_workspace(const p3d_sequence &a, size_t *bytes) {
  DeviceInfo info;
  if (int st = device_info(&info)) return st;
  const int parts = parts_of(a, info.sm_count);
  *bytes = stats_bytes(a) + norm_bytes(a) + (parts > 1 ? 2 * sizeof(float) * (size_t)parts * a.k_rows * a.kv_heads * a.dim : 0);
  return P3D_OK;
}

int launch_bwd(const p3d_sequence &a, const void *out, const float *lse, const void *dout, void *dq, void *dk, void *dv,
               void *workspace, size_t workspace_bytes, cudaStream_t s) {
  size_t need = 0;
  if (int st = bwd_workspace(a, &need)) return st;
  if (need && (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16))
    return fail(P3D_ERR_WORKSPACE, "p3d_sequence_bwd: aligned workspace of %zu bytes needed", need);
  DeviceInfo info;
  if (int st = device_info(&info)) return st;
  Params p = {};
  p.a = a;
  p.dout = dout;
  p.dq = dq, p.dk = dk, p.dv = dv;
  float2 *const stats = static_cast<float2 *>(workspace);
  p.stats = stats;
  p.parts = parts_of(a, info.sm_count);
  p.falling = falling(a, slots_of(a.k_rows, a.sequences, kTile) * a.kv_heads * p.parts, info.sm_count);
  uint8_t *const after = static_cast<uint8_t *>(workspace) + stats_bytes(a);
  if (a.dtype == P3D_F16) {
    p.dout_norm = reinterpret_cast<float *>(after);
    p.v_norm = p.dout_norm + a.q_rows * a.heads;
  }
  p.part = reinterpret_cast<float *>(after + norm_bytes(a));
  p.steps = (a.dim + 15) / 16;
  p.idesc_out = idesc_f16(128, p.steps * 16, a.dtype == P3D_BF16, true);
  p.sc = a.scale * 1.4426950408889634f;
  if (a.dtype == P3D_BF16)
    return padded(a.dim) == 64 ? launch_t<__nv_bfloat16, 64>(p, out, lse, stats, s) : launch_t<__nv_bfloat16, 128>(p, out, lse, stats, s);
  return padded(a.dim) == 64 ? launch_t<__half, 64>(p, out, lse, stats, s) : launch_t<__half, 128>(p, out, lse, stats, s);
}

int take_errors_bwd(unsigned *flags) {
  unsigned v = 0, zero = 0;
  P3D_CUDA_TRY(cudaMemcpyFromSymbol(&v, g_seq_bwd_errors, sizeof(v)));
  P3D_CUDA_TRY(cudaMemcpyToSymbol(g_seq_bwd_errors, &zero, sizeof(zero)));
  *flags |= v;
  return P3D_OK;
}

}  // namespace seq
}  // namespace p3d
