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
// these. S of 64 keys costs a third more of the pipe than half of 128, as its operands come from shared memory.
// O is rescaled only where a row's maximum has grown by more than a slack (larger weights cost no precision), after the product before
// has completed.
//
// A CTA goes through several such pairs (two thousand keys take 12 us, and setting a CTA up and taking it down 6): the next pair's
// queries, keys and first S come while this one's softmax ends and O is written. Pairs are launched the longest first, over all
// sequences, and taken over as CTAs get done. All waits go by counts that run on over the pairs.
//
// Measured, bf16, 16 heads of 128 over 4: one sequence of 8,192 without a mask 572 us, 961 TFLOP/s (64 keys of both tiles take 2,300 cycles,
// 1,280 of them products; f16 626 us), causal 292 us; causal prompts of 1,200 to 3,400 tokens, 20,011 in all, 290 us, 770. Two softmax
// warps a scheduler leave 60 % of the issue slots empty while they wait for tensor memory and for each other's exponentials.
// Looking through the values at the mask's border costs 0.2 us of three prompts of 203 tokens in all (7.1 on the GPU), nothing that shows
// of the long ones.
//
// Masks: key j counts for row i where j < seen(i); units of keys that some row of a warp does not see whole are masked by columns.
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
// The maximum may lag by 2^slack, and weights are 2^up times as large. bf16: 2^8, and as they are. f16 has no numbers below 2^-24, so the largest
// weight is between 2^10 and 2^14 (its largest number is 2^16, what is left is for the rounding of large scores): what is lost below
// 2^-35 of it, against 2^-25, is under half a step of the result for a million keys.
template <typename T> constexpr float kSlack = std::is_same<T, __half>::value ? 4.f : 8.f;
template <typename T> constexpr float kWeightUp = std::is_same<T, __half>::value ? 10.f : 0.f;
constexpr int kPoly = 2;                     // pairs of exponentials of eight that are polynomials

template <int DP>
struct Layout {
  static constexpr uint32_t kTileBytes = DP / 64 * kBox;
  static constexpr int kStages = DP == 128 ? 4 : 8;
  static constexpr uint32_t kStageOut = 8 * 4096;   // of the softmax warps, for O on its way out
  static constexpr size_t kBytes = 1024 + (2 + kStages) * (size_t)kTileBytes + kStageOut;
};

// Every wait on a barrier that completes more than once is by someone who has seen the completion before, and whose own next step the
// one after needs.
enum { kQFull, kQEmpty, kSFull, kPFull = kSFull + 4, kODone = kPFull + 2, kNext = kODone + 2, kDrain, kFull = kDrain + 2 };
template <int DP> constexpr int bars() { return kFull + 2 * Layout<DP>::kStages; }

struct Params {
  p3d_sequence a;
  void *out;
  float *lse;
  int units;       // of heads: pairs, or single ones
  int two_heads;   // a CTA's tiles are two heads
  int steps;       // of 16 columns
  int works;       // pairs of tiles
  int falling;     // their order
  uint32_t idesc_o;
  float sc;        // scale * log2(e)
};

// A pair of tiles: rows i0 (+ 128 for the second tile where the tiles are of one head) of sequence `r`.
struct Work {
  Range r;
  int row[2], head[2], kv;
  int units[2];    // 64 keys that each tile sees any of
  int whole;       // of those, the first ones that every row of both tiles sees all of
  int index;       // in the order of launches; -1: none
  __device__ __forceinline__ int most() const { return max(units[0], units[1]); }
  __device__ __forceinline__ int chunks() const { return (most() + 1) / 2; }   // tiles of keys
};
__device__ __forceinline__ Work work_of(const Params &p, int index) {
  const int slot = index / p.units, unit = index % p.units;
  const int shift = p.two_heads ? 7 : 8;   // 128 or 256 rows a slot
  const Place s = p.falling ? place_falling<false>(p.a, shift, slot)
                               : place_of<false>(p.a, shift, p.works / p.units - 1 - slot);   // the longest of each sequence first
  Work w;
  w.r = s.r;
  const int group = p.a.heads / p.a.kv_heads;
  w.index = index;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    w.head[t] = p.two_heads ? 2 * unit + t : unit;
    w.row[t] = (s.group << shift) + (p.two_heads ? 0 : t * kTile);
    w.units[t] = 0;
    if (s.group >= 0 && w.row[t] < w.r.nq)
      w.units[t] = (seen_by(w.r, min(w.row[t] + kTile, w.r.nq) - 1, p.a.causal) + kKeys - 1) / kKeys;
  }
  w.whole = w.units[0] ? seen_by(w.r, w.row[0], p.a.causal) / kKeys : 0;
  w.kv = w.head[0] / group;
  return w;
}

// P = 2^(s sc + shift) of a row's 64 scores, rounded to T and written over them; returns the row's sum.  kPoly of every eight pairs are
// polynomials, which make a finite number of a NaN and of -inf. A NaN score makes the row's maximum NaN; a score
// of +inf makes it infinite, as scores that are all -inf do. Such rows have no softmax: they become NaN at their end, whatever they held.
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
  __shared__ Work works[2];   // of a pair (by its number's last bit), as the copying warp found it
  __shared__ int odd_pair[2];   // by the same bit: the number + 1 of the last pair whose values were not all finite
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  __shared__ __align__(16) uint4 answer;
  const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
  uint8_t *const smem = smem_raw + (base - raw);
  const uint32_t ring = base + 2 * L::kTileBytes;
  auto bar = [&](int i) { return smem_u32(&bar_mem[i]); };
  auto full = [&](int s) { return bar(kFull + s); };
  auto empty = [&](int s) { return bar(kFull + NS + s); };
  if (threadIdx.x == 0) {
    for (int i = 0; i < bars<DP>(); ++i)
      mbar_init(bar(i), i == kQEmpty ? 10 : i == kPFull || i == kPFull + 1 ? 4 : i >= kFull + NS ? 2 : 1);
    fence_mbar_init();
    odd_pair[0] = odd_pair[1] = 0;
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

  int done = 0;   // pairs before this one
  if (warp == kCopyWarp) {
    // ------------------------------------------------------------------ copies; items K0, V0, K1, V1, .. of one pair after another
    bool ok = true;
    int item0 = 0, issued = 0;
    Work now = work_of(p, blockIdx.x);
    for (;; ++done) {
      // the last pair's queries have had their last product, and everybody knows of it
      if (done) ok = __all_sync(0xffffffffu, mbar_wait(bar(kQEmpty), (done - 1) & 1, &g_seq_fwd_errors, kWaitNs, kErrProducer));
      if (!ok) break;
      const int chunks = now.index < 0 ? 0 : now.chunks();
      if (lane == 0) {
        works[done & 1] = now;
        if (chunks) mbar_expect_tx(bar(kQFull), 2 * L::kTileBytes);
        else mbar_arrive(bar(kQFull));
        if (now.index >= 0) ask_for_work(smem_u32(&answer), bar(kNext));
#pragma unroll
        for (int t = 0; t < 2; ++t)
          for (int c = 0; chunks && c < DP / 64; ++c)
            tma_load_3d(base + t * L::kTileBytes + c * kBox, &tq, bar(kQFull), 64 * c, now.head[t], now.r.q0 + now.row[t]);
        for (int i = item0; i < item0 + 2 * chunks; ++i) {
          const int s = i % NS, c = (i - item0) / 2;
          if (i >= NS && !mbar_wait(empty(s), (i / NS - 1) & 1, &g_seq_fwd_errors, kWaitNs, kErrProducer)) {
            ok = false;
            break;
          }
          mbar_expect_tx(full(s), L::kTileBytes);
          for (int k = 0; k < DP / 64; ++k)
            tma_load_3d(ring + s * L::kTileBytes + k * kBox, (i - item0) % 2 ? &tv : &tk, full(s), 64 * k, now.kv, now.r.k0 + c * kTile);
          issued = i + 1;
        }
      }
      ok = __all_sync(0xffffffffu, ok);
      item0 += 2 * chunks;
      if (now.index < 0) break;
      ok = wait_warp(bar(kNext), done & 1, &g_seq_fwd_errors, kErrProducer) && ok;
      if (!ok) break;
      const int index = work_given(smem_u32(&answer));
      fence_proxy_async_smem();   // read before the next answer is written there
      if (index >= 0) now = work_of(p, index);
      else now.index = -1;
    }
    // no copy in flight into memory that is about to be given up
    if (lane == 0) {
      if (issued) mbar_wait(bar(kQFull), done & 1, &g_seq_fwd_errors, kWaitNs, kErrTeardown);
      for (int i = max(0, issued - NS); i < issued; ++i)
        mbar_wait(full(i % NS), (i / NS) & 1, &g_seq_fwd_errors, kWaitNs, kErrTeardown);
    }
  } else if (warp >= kMmaWarp) {
    // ------------------------------------------------------------------ products, of one tile
    // The whole warp runs this, with the same operands in every lane; one elected lane issues (30 cycles a product instead of 75). The
    // pipe takes four products ahead and a wait costs 70 cycles even where there is nothing to wait for: with one warp for both
    // tiles the pipe ran dry at each of them.
    const int t = warp - kMmaWarp;
    const uint32_t idesc_s = idesc_f16(128, kKeys, std::is_same<T, __nv_bfloat16>::value, false);
    const uint64_t desc_q = desc_rows(base + t * L::kTileBytes), desc_k = desc_rows(ring), desc_v = desc_cols(ring);
    const uint32_t t_s = tmem + kColS + 128 * t, t_o = tmem + kColO + 128 * t;
    int n_s = 0, n_o = 0;                  // products of this tile so far
    int item0 = 0, landed = 0;
    int give_back = -1;                    // the items whose last readers are under way: this one and the next
    bool waited = true;                    // the last O has been waited for
    auto wait = [&](uint32_t b, uint32_t parity) { return wait_warp(b, parity, &g_seq_fwd_errors, kErrMma); };
    bool ok = true;
    for (;; ++done) {
      ok = wait(bar(kQFull), done & 1);
      if (!ok) break;
      const Work &now = works[done & 1];
      if (now.index < 0) break;
      const int units = now.most(), mine = now.units[t];
      // item i is there; items are waited for in order, once
      auto wait_item = [&](int i) {
        for (; landed <= i; ++landed)
          if (!wait(full(landed % NS), (landed / NS) & 1)) return false;
        return true;
      };
      // S of unit u: into the buffer that S two before was in
      auto issue_s = [&](int u) {
        const uint64_t k = desc_k + (((uint32_t)((item0 + u / 2 * 2) % NS) * L::kTileBytes + (u & 1) * kKeys * 128) >> 4);
#pragma unroll
        for (int j = 0; j < DP / 16; ++j)
          if (j < p.steps) mma_ss_warp(t_s + 64 * (n_s & 1), desc_q + step_rows(j), k + step_rows(j), idesc_s, j > 0);
        mma_commit_warp(bar(kSFull + 2 * t + (n_s & 1)));
        ++n_s;
      };
      auto issue_o = [&](int u) {
        const uint64_t v = desc_v + ((uint32_t)((item0 + u / 2 * 2 + 1) % NS) * L::kTileBytes >> 4) + step_cols((u & 1) * (kKeys / 16));
#pragma unroll
        for (int j = 0; j < kKeys / 16; ++j)
          mma_ts_warp(t_o, t_s + 64 * (n_o & 1) + 8 * j, v + step_cols(j), p.idesc_o, u > 0 || j > 0);
        mma_commit_warp(bar(kODone + t));
        ++n_o;
        waited = false;
      };
      ok = !units || wait_item(item0);
      if (ok && mine) issue_s(0);
      for (int u = 0; ok && u < units; ++u) {
        // The last O is there, and with it its S: their keys and values may go. By a plain arrival: a commit after another one's
        // waits until the pipe has run dry. A tile that is done, or has no rows, arrives for what has landed.
        if (!waited) ok = wait(bar(kODone + t), (n_o - 1) & 1);
        waited = true;
        if (!ok) break;
        if (give_back >= 0 && lane == 0) {
          mbar_arrive(empty(give_back % NS));
          mbar_arrive(empty((give_back + 1) % NS));
        }
        give_back = -1;
        if (u + 1 < mine) {
          ok = wait_item(item0 + (u + 1) / 2 * 2);
          if (!ok) break;
          issue_s(u + 1);
        }
        ok = wait_item(item0 + u / 2 * 2 + 1);
        if (!ok) break;
        if (u < mine) {
          ok = wait(bar(kPFull + t), n_o & 1);
          if (!ok) break;
          issue_o(u);
        }
        if (u & 1 || u == units - 1) give_back = item0 + u / 2 * 2;
      }
      if (!ok) break;
      item0 += (units + 1) / 2 * 2;
      if (lane == 0) mbar_arrive(bar(kQEmpty));
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
    const int t = warp / 4;
    const uint32_t lanes = (uint32_t)((warp % 4) * 32) << 16;
    const uint32_t t_s = tmem + kColS + 128 * t + lanes, t_o = tmem + kColO + 128 * t + lanes;
    const float sc = p.sc;
    int n = 0;       // steps of this tile so far
    int item0 = 0;   // of this pair
    bool ok = true;
    uint8_t *const stage = smem + (2 + NS) * L::kTileBytes + warp * 4096;
    for (;; ++done) {
      // After the wait for a pair's queries, which come only when every warp has said that it knows of the pair before: no warp, with
      // rows or without, is a pair ahead.
      ok = wait_warp(bar(kQFull), done & 1, &g_seq_fwd_errors, kErrSoftmax);
      if (!ok) break;
      const Work now = works[done & 1];
      if (now.index < 0) break;
      const int mine = t ? now.units[1] : now.units[0], head = t ? now.head[1] : now.head[0], row0 = t ? now.row[1] : now.row[0];
      const int row = row0 + (warp % 4) * 32 + lane;
      const bool there = row0 >= 0 && row < now.r.nq;
      const int seen = there ? seen_by(now.r, row, p.a.causal) : 0;
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(kQEmpty));
      float m = -INFINITY, l = 0.f;
      for (int u = 0; u < mine; ++u, ++n) {
        const uint32_t t_u = t_s + 64 * (n & 1);
        // Keys that some row does not see: its weights are 0, and 0 times an infinity or NaN is not. The four warps clear their quarters
        // of the 64 values before this tile's product may read them. (The other tile's product may be under way: its own warps have
        // cleared them, and what is written here is what is there.) Here, as S is still being made. The wait is exact: the stage's item before
        // this one has landed, as a product of this tile that has been waited for came after it, or it was of a pair that is done.
        if (u >= now.whole) {
          const int item = item0 + u / 2 * 2 + 1;
          if (u == now.whole || u % 2 == 0) ok = wait_warp(full(item % NS), (item / NS) & 1, &g_seq_fwd_errors, kErrSoftmax);
          if (!ok) break;
          clear_not_finite<T, DP / 64, kKeys / 4>(smem + (2 + item % NS) * L::kTileBytes + ((u & 1) * 4 + warp % 4) * (kKeys / 4 * 128),
                                                  &odd_pair[done & 1], done + 1);
        }
        ok = wait_warp(bar(kSFull + 2 * t + (n & 1)), (n >> 1) & 1, &g_seq_fwd_errors, kErrSoftmax);
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
        const float best = max3_nan(m, max_nan(top[0], top[1]), max_nan(top[2], top[3]));
        // a row that has seen nothing yet has an empty O: its first maximum rescales nothing
        const bool moves = !((best - m) * sc <= kSlack<T>) && !(best == -INFINITY);
        const bool any_moves = __any_sync(0xffffffffu, moves);
        float down = 1.f;
        if (any_moves) {
          if (moves) {
            down = m == -INFINITY ? 0.f : ex2_approx((m - best) * sc);
            m = best;
          }
          l *= down;
        }
        float shift = m == -INFINITY ? 0.f : -m * sc;
        if constexpr (kWeightUp<T> != 0.f) shift += kWeightUp<T>;
        // a border's masked scores have weight 0, which the polynomial does not give
        l += masked ? weights<T, 0>(s, sc, shift, t_u) : weights<T, kPoly>(s, sc, shift, t_u);
        // O rests once the product before has completed (waited for at every step, so that the parity is exact)
        if (u > 0) {
          ok = wait_warp(bar(kODone + t), (n - 1) & 1, &g_seq_fwd_errors, kErrSoftmax);
          if (!ok) break;
          if (any_moves) {
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
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(kPFull + t));
      }
      if (!ok) break;
      if (mine) ok = wait_warp(bar(kODone + t), (n - 1) & 1, &g_seq_fwd_errors, kErrSoftmax);
      if (!ok) break;
      if (not_finite(m)) l = NAN;   // of no row whose softmax exists
      const float inv = seen > 0 ? 1.f / l : 0.f;
      const int64_t at = there ? ((int64_t)(now.r.q0 + row) * p.a.heads + head) * p.a.dim : -1;
      T *const out = static_cast<T *>(p.out);
#pragma unroll
      for (int i = 0; i < DP; i += 64) {
        if (i >= p.a.dim) continue;
        uint32_t packed[32];
#pragma unroll
        for (int h = 0; h < 64; h += 32) {
          uint32_t o[32];
          if (mine) {
            tmem_ld32(t_o + i + h, o);
            tmem_wait_ld();
          }
#pragma unroll
          for (int k = 0; k < 32; k += 2) {
            const float a = seen > 0 ? __uint_as_float(o[k]) * inv : 0.f, b = seen > 0 ? __uint_as_float(o[k + 1]) * inv : 0.f;
            packed[(h + k) / 2] = pack<T>(a, b);
          }
        }
        store_rows(stage, packed, out, at, i, p.a.dim);
      }
      if (p.lse && there)
        p.lse[(int64_t)head * p.a.q_rows + now.r.q0 + row] = seen > 0 ? (m * sc + log2f(l) - kWeightUp<T>) * 0.6931471805599453f : -INFINITY;
      // what was cleared, by this tile's warps or the other's, for the rows that see it
      if (mine && *const_cast<volatile int *>(&odd_pair[done & 1]) == done + 1)
        add_not_finite(static_cast<const T *>(p.a.v) + (int64_t)now.r.k0 * p.a.v_stride[0] + now.kv * p.a.v_stride[1], p.a.v_stride[0],
                       now.whole * kKeys, 0, p.a.dim, false, at, seen, out);
      item0 += 2 * now.chunks();
      tc_fence_before();   // O is read before the next pair's P lets a product write it
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
int launch_t(const Params &p, int grid, const CUtensorMap &tq, const CUtensorMap &tk, const CUtensorMap &tv, cudaStream_t s) {
  static size_t seen[kMaxDevices] = {};
  if (int st = smem_optin(sequence_fwd_kernel<T, DP>, Layout<DP>::kBytes, seen)) return st;
  sequence_fwd_kernel<T, DP><<<grid, kThreads, Layout<DP>::kBytes, s>>>(tq, tk, tv, p);
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
  const int64_t works = slots_of(a.q_rows, a.sequences, p.two_heads ? kTile : 2 * kTile) * p.units;
  if (works > 0x7fffffff - 4096) return fail(P3D_ERR_UNSUPPORTED, "p3d_sequence_fwd: too many tiles");
  p.works = (int)works;
  DeviceInfo info;
  if (int st = device_info(&info)) return st;
  p.falling = falling(a, works, info.sm_count);
  const int grid = p.works;
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
