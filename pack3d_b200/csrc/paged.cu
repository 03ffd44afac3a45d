// Attention of one new token of each sequence over its pages:  out = sum_t p_t v_t / sum_t p_t,  p_t = 2^(s_t - m),
// s_t = q k_t scale log2(e).
//
// Bound by HBM: every key and value that a sequence holds is read once for its group of query heads (16-bit: 4 dim bytes a token and
// head, 8-bit: half of that and two scale bytes), and little else moves.
//
// * A warp takes tiles of 16 or 32 tokens. Keys and values go from memory to registers in the layout that m16n8k16 tensor products
//   want them in, without shared memory: the products' inner indexes may be permuted, so a lane's 16 consecutive bytes of a
//   key are the columns that it contributes to two (8-bit: four) products, and 16 consecutive bytes of a value row are its
//   column in eight (sixteen) of them. The heads of a group are the products' 16 rows (padded: the tensor pipe has time to
//   spare at this intensity).
// * The next tile's keys and values are asked for as soon as this one's scores are there, before its softmax and its values' products.
//   For the registers that takes, the queries stay in shared memory. The page table is read a tile further ahead.
// * 8 bits: e4m3 goes to f16 exactly. A query is brought below 2 by a power of two, the keys' scales multiply the scores. The
//   values' scales 2^e go into the weights, which are held relative to the largest weighted scale, m = max(s_t + e_t), so that they
//   fit f16 whatever the scales; the sum of weights without them stays in fp32. In f16 (of either kind of page) the largest is 2^10,
//   so that what is below 2^-35 of it is lost, against 2^-25: tens of thousands of quiet tokens behind a loud one count.
// * Work is cut into units of four tiles (one for each warp of a CTA), laid out in one line over all sequences and KV heads, and
//   every CTA takes an equal stretch of it: one long sequence or many uneven ones fill the device alike. A head's pieces
//   are joined by a second kernel, in order; a stretch holds at most one head that began before it and one that goes on
//   after it, so two slots a CTA keep all pieces. Where no sequence can be longer than a few units, a CTA takes a whole head.
//
// Measured, 32 heads over 8 of 128, with the join: one sequence of 200,003 tokens in bf16 153 us, 5.3 TB/s (loads in flight: 255 registers
// a thread leave eight warps an SM); 64 sequences, 262,144 tokens, in 8 bits 139 us, 3.9 TB/s (the conversions' instructions, at a
// third of the issue slots, between two loads of a warp).
#include <cuda_fp8.h>
#include <math.h>

#include <algorithm>

#include "cache.cuh"
#include "kernels.cuh"
#include "sm100.cuh"

namespace p3d {
namespace {

__device__ unsigned g_paged_errors = 0;

constexpr int kWarps = 4, kRows = 16;
constexpr uint32_t kNone = 0xffffffffu, kBad = 0xfffffffeu;   // in place of a row: past the length, on a bad page

struct Params {
  p3d_cache c;
  const void *q;
  int64_t q_token, q_head;
  void *out;
  const int32_t *lengths;
  float scale;          // scale * log2(e)
  int heads, group;     // query heads, and those of one KV head
  int row_tiles;        // tiles of 16 query heads that a group takes
  int ctas;             // that the line is cut for; 0: a CTA for each head
  int wide;             // 8-bit rows are 16-byte aligned
  int exact;            // the head dim is the padded one: no piece of a row is cut
  float *parts;         // [2 * ctas][part_rows][dim + 2]
  int part_rows;
};

template <typename T> __device__ __forceinline__ uint32_t pack(float a, float b);
template <> __device__ __forceinline__ uint32_t pack<__half>(float a, float b) { return sm100::pack_f16(a, b); }
template <> __device__ __forceinline__ uint32_t pack<__nv_bfloat16>(float a, float b) { return sm100::pack_bf16(a, b); }

template <typename T>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Two e4m3 in the low half of w as f16, exactly.
__device__ __forceinline__ uint32_t e4m3x2(uint32_t w) {
  uint32_t r;
  asm("{\n\t.reg .b16 h;\n\tcvt.u16.u32 h, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, h;\n\t}" : "=r"(r) : "r"(w));
  return r;
}

__device__ __forceinline__ float two_to(uint32_t byte) { return __uint_as_float(byte ? byte << 23 : 0x400000u); }   // 2^(byte - 127)

// CTAs that an SM holds, by the registers of their tiles (two: 255 a thread; three: 168).
__host__ __device__ constexpr int per_sm(bool k8, int dp) { return k8 && dp == 64 ? 3 : 2; }

// T: the type of queries (and 16-bit pages). DP: head dim rounded up to 64 or 128. KT: 16-token steps of a tile.
template <typename T, bool k8, int DP>
struct Tile {
  using M = typename std::conditional<k8, __half, T>::type;            // what the products take
  static constexpr float kWeightUp = std::is_same<M, __half>::value ? 10.f : 0.f;
  static constexpr int KT = DP == 128 && !k8 ? 1 : 2, TT = 16 * KT, NT = 2 * KT;
  static constexpr int KC = k8 ? DP / 64 : DP / 32;                    // 16-byte pieces of a key that a lane holds
  static constexpr int VC = k8 ? 1 : DP / 64, VW = k8 && DP == 64 ? 2 : 4;   // pieces of a value row, words of each
  static constexpr int CT = DP / 8;                                    // column tiles of the output
  static constexpr int VB = VW * 4;

  // Column of the output: tile j, place x of eight.
  static __device__ __forceinline__ int column(int j, int x) {
    if constexpr (k8) return x * (DP / 8) + j;
    else return j / 8 * 64 + x * 8 + j % 8;
  }

  static constexpr int kSteps = KC * (k8 ? 4 : 2);                     // of 16 columns
  float q_scale[2];                   // of rows lane / 4 and + 8: scale and, for 8 bits, the query's power of two
  uint32_t k[NT][KC][4];
  struct Values {
    uint32_t w[KT][4][VC][VW];
  };
  float o[CT][4], m[2];
  float2 l[2];                        // of the even and odd columns that a lane has

  __device__ __forceinline__ static uint4 load16(const uint8_t *p, int at, int bytes, int wide) {
    uint4 w = make_uint4(0, 0, 0, 0);
    if (at + 16 <= bytes) {
      if (!k8 || wide) return __ldg(reinterpret_cast<const uint4 *>(p + at));
      const uint2 a = __ldg(reinterpret_cast<const uint2 *>(p + at)), b = __ldg(reinterpret_cast<const uint2 *>(p + at + 8));
      return make_uint4(a.x, a.y, b.x, b.y);
    }
    if (k8 && at < bytes) {   // eight columns left
      const uint2 a = __ldg(reinterpret_cast<const uint2 *>(p + at));
      w.x = a.x, w.y = a.y;
    }
    return w;
  }

  // The queries as A operands, in shared memory: [step][lane], written by one warp.
  __device__ __forceinline__ void load_q(const Params &p, uint4 *to, bool write, int b, int head0, int rows, int lane) {
    uint32_t q[kSteps][4];
    const int r = lane / 4, c = lane % 4, dim = p.c.dim;
    float top[2] = {0.f, 0.f};
    const T *row[2];
    bool there[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      there[i] = r + 8 * i < rows;
      row[i] = static_cast<const T *>(p.q) + b * p.q_token + (head0 + (there[i] ? r + 8 * i : 0)) * p.q_head;
    }
    if constexpr (!k8) {
#pragma unroll
      for (int s = 0; s < KC; ++s) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          uint4 w = make_uint4(0, 0, 0, 0);
          const int at = s * 32 + c * 8;
          if (there[i] && at < dim) w = *reinterpret_cast<const uint4 *>(row[i] + at);
          q[2 * s][i] = w.x, q[2 * s][2 + i] = w.y;
          q[2 * s + 1][i] = w.z, q[2 * s + 1][2 + i] = w.w;
        }
      }
      q_scale[0] = q_scale[1] = p.scale;
    } else {
      // the row's largest magnitude, then its values over that power of two, in f16
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint2 raw[KC * 4];
#pragma unroll
        for (int s = 0; s < KC * 4; ++s) {
          const int at = s / 4 * 64 + c * 16 + s % 4 * 4;
          raw[s] = there[i] && at < dim ? *reinterpret_cast<const uint2 *>(row[i] + at) : make_uint2(0, 0);
          const float2 a = unpack2<T>(raw[s].x), d = unpack2<T>(raw[s].y);
          top[i] = fmaxf(top[i], fmaxf(fmaxf(fabsf(a.x), fabsf(a.y)), fmaxf(fabsf(d.x), fabsf(d.y))));
        }
        top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 1));
        top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 2));
        const uint32_t e = min(max(__float_as_uint(top[i]) >> 23, 1u), 253u);
        const float down = __uint_as_float((254u - e) << 23);
        q_scale[i] = p.scale * __uint_as_float(e << 23);
#pragma unroll
        for (int s = 0; s < KC * 4; ++s) {
          const float2 a = unpack2<T>(raw[s].x), d = unpack2<T>(raw[s].y);
          q[s][i] = sm100::pack_f16(a.x * down, a.y * down);
          q[s][2 + i] = sm100::pack_f16(d.x * down, d.y * down);
        }
      }
    }
    if (write)
#pragma unroll
      for (int s = 0; s < kSteps; ++s) to[s * 32 + lane] = make_uint4(q[s][0], q[s][1], q[s][2], q[s][3]);
  }

  // What a lane resolves for its tile: the row of token base + lane.
  __device__ __forceinline__ static uint32_t resolve(const Params &p, int b, int g, int n, int64_t base, int lane) {
    const int64_t t = base + lane;
    if (lane >= TT || t >= n) return kNone;
    const cache::Place place = cache::place_of(p.c, b, t);
    if (place.page < 0) {
      atomicOr(&g_paged_errors, cache::kErrPage);
      return kBad;
    }
    return ((uint32_t)place.page * p.c.kv_heads + g) * p.c.page_size + place.row;
  }

  __device__ __forceinline__ const uint8_t *row_of(const void *pages, uint32_t row, int bytes) const {
    return static_cast<const uint8_t *>(pages) + (uint64_t)row * (uint32_t)bytes;
  }

  // `all`: every token of the tile is there and rows are whole, as in all tiles but a sequence's last: loads without conditions.
  __device__ __forceinline__ void load_k(const Params &p, uint32_t rows, bool all, int lane) {
    const int bytes = p.c.dim * (k8 ? 1 : 2);
    if (all) {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const uint4 *from = reinterpret_cast<const uint4 *>(
            row_of(p.c.k, __shfl_sync(0xffffffffu, rows, t * 8 + lane / 4), DP * (k8 ? 1 : 2)) + lane % 4 * 16);
#pragma unroll
        for (int s = 0; s < KC; ++s) {
          const uint4 w = __ldg(from + 4 * s);
          k[t][s][0] = w.x, k[t][s][1] = w.y, k[t][s][2] = w.z, k[t][s][3] = w.w;
        }
      }
      return;
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const uint32_t row = __shfl_sync(0xffffffffu, rows, t * 8 + lane / 4);
#pragma unroll
      for (int s = 0; s < KC; ++s) {
        uint4 w = make_uint4(0, 0, 0, 0);
        if (row < kBad) w = load16(row_of(p.c.k, row, bytes), s * 64 + lane % 4 * 16, bytes, p.wide);
        k[t][s][0] = w.x, k[t][s][1] = w.y, k[t][s][2] = w.z, k[t][s][3] = w.w;
      }
    }
  }

  __device__ __forceinline__ void load_v(const Params &p, Values &v, uint32_t rows, bool all, int lane) {
    const int bytes = p.c.dim * (k8 ? 1 : 2);
    if (all) {
#pragma unroll
      for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint8_t *from = row_of(p.c.v, __shfl_sync(0xffffffffu, rows, t * 16 + lane % 4 * 2 + i % 2 + i / 2 * 8),
                                       DP * (k8 ? 1 : 2)) + lane / 4 * VB;
#pragma unroll
          for (int s = 0; s < VC; ++s) {
            if constexpr (VW == 4) {
              const uint4 w = __ldg(reinterpret_cast<const uint4 *>(from + s * 128));
              v.w[t][i][s][0] = w.x, v.w[t][i][s][1] = w.y, v.w[t][i][s][2] = w.z, v.w[t][i][s][3] = w.w;
            } else {
              const uint2 w = __ldg(reinterpret_cast<const uint2 *>(from));
              v.w[t][i][s][0] = w.x, v.w[t][i][s][1] = w.y;
            }
          }
        }
      return;
    }
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t row = __shfl_sync(0xffffffffu, rows, t * 16 + lane % 4 * 2 + i % 2 + i / 2 * 8);
#pragma unroll
        for (int s = 0; s < VC; ++s) {
          const int at = s * 128 + lane / 4 * VB;
          if constexpr (VW == 4) {
            uint4 w = make_uint4(0, 0, 0, 0);
            if (row < kBad) w = load16(row_of(p.c.v, row, bytes), at, bytes, p.wide);
            v.w[t][i][s][0] = w.x, v.w[t][i][s][1] = w.y, v.w[t][i][s][2] = w.z, v.w[t][i][s][3] = w.w;
          } else {
            uint2 w = make_uint2(0, 0);
            if (row < kBad && at < bytes) w = __ldg(reinterpret_cast<const uint2 *>(row_of(p.c.v, row, bytes) + at));
            v.w[t][i][s][0] = w.x, v.w[t][i][s][1] = w.y;
          }
        }
      }
  }

  // Scores of the tile's tokens: columns 2c, 2c + 1 of each eight in rows r and r + 8.
  __device__ __forceinline__ void scores(float (&s)[NT][4], const uint4 *queries, int lane) const {
#pragma unroll
    for (int t = 0; t < NT; ++t) s[t][0] = s[t][1] = s[t][2] = s[t][3] = 0.f;
#pragma unroll
    for (int a = 0; a < kSteps; ++a) {
      const uint4 w = queries[a * 32 + lane];
      const uint32_t q[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        if constexpr (k8) mma<M>(s[t], q, e4m3x2(k[t][a / 4][a % 4]), e4m3x2(k[t][a / 4][a % 4] >> 16));
        else mma<M>(s[t], q, k[t][a / 2][a % 2 * 2], k[t][a / 2][a % 2 * 2 + 1]);
      }
    }
  }

  // Weights from scores, running maximum and sum, and the weighted values.  Of the lane's token: ks, vs its scales 2^e, e the value's.
  __device__ __forceinline__ void add(float (&s)[NT][4], const Values &v, uint32_t rows, bool all, float ks, float vs, float e, int lane) {
    using sm100::add2;
    using sm100::mul2;
    const int c = lane % 4;
    float2 y[NT][2], scale[NT];   // scores of rows r, r + 8; the values' scales
    float top[2] = {m[0], m[1]};
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int from = t * 8 + c * 2;
      float2 key = make_float2(1.f, 1.f), ev = make_float2(0.f, 0.f);
      if constexpr (k8) {
        key = make_float2(__shfl_sync(0xffffffffu, ks, from), __shfl_sync(0xffffffffu, ks, from + 1));
        scale[t] = make_float2(__shfl_sync(0xffffffffu, vs, from), __shfl_sync(0xffffffffu, vs, from + 1));
        ev = make_float2(__shfl_sync(0xffffffffu, e, from), __shfl_sync(0xffffffffu, e, from + 1));
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        y[t][i] = mul2(make_float2(s[t][2 * i], s[t][2 * i + 1]), make_float2(q_scale[i], q_scale[i]));
        if constexpr (k8) y[t][i] = mul2(y[t][i], key);
      }
      if (!all) {
        const uint32_t r0 = __shfl_sync(0xffffffffu, rows, from), r1 = __shfl_sync(0xffffffffu, rows, from + 1);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          y[t][i].x = r0 == kNone ? -INFINITY : r0 == kBad ? NAN : y[t][i].x;
          y[t][i].y = r1 == kNone ? -INFINITY : r1 == kBad ? NAN : y[t][i].y;
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float2 u = k8 ? add2(y[t][i], ev) : y[t][i];
        top[i] = fmaxf(top[i], fmaxf(u.x, u.y));
      }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 1));
      top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 2));
    }
    if (__any_sync(0xffffffffu, top[0] > m[0] || top[1] > m[1])) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float down = m[i] == -INFINITY ? 0.f : sm100::ex2_approx(m[i] - top[i]);
        l[i] = mul2(l[i], make_float2(down, down));
#pragma unroll
        for (int j = 0; j < CT; ++j) {
          o[j][2 * i] *= down;
          o[j][2 * i + 1] *= down;
        }
        m[i] = top[i];
      }
    }
    float2 minus[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float by = m[i] == -INFINITY ? 0.f : kWeightUp - m[i];
      minus[i] = make_float2(by, by);
    }
#pragma unroll
    for (int t = 0; t < KT; ++t) {
      uint32_t w[4];   // A operand: rows r, r + 8; tokens 2c, 2c + 1 and + 8
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float2 x = add2(y[2 * t + h][i], minus[i]);
          float2 p = make_float2(sm100::ex2_approx(x.x), sm100::ex2_approx(x.y));
          l[i] = add2(l[i], p);
          if constexpr (k8) p = mul2(p, scale[2 * t + h]);
          w[2 * h + i] = pack<M>(p.x, p.y);
        }
#pragma unroll
      for (int s4 = 0; s4 < VC; ++s4)
#pragma unroll
        for (int x = 0; x < VW; ++x) {
          if constexpr (k8) {
            // bytes of rows 2c and 2c + 1 (2c + 8 and 2c + 9) side by side, two columns a word
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const uint32_t order = half ? 0x7362 : 0x5140;
              const uint32_t lo = __byte_perm(v.w[t][0][s4][x], v.w[t][1][s4][x], order);
              const uint32_t hi = __byte_perm(v.w[t][2][s4][x], v.w[t][3][s4][x], order);
              const int j = 4 * x + 2 * half;
              mma<M>(o[j], w, e4m3x2(lo), e4m3x2(hi));
              mma<M>(o[j + 1], w, e4m3x2(lo >> 16), e4m3x2(hi >> 16));
            }
          } else {
            const int j = s4 * 8 + 2 * x;
            mma<M>(o[j], w, __byte_perm(v.w[t][0][s4][x], v.w[t][1][s4][x], 0x5410),
                   __byte_perm(v.w[t][2][s4][x], v.w[t][3][s4][x], 0x5410));
            mma<M>(o[j + 1], w, __byte_perm(v.w[t][0][s4][x], v.w[t][1][s4][x], 0x7632),
                   __byte_perm(v.w[t][2][s4][x], v.w[t][3][s4][x], 0x7632));
          }
        }
    }
  }
};

template <int DP>
struct Shared {
  uint4 q[8 * 32];
  float m[kWarps][kRows], l[kWarps][kRows], o[kWarps][kRows][DP + 4];
  int64_t sums[kWarps];
  int64_t total, before;
  int sequence;
};

// Tiles [first, last) of a warp's stride of the head, and their sums joined over the CTA's warps in shared memory: o[0], m[0], l[0].
template <typename T, bool k8, int DP>
__device__ __forceinline__ void attend(const Params &p, Shared<DP> &sh, int b, int g, int row_tile, int n, int64_t unit0, int64_t unit1) {
  using W = Tile<T, k8, DP>;
  const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
  const int head0 = g * p.group + row_tile * kRows, rows = min(kRows, p.group - row_tile * kRows);
  W w;
  w.load_q(p, sh.q, warp == 0, b, head0, rows, lane);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 2; ++i) w.m[i] = -INFINITY, w.l[i] = make_float2(0.f, 0.f);
#pragma unroll
  for (int j = 0; j < W::CT; ++j) w.o[j][0] = w.o[j][1] = w.o[j][2] = w.o[j][3] = 0.f;
  constexpr int64_t kStep = W::TT * kWarps;
  const int64_t first = unit0 * kStep + warp * W::TT, last = unit1 * kStep;
  // a lane's token's scales; a value's exponent below -80 does not set the reference, so that the sum of weights (2^(80 + 10) of up to 2^31
  // tokens) stays finite
  float ks = 1.f, vs = 1.f, e = 0.f;
  auto scales = [&](uint32_t row, uint32_t &kb, uint32_t &vb) {
    kb = vb = 127;
    if (k8 && row < kBad) kb = __ldg(p.c.k_scales + row), vb = __ldg(p.c.v_scales + row);
  };
  auto all_there = [&](uint32_t row) { return p.exact && __all_sync(0xffffffffu, row < kBad || lane >= W::TT); };
  uint32_t now = W::resolve(p, b, g, n, first, lane), next = W::resolve(p, b, g, last > first + kStep ? n : 0, first + kStep, lane);
  uint32_t kb, vb;
  bool all = all_there(now);
  w.load_k(p, now, all, lane);
  typename W::Values even, odd;
  w.load_v(p, even, now, all, lane);
  scales(now, kb, vb);
  int64_t at = first;
  auto tile = [&](const typename W::Values &v, typename W::Values &coming) {
    float s[W::NT][4];
    w.scores(s, sh.q, lane);
    if constexpr (k8) {
      ks = two_to(kb), vs = two_to(vb);
      e = fmaxf((float)(int)vb - 127.f, -80.f);
    }
    const bool next_all = all_there(next);
    w.load_k(p, next, next_all, lane);
    w.load_v(p, coming, next, next_all, lane);
    scales(next, kb, vb);
    const uint32_t after = W::resolve(p, b, g, at + 2 * kStep < last ? n : 0, at + 2 * kStep, lane);
    w.add(s, v, now, all, ks, vs, e, lane);
    now = next, next = after, all = next_all;
    at += kStep;
  };
  while (at < last) {
    tile(even, odd);
    if constexpr (k8) {
      // a copy, which waits for the values: twice the code instead costs more (the 64 sequences: 140 -> 184 us), as it leaves the
      // instruction cache
      even = odd;
    } else {
      if (at >= last) break;
      tile(odd, even);   // the long sequence: 205 -> 156 us
    }
  }
  const int r = lane / 4, c = lane % 4;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float l = w.l[i].x + w.l[i].y;
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    if (c == 0) sh.m[warp][r + 8 * i] = w.m[i], sh.l[warp][r + 8 * i] = l;
#pragma unroll
    for (int j = 0; j < W::CT; ++j)
#pragma unroll
      for (int x = 0; x < 2; ++x)
        if (r + 8 * i < rows) sh.o[warp][r + 8 * i][W::column(j, 2 * c + x)] = w.o[j][2 * i + x];
  }
  __syncthreads();
  for (int e = threadIdx.x; e < rows * DP; e += kWarps * 32) {
    const int row = e / DP, col = e % DP;
    float top = sh.m[0][row];
#pragma unroll
    for (int i = 1; i < kWarps; ++i) top = fmaxf(top, sh.m[i][row]);
    const float ref = top == -INFINITY ? 0.f : top;
    float o = 0.f, l = 0.f;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
      const float f = sm100::ex2_approx(sh.m[i][row] - ref);   // a warp without tokens: 2^-inf = 0
      o += f * sh.o[i][row][col];
      l += f * sh.l[i][row];
    }
    sh.o[0][row][col] = o;
    if (col == 0) sh.o[0][row][DP] = top, sh.o[0][row][DP + 1] = l;
  }
  __syncthreads();
}

template <typename T, int DP>
__device__ __forceinline__ void finish(const Params &p, Shared<DP> &sh, int b, int g, int row_tile, bool empty) {
  const int head0 = g * p.group + row_tile * kRows, rows = min(kRows, p.group - row_tile * kRows);
  T *out = static_cast<T *>(p.out) + ((int64_t)b * p.heads + head0) * p.c.dim;
  for (int e = threadIdx.x; e < rows * p.c.dim; e += kWarps * 32) {
    const int row = e / p.c.dim, col = e - row * p.c.dim;
    out[e] = from_f32<T>(empty ? 0.f : sh.o[0][row][col] / sh.o[0][row][DP + 1]);
  }
}

// Tokens of a sequence; one past its table's places, where the length says more, stands for all of those.
__device__ __forceinline__ int length_of(const Params &p, int b) {
  return (int)min((int64_t)max(p.lengths[b], 0), (int64_t)p.c.table_width * p.c.page_size + 1);
}
// The line is cut for as many CTAs as it has units, at most p.ctas: each of those has one unit or more.
__device__ __forceinline__ int64_t line_ctas(const Params &p, int64_t total) { return min((int64_t)p.ctas, total); }
__device__ __forceinline__ int64_t line_begin(const Params &p, int64_t total, int cta) {
  const int64_t n = line_ctas(p, total);
  return n ? total * min((int64_t)cta, n) / n : 0;
}

// The line of units: how many in all, and where a CTA's stretch begins: the sequence there and the units before that. Every
// thread sums a run of sequences.
template <int DP>
__device__ __forceinline__ void find(const Params &p, Shared<DP> &sh, int unit, int heads, int cta) {
  const int per = (p.c.sequences + kWarps * 32 - 1) / (kWarps * 32), b0 = threadIdx.x * per, b1 = min(b0 + per, p.c.sequences);
  int64_t mine = 0;
  for (int b = b0; b < b1; ++b) mine += (length_of(p, b) + (int64_t)unit - 1) / unit;
  mine *= heads;
  int64_t upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t v = __shfl_up_sync(0xffffffffu, upto, o);
    if ((int)(threadIdx.x & 31) >= o) upto += v;
  }
  if ((threadIdx.x & 31) == 31) sh.sums[threadIdx.x / 32] = upto;
  __syncthreads();
  int64_t total = 0, before = 0;
#pragma unroll
  for (int i = 0; i < kWarps; ++i) {
    if (i < (int)threadIdx.x / 32) before += sh.sums[i];
    total += sh.sums[i];
  }
  before += upto - mine;
  const int64_t at = line_begin(p, total, cta);
  if (threadIdx.x == 0) sh.total = total;
  if (at >= before && at < before + mine) {
    int b = b0;
    for (;; ++b) {
      const int64_t n = (length_of(p, b) + (int64_t)unit - 1) / unit * heads;
      if (at < before + n) break;
      before += n;
    }
    sh.sequence = b;
    sh.before = before;
  }
  __syncthreads();
}

template <typename T, bool k8, int DP>
__global__ void __launch_bounds__(kWarps * 32, per_sm(k8, DP)) paged_kernel(const __grid_constant__ Params p) {
  extern __shared__ __align__(16) uint8_t raw[];
  Shared<DP> &sh = *reinterpret_cast<Shared<DP> *>(raw);
  constexpr int unit = Tile<T, k8, DP>::TT * kWarps;
  const int heads = p.c.kv_heads * p.row_tiles;
  if (p.ctas == 0) {
    const int b = blockIdx.x / heads, h = blockIdx.x % heads, n = length_of(p, b);
    if (n > 0) attend<T, k8, DP>(p, sh, b, h / p.row_tiles, h % p.row_tiles, n, 0, (n + (int64_t)unit - 1) / unit);
    finish<T, DP>(p, sh, b, h / p.row_tiles, h % p.row_tiles, n == 0);
    return;
  }
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  find<DP>(p, sh, unit, heads, blockIdx.x);
  int64_t at = line_begin(p, sh.total, blockIdx.x);
  const int64_t end = line_begin(p, sh.total, blockIdx.x + 1);
  int64_t before = sh.before;
  for (int b = sh.sequence; at < end;) {
    const int n = length_of(p, b);
    const int64_t units = (n + (int64_t)unit - 1) / unit;
    if (at >= before + units * heads) {   // the next sequence
      before += units * heads;
      ++b;
      continue;
    }
    const int h = (int)((at - before) / units), g = h / p.row_tiles, row_tile = h % p.row_tiles;
    const int64_t u0 = at - before - h * units, u1 = min(units, u0 + end - at);
    attend<T, k8, DP>(p, sh, b, g, row_tile, n, u0, u1);
    if (u0 == 0 && u1 == units) {
      finish<T, DP>(p, sh, b, g, row_tile, false);
    } else {
      const int rows = min(kRows, p.group - row_tile * kRows), dim = p.c.dim;
      float *part = p.parts + (int64_t)(2 * blockIdx.x + (u0 == 0)) * p.part_rows * (dim + 2);
      for (int e = threadIdx.x; e < rows * (dim + 2); e += kWarps * 32) {
        const int row = e / (dim + 2), col = e - row * (dim + 2);
        part[e] = sh.o[0][row][col < dim ? col : DP + col - dim];
      }
    }
    __syncthreads();
    at += u1 - u0;
  }
}

// The pieces of one query head (a block), added in the order of the line; empty sequences get 0.
constexpr int kMaxPieces = 1024;
template <typename T>
__global__ void __launch_bounds__(kWarps * 32) join_kernel(const __grid_constant__ Params p, int unit) {
  __shared__ int64_t sums[2][kWarps];
  __shared__ float weight[kMaxPieces], reduced[2][kWarps];
  const int b = blockIdx.x / p.heads, head = blockIdx.x % p.heads, g = head / p.group, in_group = head % p.group;
  const int heads = p.c.kv_heads * p.row_tiles, h = g * p.row_tiles + in_group / kRows, row = in_group % kRows, dim = p.c.dim;
  const int warp = threadIdx.x / 32;
  // the units before sequence b, and all of them
  int64_t before = 0, total = 0;
  for (int i = threadIdx.x; i < p.c.sequences; i += kWarps * 32) {
    const int64_t n = (length_of(p, i) + (int64_t)unit - 1) / unit;
    total += n;
    if (i < b) before += n;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    before += __shfl_xor_sync(0xffffffffu, before, o);
    total += __shfl_xor_sync(0xffffffffu, total, o);
  }
  if ((threadIdx.x & 31) == 0) sums[0][warp] = before, sums[1][warp] = total;
  __syncthreads();
  before = total = 0;
#pragma unroll
  for (int i = 0; i < kWarps; ++i) before += sums[0][i], total += sums[1][i];
  const int64_t units = (length_of(p, b) + (int64_t)unit - 1) / unit;
  T *const out = static_cast<T *>(p.out) + ((int64_t)b * p.heads + head) * dim;
  // in every block: this kernel's end stands for the first one's too
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (units == 0) {
    for (int col = threadIdx.x; col < dim; col += kWarps * 32) out[col] = from_f32<T>(0.f);
    return;
  }
  before = before * heads + h * units;
  total *= heads;
  // CTA i of n has the places from total * i / n on
  const int64_t n = line_ctas(p, total);
  const int first = (int)(((before + 1) * n - 1) / total), pieces = (int)(((before + units) * n - 1) / total) - first + 1;
  if (pieces == 1) return;
  const int64_t size = (int64_t)p.part_rows * (dim + 2);
  auto part = [&](int i) { return p.parts + (2 * (first + i) + (i == 0)) * size + (int64_t)row * (dim + 2); };
  auto all = [&](float v, bool largest, int which) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float u = __shfl_xor_sync(0xffffffffu, v, o);
      v = largest ? fmaxf(v, u) : v + u;
    }
    if ((threadIdx.x & 31) == 0) reduced[which][warp] = v;
    __syncthreads();
    v = reduced[which][0];
#pragma unroll
    for (int i = 1; i < kWarps; ++i) v = largest ? fmaxf(v, reduced[which][i]) : v + reduced[which][i];
    return v;
  };
  float top = -INFINITY, l = 0.f;
  for (int i = threadIdx.x; i < pieces; i += kWarps * 32) top = fmaxf(top, weight[i] = part(i)[dim]);
  top = all(top, true, 0);
  const float ref = top == -INFINITY ? 0.f : top;
  for (int i = threadIdx.x; i < pieces; i += kWarps * 32) {
    weight[i] = sm100::ex2_approx(weight[i] - ref);
    l += weight[i] * part(i)[dim + 1];
  }
  l = all(l, false, 1);   // and the weights are there
  for (int col = threadIdx.x; col < dim; col += kWarps * 32) {
    float o = 0.f;
#pragma unroll 8
    for (int i = 0; i < pieces; ++i) o = fmaf(weight[i], part(i)[col], o);
    out[col] = from_f32<T>(o / l);
  }
}

// ------------------------------------------------------------------------------- host
int padded(int dim) { return dim <= 64 ? 64 : 128; }
int unit_of(const p3d_cache &c) { return (padded(c.dim) == 128 && c.dtype != P3D_E4M3 ? 16 : 32) * kWarps; }

struct Plan {
  int row_tiles, part_rows, ctas;
};
int plan(const p3d_cache *c, int heads, Plan *out) {
  const int group = heads / c->kv_heads;
  out->row_tiles = (group + kRows - 1) / kRows;
  out->part_rows = std::min(group, kRows);
  DeviceInfo info;
  if (int st = device_info(&info)) return st;
  // as far as the tables reach: a few units a head are done by one CTA, which costs less than a second kernel
  const int64_t unit = unit_of(*c), most = ((int64_t)c->table_width * c->page_size + unit - 1) / unit;
  const int64_t all = most * c->sequences * c->kv_heads * out->row_tiles;
  out->ctas = most <= 4 ? 0 : (int)std::min<int64_t>(std::min<int64_t>(all, kMaxPieces), (int64_t)info.sm_count * per_sm(c->dtype == P3D_E4M3, padded(c->dim)));
  return P3D_OK;
}

template <typename T, bool k8, int DP>
int launch(const Params &p, cudaStream_t s) {
  static size_t seen[kMaxDevices] = {};
  const size_t bytes = sizeof(Shared<DP>);
  if (int st = smem_optin(paged_kernel<T, k8, DP>, bytes, seen)) return st;
  const int heads = p.c.kv_heads * p.row_tiles;
  paged_kernel<T, k8, DP><<<p.ctas ? p.ctas : p.c.sequences * heads, kWarps * 32, bytes, s>>>(p);
  P3D_LAUNCH_CHECK();
  if (!p.ctas) return P3D_OK;
  // starts while the first kernel still runs, and waits in the kernel for what it wrote
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.c.sequences * p.heads);
  cfg.blockDim = dim3(kWarps * 32);
  cfg.stream = s;
  cudaLaunchAttribute attr = {};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  P3D_CUDA_TRY(cudaLaunchKernelEx(&cfg, join_kernel<T>, p, (int)(Tile<T, k8, DP>::TT * kWarps)));
  return P3D_OK;
}

template <typename T>
int launch_t(const Params &p, cudaStream_t s) {
  const bool k8 = p.c.dtype == P3D_E4M3;
  if (padded(p.c.dim) == 64) return k8 ? launch<T, true, 64>(p, s) : launch<T, false, 64>(p, s);
  return k8 ? launch<T, true, 128>(p, s) : launch<T, false, 128>(p, s);
}

int check(const p3d_cache *c, int heads) {
  if (int st = cache::check(c, "p3d_paged_attention")) return st;
  P3D_CHECK_ARG(c->dim <= 128, "p3d_paged_attention: head dim up to 128");
  P3D_CHECK_ARG(heads >= 1 && heads % c->kv_heads == 0 && heads <= 65535,
                "p3d_paged_attention: query heads must be a multiple of the cache's heads");
  if ((__int128)c->pages * c->kv_heads * c->page_size >= (int64_t)kBad || (int64_t)c->sequences * heads >= (1ll << 31))
    return fail(P3D_ERR_UNSUPPORTED, "p3d_paged_attention: at most 2^32 - 3 rows in the pages and 2^31 - 1 queries");
  return P3D_OK;
}

}  // namespace

int take_paged_errors(unsigned *flags) {
  unsigned v = 0, zero = 0;
  P3D_CUDA_TRY(cudaMemcpyFromSymbol(&v, g_paged_errors, sizeof(v)));
  P3D_CUDA_TRY(cudaMemcpyToSymbol(g_paged_errors, &zero, sizeof(zero)));
  *flags |= v;
  return P3D_OK;
}

}  // namespace p3d

using namespace p3d;

extern "C" {

size_t p3d_paged_attention_workspace(const p3d_cache *c, int heads) {
  Plan pl;
  if (check(c, heads) != P3D_OK || c->sequences == 0 || plan(c, heads, &pl) != P3D_OK) return 0;
  return sizeof(float) * 2 * (size_t)pl.ctas * pl.part_rows * (c->dim + 2);
}

int p3d_paged_attention(const p3d_cache *c, const void *q, const int64_t q_stride[2], int dtype, int heads,
                        const int32_t *lengths, float scale, void *out, void *workspace, size_t workspace_bytes,
                        void *stream) {
  if (int st = check(c, heads)) return st;
  P3D_CHECK_ARG(dtype == P3D_F16 || dtype == P3D_BF16, "p3d_paged_attention: f16 or bf16 queries only");
  P3D_CHECK_ARG(c->dtype == dtype || c->dtype == P3D_E4M3, "p3d_paged_attention: queries must be of the cache's dtype");
  P3D_CHECK_ARG(isfinite(scale) && scale > 0, "p3d_paged_attention: scale must be finite and positive");
  if (c->sequences == 0) return P3D_OK;
  P3D_CHECK_ARG(q && q_stride && lengths && out, "p3d_paged_attention: null argument");
  P3D_CHECK_ARG((uintptr_t)q % 16 == 0 && q_stride[0] % 8 == 0 && q_stride[1] % 8 == 0,
                "p3d_paged_attention: queries must be 16-byte aligned");
  Plan pl;
  if (int st = plan(c, heads, &pl)) return st;
  const size_t need = sizeof(float) * 2 * (size_t)pl.ctas * pl.part_rows * (c->dim + 2);
  if (need && (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16))
    return fail(P3D_ERR_WORKSPACE, "p3d_paged_attention: aligned workspace of %zu bytes needed", need);
  Params p = {};
  p.c = *c;
  p.q = q, p.q_token = q_stride[0], p.q_head = q_stride[1], p.out = out, p.lengths = lengths;
  p.scale = scale * 1.4426950408889634f;
  p.heads = heads, p.group = heads / c->kv_heads, p.row_tiles = pl.row_tiles, p.ctas = pl.ctas, p.part_rows = pl.part_rows;
  p.wide = c->dtype != P3D_E4M3 || c->dim % 16 == 0;
  p.exact = c->dim == padded(c->dim);
  p.parts = static_cast<float *>(workspace);
  return dtype == P3D_F16 ? launch_t<__half>(p, (cudaStream_t)stream) : launch_t<__nv_bfloat16>(p, (cudaStream_t)stream);
}

}  // extern "C"
