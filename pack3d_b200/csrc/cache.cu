// Keys and values written into pages as they are or in 8 bits, and read back.
//
//     8 bits: e the smallest integer from -126 on with amax / 2^e <= 448 over a token's dim values of one head, e4m3(x / 2^e) and a
//     byte e + 127
//
// The scale is a power of two, so scaling is exact and e4m3's rounding the only one; it belongs to one token and head, so that a
// token is written once and its neighbours in the page never change.
//
// Bound by HBM: each value is read once and written once. A row (token, head, key or value) is S = dim / 8 lanes (up to a power
// of two), and a pass is 32 / S rows. What page a token goes to is a chain of loads (offsets, start, table), so a warp takes up to
// 32 consecutive tokens, each lane follows the chain for one of them, and the places are handed round by shuffles. Tokens and
// heads are cut so that the warps that the device holds have about one item each.
//
// A kernel reads in the order in which its input lies: append takes the heads of one token (four passes in flight), read takes
// consecutive tokens of one head, which are neighbours in a page (eight). With 8 heads of 128
// between bf16 and 8 bits, append takes 54 us for 40,001 tokens, 4.6 TB/s (by tokens of one head 107), and read 65 us for 50,001,
// 4.7 TB/s (by heads of one token 83). What is left in both is the wait for loads: 64 registers leave an SM 32 warps.
// They are too few for eight passes of some types: from e4m3 or 16 bits read spills 28 to 116 bytes a thread, from fp32 pages 540 to 624, and
// append of fp32 rows 64 (none of these is measured but e4m3 to bf16).
#include "cache.cuh"

#include <cuda_fp8.h>

#include <algorithm>

#include "fp8_quant.cuh"
#include "kernels.cuh"

namespace p3d {
namespace {

__device__ unsigned g_cache_errors = 0;

constexpr int kWarps = 8, kAppendPasses = 4;
constexpr int read_passes(int s) { return s < 8 ? s : 8; }

struct Params {
  p3d_cache c;
  const void *in[2];
  int64_t token_stride[2], head_stride[2];
  void *out[2];
  const int32_t *starts, *offsets;
  int rows;          // packed rows
  int run;           // tokens of a warp's item
  int group, groups; // its rows of each of them, and how many such groups the 2 * kv_heads rows make
  int shift;         // log2 of the lanes of a row
};

// What a lane knows of one token: its place, or why it has none.
enum { kOutside = -1, kBad = -2 };
__device__ __forceinline__ cache::Place find(const Params &p, int t) {
  cache::Place place = {kOutside, 0};
  if (t >= p.rows) return place;
  const int b = cache::sequence_of(p.offsets, p.c.sequences, p.rows, t);
  if (t >= cache::offset_at(p.offsets, b + 1, p.rows)) return place;
  place = cache::place_of(p.c, b, (p.starts ? p.starts[b] : 0) + (int64_t)(t - cache::offset_at(p.offsets, b, p.rows)));
  if (place.page < 0) {
    place.page = kBad;
    atomicOr(&g_cache_errors, cache::kErrPage);
  }
  return place;
}

// S: lanes of a row.
template <typename T, bool k8, int S>
__global__ void __launch_bounds__(kWarps * 32, 4) append_kernel(const __grid_constant__ Params p) {
  constexpr int U = kAppendPasses, kPerPass = 32 / S;
  const int lane = threadIdx.x & 31, col = lane % S * 8, rows = 2 * p.c.kv_heads;
  const int64_t items = (int64_t)((p.rows + p.run - 1) / p.run) * p.groups;
  for (int64_t item = (int64_t)blockIdx.x * kWarps + threadIdx.x / 32; item < items; item += (int64_t)gridDim.x * kWarps) {
    const int run = (int)(item / p.groups), t0 = run * p.run;
    const int first = (int)(item - (int64_t)run * p.groups) * U * kPerPass + lane / S;
    const cache::Place mine = find(p, lane < p.run ? t0 + lane : p.rows);
    // a lane's rows of every token of the run: the same heads
    const T *in[U];
    int64_t to[U];   // row of the pages, less the page and the place in it
    bool on[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int r = first + u * kPerPass, which = r >= p.c.kv_heads, head = r - which * p.c.kv_heads;
      on[u] = r < rows && col < p.c.dim;
      to[u] = (int64_t)head * p.c.page_size;
      in[u] = static_cast<const T *>(which ? p.in[1] : p.in[0]) + (int64_t)t0 * (which ? p.token_stride[1] : p.token_stride[0]) +
              head * (which ? p.head_stride[1] : p.head_stride[0]) + col;
    }
    for (int i = 0; i < p.run && t0 + i < p.rows; ++i) {
      const int page = __shfl_sync(0xffffffffu, mine.page, i), at = __shfl_sync(0xffffffffu, mine.row, i);
      quant::Raw<T> raw[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        raw[u] = quant::load8<T, true>(in[u], 0, on[u] && page >= 0 ? 8 : 0);
        in[u] += first + u * kPerPass >= p.c.kv_heads ? p.token_stride[1] : p.token_stride[0];
      }
      if (page < 0) continue;
      const int64_t place = (int64_t)page * p.c.kv_heads * p.c.page_size + at;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const bool values = first + u * kPerPass >= p.c.kv_heads;
        if constexpr (k8) {
          uint32_t m = quant::largest8<T>(raw[u]);
#pragma unroll
          for (int o = S / 2; o > 0; o >>= 1) m = quant::larger<T>(m, __shfl_xor_sync(0xffffffffu, m, o));
          const bool odd = __any_sync(0xffffffffu, quant::infinite<T>(m));   // infinities or NaN among the warp's rows
          if (odd) {
            m = quant::finite_largest8<T>(raw[u]);
#pragma unroll
            for (int o = S / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
          } else {
            m = quant::widest<T>(m);
          }
          const uint32_t byte = m ? quant::scale_byte(m) : 1u;
          const float inv = quant::inverse_scale(byte);
          const uint2 w = odd ? quant::quantize8<true, T>(raw[u], inv) : quant::quantize8<false, T>(raw[u], inv);
          if (on[u]) {
            *reinterpret_cast<uint2 *>(static_cast<uint8_t *>(values ? p.c.v : p.c.k) + (place + to[u]) * p.c.dim + col) = w;
            if (col == 0) (values ? p.c.v_scales : p.c.k_scales)[place + to[u]] = (uint8_t)byte;
          }
        } else if (on[u]) {
          T *dst = static_cast<T *>(values ? p.c.v : p.c.k) + (place + to[u]) * p.c.dim + col;
#pragma unroll
          for (int q = 0; q < quant::Raw<T>::kWords / 4; ++q)
            reinterpret_cast<uint4 *>(dst)[q] =
                make_uint4(raw[u].w[4 * q], raw[u].w[4 * q + 1], raw[u].w[4 * q + 2], raw[u].w[4 * q + 3]);
        }
      }
    }
  }
}

struct E4m3 {};
template <typename C> struct Stored { using Raw = quant::Raw<C>; };
template <> struct Stored<E4m3> {
  struct Raw { uint2 w; };
};

template <typename C, typename T, int S>
__global__ void __launch_bounds__(kWarps * 32, 4) read_kernel(const __grid_constant__ Params p) {
  constexpr bool k8 = std::is_same<C, E4m3>::value;
  constexpr int U = read_passes(S), kTokens = 32 / S;
  const int lane = threadIdx.x & 31, col = lane % S * 8;
  const bool on = col < p.c.dim;
  const int64_t items = (int64_t)((p.rows + p.run - 1) / p.run) * p.groups;
  for (int64_t item = (int64_t)blockIdx.x * kWarps + threadIdx.x / 32; item < items; item += (int64_t)gridDim.x * kWarps) {
    const int run = (int)(item / p.groups), t0 = run * p.run, n = min(p.run, p.rows - t0), r0 = (int)(item - (int64_t)run * p.groups) * p.group;
    const cache::Place place = find(p, lane < n ? t0 + lane : p.rows);
    // the token's row of the pages' first head, or why it has none
    const int64_t mine = place.page < 0 ? place.page : (int64_t)place.page * p.c.kv_heads * p.c.page_size + place.row;
    for (int r = r0; r < min(r0 + p.group, 2 * p.c.kv_heads); ++r) {
      const bool values = r >= p.c.kv_heads;
      const int head = values ? r - p.c.kv_heads : r;
      using Element = std::conditional_t<k8, uint8_t, C>;
      const Element *const from = static_cast<const Element *>(values ? p.c.v : p.c.k) + (int64_t)head * p.c.page_size * p.c.dim + col;
      const uint8_t *const scales = (values ? p.c.v_scales : p.c.k_scales) + (int64_t)head * p.c.page_size;
      T *dst = static_cast<T *>(values ? p.out[1] : p.out[0]) + ((int64_t)(t0 + lane / S) * p.c.kv_heads + head) * p.c.dim + col;
      const int64_t step = (int64_t)kTokens * p.c.kv_heads * p.c.dim;
      for (int i0 = 0; i0 < n; i0 += U * kTokens) {
        typename Stored<C>::Raw raw[U];
        uint32_t byte[U];
        int state[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int i = i0 + u * kTokens + lane / S;
          const int64_t at = __shfl_sync(0xffffffffu, mine, i & 31);
          const bool there = at >= 0 && i < n && on;
          state[u] = at < 0 ? (int)at : 0;
          if constexpr (k8) {
            raw[u].w = make_uint2(0, 0);
            byte[u] = 127;
            if (there) {
              raw[u].w = *reinterpret_cast<const uint2 *>(from + at * p.c.dim);
              byte[u] = scales[at];
            }
          } else {
            raw[u] = quant::load8<C, true>(from + (there ? at : 0) * p.c.dim, 0, there ? 8 : 0);
          }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int i = i0 + u * kTokens + lane / S;
          T *const to = dst;
          dst += step;
          if (i >= n || !on) continue;
          float v[8];
          if constexpr (k8) {
            const float scale = __uint_as_float(byte[u] ? byte[u] << 23 : 0x400000u);   // 2^(byte - 127); byte 0 is 2^-127
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const uint32_t w = q < 2 ? raw[u].w.x : raw[u].w.y;
              const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> 16 * (q % 2)), __NV_E4M3);
              const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&h));
              v[2 * q] = f.x * scale;
              v[2 * q + 1] = f.y * scale;
            }
          } else {
#pragma unroll
            for (int q = 0; q < 8; ++q) v[q] = quant::value(raw[u], q);
          }
          if (state[u] == kBad)
#pragma unroll
            for (int q = 0; q < 8; ++q) v[q] = __uint_as_float(0x7fffffffu);
          alignas(16) T packed[8];
#pragma unroll
          for (int q = 0; q < 8; ++q) packed[q] = from_f32<T>(v[q]);
#pragma unroll
          for (int q = 0; q < (int)sizeof(T) / 2; ++q)
            reinterpret_cast<uint4 *>(to)[q] = reinterpret_cast<const uint4 *>(packed)[q];
        }
      }
    }
  }
}

// Cuts tokens and rows into items. Append: the rows of four passes each, and as many tokens as leave the warps that the device
// holds one item each. Read: one pass of tokens and one row, and while there are more items than warps, more tokens up to 32,
// then more rows.
int fill(Params *p, const p3d_cache *c, int64_t rows, bool read) {
  p->c = *c;
  p->rows = (int)rows;
  p->shift = 0;
  while (8 << p->shift < c->dim) ++p->shift;
  DeviceInfo info;
  if (int st = device_info(&info)) return st;
  const int64_t warps = (int64_t)info.sm_count * 32, heads = 2 * (int64_t)c->kv_heads;
  const int per_pass = 32 >> p->shift;
  if (read) {
    p->run = per_pass;
    while (p->run < 32 && (rows + p->run - 1) / p->run * heads > warps) p->run *= 2;
    const int64_t runs = (rows + p->run - 1) / p->run;
    p->group = (int)std::min(heads, std::max<int64_t>(1, (runs * heads + warps - 1) / warps));
  } else {
    p->group = per_pass * kAppendPasses;
  }
  p->groups = (int)((heads + p->group - 1) / p->group);
  if (!read) p->run = (int)std::min<int64_t>(32, std::max<int64_t>(1, (rows * p->groups + warps - 1) / warps));
  return P3D_OK;
}
int blocks_of(const Params &p) {
  const int64_t items = (int64_t)((p.rows + p.run - 1) / p.run) * p.groups;
  return (int)std::min<int64_t>((items + kWarps - 1) / kWarps, 1 << 20);
}
template <typename F>
void by_lanes(int shift, F go) {
  switch (shift) {
    case 0: return go(std::integral_constant<int, 1>());
    case 1: return go(std::integral_constant<int, 2>());
    case 2: return go(std::integral_constant<int, 4>());
    case 3: return go(std::integral_constant<int, 8>());
    case 4: return go(std::integral_constant<int, 16>());
    default: return go(std::integral_constant<int, 32>());
  }
}

bool aligned(const void *q) { return (uintptr_t)q % 16 == 0; }

}  // namespace

namespace cache {

int check(const p3d_cache *c, const char *what) {
  P3D_CHECK_ARG(c != nullptr, "%s: null cache", what);
  P3D_CHECK_ARG(dtype_ok(c->dtype) || c->dtype == P3D_E4M3, "%s: unknown cache dtype %d", what, c->dtype);
  P3D_CHECK_ARG(c->dim >= 8 && c->dim <= 256 && c->dim % 8 == 0, "%s: head dim must be a multiple of 8 up to 256, got %d", what,
                c->dim);
  P3D_CHECK_ARG(c->kv_heads >= 1 && c->kv_heads <= 65535 && c->page_size >= 1 && c->pages >= 1,
                "%s: pages, heads and page size must be positive", what);
  P3D_CHECK_ARG(c->pages < (1ll << 31) && c->page_size < (1 << 30), "%s: at most 2^31 - 1 pages of 2^30 - 1 tokens", what);
  P3D_CHECK_ARG(c->sequences >= 0 && c->table_width >= 0, "%s: sequences and table width must not be negative", what);
  P3D_CHECK_ARG((int64_t)c->table_width * c->page_size < (1ll << 31), "%s: a sequence has at most 2^31 - 1 places", what);
  P3D_CHECK_ARG(c->k && c->v && aligned(c->k) && aligned(c->v), "%s: pages must be given and 16-byte aligned", what);
  P3D_CHECK_ARG((c->k_scales && c->v_scales) || c->dtype != P3D_E4M3, "%s: 8-bit pages need their scales", what);
  P3D_CHECK_ARG(c->table || !c->sequences || !c->table_width, "%s: null page table", what);
  return P3D_OK;
}

}  // namespace cache

int take_cache_errors(unsigned *flags) {
  unsigned v = 0, zero = 0;
  P3D_CUDA_TRY(cudaMemcpyFromSymbol(&v, g_cache_errors, sizeof(v)));
  P3D_CUDA_TRY(cudaMemcpyToSymbol(g_cache_errors, &zero, sizeof(zero)));
  *flags |= v;
  return P3D_OK;
}

}  // namespace p3d

using namespace p3d;

extern "C" {

int p3d_cache_append(const p3d_cache *c, const void *new_k, const int64_t k_stride[2], const void *new_v,
                     const int64_t v_stride[2], int dtype, int64_t rows, const int32_t *starts, const int32_t *offsets,
                     void *stream) {
  if (int st = cache::check(c, "p3d_cache_append")) return st;
  P3D_CHECK_ARG(dtype_ok(dtype) && (c->dtype == P3D_E4M3 || c->dtype == dtype),
                "p3d_cache_append: new rows must be of the cache's dtype, or fp32, f16 or bf16 for an 8-bit cache");
  P3D_CHECK_ARG(rows >= 0 && rows < (1ll << 31) - 64, "p3d_cache_append: row count out of range");
  if (rows == 0 || c->sequences == 0) return P3D_OK;
  P3D_CHECK_ARG(new_k && new_v && k_stride && v_stride && starts && offsets, "p3d_cache_append: null input");
  const int unit = 16 / dtype_size(dtype);
  P3D_CHECK_ARG(aligned(new_k) && aligned(new_v) && k_stride[0] % unit == 0 && k_stride[1] % unit == 0 &&
                    v_stride[0] % unit == 0 && v_stride[1] % unit == 0,
                "p3d_cache_append: rows must be 16-byte aligned");
  Params p = {};
  if (int st = fill(&p, c, rows, false)) return st;
  p.in[0] = new_k, p.in[1] = new_v;
  for (int i = 0; i < 2; ++i) {
    p.token_stride[i] = (i ? v_stride : k_stride)[0];
    p.head_stride[i] = (i ? v_stride : k_stride)[1];
  }
  p.starts = starts, p.offsets = offsets;
  const int blocks = blocks_of(p);
  const cudaStream_t s = (cudaStream_t)stream;
  auto go = [&](auto type) {
    using T = decltype(type);
    by_lanes(p.shift, [&](auto lanes) {
      constexpr int S = decltype(lanes)::value;
      if (c->dtype == P3D_E4M3) append_kernel<T, true, S><<<blocks, kWarps * 32, 0, s>>>(p);
      else append_kernel<T, false, S><<<blocks, kWarps * 32, 0, s>>>(p);
    });
  };
  dtype == P3D_F32 ? go(float()) : dtype == P3D_F16 ? go(__half()) : go(__nv_bfloat16());
  P3D_LAUNCH_CHECK();
  return P3D_OK;
}

int p3d_cache_read(const p3d_cache *c, const int32_t *starts, const int32_t *offsets, int64_t rows, void *out_k, void *out_v,
                   int dtype, void *stream) {
  if (int st = cache::check(c, "p3d_cache_read")) return st;
  P3D_CHECK_ARG(dtype_ok(dtype), "p3d_cache_read: unknown dtype %d", dtype);
  P3D_CHECK_ARG(rows >= 0 && rows < (1ll << 31) - 64, "p3d_cache_read: row count out of range");
  if (rows == 0) return P3D_OK;
  P3D_CHECK_ARG(c->sequences >= 1, "p3d_cache_read: no sequences");
  P3D_CHECK_ARG(out_k && out_v && offsets, "p3d_cache_read: null argument");
  P3D_CHECK_ARG(aligned(out_k) && aligned(out_v), "p3d_cache_read: outputs must be 16-byte aligned");
  Params p = {};
  if (int st = fill(&p, c, rows, true)) return st;
  p.out[0] = out_k, p.out[1] = out_v;
  p.starts = starts, p.offsets = offsets;
  const int blocks = blocks_of(p);
  const cudaStream_t s = (cudaStream_t)stream;
  auto go = [&](auto type) {
    using T = decltype(type);
    by_lanes(p.shift, [&](auto lanes) {
      constexpr int S = decltype(lanes)::value;
      switch (c->dtype) {
        case P3D_F32: read_kernel<float, T, S><<<blocks, kWarps * 32, 0, s>>>(p); break;
        case P3D_F16: read_kernel<__half, T, S><<<blocks, kWarps * 32, 0, s>>>(p); break;
        case P3D_BF16: read_kernel<__nv_bfloat16, T, S><<<blocks, kWarps * 32, 0, s>>>(p); break;
        default: read_kernel<E4m3, T, S><<<blocks, kWarps * 32, 0, s>>>(p);
      }
    });
  };
  dtype == P3D_F32 ? go(float()) : dtype == P3D_F16 ? go(__half()) : go(__nv_bfloat16());
  P3D_LAUNCH_CHECK();
  return P3D_OK;
}

}  // extern "C"
