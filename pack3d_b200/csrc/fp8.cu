// e4m3 values with one power-of-two scale for each block of 128: the quantiser.
//
// A block's exponent e is the smallest integer with amax / 2^e <= 448 (amax: its largest finite
// magnitude; e >= -126; 0 for a block of zeros), so the division is exact and the only rounding is the
// one to e4m3.  NaN and infinities become e4m3's NaN (it has no infinity) and set no scale.
//
// Scales are bytes e + 127 (the exponent format the tensor cores take), stored as they read
// them: for every 128 rows and every four blocks 512 consecutive bytes, row r's block b at
// (r % 32) * 16 + (r % 128) / 32 * 4 + b % 4.
//
// Meant to be bound by HBM: 2 or 4 bytes read and one written an element; with the transposed copy (blocks of
// 128 rows, for a product that sums over the rows) one more, from the same read.  Measured on B200 (bf16): rows
// 262144 x 192 33 us (4.5 TB/s), both copies of 16384 x 8192 about 110 us (4.9 TB/s): unpacking,
// scaling and rounding take about as many issue slots (65 %) as the bytes take time.
#include <algorithm>

#include "common.cuh"
#include "fp8_quant.cuh"
#include "kernels.cuh"

namespace p3d {
namespace {

using namespace quant;

struct QuantArgs {
  const void *x;
  int64_t rows, cols;
  uint8_t *q, *scales;     // [rows, pitch]
  int64_t pitch;
  uint8_t *qt, *t_scales;  // [cols, t_pitch]
  int64_t t_pitch;
  float *sums;             // [row tiles, cols] partial column sums
};

// 1 x 128 blocks along the rows: eight lanes a block, sixteen elements each (three steps to the block's maximum and one
// scale for four blocks a warp); a CTA takes 32 rows and 32 more gridDim.x groups further on, so that more
// loads are on their way, and walks their blocks from blockIdx.y on.
template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const QuantArgs a) {
  constexpr int kRowsAtOnce = 32;
  const int blocks = (int)((a.cols + kBlock - 1) / kBlock), groups = (blocks + 3) / 4;
  const int sub = threadIdx.x & 7;
  const int64_t step = (int64_t)gridDim.x * kRowsAtOnce;
  struct Pair {
    Raw<T> r[2];
  };
  auto load = [&](int64_t row, int64_t col) {
    const T *x = static_cast<const T *>(a.x) + row * a.cols;
    Pair p;
    p.r[0] = load8<T, ALIGNED>(x, row < a.rows ? col : a.cols, a.cols);
    p.r[1] = load8<T, ALIGNED>(x, row < a.rows ? col + 8 : a.cols, a.cols);
    return p;
  };
  auto write = [&](const Pair &p, int64_t row, int b, int64_t col) {
    uint32_t m = larger<T>(largest8<T>(p.r[0]), largest8<T>(p.r[1]));
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) m = larger<T>(m, __shfl_xor_sync(0xffffffffu, m, o));
    const bool odd = __any_sync(0xffffffffu, infinite<T>(m));
    if (odd) {
      m = max(finite_largest8<T>(p.r[0]), finite_largest8<T>(p.r[1]));
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    } else {
      m = widest<T>(m);
    }
    const uint32_t byte = scale_byte(m);
    if (row < a.rows) {
      const float inv = inverse_scale(byte);
      if (col < a.pitch) {   // the pitch is whole 16-byte pieces
        const uint2 lo = odd ? quantize8<true, T>(p.r[0], inv) : quantize8<false, T>(p.r[0], inv);
        const uint2 hi = odd ? quantize8<true, T>(p.r[1], inv) : quantize8<false, T>(p.r[1], inv);
        *reinterpret_cast<uint4 *>(a.q + row * a.pitch + col) = make_uint4(lo.x, lo.y, hi.x, hi.y);
      }
      if (sub == 0) a.scales[scale_at(row, b, groups)] = (uint8_t)byte;
    }
  };
  // the loop is the same for the whole CTA: the shuffles take whole warps
  for (int64_t r0 = (int64_t)blockIdx.x * kRowsAtOnce; r0 < a.rows; r0 += 2 * step) {
    const int64_t row = r0 + threadIdx.x / 8, next = row + step;
    for (int b = blockIdx.y; b < blocks; b += gridDim.y) {
      const int64_t col = (int64_t)b * kBlock + sub * 16;
      const Pair u = load(row, col), v = load(next, col);
      write(u, row, b, col);
      if (r0 + step < a.rows) write(v, next, b, col);
    }
  }
}

// What follows the loads of a tile.  CHECK: the tile has infinities.  FULL: all its rows and columns exist.
template <typename T, bool SQUARE, bool CHECK, bool FULL>
__device__ __forceinline__ void quantize_loaded(const QuantArgs &a, int tile_row, const Raw<T> (&v)[8],
                                                const uint32_t (&largest)[8], T *tile, uint32_t (&s_max)[4][kBlock],
                                                float (&s_sum)[4][kBlock]) {
  constexpr int kPitch = kBlock + 16 / sizeof(T);
  const int64_t k0 = (int64_t)blockIdx.x * kBlock, m0 = (int64_t)tile_row * kBlock;
  const int tid = threadIdx.x, sub = tid & 15, r0 = tid / 16;
  uint32_t all = 0;
  if constexpr (SQUARE) {
#pragma unroll
    for (int i = 0; i < 8; ++i) all = max(all, CHECK ? finite_largest8<T>(v[i]) : widest<T>(largest[i]));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) all = max(all, __shfl_xor_sync(0xffffffffu, all, o));
    if ((tid & 31) == 0) s_max[0][tid / 32] = all;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) all = max(all, s_max[0][w]);
  }
  if (a.q) {
    uint32_t byte[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      uint32_t m = all;
      if constexpr (!SQUARE) {
        m = CHECK ? finite_largest8<T>(v[i]) : largest[i];
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) {
          const uint32_t other = __shfl_xor_sync(0xffffffffu, m, o);
          m = CHECK ? max(m, other) : larger<T>(m, other);
        }
        if constexpr (!CHECK) m = widest<T>(m);
      }
      byte[i] = scale_byte(m);
    }
    const int64_t col = k0 + sub * 8;
    uint8_t *q = a.q + (m0 + r0) * a.pitch + col;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (FULL || (m0 + r0 + 16 * i < a.rows && col < a.pitch))
        *reinterpret_cast<uint2 *>(q + 16 * i * a.pitch) = quantize8<CHECK, T>(v[i], inverse_scale(byte[i]));
    if (sub == 0) {   // rows r0 + 16 i, r0 < 16: 256 bytes on for odd i, four for every second i (see scale_at)
      uint8_t *to = a.scales + scale_at(m0 + r0, blockIdx.x, ((a.cols + kBlock - 1) / kBlock + 3) / 4);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (FULL || m0 + r0 + 16 * i < a.rows) to[(i & 1) * 256 + (i >> 1) * 4] = (uint8_t)byte[i];
    }
  }
  if (!a.qt && !a.sums) return;
  // a pair of columns and a quarter of the rows a thread: x[r] is row r's pair
  const int c = (tid & 63) * 2, quarter = tid / 64;
  const T *from = tile + quarter * 32 * kPitch + c;
  constexpr int kPair = sizeof(T) / 2;   // words of a pair
  uint32_t x[32 * kPair], m0w = 0, m1w = 0;   // 16 bits: both columns' magnitudes share m0w
#pragma unroll
  for (int r = 0; r < 32; ++r) {
    if constexpr (kPair == 1) {
      x[r] = *reinterpret_cast<const uint32_t *>(from + r * kPitch);
      m0w = larger<T>(m0w, x[r]);
    } else {
      const uint2 w = *reinterpret_cast<const uint2 *>(from + r * kPitch);
      x[2 * r] = w.x;
      x[2 * r + 1] = w.y;
      m0w = larger<T>(m0w, w.x);
      m1w = larger<T>(m1w, w.y);
    }
  }
  auto pair = [&](int r) {
    if constexpr (kPair == 1) return unpack2<T>(x[r]);
    else return make_float2(__uint_as_float(x[2 * r]), __uint_as_float(x[2 * r + 1]));
  };
  if (a.sums) {
    float2 s = pair(0);
#pragma unroll
    for (int r = 1; r < 32; ++r) s = sm100::add2(s, pair(r));
    *reinterpret_cast<float2 *>(&s_sum[quarter][c]) = s;
  }
  if constexpr (!SQUARE) {
    uint2 m;
    if constexpr (CHECK) {
      m = make_uint2(0u, 0u);
#pragma unroll
      for (int r = 0; r < 32; ++r) {
        const float2 f = pair(r);
        m.x = max(m.x, finite_bits(f.x));
        m.y = max(m.y, finite_bits(f.y));
      }
    } else if constexpr (kPair == 1) {
      m = make_uint2(widest<T>(m0w & 0x7fffu), widest<T>(m0w >> 16 & 0x7fffu));
    } else {
      m = make_uint2(widest<T>(m0w), widest<T>(m1w));
    }
    *reinterpret_cast<uint2 *>(&s_max[quarter][c]) = m;
  }
  __syncthreads();
  if (a.sums && tid < kBlock && k0 + tid < a.cols)
    a.sums[(int64_t)tile_row * a.cols + k0 + tid] = s_sum[0][tid] + s_sum[1][tid] + s_sum[2][tid] + s_sum[3][tid];
  if (!a.qt) return;
  uint32_t byte[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if constexpr (!SQUARE) all = max(max(s_max[0][c + h], s_max[1][c + h]), max(s_max[2][c + h], s_max[3][c + h]));
    byte[h] = scale_byte(all);
  }
  if (quarter == 0) {   // rows c and c + 1 of the transposed matrix: sixteen bytes apart (c is even)
    uint8_t *to = a.t_scales + scale_at(k0 + c, tile_row, ((a.rows + kBlock - 1) / kBlock + 3) / 4);
    if (FULL || k0 + c < a.cols) to[0] = (uint8_t)byte[0];
    if (FULL || k0 + c + 1 < a.cols) to[16] = (uint8_t)byte[1];
  }
  const float2 inv = make_float2(inverse_scale(byte[0]), inverse_scale(byte[1]));
  // over the tile, whose values are in registers now: the transposed bytes, rows of 144 bytes apart, from which
  // whole 128-byte lines go out (16 bytes at a row's pitch would touch as many half sectors)
  constexpr int kOut = kBlock + 16;
  uint8_t *out = reinterpret_cast<uint8_t *>(tile);
#pragma unroll
  for (int i = 0; i < 2; ++i) {   // sixteen rows: sixteen bytes of either column
    uint32_t w[2][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t h[2][2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const float2 p = pair(16 * i + 4 * j + 2 * k), n = pair(16 * i + 4 * j + 2 * k + 1);
        h[0][k] = to_e4m3x2<CHECK>(make_float2(p.x, n.x), inv.x);
        h[1][k] = to_e4m3x2<CHECK>(make_float2(p.y, n.y), inv.y);
      }
      w[0][j] = __byte_perm(h[0][0], h[0][1], 0x5410);
      w[1][j] = __byte_perm(h[1][0], h[1][1], 0x5410);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
      *reinterpret_cast<uint4 *>(out + (c + h) * kOut + quarter * 32 + i * 16) = make_uint4(w[h][0], w[h][1], w[h][2], w[h][3]);
  }
  __syncthreads();
  const int piece = (tid & 7) * 16;
  uint8_t *qt = a.qt + k0 * a.t_pitch + m0 + piece;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int col = tid / 8 + 32 * i;
    if (FULL || (k0 + col < a.cols && m0 + piece < a.t_pitch))
      *reinterpret_cast<uint4 *>(qt + (int64_t)col * a.t_pitch) = *reinterpret_cast<const uint4 *>(out + col * kOut + piece);
  }
}

// A tile with infinities: its values are read again, so that the kernel's own path keeps its registers.
template <typename T, bool SQUARE>
__device__ __noinline__ void quantize_odd(const QuantArgs &a, int tile_row, T *tile, uint32_t (&s_max)[4][kBlock],
                                          float (&s_sum)[4][kBlock]) {
  const int64_t m0 = (int64_t)tile_row * kBlock + threadIdx.x / 16, col = (int64_t)blockIdx.x * kBlock + (threadIdx.x & 15) * 8;
  Raw<T> v[8];
  const uint32_t none[8] = {};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t row = m0 + 16 * i;
    v[i] = load8<T, false>(static_cast<const T *>(a.x) + row * a.cols, row < a.rows ? col : a.cols, a.cols);
  }
  quantize_loaded<T, SQUARE, true, false>(a, tile_row, v, none, tile, s_max, s_sum);
}

// One 128 x 128 tile a CTA, read once.  Row output: 1 x 128 blocks, or the whole tile as one block
// (SQUARE).  Transposed output: blocks of 128 rows of a column (or the same whole tile), from
// the tile's copy in shared memory.  Column sums of the tile where asked for.
template <typename T, bool ALIGNED, bool SQUARE>
__device__ __forceinline__ void quantize_tile(const QuantArgs &a, int tile_row, T *tile, uint32_t (&s_max)[4][kBlock],
                                              float (&s_sum)[4][kBlock]) {
  constexpr int kPitch = kBlock + 16 / sizeof(T);   // 16 bytes past 128 values: rows start on other banks
  const int64_t k0 = (int64_t)blockIdx.x * kBlock, m0 = (int64_t)tile_row * kBlock;
  const int tid = threadIdx.x, sub = tid & 15, r0 = tid / 16;
  const bool full = m0 + kBlock <= a.rows && k0 + kBlock <= a.cols;
  Raw<T> v[8];
  uint32_t largest[8];
  bool odd = false;
  const T *x = static_cast<const T *>(a.x) + (m0 + r0) * a.cols;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    v[i] = load8<T, ALIGNED>(x + 16 * i * a.cols, full || m0 + r0 + 16 * i < a.rows ? k0 + sub * 8 : a.cols, a.cols);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (a.qt || a.sums) {
      uint4 *to = reinterpret_cast<uint4 *>(tile + (r0 + 16 * i) * kPitch + sub * 8);
#pragma unroll
      for (int j = 0; j < Raw<T>::kWords / 4; ++j)
        to[j] = make_uint4(v[i].w[4 * j], v[i].w[4 * j + 1], v[i].w[4 * j + 2], v[i].w[4 * j + 3]);
    }
    largest[i] = largest8<T>(v[i]);
    odd |= infinite<T>(largest[i]);
  }
  odd = __syncthreads_or(odd);   // and the tile is there
  if (odd) quantize_odd<T, SQUARE>(a, tile_row, tile, s_max, s_sum);
  else if (full) quantize_loaded<T, SQUARE, false, true>(a, tile_row, v, largest, tile, s_max, s_sum);
  else quantize_loaded<T, SQUARE, false, false>(a, tile_row, v, largest, tile, s_max, s_sum);
}

template <typename T> constexpr size_t tile_bytes() { return (size_t)kBlock * (kBlock + 16 / sizeof(T)) * sizeof(T); }

// kBoth: the first x_tiles rows of tiles are x's, with blocks along its rows, the others w's, as square blocks.
enum : int { kRowBlocks = 0, kSquare = 1, kBoth = 2 };
template <typename T, bool ALIGNED, int BLOCKS>
__global__ void __launch_bounds__(256, sizeof(T) == 2 ? 4 : 2)
    quantize_tile_kernel(const __grid_constant__ QuantArgs x, const __grid_constant__ QuantArgs w, int x_tiles) {
  extern __shared__ __align__(16) unsigned char s_raw[];
  T *tile = reinterpret_cast<T *>(s_raw);
  __shared__ __align__(16) uint32_t s_max[4][kBlock];
  __shared__ __align__(16) float s_sum[4][kBlock];
  const int tile_row = blockIdx.y;
  if (BLOCKS == kRowBlocks || (BLOCKS == kBoth && tile_row < x_tiles))
    quantize_tile<T, ALIGNED, false>(x, tile_row, tile, s_max, s_sum);
  else
    quantize_tile<T, ALIGNED, true>(w, tile_row - x_tiles, tile, s_max, s_sum);
}

// x or w may be without rows.
template <typename T, bool ALIGNED, int BLOCKS>
int launch_tile(const QuantArgs &x, const QuantArgs &w, cudaStream_t s) {
  static size_t seen[kMaxDevices] = {};
  if (int st = smem_optin(quantize_tile_kernel<T, ALIGNED, BLOCKS>, tile_bytes<T>(), seen)) return st;
  const int64_t x_tiles = (x.rows + kBlock - 1) / kBlock, w_tiles = (w.rows + kBlock - 1) / kBlock;
  const dim3 grid((unsigned)((std::max(x.cols, w.cols) + kBlock - 1) / kBlock), (unsigned)(x_tiles + w_tiles));
  quantize_tile_kernel<T, ALIGNED, BLOCKS><<<grid, 256, tile_bytes<T>(), s>>>(x, w, (int)x_tiles);
  P3D_LAUNCH_CHECK();
  return P3D_OK;
}

template <typename T>
int run_quantize(const QuantArgs &a, bool square, int sms, cudaStream_t s) {
  const bool aligned = a.cols % 8 == 0 && ((uintptr_t)a.x & 15) == 0;
  if (!square && !a.qt && !a.sums) {
    // as many CTAs as the SMs hold; few rows: their blocks are dealt out to more CTAs
    const int64_t across = std::min<int64_t>((a.rows + 31) / 32, sms * 6), blocks = (a.cols + kBlock - 1) / kBlock;
    const dim3 grid((unsigned)across, (unsigned)std::min<int64_t>(blocks, std::max<int64_t>(1, sms * 8 / across)));
    if (aligned) quantize_rows_kernel<T, true><<<grid, 256, 0, s>>>(a);
    else quantize_rows_kernel<T, false><<<grid, 256, 0, s>>>(a);
    P3D_LAUNCH_CHECK();
    return P3D_OK;
  }
  const QuantArgs none = {};
  if (square) return aligned ? launch_tile<T, true, kSquare>(none, a, s) : launch_tile<T, false, kSquare>(none, a, s);
  return aligned ? launch_tile<T, true, kRowBlocks>(a, none, s) : launch_tile<T, false, kRowBlocks>(a, none, s);
}

template <typename T>
int run_both(const QuantArgs &x, const QuantArgs &w, cudaStream_t s) {
  const bool aligned = x.cols % 8 == 0 && (((uintptr_t)x.x | (uintptr_t)w.x) & 15) == 0;
  return aligned ? launch_tile<T, true, kBoth>(x, w, s) : launch_tile<T, false, kBoth>(x, w, s);
}

}  // namespace

int launch_quantize_both(const QuantOperand &x, const QuantOperand &w, int64_t cols, int dtype, cudaStream_t s) {
  auto args = [&](const QuantOperand &m) {
    QuantArgs a = {};
    a.x = m.x;
    a.rows = m.rows;
    a.cols = cols;
    a.q = static_cast<uint8_t *>(m.q);
    a.scales = static_cast<uint8_t *>(m.scales);
    a.pitch = m.pitch;
    a.qt = static_cast<uint8_t *>(m.qt);
    a.t_scales = static_cast<uint8_t *>(m.t_scales);
    a.t_pitch = m.t_pitch;
    return a;
  };
  if (dtype == P3D_F32) return run_both<float>(args(x), args(w), s);
  if (dtype == P3D_F16) return run_both<__half>(args(x), args(w), s);
  return run_both<__nv_bfloat16>(args(x), args(w), s);
}

}  // namespace p3d

using namespace p3d;

extern "C" int64_t p3d_fp8_scale_bytes(int64_t rows, int64_t cols) {
  if (rows < 0 || cols < 0) return 0;
  return (rows + 127) / 128 * (((cols + 127) / 128 + 3) / 4) * 512;
}

extern "C" size_t p3d_fp8_quantize_workspace(int64_t rows, int64_t cols) {
  if (rows < 0 || cols < 0) return 0;
  return (size_t)((rows + 127) / 128 * cols) * sizeof(float);
}

extern "C" int p3d_fp8_quantize(const void *x, int dtype, int64_t rows, int64_t cols, int square, void *q, int64_t pitch,
                                void *scales, void *qt, int64_t t_pitch, void *t_scales, void *col_sum,
                                int col_sum_dtype, void *workspace, size_t workspace_bytes, void *stream) {
  P3D_CHECK_ARG(dtype_ok(dtype), "p3d_fp8_quantize: unknown dtype %d", dtype);
  P3D_CHECK_ARG(rows >= 1 && cols >= 1, "p3d_fp8_quantize: rows and cols must be positive");
  if (rows > 65535LL * kBlock || cols > 65535LL * kBlock)
    return fail(P3D_ERR_UNSUPPORTED, "p3d_fp8_quantize: extents above %lld", 65535LL * kBlock);
  P3D_CHECK_ARG(x && (q || qt || col_sum), "p3d_fp8_quantize: null pointer");
  P3D_CHECK_ARG(!q || (scales && pitch >= cols && pitch % 16 == 0 && ((uintptr_t)q & 15) == 0),
                "p3d_fp8_quantize: values need scales and a pitch of at least cols, both aligned to 16 bytes");
  P3D_CHECK_ARG(!qt || (t_scales && t_pitch >= rows && t_pitch % 16 == 0 && ((uintptr_t)qt & 15) == 0),
                "p3d_fp8_quantize: transposed values need scales and a pitch of at least rows, aligned to 16 bytes");
  P3D_CHECK_ARG(!col_sum || dtype_ok(col_sum_dtype), "p3d_fp8_quantize: unknown dtype of the column sums");
  const size_t need = col_sum ? p3d_fp8_quantize_workspace(rows, cols) : 0;
  if (need && (!workspace || workspace_bytes < need))
    return fail(P3D_ERR_WORKSPACE, "p3d_fp8_quantize: workspace of %zu bytes, %zu needed", workspace_bytes, need);
  DeviceInfo info;
  if (int st = device_info(&info)) return st;
  QuantArgs a = {};
  a.x = x;
  a.rows = rows;
  a.cols = cols;
  a.q = static_cast<uint8_t *>(q);
  a.scales = static_cast<uint8_t *>(scales);
  a.pitch = pitch;
  a.qt = static_cast<uint8_t *>(qt);
  a.t_scales = static_cast<uint8_t *>(t_scales);
  a.t_pitch = t_pitch;
  a.sums = col_sum ? static_cast<float *>(workspace) : nullptr;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  int st;
  if (dtype == P3D_F32) st = run_quantize<float>(a, square != 0, info.sm_count, s);
  else if (dtype == P3D_F16) st = run_quantize<__half>(a, square != 0, info.sm_count, s);
  else st = run_quantize<__nv_bfloat16>(a, square != 0, info.sm_count, s);
  if (st != P3D_OK || !col_sum) return st;
  return launch_column_join(a.sums, col_sum, col_sum_dtype, (rows + 127) / 128, (int)cols, s);
}
