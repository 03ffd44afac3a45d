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
// Bound by HBM: 2 or 4 bytes read and one written an element; with the transposed copy (blocks of
// 128 rows, for a product that sums over the rows) one more, from the same read.
#include <algorithm>

#include "common.cuh"
#include "kernels.cuh"

namespace p3d {
namespace {

constexpr int kBlock = 128;

__device__ __forceinline__ uint32_t finite_bits(float v) {
  const uint32_t b = __float_as_uint(v) & 0x7fffffffu;
  return b < 0x7f800000u ? b : 0u;
}

// e + 127 of a block whose largest finite magnitude has these bits: 448 = 1.75 * 2^8.
__device__ __forceinline__ uint32_t scale_byte(uint32_t amax_bits) {
  if (amax_bits == 0u) return 127u;
  const int e = (int)(amax_bits >> 23) - 8 + ((amax_bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return (uint32_t)max(e, 1);
}
// 2^-e
__device__ __forceinline__ float inverse_scale(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }

// Two values to e4m3 (lo in the low byte).  x * inv + (x - x): the second term is 0 for finite x and
// NaN otherwise.
__device__ __forceinline__ uint32_t to_e4m3x2(float lo, float hi, float inv) {
  lo = fmaf(lo, inv, lo - lo);
  hi = fmaf(hi, inv, hi - hi);
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t to_e4m3x4(float a, float b, float c, float d, float inv) {
  return to_e4m3x2(a, b, inv) | to_e4m3x2(c, d, inv) << 16;
}

// Where the scale byte of row `r`, block `b` lies; groups = ceil(blocks / 4).
__device__ __forceinline__ int64_t scale_at(int64_t r, int64_t b, int64_t groups) {
  return ((r / 128) * groups + b / 4) * 512 + (r % 32) * 16 + (r % 128) / 32 * 4 + b % 4;
}

// Eight elements of a row from column `col` on, zero past its end.
template <typename T, bool ALIGNED>
__device__ __forceinline__ void load8(T (&v)[8], const T *row, int64_t col, int64_t cols) {
  if constexpr (ALIGNED) {
    if (col < cols) {
      constexpr int n = sizeof(v) / 16;
      uint4 raw[n];
#pragma unroll
      for (int i = 0; i < n; ++i) raw[i] = reinterpret_cast<const uint4 *>(row + col)[i];
      memcpy(v, raw, sizeof(v));
      return;
    }
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = !ALIGNED && col + j < cols ? row[col + j] : from_f32<T>(0.f);
}

template <typename T>
__device__ __forceinline__ uint32_t amax8(const T (&v)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) m = max(m, finite_bits(to_f32<T>(v[j])));
  return m;
}
template <typename T>
__device__ __forceinline__ uint2 quantize8(const T (&v)[8], float inv) {
  return make_uint2(to_e4m3x4(to_f32<T>(v[0]), to_f32<T>(v[1]), to_f32<T>(v[2]), to_f32<T>(v[3]), inv),
                    to_e4m3x4(to_f32<T>(v[4]), to_f32<T>(v[5]), to_f32<T>(v[6]), to_f32<T>(v[7]), inv));
}

struct QuantArgs {
  const void *x;
  int64_t rows, cols;
  uint8_t *q, *scales;     // [rows, pitch]
  int64_t pitch;
  uint8_t *qt, *t_scales;  // [cols, t_pitch]
  int64_t t_pitch;
  float *sums;             // [row tiles, cols] partial column sums
};

// 1 x 128 blocks along the rows: sixteen lanes a block, eight elements each.
template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const QuantArgs a) {
  const int64_t blocks = (a.cols + kBlock - 1) / kBlock, groups = (blocks + 3) / 4, total = a.rows * blocks;
  const int sub = threadIdx.x & 15;
  const int64_t step = (int64_t)gridDim.x * 16;
  for (int64_t i0 = (int64_t)blockIdx.x * 16; i0 < total; i0 += step) {   // uniform: the shuffles take whole warps
    const int64_t i = i0 + threadIdx.x / 16, row = i / blocks, b = i - row * blocks, col = b * kBlock + sub * 8;
    T v[8];
    load8<T, ALIGNED>(v, static_cast<const T *>(a.x) + row * a.cols, i < total ? col : a.cols, a.cols);
    uint32_t m = amax8<T>(v);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    const uint32_t byte = scale_byte(m);
    if (i < total) {
      if (col < a.pitch) *reinterpret_cast<uint2 *>(a.q + row * a.pitch + col) = quantize8<T>(v, inverse_scale(byte));
      if (sub == 0) a.scales[scale_at(row, b, groups)] = (uint8_t)byte;
    }
  }
}

// One 128 x 128 tile a CTA, read once.  Row output: 1 x 128 blocks, or the whole tile as one block
// (SQUARE).  Transposed output: blocks of 128 rows of a column (or the same whole tile), from
// the tile's copy in shared memory.  Column sums of the tile where asked for.
template <typename T, bool ALIGNED, bool SQUARE>
__global__ void __launch_bounds__(256) quantize_tile_kernel(const QuantArgs a) {
  constexpr int kPitch = kBlock + 16 / sizeof(T);   // 16 bytes past 128 values: rows start on other banks
  extern __shared__ __align__(16) unsigned char s_raw[];
  T *tile = reinterpret_cast<T *>(s_raw);
  __shared__ uint32_t s_max[4][kBlock];
  __shared__ float s_sum[4][kBlock];
  const int64_t k0 = (int64_t)blockIdx.x * kBlock, m0 = (int64_t)blockIdx.y * kBlock;
  const int tid = threadIdx.x, sub = tid & 15, r0 = tid / 16;
  const int64_t groups = ((a.cols + kBlock - 1) / kBlock + 3) / 4;
  T v[8][8];
  uint32_t all = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t row = m0 + r0 + 16 * i;
    load8<T, ALIGNED>(v[i], static_cast<const T *>(a.x) + row * a.cols, row < a.rows ? k0 + sub * 8 : a.cols, a.cols);
    if (a.qt || a.sums) memcpy(tile + (r0 + 16 * i) * kPitch + sub * 8, v[i], sizeof(v[i]));
    if (SQUARE) all = max(all, amax8<T>(v[i]));
  }
  if (SQUARE) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) all = max(all, __shfl_xor_sync(0xffffffffu, all, o));
    if ((tid & 31) == 0) s_max[0][tid / 32] = all;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) all = max(all, s_max[0][w]);
  }
  if (a.q) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      uint32_t m = all;
      if (!SQUARE) {
        m = amax8<T>(v[i]);
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
      }
      const uint32_t byte = scale_byte(m);
      const int64_t row = m0 + r0 + 16 * i, col = k0 + sub * 8;
      if (row < a.rows) {
        if (col < a.pitch) *reinterpret_cast<uint2 *>(a.q + row * a.pitch + col) = quantize8<T>(v[i], inverse_scale(byte));
        if (sub == 0) a.scales[scale_at(row, blockIdx.x, groups)] = (uint8_t)byte;
      }
    }
  }
  if (!a.qt && !a.sums) return;
  __syncthreads();
  // a pair of columns and a quarter of the rows a thread
  const int c = (tid & 63) * 2, quarter = tid / 64;
  float x[2][32];
  uint32_t m[2] = {0u, 0u};
  float s[2] = {0.f, 0.f};
#pragma unroll
  for (int r = 0; r < 32; ++r) {
    const T *at = tile + (quarter * 32 + r) * kPitch + c;
    if constexpr (sizeof(T) == 2) {
      const float2 f = unpack2<T>(*reinterpret_cast<const uint32_t *>(at));
      x[0][r] = f.x;
      x[1][r] = f.y;
    } else {
      const float2 f = *reinterpret_cast<const float2 *>(at);
      x[0][r] = f.x;
      x[1][r] = f.y;
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      m[h] = max(m[h], finite_bits(x[h][r]));
      s[h] += x[h][r];
    }
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if (!SQUARE) s_max[quarter][c + h] = m[h];
    s_sum[quarter][c + h] = s[h];
  }
  __syncthreads();
  if (a.sums && tid < kBlock && k0 + tid < a.cols)
    a.sums[(int64_t)blockIdx.y * a.cols + k0 + tid] = s_sum[0][tid] + s_sum[1][tid] + s_sum[2][tid] + s_sum[3][tid];
  if (!a.qt) return;
  const int64_t t_groups = ((a.rows + kBlock - 1) / kBlock + 3) / 4;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int64_t col = k0 + c + h;
    if (!SQUARE) all = max(max(s_max[0][c + h], s_max[1][c + h]), max(s_max[2][c + h], s_max[3][c + h]));
    const uint32_t byte = scale_byte(all);
    const float inv = inverse_scale(byte);
    if (col < a.cols) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int64_t at = m0 + quarter * 32 + i * 16;
        uint4 w;
        w.x = to_e4m3x4(x[h][16 * i], x[h][16 * i + 1], x[h][16 * i + 2], x[h][16 * i + 3], inv);
        w.y = to_e4m3x4(x[h][16 * i + 4], x[h][16 * i + 5], x[h][16 * i + 6], x[h][16 * i + 7], inv);
        w.z = to_e4m3x4(x[h][16 * i + 8], x[h][16 * i + 9], x[h][16 * i + 10], x[h][16 * i + 11], inv);
        w.w = to_e4m3x4(x[h][16 * i + 12], x[h][16 * i + 13], x[h][16 * i + 14], x[h][16 * i + 15], inv);
        if (at < a.t_pitch) *reinterpret_cast<uint4 *>(a.qt + col * a.t_pitch + at) = w;
      }
      if (quarter == 0) a.t_scales[scale_at(col, blockIdx.y, t_groups)] = (uint8_t)byte;
    }
  }
}

template <typename T, bool ALIGNED, bool SQUARE>
int launch_tile(const QuantArgs &a, cudaStream_t s) {
  static size_t seen[kMaxDevices] = {};
  const size_t smem = (size_t)kBlock * (kBlock + 16 / sizeof(T)) * sizeof(T);
  if (int st = smem_optin(quantize_tile_kernel<T, ALIGNED, SQUARE>, smem, seen)) return st;
  const dim3 grid((unsigned)((a.cols + kBlock - 1) / kBlock), (unsigned)((a.rows + kBlock - 1) / kBlock));
  quantize_tile_kernel<T, ALIGNED, SQUARE><<<grid, 256, smem, s>>>(a);
  P3D_LAUNCH_CHECK();
  return P3D_OK;
}

template <typename T>
int run_quantize(const QuantArgs &a, bool square, int sms, cudaStream_t s) {
  const bool aligned = a.cols % 8 == 0 && ((uintptr_t)a.x & 15) == 0;
  if (!square && !a.qt && !a.sums) {
    const int64_t total = a.rows * ((a.cols + kBlock - 1) / kBlock);
    const unsigned grid = (unsigned)std::min<int64_t>((total + 15) / 16, (int64_t)sms * 16);
    if (aligned) quantize_rows_kernel<T, true><<<grid, 256, 0, s>>>(a);
    else quantize_rows_kernel<T, false><<<grid, 256, 0, s>>>(a);
    P3D_LAUNCH_CHECK();
    return P3D_OK;
  }
  if (square) return aligned ? launch_tile<T, true, true>(a, s) : launch_tile<T, false, true>(a, s);
  return aligned ? launch_tile<T, true, false>(a, s) : launch_tile<T, false, false>(a, s);
}

}  // namespace
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
