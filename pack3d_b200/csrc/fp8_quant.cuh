// Device pieces of the e4m3 quantiser (see fp8.cu): block maxima, scale bytes, rounding, scale addresses.
#pragma once

#include <type_traits>

#include "common.cuh"
#include "sm100.cuh"

namespace p3d {
namespace quant {

constexpr int kBlock = 128;

__device__ __forceinline__ uint32_t finite_bits(float v) {
  const uint32_t b = __float_as_uint(v) & 0x7fffffffu;
  return b < 0x7f800000u ? b : 0u;
}

// Magnitudes of a block are compared two 16-bit ones at a time, NaN left out; a word is `infinite` where either half is
// infinite (or both operands were NaN), and then the block is gone over again with infinities left out.
template <typename T> __device__ __forceinline__ bool infinite(uint32_t m) {
  constexpr uint32_t top = std::is_same<T, __nv_bfloat16>::value ? 0x7f80u : 0x7c00u;
  return (m & 0x7fffu) >= top || (m >> 16 & 0x7fffu) >= top;
}
template <> __device__ __forceinline__ bool infinite<float>(uint32_t m) { return (m & 0x7fffffffu) >= 0x7f800000u; }

// The larger magnitude of two words, half by half for 16-bit types; the sign bits of the result mean nothing.
template <typename T> __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {
  uint32_t r;
  if constexpr (std::is_same<T, __nv_bfloat16>::value) asm("max.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else if constexpr (std::is_same<T, __half>::value) asm("max.xorsign.abs.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else r = __float_as_uint(fmaxf(fabsf(__uint_as_float(a)), fabsf(__uint_as_float(b))));
  return r;
}
// fp32 bits of the larger half.
template <typename T> __device__ __forceinline__ uint32_t widest(uint32_t m) {
  if constexpr (sizeof(T) == 4) return m & 0x7fffffffu;
  const uint32_t h = max(m & 0x7fffu, m >> 16 & 0x7fffu);
  if constexpr (std::is_same<T, __nv_bfloat16>::value) return h << 16;
  else return __float_as_uint(__half2float(__ushort_as_half((unsigned short)h)));
}

// Eight values of a row as they lie in memory.
template <typename T> struct Raw {
  static constexpr int kWords = 2 * sizeof(T);
  uint32_t w[kWords];
};

template <typename T, bool ALIGNED>
__device__ __forceinline__ Raw<T> load8(const T *row, int64_t col, int64_t cols) {
  Raw<T> r;
  if constexpr (ALIGNED) {
    if (col < cols) {
#pragma unroll
      for (int i = 0; i < Raw<T>::kWords / 4; ++i) {
        const uint4 v = reinterpret_cast<const uint4 *>(row + col)[i];
        r.w[4 * i] = v.x;
        r.w[4 * i + 1] = v.y;
        r.w[4 * i + 2] = v.z;
        r.w[4 * i + 3] = v.w;
      }
      return r;
    }
  }
  alignas(16) T v[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = !ALIGNED && col + j < cols ? row[col + j] : from_f32<T>(0.f);
  memcpy(r.w, v, sizeof(r.w));
  return r;
}
template <typename T> __device__ __forceinline__ float value(const Raw<T> &r, int j) {
  if constexpr (sizeof(T) == 4) return __uint_as_float(r.w[j]);
  else {
    const float2 f = unpack2<T>(r.w[j / 2]);
    return j & 1 ? f.y : f.x;
  }
}
template <typename T> __device__ __forceinline__ uint32_t largest8(const Raw<T> &r) {
  uint32_t m = larger<T>(r.w[0], r.w[1]);
#pragma unroll
  for (int i = 2; i < Raw<T>::kWords; ++i) m = larger<T>(m, r.w[i]);
  return m;
}
template <typename T> __device__ __forceinline__ uint32_t finite_largest8(const Raw<T> &r) {   // in fp32 bits
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) m = max(m, finite_bits(value(r, j)));
  return m;
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
// NaN otherwise; a block without infinities needs only the product (NaN stays NaN).
template <bool CHECK> __device__ __forceinline__ uint32_t to_e4m3x2(float2 v, float inv) {
  if constexpr (CHECK) {
    v.x = fmaf(v.x, inv, v.x - v.x);
    v.y = fmaf(v.y, inv, v.y - v.y);
  } else {
    v = sm100::mul2(v, make_float2(inv, inv));
  }
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(v.y), "f"(v.x));
  return r;
}
template <bool CHECK> __device__ __forceinline__ uint32_t to_e4m3x4(float2 lo, float2 hi, float inv) {
  return __byte_perm(to_e4m3x2<CHECK>(lo, inv), to_e4m3x2<CHECK>(hi, inv), 0x5410);
}
template <bool CHECK, typename T> __device__ __forceinline__ uint2 quantize8(const Raw<T> &r, float inv) {
  float2 v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 2) v[i] = unpack2<T>(r.w[i]);
    else v[i] = make_float2(__uint_as_float(r.w[2 * i]), __uint_as_float(r.w[2 * i + 1]));
  }
  return make_uint2(to_e4m3x4<CHECK>(v[0], v[1], inv), to_e4m3x4<CHECK>(v[2], v[3], inv));
}

// Where the scale byte of row `r`, block `b` lies; groups = ceil(blocks / 4).
__device__ __forceinline__ int64_t scale_at(int64_t r, int64_t b, int64_t groups) {
  return ((r / 128) * groups + b / 4) * 512 + (r % 32) * 16 + (r % 128) / 32 * 4 + b % 4;
}

// The largest magnitude (fp32 bits, infinities left out) of a 128-element block that sixteen lanes hold; *odd
// says whether it has infinities or NaN.
template <typename T>
__device__ __forceinline__ uint32_t block_amax(const Raw<T> &r, bool *odd) {
  uint32_t m = largest8<T>(r);
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) m = larger<T>(m, __shfl_xor_sync(0xffffffffu, m, o));
  *odd = __any_sync(0xffffffffu, infinite<T>(m));   // either half of the warp: both then check every value
  if (*odd) {
    m = finite_largest8<T>(r);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    return m;
  }
  return widest<T>(m);
}

}  // namespace quant
}  // namespace p3d
