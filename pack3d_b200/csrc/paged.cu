// Attention of one new token of each sequence over its pages, a warp to a head.
#include <cuda_fp8.h>
#include <math.h>

#include "cache.cuh"

namespace p3d {
namespace {

constexpr int kWarps = 8;

struct Params {
  p3d_cache c;
  const void *q;
  int64_t stride[2];
  int dtype, heads;
  const int32_t *lengths;
  float scale;
  void *out;
};

__device__ __forceinline__ float cached(const p3d_cache &c, const void *pages, const uint8_t *scales, int64_t row, int col) {
  if (c.dtype != P3D_E4M3) return load_any(pages, c.dtype, row * c.dim + col);
  const __half_raw h = __nv_cvt_fp8_to_halfraw(static_cast<const uint8_t *>(pages)[row * c.dim + col], __NV_E4M3);
  const uint32_t byte = scales[row];
  return __half2float(h) * __uint_as_float(byte ? byte << 23 : 0x400000u);
}

__global__ void paged_kernel(const __grid_constant__ Params p) {
  const int item = blockIdx.x * kWarps + threadIdx.x / 32, lane = threadIdx.x & 31, b = item / p.heads, h = item % p.heads;
  if (b >= p.c.sequences) return;
  const int g = h / (p.heads / p.c.kv_heads), n = p.lengths[b];
  float q[4], o[4] = {0.f, 0.f, 0.f, 0.f}, m = -INFINITY, l = 0.f;
  for (int i = 0; i < 4; ++i)
    q[i] = lane * 4 + i < p.c.dim ? load_any(p.q, p.dtype, b * p.stride[0] + h * p.stride[1] + lane * 4 + i) : 0.f;
  for (int j = 0; j < n; ++j) {
    const cache::Place place = cache::place_of(p.c, b, j);
    const int64_t row = ((int64_t)place.page * p.c.kv_heads + g) * p.c.page_size + place.row;
    float k[4], v[4];
    for (int i = 0; i < 4; ++i) {
      const bool there = lane * 4 + i < p.c.dim;
      k[i] = !there ? 0.f : place.page < 0 ? NAN : cached(p.c, p.c.k, p.c.k_scales, row, lane * 4 + i);
      v[i] = !there ? 0.f : place.page < 0 ? NAN : cached(p.c, p.c.v, p.c.v_scales, row, lane * 4 + i);
    }
    const float s = warp_sum(q[0] * k[0] + q[1] * k[1] + q[2] * k[2] + q[3] * k[3]) * p.scale;
    const float top = fmaxf(m, s), old = m == -INFINITY ? 0.f : expf(m - top), w = expf(s - top);
    l = l * old + w;
    m = top;
    for (int i = 0; i < 4; ++i) o[i] = o[i] * old + w * v[i];
  }
  for (int i = 0; i < 4; ++i)
    if (lane * 4 + i < p.c.dim)
      store_any(p.out, p.dtype, ((int64_t)b * p.heads + h) * p.c.dim + lane * 4 + i, n > 0 ? o[i] / l : 0.f);
}

}  // namespace
}  // namespace p3d

using namespace p3d;

extern "C" {

size_t p3d_paged_attention_workspace(const p3d_cache *cache, int heads) { return 0; }

int p3d_paged_attention(const p3d_cache *c, const void *q, const int64_t q_stride[2], int dtype, int heads,
                        const int32_t *lengths, float scale, void *out, void *workspace, size_t workspace_bytes,
                        void *stream) {
  if (int st = cache::check(c, "p3d_paged_attention")) return st;
  P3D_CHECK_ARG(dtype == P3D_F16 || dtype == P3D_BF16, "p3d_paged_attention: f16 or bf16 queries only");
  P3D_CHECK_ARG(c->dtype == dtype || c->dtype == P3D_E4M3, "p3d_paged_attention: queries must be of the cache's dtype");
  P3D_CHECK_ARG(c->dim <= 128, "p3d_paged_attention: head dim up to 128");
  P3D_CHECK_ARG(heads >= 1 && heads % c->kv_heads == 0 && heads <= 65535,
                "p3d_paged_attention: query heads must be a multiple of the cache's heads");
  P3D_CHECK_ARG(isfinite(scale) && scale > 0, "p3d_paged_attention: scale must be finite and positive");
  if (c->sequences == 0) return P3D_OK;
  P3D_CHECK_ARG(q && q_stride && lengths && out, "p3d_paged_attention: null argument");
  Params p = {*c, q, {q_stride[0], q_stride[1]}, dtype, heads, lengths, scale, out};
  paged_kernel<<<((int64_t)c->sequences * heads + kWarps - 1) / kWarps, kWarps * 32, 0, (cudaStream_t)stream>>>(p);
  P3D_LAUNCH_CHECK();
  return P3D_OK;
}

}  // extern "C"
