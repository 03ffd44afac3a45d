// Product of two e4m3 matrices with power-of-two scales for each block of 128 (see fp8.cu):
//     out[m, n] = sum over k of a[m, k] 2^ea[m, k / 128] b[n, k] 2^eb[n, k / 128]  (+ bias[n])
// Both operands lie along k.  The tensor cores take the scales themselves (tcgen05.mma, block-scaled 8-bit
// kind): products of e4m3 and their powers of two are exact in fp32, so nothing but the fp32
// accumulation and the last rounding is inexact, and no accumulator leaves TMEM before its tile is done.
//
// Two kernels share the scheme: warp 0 is the TMA producer (a ring of 128-column slices of the operands, 128-byte rows,
// SWIZZLE_128B, with the scale bytes of four slices when a new four begin), warp 1 the MMA issuer (it
// copies those bytes to TMEM, where one byte of a row's word scales one slice, and issues the
// products), the others the epilogue (one row a thread).  Producer and issuer run as whole warps on
// values that the compiler knows to be uniform, one elected lane issuing: as single threads they took
// about 600 cycles a slice to bring operands to uniform registers, more than the products.
//   pair kernel     256 x 256 (or 128) tiles of a pair of SMs, each holding half of either operand, CTAs
//                   walking tiles (or, where there are fewer tiles than pairs, parts of k, which go to fp32
//                   partials that a second kernel adds in order).  The accumulator of 256 columns has
//                   no room for a second beside the scales: the epilogue takes it to registers at
//                   once and frees it.  Rows go out through shared memory by TMA.  Measured on B200:
//                   16384 x 2048 x 8192 177 us (3.1 PFLOP/s), 16384 x 8192 x 2048 209 us (2.6),
//                   262144 x 768 x 192 122 us (bound by the 402 MB it writes: 105 us at the 3.8 TB/s of a fill).
//   narrow kernel   up to 128 rows of `a` (tokens of a decode step) are the N side: the weight's rows
//                   fill the 128 lanes and the token count only sets N.  The CTAs of a cluster each take a
//                   part of k and add them through each other's shared memory.  Up to 32 tokens
//                   may come unquantised.
//
// Every wait is bounded (2 s): on a timeout the kernel records an error bit (p3d_device_errors), drains its
// copies and MMAs and frees TMEM.
#include <algorithm>

#include "common.cuh"
#include "fp8_quant.cuh"
#include "kernels.cuh"
#include "sm100.cuh"
#include "tma_host.cuh"

namespace p3d {
namespace {

using namespace sm100;

__device__ unsigned g_fp8_errors = 0;

constexpr int kTileM = 128, kSlice = 128;
constexpr int kProducerWarp = 0, kMmaWarp = 1;
constexpr uint64_t kWaitNs = 2000000000ull;
constexpr int kMaxStages = 12;

// mbar_wait that first sleeps on the barrier for up to 2 x 20 us without counting: reading the timer takes
// longer than the wait for a ring's next stage should.
__device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity, unsigned role) {
  if (mbar_test_wait(bar, parity) || mbar_try_wait_sleep(bar, parity, 20000u) ||
      mbar_try_wait_sleep(bar, parity, 20000u))
    return true;
  return mbar_wait(bar, parity, &g_fp8_errors, kWaitNs, role);
}
// The same by a converged warp, with an answer that the compiler knows to be uniform: what follows then
// lives in uniform registers, which TMA and MMA instructions take their operands from.
__device__ __forceinline__ bool wait_warp(uint32_t bar, uint32_t parity, unsigned role) {
  return __all_sync(0xffffffffu, wait(bar, parity, role));
}

// In what follows a converged warp calls with uniform operands and one elected lane, always the same, issues.
__device__ __forceinline__ void expect_tx_warp(uint32_t bar, uint32_t bytes) {
  asm volatile(
      "{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
      "@e mbarrier.arrive.expect_tx.release.cta.shared::cta.b64 _, [%0], %1;\n\t}" ::"r"(bar),
      "r"(bytes)
      : "memory");
}
__device__ __forceinline__ void load_2d_warp(uint32_t dst, const CUtensorMap *map, uint32_t bar, int c0, int c1) {
  asm volatile(
      "{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
      "@e cp.async.bulk.tensor.2d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];\n\t}" ::
          "r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1)
      : "memory");
}
// D[tmem] (+)= A[smem desc] * B[smem desc]^T, e4m3, each row of A and of B times the power of two in its
// byte of the scale words in TMEM; K = 32.
__device__ __forceinline__ void mma_scaled_warp(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sa, uint32_t sb,
                                                uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred e, p;\n\telect.sync _|e, 0xffffffff;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate)
      : "memory");
}
// 32 rows of 16 bytes from shared memory to four columns of TMEM, repeated in every quarter of its lanes.
__device__ __forceinline__ void copy_scales_warp(uint32_t tmem, uint64_t desc) {
  asm volatile(
      "{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
      "@e tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;\n\t}" ::"r"(tmem),
      "l"(desc)
      : "memory");
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t in_cta(uint32_t smem, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem), "r"(rank));
  return r;
}

// Unswizzled descriptor of 512 scale bytes: 8-row groups of 16-byte rows, 128 bytes apart.
__device__ __forceinline__ uint64_t desc_scales(uint32_t smem) {
  return (uint64_t)((smem >> 4) & 0x3FFFu) | (uint64_t)(128 >> 4) << 32 | (uint64_t)1 << 46;
}

// Instruction descriptor: e4m3 operands along k, power-of-two scales; the byte of the scale words
// that a slice uses is or-ed in.
__host__ __device__ constexpr uint32_t idesc_scaled(int m, int n) {
  return (uint32_t)(n >> 3) << 17 | 1u << 23 | (uint32_t)(m >> 7) << 27;
}
__device__ __forceinline__ uint32_t scale_ids(int byte) { return (uint32_t)byte << 4 | (uint32_t)byte << 29; }

struct GemmParams {
  int rows, cols;
  int slices, last_steps;  // ceil(k / 128); ceil(k / 32) of the last one
  int tiles_m, tiles_n, splits;
  const uint8_t *scales_a, *scales_b;
  void *out;               // [rows, cols] of out_type, or the partials [splits][rows, cols] fp32
  int64_t pitch;           // elements between out's rows
  int64_t split_stride;    // elements between partials
  const void *bias;        // over out's columns, of bias_type, or null
  int out_type, bias_type, vector;   // vector: rows are whole, aligned 16-byte pieces
  int stages;
};

// Which tile and slices a unit is: units of one tile follow each other, tiles go down groups of eight
// tile rows so that the operands of CTAs at work together stay in L2.
struct Unit {
  int tm, tn, split, begin, end;
};
__device__ __forceinline__ Unit unit_of(const GemmParams &p, int u) {
  Unit r;
  r.split = u % p.splits;
  const int t = u / p.splits, group = 8 * p.tiles_n, g = t / group, in = t - g * group;
  const int height = min(8, p.tiles_m - 8 * g);
  r.tm = 8 * g + in % height;
  r.tn = in / height;
  r.begin = (int)((int64_t)p.slices * r.split / p.splits);
  r.end = (int)((int64_t)p.slices * (r.split + 1) / p.splits);
  return r;
}

// ------------------------------------------------------------------------ the narrow kernel
constexpr int kNarrowThreads = 192;   // producer, MMA issuer, four epilogue warps
constexpr int kMaxSplits = 8;         // CTAs of a cluster

// Up to BN rows of a (tokens) against 128 rows of b a CTA; the CTAs of a cluster each take a part of k.
// FUSED: a comes in its own type and the epilogue warps, which have nothing else to do yet, quantise this CTA's
// part of it into shared memory while the first slices of b are on their way.
struct NarrowParams {
  int rows, cols;          // of b (the weight) and of a (the tokens)
  int slices, last_steps;  // ceil(k / 128); ceil(k / 32) of the last one
  int64_t k;
  const uint8_t *scales_b, *scales_a;
  const void *x;           // FUSED: a [cols, k] of x_type
  int x_type, x_slices;    // slices of a that a CTA holds
  void *out;               // [cols, rows] of out_type
  const void *bias;
  int out_type, bias_type, stages;
};

// Blocks of x in slices [begin, end) into the layout that TMA would give them: 128-byte rows, 16-byte piece j of row r
// at j ^ (r % 8); scale bytes in the order of fp8.cu's, from group begin / 4 on.
template <typename T, int BN>
__device__ __forceinline__ void quantize_tokens(const NarrowParams &p, char *values, char *scales, int begin, int end, int t) {
  using namespace quant;
  const bool aligned = p.k % 8 == 0 && (reinterpret_cast<uintptr_t>(p.x) & 15) == 0;
  const int sub = t & 15, n = end - begin, total = p.cols * n;
  for (int i0 = 0; i0 < total; i0 += 8) {   // eight blocks at a time, a half warp each
    const int i = i0 + t / 16, row = i / n, kb = i - row * n + begin;
    const bool inside = i < total;
    const T *x = static_cast<const T *>(p.x) + (int64_t)(inside ? row : 0) * p.k;
    const int64_t col = inside ? (int64_t)kb * kSlice + sub * 8 : p.k;
    const Raw<T> r = aligned ? load8<T, true>(x, col, p.k) : load8<T, false>(x, col, p.k);
    bool odd;
    const uint32_t byte = scale_byte(block_amax<T>(r, &odd));
    if (inside) {
      const float inv = inverse_scale(byte);
      const uint2 v = odd ? quantize8<true, T>(r, inv) : quantize8<false, T>(r, inv);
      char *at = values + (kb - begin) * (BN * kSlice) + row * kSlice;
      *reinterpret_cast<uint2 *>(at + (((sub >> 1) ^ (row & 7)) * 16) + (sub & 1) * 8) = v;
      if (sub == 0) scales[(kb / 4 - begin / 4) * 512 + (row % 32) * 16 + row / 32 * 4 + kb % 4] = (char)byte;
    }
  }
}

template <int BN, bool FUSED>
__global__ void __launch_bounds__(kNarrowThreads, 1)
    fp8_narrow_kernel(const __grid_constant__ CUtensorMap tb, const __grid_constant__ CUtensorMap ta, const NarrowParams p) {
  constexpr uint32_t kBytesW = kTileM * kSlice, kBytesX = FUSED ? 0 : BN * kSlice;
  constexpr uint32_t kStageBytes = kBytesW + kBytesX + 1024u;   // and the scale bytes of either
  constexpr int kAccCols = BN < 32 ? 32 : BN, kUsed = kAccCols + 16;
  constexpr int kTmemCols = kUsed <= 64 ? 64 : kUsed <= 128 ? 128 : 256;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  __shared__ __align__(8) uint64_t s_bars[2 * kMaxStages + 2];
  __shared__ uint32_t tmem_holder;
  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  uint32_t splits;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(splits));
  const uint32_t split = __shfl_sync(0xffffffffu, cluster_rank(), 0);
  const int tile = blockIdx.x / splits;
  const int begin = (int)((int64_t)p.slices * split / splits), end = (int)((int64_t)p.slices * (split + 1) / splits);
  const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
  const uint32_t bars = smem_u32(s_bars);
  const int S = p.stages;
  const uint32_t x_at = base + S * kStageBytes, xs_at = x_at + p.x_slices * (BN * kSlice);   // FUSED
  auto full = [&](int s) { return bars + 8u * s; };
  auto empty = [&](int s) { return bars + 8u * (kMaxStages + s); };
  const uint32_t acc_full = bars + 8u * (2 * kMaxStages), x_full = acc_full + 8u;
  const int groups = (p.slices + 3) / 4;

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), 1);
    }
    mbar_init(acc_full, 1);
    mbar_init(x_full, 4);
    fence_mbar_init();
  }
  if (warp == kMmaWarp) {
    tmem_alloc(smem_u32(&tmem_holder), kTmemCols);
    tmem_relinquish();
  }
  if (warp == kProducerWarp && lane == 0) {
    prefetch_tmap(&tb);
    if (!FUSED) prefetch_tmap(&ta);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_holder, 0);

  bool done = true;   // of the epilogue warps: the products are there
  if (warp == kProducerWarp) {
    // ------------------------------------------------------------------ TMA producer
    int s = 0, it = 0;
    uint32_t turn = 1;
    for (int kb = begin; kb < end; ++kb, ++it) {
      if (it >= S && !wait_warp(empty(s), turn, kErrProducer)) break;
      const uint32_t st = base + s * kStageBytes, at = st + kBytesW + kBytesX;
      const bool scales = kb == begin || kb % 4 == 0;
      expect_tx_warp(full(s), kBytesW + kBytesX + (scales ? (FUSED ? 512u : 1024u) : 0u));
      load_2d_warp(st, &tb, full(s), kb * kSlice, tile * kTileM);
      if (!FUSED) load_2d_warp(st + kBytesW, &ta, full(s), kb * kSlice, 0);
      if (scales && lane == 0) {
        bulk_load(at, p.scales_b + ((int64_t)tile * groups + kb / 4) * 512, 512u, full(s));
        if (!FUSED) bulk_load(at + 512u, p.scales_a + (int64_t)(kb / 4) * 512, 512u, full(s));
      }
      __syncwarp();
      if (++s == S) {
        s = 0;
        turn ^= 1;
      }
    }
    // every stage used: its products are done, so its copies are too
    for (int i = it > S ? it - S : 0; i < it; ++i)
      mbar_wait(empty(i % S), (i / S) & 1, &g_fp8_errors, kWaitNs, kErrTeardown);
  } else if (warp == kMmaWarp) {
    // ------------------------------------------------------------------ MMA issuer
    constexpr uint32_t idesc = idesc_scaled(kTileM, BN);
    const uint32_t scale_cols = tmem + kAccCols;
    const uint64_t desc_w = desc_sw128(base, 1024), desc_x = desc_sw128(FUSED ? x_at : base + kBytesW, 1024);
    const uint64_t desc_s = desc_scales(base + kBytesW + kBytesX), desc_xs = desc_scales(FUSED ? xs_at : 0u);
    bool ok = !FUSED || wait_warp(x_full, 0, kErrMma);
    int s = 0, copied = 0;
    uint32_t turn = 0;
    for (int kb = begin; ok && kb < end; ++kb) {
      ok = wait_warp(full(s), turn, kErrMma);
      if (!ok) break;
      tc_fence_after();
      const uint64_t off = (uint64_t)(s * kStageBytes >> 4);
      if (kb == begin || kb % 4 == 0) {
        // the other buffer: products of the four slices before may still read theirs
        const uint32_t to = scale_cols + (copied & 1) * 8;
        copy_scales_warp(to, desc_s + off);
        copy_scales_warp(to + 4, FUSED ? desc_xs + (uint64_t)((kb / 4 - begin / 4) * 512 >> 4) : desc_s + off + 32u);
        ++copied;
      }
      const uint32_t sc = scale_cols + ((copied - 1) & 1) * 8, id = idesc | scale_ids(kb % 4);
      const uint64_t x_off = FUSED ? (uint64_t)((kb - begin) * (BN * kSlice) >> 4) : off;
      // 32 columns: 32 bytes along the 128-byte rows; the last slice may have fewer than four
      const int steps = kb + 1 < p.slices ? 4 : p.last_steps;
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (k < steps)
          mma_scaled_warp(tmem, desc_w + off + 2 * k, desc_x + x_off + 2 * k, id, sc, sc + 4, kb > begin || k > 0 ? 1u : 0u);
      mma_commit_warp(empty(s));
      if (++s == S) {
        s = 0;
        turn ^= 1;
      }
    }
    mma_commit_warp(acc_full);
    mbar_wait(acc_full, 0, &g_fp8_errors, kWaitNs, kErrTeardown);
  } else {
    // ------------------------------------------------------------------ quantiser, then epilogue
    if constexpr (FUSED) {
      const int t = threadIdx.x - 64;
      char *const values = reinterpret_cast<char *>(smem_raw) + (x_at - raw);
      char *const scales = reinterpret_cast<char *>(smem_raw) + (xs_at - raw);
      if (p.x_type == P3D_BF16) quantize_tokens<__nv_bfloat16, BN>(p, values, scales, begin, end, t);
      else if (p.x_type == P3D_F16) quantize_tokens<__half, BN>(p, values, scales, begin, end, t);
      else quantize_tokens<float, BN>(p, values, scales, begin, end, t);
      fence_proxy_async_smem();   // written here, read by the tensor core
      __syncwarp();
      if (lane == 0) mbar_arrive(x_full);
    }
    done = __all_sync(0xffffffffu, wait(acc_full, 0, kErrSoftmax));
    tc_fence_after();
  }
  // a thread's row of b; columns are tokens
  const int quarter = warp & 3, r = quarter * 32 + lane, row = tile * kTileM + r;
  const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
  float *const part = reinterpret_cast<float *>(smem_raw + (base - raw));   // [BN][128], over the ring, which is done with
  const float add = warp >= 2 && p.bias && row < p.rows ? load_any(p.bias, p.bias_type, row) : 0.f;
  if (warp >= 2 && done) {
#pragma unroll 1
    for (int c0 = 0; c0 < p.cols; c0 += 32) {
      uint32_t v[32];
      tmem_ld32(lanes + c0, v);
      tmem_wait_ld();
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (c0 + j < p.cols) {
          if (splits > 1) part[(c0 + j) * kTileM + r] = __uint_as_float(v[j]);
          else if (row < p.rows) store_any(p.out, p.out_type, (int64_t)(c0 + j) * p.rows + row, __uint_as_float(v[j]) + add);
        }
      __syncwarp();
    }
  }
  __syncwarp();
  tc_fence_before();
  if (splits > 1) {
    // tokens split, split + splits, ..: the parts of k in order, from each CTA's shared memory
    cluster_sync();
    if (warp >= 2 && done && row < p.rows) {
      for (int c = split; c < p.cols; c += splits) {
        const uint32_t at = smem_u32(part + c * kTileM + r);
        float sum = 0.f;
        for (uint32_t q = 0; q < splits; ++q) {
          float v;
          asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(in_cta(at, q)) : "memory");
          sum += v;
        }
        store_any(p.out, p.out_type, (int64_t)c * p.rows + row, sum + add);
      }
    }
    __syncwarp();
    cluster_sync();   // nobody reads this CTA's shared memory any more
  }
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

// ------------------------------------------------------------------------ the pair kernel
constexpr int kPairRows = 256;
constexpr int kWarpCols = 64;          // columns of an epilogue warp
constexpr int epilogue_warps(int bn) { return 4 * bn / kWarpCols; }

__device__ __forceinline__ void arrive_at(uint32_t cluster_bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_bar) : "memory");
}
// A warp's wait on arrivals of the other CTA too (acquired over the cluster).
__device__ __forceinline__ bool wait_cluster(uint32_t bar, uint32_t parity, unsigned role) {
  const bool ok = wait(bar, parity, role);
  uint32_t done;   // the phase is over: this only orders
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done)
      : "r"(bar), "r"(parity)
      : "memory");
  return __all_sync(0xffffffffu, ok && done);
}
// Into this CTA's shared memory, signalling a barrier of the pair's first CTA.
__device__ __forceinline__ void pair_load_2d(uint32_t dst, const CUtensorMap *map, uint32_t bar, int c0, int c1) {
  asm volatile(
      "{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
      "@e cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, "
      "%4}], [%2];\n\t}" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1)
      : "memory");
}
__device__ __forceinline__ void store_3d(const CUtensorMap *map, uint32_t src, int c0, int c1, int c2) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(src), "r"(c0), "r"(c1), "r"(c2)
               : "memory");
}
__device__ __forceinline__ void pair_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sa, uint32_t sb,
                                         uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred e, p;\n\telect.sync _|e, 0xffffffff;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "@e tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void pair_copy_scales(uint32_t tmem, uint64_t desc) {
  asm volatile(
      "{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
      "@e tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;\n\t}" ::"r"(tmem),
      "l"(desc)
      : "memory");
}
// Arrives at the same barrier of both CTAs once all MMAs and copies issued so far are done.
__device__ __forceinline__ void pair_commit(uint32_t bar) {
  asm volatile(
      "{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
      "@e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n\t}" ::"r"(bar),
      "h"((uint16_t)3)
      : "memory");
}

constexpr int kStageRow = 64;   // bytes of a row that the epilogue stages at a time (what leaves room for five stages)

// 16-byte pieces of a thread's row segment, as the 64-byte swizzle lays them out, from fp32 values.
template <typename T>
__device__ __forceinline__ void stage_row(char *row_base, int row, const float *v) {
  constexpr int n = 16 / sizeof(T);
#pragma unroll
  for (int i = 0; i < kStageRow / 16; ++i) {
    uint4 w;
    if constexpr (sizeof(T) == 4) {
      w = make_uint4(__float_as_uint(v[4 * i]), __float_as_uint(v[4 * i + 1]), __float_as_uint(v[4 * i + 2]),
                     __float_as_uint(v[4 * i + 3]));
    } else {
      uint32_t h[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (std::is_same<T, __nv_bfloat16>::value) h[j] = pack_bf16(v[n * i + 2 * j], v[n * i + 2 * j + 1]);
        else h[j] = pack_f16(v[n * i + 2 * j], v[n * i + 2 * j + 1]);
      }
      w = make_uint4(h[0], h[1], h[2], h[3]);
    }
    *reinterpret_cast<uint4 *>(row_base + ((i ^ (row >> 1 & 3)) * 16)) = w;
  }
}

// A warp's 32 rows x 64 columns through shared memory, BOXES times 64 bytes of every row at a time.  Boxes end at
// out's own rows and columns.
template <typename T, int BOXES>
__device__ __forceinline__ void pair_epilogue(const CUtensorMap *tout, const GemmParams &p, const Unit &w,
                                              const float (&v)[kWarpCols], int row0, int col0, int lane, char *stage) {
  constexpr int kCols = kStageRow / sizeof(T), kBox = 32 * kStageRow;
  if (p.vector) {
#pragma unroll
    for (int c = 0; c < kWarpCols; c += kCols * BOXES) {
      if (col0 + c >= p.cols || row0 >= p.rows) break;   // the same in the whole warp
      if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
      __syncwarp();
#pragma unroll
      for (int b = 0; b < BOXES; ++b) stage_row<T>(stage + b * kBox + lane * kStageRow, lane, v + c + b * kCols);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
#pragma unroll
        for (int b = 0; b < BOXES; ++b)
          if (b == 0 || col0 + c + b * kCols < p.cols)
            store_3d(tout, smem_u32(stage) + b * kBox, col0 + c + b * kCols, row0, w.split);
        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
      }
    }
  } else if (row0 + lane < p.rows) {
    T *dst = static_cast<T *>(p.out) + (int64_t)(row0 + lane) * p.pitch + col0 + (int64_t)w.split * p.split_stride;
#pragma unroll
    for (int j = 0; j < kWarpCols; ++j)
      if (col0 + j < p.cols) dst[j] = from_f32<T>(v[j]);
  }
}

template <int BN, int BOXES>
__global__ void __launch_bounds__(64 + 32 * epilogue_warps(BN), 1) __cluster_dims__(2, 1, 1)
    fp8_pair_kernel(const __grid_constant__ CUtensorMap ta, const __grid_constant__ CUtensorMap tb,
                    const __grid_constant__ CUtensorMap tsa, const __grid_constant__ CUtensorMap tsb,
                    const __grid_constant__ CUtensorMap tout, const GemmParams p) {
  constexpr int kChunksB = BN / 128;
  constexpr uint32_t kBytesA = kTileM * kSlice, kBytesB = BN / 2 * kSlice, kBytesS = 512u * (1 + kChunksB);
  constexpr uint32_t kStageBytes = kBytesA + kBytesB + 2048u;   // the scale bytes in the last 2048
  constexpr int kScaleCols = 4 + 4 * kChunksB;
  constexpr int kAccs = 2 * BN + 2 * kScaleCols <= 512 ? 2 : 1;
  constexpr int kTmemCols = 512;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  __shared__ __align__(8) uint64_t s_bars[2 * kMaxStages + 5];
  __shared__ uint32_t tmem_holder;
  __shared__ __align__(16) float s_bias[epilogue_warps(BN)][kWarpCols];
  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t rank = __shfl_sync(0xffffffffu, cluster_rank(), 0);
  const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
  const uint32_t bars = smem_u32(s_bars);
  const int S = p.stages;
  auto full = [&](int s) { return bars + 8u * s; };      // the first CTA's, for both
  auto empty = [&](int s) { return bars + 8u * (kMaxStages + s); };
  auto acc_full = [&](int a) { return bars + 8u * (2 * kMaxStages + a); };
  auto acc_empty = [&](int a) { return bars + 8u * (2 * kMaxStages + 2 + a); };   // the first CTA's, for both
  const uint32_t drain = bars + 8u * (2 * kMaxStages + 4);
  const int units = p.tiles_m * p.tiles_n * p.splits, pairs = gridDim.x / 2, pair = blockIdx.x / 2;

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(acc_full(a), 1);
      mbar_init(acc_empty(a), 2 * epilogue_warps(BN));
    }
    mbar_init(drain, 1);
    fence_mbar_init();
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_holder)),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  if (warp == kProducerWarp && lane == 0) {
    prefetch_tmap(&ta);
    prefetch_tmap(&tb);
    prefetch_tmap(&tsa);
    prefetch_tmap(&tsb);
    if (p.vector) prefetch_tmap(&tout);
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem = tmem_holder;

  if (warp == kProducerWarp) {
    // ------------------------------------------------------------------ TMA producer, one in each CTA
    const int groups = (p.slices + 3) / 4;
    const uint32_t full0 = in_cta(bars, 0);   // the first CTA's full barriers
    int it = 0, s = 0;
    uint32_t turn = 1;   // parity of the empty phase to wait for
    bool ok = true;
    for (int u = pair; ok && u < units; u += pairs) {
      const Unit w = unit_of(p, u);
      const int m0 = 2 * w.tm + (int)rank;   // this CTA's 128 rows; past the end everything reads as zero
      const int rows_b = w.tn * BN + (int)rank * (BN / 2);
      for (int kb = w.begin; kb < w.end; ++kb, ++it) {
        if (it >= S && !wait_warp(empty(s), turn, kErrProducer)) {
          ok = false;
          break;
        }
        const uint32_t st = base + s * kStageBytes, bar = full0 + 8u * s;
        const bool scales = kb == w.begin || kb % 4 == 0;
        if (rank == 0) expect_tx_warp(full(s), 2 * (kBytesA + kBytesB + (scales ? kBytesS : 0u)));
        pair_load_2d(st, &ta, bar, kb * kSlice, m0 * 128);
        pair_load_2d(st + kBytesA, &tb, bar, kb * kSlice, rows_b);
        if (scales) {
          const uint32_t at = st + kStageBytes - 2048u;
          pair_load_2d(at, &tsa, bar, 0, m0 * groups + kb / 4);
#pragma unroll
          for (int c = 0; c < kChunksB; ++c)
            pair_load_2d(at + 512u * (1 + c), &tsb, bar, 0, (w.tn * kChunksB + c) * groups + kb / 4);
        }
        if (++s == S) {
          s = 0;
          turn ^= 1;
        }
      }
    }
    // every stage used: its products are done, so its copies are too
    for (int i = it > S ? it - S : 0; i < it; ++i)
      mbar_wait(empty(i % S), (i / S) & 1, &g_fp8_errors, kWaitNs, kErrTeardown);
  } else if (warp == kMmaWarp) {
    // ------------------------------------------------------------------ MMA issuer, of the first CTA for both
    if (rank == 0) {
      constexpr uint32_t idesc = idesc_scaled(kPairRows, BN);
      const uint32_t acc = __shfl_sync(0xffffffffu, tmem, 0), scale_cols = acc + kAccs * BN;
      const uint64_t desc_a = desc_sw128(base, 1024), desc_b = desc_sw128(base + kBytesA, 1024);
      const uint64_t desc_s = desc_scales(base + kStageBytes - 2048u);
      int n = 0, groups = 0, s = 0;
      uint32_t turn = 0;
      bool ok = true;
      for (int u = pair; ok && u < units; u += pairs, ++n) {
        const Unit w = unit_of(p, u);
        const int a = n % kAccs;
        if (n >= kAccs && !wait_cluster(acc_empty(a), (n / kAccs - 1) & 1, kErrMma)) break;
        tc_fence_after();
        for (int kb = w.begin; kb < w.end; ++kb) {
          if (!wait_warp(full(s), turn, kErrMma)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint64_t off = (uint64_t)(s * kStageBytes >> 4);
          if (kb == w.begin || kb % 4 == 0) {
            // the other buffer: products of the four slices before may still read theirs
            const uint32_t to = scale_cols + (groups & 1) * kScaleCols;
#pragma unroll
            for (int c = 0; c < 1 + kChunksB; ++c) pair_copy_scales(to + 4 * c, desc_s + off + 32u * c);
            ++groups;
          }
          const uint32_t sc = scale_cols + ((groups - 1) & 1) * kScaleCols;
          const uint32_t id = idesc | scale_ids(kb % 4);
          // 32 columns: 32 bytes along the 128-byte rows; the last slice may have fewer than four
          const int steps = kb + 1 < p.slices ? 4 : p.last_steps;
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (k < steps) pair_mma(acc + a * BN, desc_a + off + 2 * k, desc_b + off + 2 * k, id, sc, sc + 4,
                     kb > w.begin || k > 0 ? 1u : 0u);
          pair_commit(empty(s));
          if (++s == S) {
            s = 0;
            turn ^= 1;
          }
        }
        if (!ok) break;
        pair_commit(acc_full(a));
      }
      pair_commit(drain);
      mbar_wait(drain, 0, &g_fp8_errors, kWaitNs, kErrTeardown);
    }
  } else {
    // ------------------------------------------------------------------ epilogue
    const int quarter = warp & 3, part = (warp - 2) >> 2;   // TMEM lanes and columns of this warp
    const uint32_t from = tmem + ((uint32_t)(quarter * 32) << 16) + part * kWarpCols;
    char *const stage = reinterpret_cast<char *>(smem_raw) + (base - raw) + S * kStageBytes + (warp - 2) * BOXES * 32 * kStageRow;
    float *const bias = s_bias[warp - 2];
    int n = 0;
    for (int u = pair; u < units; u += pairs, ++n) {
      const Unit w = unit_of(p, u);
      const int a = n % kAccs;
      const int row0 = w.tm * kPairRows + (int)rank * 128 + quarter * 32, col0 = w.tn * BN + part * kWarpCols;
      if (p.bias) {
#pragma unroll
        for (int i = lane; i < kWarpCols; i += 32)
          bias[i] = col0 + i < p.cols ? load_any(p.bias, p.bias_type, col0 + i) : 0.f;
      }
      const bool ready = wait(acc_full(a), (n / kAccs) & 1, kErrSoftmax);
      if (!__all_sync(0xffffffffu, ready)) break;
      tc_fence_after();
      uint32_t r[kWarpCols];
#pragma unroll
      for (int c = 0; c < kWarpCols; c += 32) tmem_ld32(from + a * BN + c, r + c);
      tmem_wait_ld();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) arrive_at(in_cta(acc_empty(a), 0));
      float v[kWarpCols];
#pragma unroll
      for (int j = 0; j < kWarpCols; ++j) v[j] = __uint_as_float(r[j]);
      if (p.bias) {
#pragma unroll
        for (int j = 0; j < kWarpCols; j += 4) {
          const float4 b = *reinterpret_cast<const float4 *>(bias + j);
          v[j] += b.x;
          v[j + 1] += b.y;
          v[j + 2] += b.z;
          v[j + 3] += b.w;
        }
      }
      if (p.out_type == P3D_BF16) pair_epilogue<__nv_bfloat16, BOXES>(&tout, p, w, v, row0, col0, lane, stage);
      else if (p.out_type == P3D_F16) pair_epilogue<__half, BOXES>(&tout, p, w, v, row0, col0, lane, stage);
      else pair_epilogue<float, BOXES>(&tout, p, w, v, row0, col0, lane, stage);
      __syncwarp();
    }
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  cluster_sync();   // the other CTA's barriers, shared memory and TMEM are in use until here
  if (warp == kMmaWarp) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
  }
}

// out = the partials added in slice order, plus the bias.
__global__ void __launch_bounds__(256) add_splits_kernel(const float *part, int splits, int64_t rows, int64_t cols,
                                                         const void *bias, int bias_type, void *out, int out_type,
                                                         int64_t pitch) {
  const int64_t total = rows * cols, step = (int64_t)gridDim.x * blockDim.x;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += step) {
    const int64_t r = i / cols, c = i - r * cols;
    float v = part[i];
    for (int s = 1; s < splits; ++s) v += part[s * total + i];
    if (bias) v += load_any(bias, bias_type, c);
    store_any(out, out_type, r * pitch + c, v);
  }
}

struct Plan {
  int bn;
  bool pair;
  int tiles_m, tiles_n, splits;
};

// Up to 128 rows (tokens) are the narrow kernel's; more go to the pair kernel, with the narrower tile where that
// makes less work of the last wave (a tile costs its columns and about 64 more for filling the
// pipeline).  Splits: as many parts of k as fill the SMs, each of at least two 128-column slices (four for
// a pair); the narrow kernel's are a cluster, at most eight.  The pair kernel's parts cost a second kernel
// (5 us with its launch, as long as about 30 slices): they have to save more.
constexpr int kWorthSplitting = 32;
Plan plan_of(int64_t rows, int64_t cols, int64_t k, int sms) {
  Plan p;
  const int64_t slices = (k + kSlice - 1) / kSlice;
  p.pair = rows > 128;
  if (!p.pair) {
    p.bn = rows <= 16 ? 16 : rows <= 32 ? 32 : rows <= 64 ? 64 : 128;
    p.tiles_m = (int)((cols + kTileM - 1) / kTileM);
    p.tiles_n = 1;
    p.splits = 1;
    while (p.splits < kMaxSplits && (int64_t)p.tiles_m * p.splits * 2 <= sms && slices >= 4 * p.splits) p.splits *= 2;
    return p;
  }
  const int64_t slots = sms / 2;
  p.tiles_m = (int)((rows + kPairRows - 1) / kPairRows);
  auto cost = [&](int bn) { return (p.tiles_m * ((cols + bn - 1) / bn) + slots - 1) / slots * (bn + 64); };
  p.bn = cost(128) < cost(256) ? 128 : 256;
  p.tiles_n = (int)((cols + p.bn - 1) / p.bn);
  const int64_t tiles = (int64_t)p.tiles_m * p.tiles_n;
  p.splits = (int)std::max<int64_t>(1, std::min<int64_t>({slots / std::max<int64_t>(1, tiles), slices / 4, 64}));
  if (slices - slices / p.splits < kWorthSplitting) p.splits = 1;
  return p;
}

size_t partial_bytes(const Plan &p, int64_t rows, int64_t cols) {
  return p.pair && p.splits > 1 ? (size_t)p.splits * rows * cols * sizeof(float) : 0;
}

template <int BN, int BOXES>
int launch_pair(const CUtensorMap &ta, const CUtensorMap &tb, const CUtensorMap &tsa, const CUtensorMap &tsb,
                const CUtensorMap &tout, GemmParams g, int sms, cudaStream_t s) {
  constexpr size_t stage = kTileM * kSlice + BN / 2 * kSlice + 2048, staging = epilogue_warps(BN) * BOXES * 32 * kStageRow;
  g.stages = (int)std::min<size_t>(kMaxStages, (220 * 1024 - staging - 1024) / stage);
  const size_t smem = g.stages * stage + staging + 1024;
  static size_t seen[kMaxDevices] = {};
  if (int st = smem_optin(fp8_pair_kernel<BN, BOXES>, smem, seen)) return st;
  const int64_t units = (int64_t)g.tiles_m * g.tiles_n * g.splits;
  const unsigned grid = 2u * (unsigned)std::min<int64_t>(units, sms / 2);
  fp8_pair_kernel<BN, BOXES><<<grid, 64 + 32 * epilogue_warps(BN), smem, s>>>(ta, tb, tsa, tsb, tout, g);
  P3D_LAUNCH_CHECK();
  return P3D_OK;
}

// What a narrow launch holds: a ring of at least three stages and, fused, its part of the tokens.
template <int BN, bool FUSED>
int launch_narrow(const CUtensorMap &tb, const CUtensorMap &ta, NarrowParams g, int tiles, int splits, cudaStream_t s) {
  constexpr size_t stage = kTileM * kSlice + (FUSED ? 0 : BN * kSlice) + 1024;
  const size_t x_bytes = FUSED ? (size_t)g.x_slices * BN * kSlice + ((size_t)g.x_slices / 4 + 2) * 512 : 0;
  const size_t part = (size_t)BN * kTileM * sizeof(float);
  g.stages = (int)std::min<size_t>(kMaxStages, (216 * 1024 - 1024 - x_bytes) / stage);
  const size_t smem = std::max(g.stages * stage + x_bytes, splits > 1 ? part : (size_t)0) + 1024;
  static size_t seen[kMaxDevices] = {};
  // always the same amount: calls of several threads then cannot lower each other's
  if (int st = smem_optin(fp8_narrow_kernel<BN, FUSED>, std::max<size_t>(smem, 224 * 1024), seen)) return st;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(tiles * splits));
  cfg.blockDim = dim3(kNarrowThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)splits;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  P3D_CUDA_TRY(cudaLaunchKernelEx(&cfg, fp8_narrow_kernel<BN, FUSED>, tb, ta, g));
  return P3D_OK;
}

int check_extents(int64_t rows, int64_t cols, int64_t k, const char *what) {
  P3D_CHECK_ARG(rows >= 1 && cols >= 1 && k >= 1, "%s: extents must be positive", what);
  const int64_t most = (int64_t)1 << 30;
  if (rows > most || cols > most || k > most || ((rows + 127) / 128) * ((cols + 127) / 128) > most)
    return fail(P3D_ERR_UNSUPPORTED, "%s: extents too large", what);
  return P3D_OK;
}

}  // namespace

int take_fp8_errors(unsigned *flags) {
  unsigned v = 0, zero = 0;
  P3D_CUDA_TRY(cudaMemcpyFromSymbol(&v, g_fp8_errors, sizeof(v)));
  P3D_CUDA_TRY(cudaMemcpyToSymbol(g_fp8_errors, &zero, sizeof(zero)));
  *flags |= v;
  return P3D_OK;
}

}  // namespace p3d

using namespace p3d;

namespace {

// The narrow product: tokens a (8-bit, with a_scales) or x (of x_type), against b.
int run_narrow(const Plan &p, const void *x, int x_type, const void *a, int64_t a_pitch, const void *a_scales, const void *b,
               int64_t b_pitch, const void *b_scales, int64_t rows, int64_t cols, int64_t k, const void *bias,
               int bias_type, void *out, int out_type, cudaStream_t s) {
  CUtensorMap tb, ta = {};
  {
    const uint64_t dims[2] = {(uint64_t)k, (uint64_t)cols}, strides[1] = {(uint64_t)b_pitch};
    const uint32_t box[2] = {kSlice, kTileM};
    if (int st = encode_tiled(&tb, CU_TENSOR_MAP_DATA_TYPE_UINT8, b, 2, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B)) return st;
  }
  if (!x) {
    const uint64_t dims[2] = {(uint64_t)k, (uint64_t)rows}, strides[1] = {(uint64_t)a_pitch};
    const uint32_t box[2] = {kSlice, (uint32_t)p.bn};
    if (int st = encode_tiled(&ta, CU_TENSOR_MAP_DATA_TYPE_UINT8, a, 2, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B)) return st;
  }
  NarrowParams g = {};
  g.rows = (int)cols;
  g.cols = (int)rows;
  g.k = k;
  g.slices = (int)((k + kSlice - 1) / kSlice);
  g.last_steps = (int)((k - (int64_t)(g.slices - 1) * kSlice + 31) / 32);
  g.scales_b = static_cast<const uint8_t *>(b_scales);
  g.scales_a = static_cast<const uint8_t *>(a_scales);
  g.x = x;
  g.x_type = x_type;
  g.x_slices = x ? (g.slices + p.splits - 1) / p.splits : 0;
  g.out = out;
  g.out_type = out_type;
  g.bias = bias;
  g.bias_type = bias_type;
  if (x) return p.bn == 16 ? launch_narrow<16, true>(tb, ta, g, p.tiles_m, p.splits, s)
                           : launch_narrow<32, true>(tb, ta, g, p.tiles_m, p.splits, s);
  switch (p.bn) {
    case 16: return launch_narrow<16, false>(tb, ta, g, p.tiles_m, p.splits, s);
    case 32: return launch_narrow<32, false>(tb, ta, g, p.tiles_m, p.splits, s);
    case 64: return launch_narrow<64, false>(tb, ta, g, p.tiles_m, p.splits, s);
    default: return launch_narrow<128, false>(tb, ta, g, p.tiles_m, p.splits, s);
  }
}

}  // namespace

namespace p3d {

// Whether launch_fp8_tokens takes these extents: up to 32 tokens of which a CTA's part fits beside the ring, and few
// enough weight tiles that quantising the tokens in each of them does not outweigh the launch that it saves.
bool fp8_tokens_fit(int64_t rows, int64_t cols, int64_t k) {
  DeviceInfo info;
  if (rows > 32 || check_extents(rows, cols, k, "p3d_fp8_linear_fwd") || device_info(&info)) return false;
  const Plan p = plan_of(rows, cols, k, info.sm_count);
  const int64_t slices = ((k + kSlice - 1) / kSlice + p.splits - 1) / p.splits;
  return slices * p.bn * kSlice <= 64 * 1024 && rows * slices <= 256 && p.tiles_m * p.splits <= 2 * info.sm_count;
}

int launch_fp8_tokens(const void *x, int x_type, const void *b, int64_t b_pitch, const void *b_scales, int64_t rows,
                      int64_t cols, int64_t k, const void *bias, int bias_type, void *out, int out_type, cudaStream_t s) {
  DeviceInfo info;
  if (int st = device_info(&info)) return st;
  if (info.major != 10) return fail(P3D_ERR_DEVICE, "p3d_fp8_linear_fwd needs an sm_100 device");
  P3D_CHECK_ARG(b_pitch >= k && b_pitch % 16 == 0 && (((uintptr_t)b | (uintptr_t)b_scales) & 15) == 0,
                "p3d_fp8_linear_fwd: the weight's pitch must be a multiple of 16 and hold k columns, aligned to 16 bytes");
  return run_narrow(plan_of(rows, cols, k, info.sm_count), x, x_type, nullptr, 0, nullptr, b, b_pitch, b_scales, rows, cols, k,
                    bias, bias_type, out, out_type, s);
}

}  // namespace p3d

extern "C" size_t p3d_fp8_matmul_workspace(int64_t rows, int64_t cols, int64_t k) {
  DeviceInfo info;
  if (check_extents(rows, cols, k, "p3d_fp8_matmul_workspace") || device_info(&info)) return 0;
  return partial_bytes(plan_of(rows, cols, k, info.sm_count), rows, cols);
}

extern "C" int p3d_fp8_matmul(const void *a, int64_t a_pitch, const void *a_scales, const void *b, int64_t b_pitch,
                              const void *b_scales, int64_t rows, int64_t cols, int64_t k, const void *bias,
                              int bias_dtype, void *out, int out_dtype, void *workspace, size_t workspace_bytes,
                              void *stream) {
  if (int st = check_extents(rows, cols, k, "p3d_fp8_matmul")) return st;
  P3D_CHECK_ARG(a && a_scales && b && b_scales && out, "p3d_fp8_matmul: null pointer");
  P3D_CHECK_ARG(dtype_ok(out_dtype) && (!bias || dtype_ok(bias_dtype)), "p3d_fp8_matmul: unknown dtype");
  P3D_CHECK_ARG(a_pitch >= k && b_pitch >= k && a_pitch % 16 == 0 && b_pitch % 16 == 0,
                "p3d_fp8_matmul: pitches must be multiples of 16 and hold k columns");
  P3D_CHECK_ARG((((uintptr_t)a | (uintptr_t)b | (uintptr_t)a_scales | (uintptr_t)b_scales | (uintptr_t)workspace) & 15) == 0,
                "p3d_fp8_matmul: operands, scales and workspace must be 16-byte aligned");
  DeviceInfo info;
  if (int st = device_info(&info)) return st;
  if (info.major != 10) return fail(P3D_ERR_DEVICE, "p3d_fp8_matmul needs an sm_100 device");
  const Plan p = plan_of(rows, cols, k, info.sm_count);
  const size_t need = partial_bytes(p, rows, cols);
  if (need && (!workspace || workspace_bytes < need))
    return fail(P3D_ERR_WORKSPACE, "p3d_fp8_matmul: workspace of %zu bytes, %zu needed", workspace_bytes, need);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (!p.pair)
    return run_narrow(p, nullptr, 0, a, a_pitch, a_scales, b, b_pitch, b_scales, rows, cols, k, bias, bias_dtype, out, out_dtype,
                      s);
  CUtensorMap ta, tb;
  {
    const uint64_t dims[2] = {(uint64_t)k, (uint64_t)rows}, strides[1] = {(uint64_t)a_pitch};
    const uint32_t box[2] = {kSlice, kTileM};
    if (int st = encode_tiled(&ta, CU_TENSOR_MAP_DATA_TYPE_UINT8, a, 2, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B)) return st;
  }
  {
    const uint64_t dims[2] = {(uint64_t)k, (uint64_t)cols}, strides[1] = {(uint64_t)b_pitch};
    const uint32_t box[2] = {kSlice, (uint32_t)p.bn / 2};
    if (int st = encode_tiled(&tb, CU_TENSOR_MAP_DATA_TYPE_UINT8, b, 2, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B)) return st;
  }
  GemmParams g = {};
  g.rows = (int)rows;
  g.cols = (int)cols;
  g.slices = (int)((k + kSlice - 1) / kSlice);
  g.last_steps = (int)((k - (int64_t)(g.slices - 1) * kSlice + 31) / 32);
  g.tiles_m = p.tiles_m;
  g.tiles_n = p.tiles_n;
  g.splits = p.splits;
  g.scales_a = static_cast<const uint8_t *>(a_scales);
  g.scales_b = static_cast<const uint8_t *>(b_scales);
  g.out = p.splits > 1 ? workspace : out;
  g.out_type = p.splits > 1 ? (int)P3D_F32 : out_dtype;
  g.pitch = cols;
  g.split_stride = p.splits > 1 ? rows * cols : 0;
  g.bias = p.splits > 1 ? nullptr : bias;
  g.bias_type = bias_dtype;
  g.vector = (cols * dtype_size(g.out_type)) % 16 == 0 && ((uintptr_t)g.out & 15) == 0;
  int st;
  {
    CUtensorMap tout = {};
    if (g.vector) {
      const int size = dtype_size(g.out_type);
      const uint64_t dims[3] = {(uint64_t)cols, (uint64_t)rows, (uint64_t)p.splits};
      const uint64_t strides[2] = {(uint64_t)(cols * size), (uint64_t)(rows * cols * size)};
      const uint32_t box[3] = {(uint32_t)(kStageRow / size), 32, 1};
      const CUtensorMapDataType type = g.out_type == P3D_F32   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                       : g.out_type == P3D_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                               : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
      if (int e = encode_tiled(&tout, type, g.out, 3, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_64B)) return e;
    }
    CUtensorMap ts[2];   // scale bytes, a row for each 512-byte chunk
    for (int i = 0; i < 2; ++i) {
      const uint64_t chunks = (uint64_t)p3d_fp8_scale_bytes(i ? cols : rows, k) / 512;
      const uint64_t dims[2] = {128, chunks}, strides[1] = {512};
      const uint32_t box[2] = {128, 1};
      if (int e = encode_tiled(&ts[i], CU_TENSOR_MAP_DATA_TYPE_UINT32, i ? g.scales_b : g.scales_a, 2, dims, strides, box,
                               CU_TENSOR_MAP_SWIZZLE_NONE))
        return e;
    }
    // a short k makes the epilogue the longer part: it then stages whole 128-byte segments, which costs a stage
    st = p.bn == 128   ? launch_pair<128, 2>(ta, tb, ts[0], ts[1], tout, g, info.sm_count, s)
         : g.slices <= 8 ? launch_pair<256, 2>(ta, tb, ts[0], ts[1], tout, g, info.sm_count, s)
                         : launch_pair<256, 1>(ta, tb, ts[0], ts[1], tout, g, info.sm_count, s);
  }
  if (st != P3D_OK || p.splits == 1) return st;
  const unsigned grid = (unsigned)std::min<int64_t>((rows * cols + 255) / 256, (int64_t)info.sm_count * 8);
  add_splits_kernel<<<grid, 256, 0, s>>>(static_cast<const float *>(workspace), p.splits, rows, cols, bias, bias_dtype,
                                         out, out_dtype, cols);
  P3D_LAUNCH_CHECK();
  return P3D_OK;
}
