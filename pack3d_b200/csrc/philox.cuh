// Counter-based random bits for dropout: Philox-4x32 with ten rounds (Salmon, Moraes, Dror,
// Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC 2011).  A 128-bit counter under a
// 64-bit key gives 128 bits, so any element's bits can be made again from its position alone
// and no mask is ever stored.
#pragma once

#include <stdint.h>

namespace p3d {

struct PhiloxKey {
  uint64_t seed, offset;
};

// Seed and offset of a call: by value, or from device memory when `rng` is not null (a captured
// graph then draws new bits at each replay that advances it).
__device__ __forceinline__ PhiloxKey philox_key(const uint64_t *rng, uint64_t seed, uint64_t offset) {
  if (rng != nullptr) return PhiloxKey{rng[0], rng[1]};
  return PhiloxKey{seed, offset};
}

__device__ __forceinline__ void philox_round(uint4 &c, uint32_t k0, uint32_t k1) {
  const uint64_t p0 = (uint64_t)0xD2511F53u * c.x, p1 = (uint64_t)0xCD9E8D57u * c.z;
  c = make_uint4((uint32_t)(p1 >> 32) ^ c.y ^ k0, (uint32_t)p1, (uint32_t)(p0 >> 32) ^ c.w ^ k1, (uint32_t)p0);
}

// The keys of the ten rounds, in shared memory: for kernels that draw a block a row, five loads instead of twenty
// additions each time.
struct RoundKeys {
  uint4 pair[5];   // (k0, k1) of rounds 2 i and 2 i + 1
  uint32_t offset[2];
  // By the CTA's first threads, before a barrier.
  __device__ __forceinline__ void set(PhiloxKey key) {
    const uint32_t r = threadIdx.x;
    if (r < 10) {
      reinterpret_cast<uint2 *>(pair)[r] =
          make_uint2((uint32_t)key.seed + r * 0x9E3779B9u, (uint32_t)(key.seed >> 32) + r * 0xBB67AE85u);
      if (r < 2) offset[r] = (uint32_t)(key.offset >> (32 * r));
    }
  }
};

__device__ __forceinline__ uint4 philox(PhiloxKey key, uint64_t block) {
  uint4 c = make_uint4((uint32_t)block, (uint32_t)(block >> 32), (uint32_t)key.offset, (uint32_t)(key.offset >> 32));
  uint32_t k0 = (uint32_t)key.seed, k1 = (uint32_t)(key.seed >> 32);
#pragma unroll
  for (int round = 0; round < 10; ++round) {
    philox_round(c, k0, k1);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return c;
}
__device__ __forceinline__ uint4 philox(const RoundKeys &keys, uint64_t block) {
  uint4 c = make_uint4((uint32_t)block, (uint32_t)(block >> 32), keys.offset[0], keys.offset[1]);
#pragma unroll
  for (int i = 0; i < 5; ++i) {
    const uint4 k = keys.pair[i];
    philox_round(c, k.x, k.y);
    philox_round(c, k.z, k.w);
  }
  return c;
}

// Element j of a block is kept when its 16-bit field (field j % 2 of word j / 2, low half first) is at least
// `threshold`, so the drop probability is threshold / 65536.  Sixteen bits an element instead of 32 halve
// the rounds; the probability asked for is met within 2^-17.  A field is compared in the upper half of a
// word, where the bits below it change nothing: the high field as it lies, the low one shifted up.
struct Keep {
  uint32_t bound;   // threshold << 16; with threshold 65536 no word reaches it
  bool none;        // everything is dropped
  __device__ __forceinline__ explicit Keep(uint32_t threshold)
      : bound(threshold >= 65536u ? 0xffffffffu : threshold << 16), none(threshold >= 65536u) {}
  template <typename Keys>
  __device__ __forceinline__ void words(const Keys &keys, uint64_t block, uint32_t *w) const {
    const uint4 r = philox(keys, block);
    w[0] = none ? 0u : r.x;
    w[1] = none ? 0u : r.y;
    w[2] = none ? 0u : r.z;
    w[3] = none ? 0u : r.w;
  }
  __device__ __forceinline__ bool low(uint32_t word) const { return (word << 16) >= bound; }
  __device__ __forceinline__ bool high(uint32_t word) const { return word >= bound; }
  // The eight decisions as bits.
  template <typename Keys>
  __device__ __forceinline__ uint32_t bits(const Keys &keys, uint64_t block) const {
    uint32_t w[4], b = 0;
    words(keys, block, w);
#pragma unroll
    for (int i = 0; i < 4; ++i) b |= (low(w[i]) ? 1u << (2 * i) : 0u) | (high(w[i]) ? 2u << (2 * i) : 0u);
    return b;
  }
};

// 1 / (1 - p) of the probability actually used; 0 when everything is dropped.
__host__ __device__ inline float keep_scale(uint32_t threshold) {
  return threshold >= 65536u ? 0.f : 65536.f / (float)(65536u - threshold);
}

}  // namespace p3d
