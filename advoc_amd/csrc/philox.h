// Philox-4x32-10 (Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC 2011): word i % 4 of the
// block at counter i / 4 under a 64-bit key is a pure function of (key, i), so what is drawn for an element does not depend
// on which thread, launch, GPU or direction draws it.  One stream for every user in the library: the stored masks of
// train_ops.hip, the mask-free dropout of dropout.hip and the dropout inside residual_norm_*.hip.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace advoc {

// Both halves of a 32 x 32-bit product in one instruction; the compiler issues two, each at a quarter of the vector rate, and they
// are what the generator's time goes to.
__device__ __forceinline__ void mul64(uint64_t& p, uint32_t a, uint32_t b) {
  uint64_t carry;
  asm("v_mad_u64_u32 %0, %1, %2, %3, 0" : "=v"(p), "=s"(carry) : "s"(a), "v"(b));
}

__device__ __forceinline__ uint4 philox4x32(uint4 ctr, uint2 key) {
  const uint32_t M0 = 0xD2511F53u, M1 = 0xCD9E8D57u, W0 = 0x9E3779B9u, W1 = 0xBB67AE85u;
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    uint64_t p0, p1;
    mul64(p0, M0, ctr.x);
    mul64(p1, M1, ctr.z);
    ctr = make_uint4((uint32_t)(p1 >> 32) ^ ctr.y ^ key.x, (uint32_t)p1, (uint32_t)(p0 >> 32) ^ ctr.w ^ key.y, (uint32_t)p0);
    key.x += W0;
    key.y += W1;
  }
  return ctr;
}

// What a dropout kernel needs to draw: word i is kept when it is >= thresh (0: everything is kept and nothing is drawn).
struct DropKey {
  uint64_t seed, offset;        // offset is a multiple of 4
  const uint64_t* seed_dev;     // added to the seed when not NULL: read by the kernel, so a replayed graph draws anew
  uint32_t thresh;
  float scale;                  // 1 / keep
};

// (1 - keep) 2^32 in fp32, as dropout_mask_kernel (train_ops.hip) computes it on the device, where the conversion to an
// integer saturates; done on the host in a form that is defined there
static inline DropKey make_drop_key(float keep, uint64_t seed, uint64_t offset, const uint64_t* seed_dev) {
  DropKey k;
  const float t = (1.0f - keep) * 4294967296.0f;
  k.thresh = !(t > 0.f) ? 0u : t >= 4294967296.0f ? 0xffffffffu : (uint32_t)t;
  k.scale = (float)(1.0 / (double)keep);
  k.seed = seed;
  k.offset = offset;
  k.seed_dev = seed_dev;
  return k;
}

__device__ __forceinline__ uint2 drop_key_words(const DropKey& k) {
  const uint64_t s = k.seed + (k.seed_dev ? *k.seed_dev : 0);
  return make_uint2((uint32_t)s, (uint32_t)(s >> 32));
}

// words 4 q .. 4 q + 3
__device__ __forceinline__ uint4 drop_quad(uint64_t q, uint2 key) {
  return philox4x32(make_uint4((uint32_t)q, (uint32_t)(q >> 32), 0u, 0u), key);
}

// bit k set: element i + k of the stream is kept, k < 8.  i = offset + index; any alignment (a third block only where i is no
// multiple of 4, and `aligned` -- uniform over the launch -- says that none is).
__device__ __forceinline__ uint32_t drop_keep8(uint64_t i, bool aligned, uint2 key, uint32_t thresh) {
  const uint64_t q = i >> 2;
  const uint4 a = drop_quad(q, key), b = drop_quad(q + 1, key);
  uint32_t bits = (a.x >= thresh) | (a.y >= thresh) << 1 | (a.z >= thresh) << 2 | (a.w >= thresh) << 3 |
                  (b.x >= thresh) << 4 | (b.y >= thresh) << 5 | (b.z >= thresh) << 6 | (b.w >= thresh) << 7;
  if (!aligned) {
    const uint4 c = drop_quad(q + 2, key);
    bits |= (c.x >= thresh) << 8 | (c.y >= thresh) << 9 | (c.z >= thresh) << 10 | (c.w >= thresh) << 11;
    bits >>= (uint32_t)i & 3u;
  }
  return bits;
}

__device__ __forceinline__ uint32_t drop_keep1(uint64_t i, uint2 key, uint32_t thresh) {
  const uint4 a = drop_quad(i >> 2, key);
  const uint32_t w = (i & 2) ? ((i & 1) ? a.w : a.z) : ((i & 1) ? a.y : a.x);
  return w >= thresh;
}

}  // namespace advoc
