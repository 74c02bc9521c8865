// Philox-4x32-10 (Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC 2011): word i % 4 of the
// block at counter i / 4 under a 64-bit key is a pure function of (key, i), so what is drawn for an element does not depend
// on which thread, launch, GPU or direction draws it.  One stream for every user in the library: the stored masks of
// train_ops.hip, the mask-free dropout of dropout.hip and the dropout inside residual_norm_*.hip.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace advoc {

// Both halves of a 32 x 32-bit product in one instruction where the compiler issues two (with the first round's product that is
// known to be zero left out and the words compared directly, 65536 x 1024 bf16 elements: 60 -> 54 us).
__device__ __forceinline__ void mul64(uint64_t& p, uint32_t a, uint32_t b) {
  uint64_t carry;
  asm("v_mad_u64_u32 %0, %1, %2, %3, 0" : "=v"(p), "=s"(carry) : "s"(a), "v"(b));
}

// Counter (c, 0): the first round multiplies one word only.
__device__ __forceinline__ uint4 philox4x32(uint64_t c, uint2 key) {
  const uint32_t M0 = 0xD2511F53u, M1 = 0xCD9E8D57u, W0 = 0x9E3779B9u, W1 = 0xBB67AE85u;
  uint64_t p0, p1;
  mul64(p0, M0, (uint32_t)c);
  uint4 ctr = make_uint4((uint32_t)(c >> 32) ^ key.x, 0u, (uint32_t)(p0 >> 32) ^ key.y, (uint32_t)p0);
#pragma unroll
  for (int r = 1; r < 10; ++r) {
    key.x += W0;
    key.y += W1;
    mul64(p0, M0, ctr.x);
    mul64(p1, M1, ctr.z);
    ctr = make_uint4((uint32_t)(p1 >> 32) ^ ctr.y ^ key.x, (uint32_t)p1, (uint32_t)(p0 >> 32) ^ ctr.w ^ key.y, (uint32_t)p0);
  }
  return ctr;
}

// What a dropout kernel needs to draw: word i is kept when it is >= thresh (0: everything is kept and nothing is drawn).
struct DropKey {
  uint64_t seed, offset;        // offset is a multiple of 4
  const uint64_t* seed_dev;     // added to the seed when not NULL: read by the kernel, so a replayed graph draws anew
  uint32_t thresh;
  float scale;                  // 1 / keep, rounded once: what is kept is multiplied by it (1.5 units of fp32 off x / keep at most, a
                                // division would be 0.5 and a dozen instructions; nothing where keep is a power of two)
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

// The words of elements i ... i + N - 1 of the stream, N = 8 or 9: element k is kept when words[k] >= thresh.  i = offset + index, of
// any alignment: a third block is drawn only where i is no multiple of 4, which `aligned` -- uniform over the launch -- rules out, or
// for a ninth word.
template <int N>
__device__ __forceinline__ void drop_words(uint32_t (&words)[N], uint64_t i, bool aligned, uint2 key) {
  const uint64_t q = i >> 2;
  const uint4 a = philox4x32(q, key), b = philox4x32(q + 1, key);
  if (N == 8 && aligned) {
    words[0] = a.x, words[1] = a.y, words[2] = a.z, words[3] = a.w;
    words[4] = b.x, words[5] = b.y, words[6] = b.z, words[7] = b.w;
  } else {
    const uint4 c = philox4x32(q + 2, key);
    const uint32_t w[12] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w, c.x, c.y, c.z, c.w};
    uint32_t v[11];
    // by masks: a choice between neighbours of an array becomes a load at a chosen address, from memory of the lane's own
    const uint32_t one = 0u - (uint32_t)(i & 1), two = 0u - (uint32_t)(i >> 1 & 1);
#pragma unroll
    for (int k = 0; k < 11; ++k) v[k] = (w[k + 1] & one) | (w[k] & ~one);
#pragma unroll
    for (int k = 0; k < N; ++k) words[k] = (v[k + 2] & two) | (v[k] & ~two);
  }
}

__device__ __forceinline__ uint32_t drop_word(uint64_t i, uint2 key) {
  const uint4 a = philox4x32(i >> 2, key);
  return (i & 2) ? ((i & 1) ? a.w : a.z) : ((i & 1) ? a.y : a.x);
}

}  // namespace advoc
