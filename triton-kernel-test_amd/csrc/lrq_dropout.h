// Dropout's random numbers: the counter-based generator Philox4x32-10 (Salmon, Moraes, Dror and Shaw,
// "Parallel random numbers: as easy as 1, 2, 3", SC 2011), so a mask is a function of (seed, offset,
// position) and is drawn again wherever it is needed instead of being stored.
//
// Element (row, col) of a tensor of n columns takes 16 bits: number col % 8 of the block with
// counter (q, offset), q = row * ceil(n / 8) + col / 8.  One block serves a chunk of 8 elements, whatever
// the row's alignment.  16 bits an element keep the ten rounds (20 wide multiplies at a quarter of the vector rate) at
// half the cost of 32-bit numbers; probabilities are multiples of 1 / 65536, and the scale 65536 / keep is
// that of the probability actually drawn with.
#pragma once

#include "lrq_elem.h"
#include "lrq_host.h"

namespace lrq {

struct Drop {
  uint32_t keep;          // kept where the 16-bit number is below it; 65536: keep all (no numbers drawn)
  float scale;            // 65536 / keep, 0 where keep is 0
  uint64_t seed, offset;
  const uint64_t* state;  // device words (seed, offset) that replace seed and are added to offset; may be NULL
};

static inline Drop make_drop(const lrq_dropout* d) {
  if (d == nullptr) return Drop{65536u, 1.f, 0, 0, nullptr};
  const float scale = d->keep == 0 ? 0.f : (float)(65536.0 / d->keep);
  return Drop{d->keep, scale, d->seed, d->offset, (const uint64_t*)d->state};
}

static inline int validate_dropout(const lrq_dropout* d) {
  if (d == nullptr) return LRQ_OK;
  if (d->keep > 65536u) return LRQ_ERR_SHAPE;
  if (!aligned(d->state, 8)) return LRQ_ERR_ALIGN;
  return LRQ_OK;
}

struct DropKey {
  uint32_t k0, k1, c2, c3;
};

__device__ __forceinline__ DropKey drop_key(const Drop& d) {
  uint64_t seed = d.seed, off = d.offset;
  if (d.state != nullptr) {
    seed = d.state[0];
    off += d.state[1];
  }
  return DropKey{(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)seed),
                 (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(seed >> 32)),
                 (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)off),
                 (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(off >> 32))};
}

__device__ __forceinline__ uint32_t xor3(uint32_t a, uint32_t b, uint32_t c) {
  return __builtin_amdgcn_bitop3_b32(a, b, c, 0x96);
}

__device__ __forceinline__ u32x4 philox(uint64_t q, const DropKey& key) {
  uint32_t c0 = (uint32_t)q, c1 = (uint32_t)(q >> 32), c2 = key.c2, c3 = key.c3, k0 = key.k0, k1 = key.k1;
  // opaque, or the rounds' twenty keys are kept in scalar registers over the caller's loop and crowd out its own values
  asm volatile("" : "+s"(k0), "+s"(k1));
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t p0 = (uint64_t)c0 * 0xD2511F53u, p1 = (uint64_t)c2 * 0xCD9E8D57u;
    c0 = xor3((uint32_t)(p1 >> 32), c1, k0);
    c1 = (uint32_t)p1;
    c2 = xor3((uint32_t)(p0 >> 32), c3, k1);
    c3 = (uint32_t)p0;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return u32x4{c0, c1, c2, c3};
}

// f[e] = kept ? f[e] * scale : 0 for a chunk with the block w (a dropped NaN or infinity gives 0).
__device__ __forceinline__ void drop_words(const Drop& d, const u32x4& w, float* f) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t u = (e & 1) ? w[e / 2] >> 16 : w[e / 2] & 0xffffu;
    f[e] = u < d.keep ? f[e] * d.scale : 0.f;
  }
}
__device__ __forceinline__ void drop_chunk(const Drop& d, const DropKey& key, uint64_t q, float* f) {
  drop_words(d, philox(q, key), f);
}

}  // namespace lrq
