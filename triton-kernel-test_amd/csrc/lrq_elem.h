// Element types and 8-element accesses of the layer-norm, dropout and MXFP4 kernels.
//
// Rows are walked in chunks of 8 elements (16 bytes of bf16 / fp16, 32 of fp32) from the row's first
// element, so a row of any width has one partial chunk at most, its last.  Global vector accesses
// need no alignment beyond the element's on gfx950 (unaligned access mode is part of the HSA ABI), so rows that
// start on an odd element take the same 16-byte loads and stores as aligned ones.
#pragma once

#include "lrq_common.h"

namespace lrq {

enum { kBf16 = 0, kF16 = 1, kF32 = 2 };  // LRQ_BF16, LRQ_F16, LRQ_F32

template <int DT>
struct Elem {
  static constexpr int kBytes = DT == kF32 ? 4 : 2;
  static constexpr int kVecs = DT == kF32 ? 2 : 1;  // 16-byte vectors a chunk
};

// One chunk as stored.
template <int DT>
struct Chunk {
  u32x4 v[Elem<DT>::kVecs];
};

typedef u32x4 u32x4_any __attribute__((aligned(2)));

template <int DT>
__device__ __forceinline__ void pin(Chunk<DT>& c) {
#pragma unroll
  for (int k = 0; k < Elem<DT>::kVecs; ++k) pin(c.v[k]);
}

// What is compared with v is compared afresh behind this: a partial chunk's seven comparisons and the tests of a whole one,
// kept over a loop, take a pair of scalar registers each, for every chunk of a thread.
__device__ __forceinline__ void opaque(int& v) { asm volatile("" : "+v"(v)); }

// `valid` elements of the chunk at p (8 or more: the whole chunk; 0 or less: none); the others are 0.
template <int DT, bool STREAM = false>
__device__ __forceinline__ Chunk<DT> ld_chunk(const char* p, int valid) {
  Chunk<DT> c;
#pragma unroll
  for (int k = 0; k < Elem<DT>::kVecs; ++k) c.v[k] = u32x4{0u, 0u, 0u, 0u};
  if (valid >= 8) {
#pragma unroll
    for (int k = 0; k < Elem<DT>::kVecs; ++k) {
      const u32x4_any* q = reinterpret_cast<const u32x4_any*>(p) + k;
      c.v[k] = STREAM ? __builtin_nontemporal_load(q) : *q;
    }
  } else if (valid > 0) {
#pragma unroll
    for (int e = 0; e < 7; ++e) {
      if (e < valid) {
        if constexpr (DT == kF32) c.v[e / 4][e % 4] = reinterpret_cast<const uint32_t*>(p)[e];
        else c.v[0][e / 2] |= (uint32_t)reinterpret_cast<const uint16_t*>(p)[e] << (16 * (e & 1));
      }
    }
  }
  return c;
}

template <int DT, bool STREAM = false>
__device__ __forceinline__ void st_chunk(char* p, const Chunk<DT>& c, int valid) {
  if (valid >= 8) {
#pragma unroll
    for (int k = 0; k < Elem<DT>::kVecs; ++k) {
      u32x4_any* q = reinterpret_cast<u32x4_any*>(p) + k;
      if (STREAM) __builtin_nontemporal_store(c.v[k], q);
      else *q = c.v[k];
    }
  } else if (valid > 0) {
#pragma unroll
    for (int e = 0; e < 7; ++e) {
      if (e < valid) {
        if constexpr (DT == kF32) reinterpret_cast<uint32_t*>(p)[e] = c.v[e / 4][e % 4];
        else reinterpret_cast<uint16_t*>(p)[e] = (uint16_t)(c.v[0][e / 2] >> (16 * (e & 1)));
      }
    }
  }
}

template <int DT>
__device__ __forceinline__ void widen(const Chunk<DT>& c, float* f) {
  if constexpr (DT == kF32) {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = __uint_as_float(c.v[e / 4][e % 4]);
  } else if constexpr (DT == kBf16) {
    unpack8(c.v[0], f);
  } else {
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      f[2 * d] = f16_val(c.v[0][d] & 0xffffu);
      f[2 * d + 1] = f16_val(c.v[0][d] >> 16);
    }
  }
}

// How many elements of a chunk to load: a row's partial chunk is read whole, up to 7 elements into what follows the row,
// where a further row keeps that inside the tensor (element loads are joined as they arrive, so a thread that waits for
// them holds up the rows in flight: layer norm of bf16 [8192, 5003] backward 103 in place of 59 us).  mask_chunk takes away
// what lies past the row where that matters.
__device__ __forceinline__ int load_size(int valid, bool more_rows) { return more_rows && valid > 0 ? 8 : valid; }

template <int DT>
__device__ __forceinline__ void mask_chunk(Chunk<DT>& c, int valid) {
  if (valid >= 8) return;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    if constexpr (DT == kF32) c.v[e / 4][e % 4] = e < valid ? c.v[e / 4][e % 4] : 0u;
    else c.v[0][e / 2] &= e < valid ? ~0u : (e & 1) ? 0xffffu : 0xffff0000u;
  }
}

// Element e of those at p.
template <int DT>
__device__ __forceinline__ float ld_elem(const char* p, int e) {
  if constexpr (DT == kF32) return reinterpret_cast<const float*>(p)[e];
  const uint32_t v = reinterpret_cast<const uint16_t*>(p)[e];
  return DT == kBf16 ? __uint_as_float(v << 16) : f16_val(v);
}

// Rounds to the element type, nearest even.
template <int DT>
__device__ __forceinline__ Chunk<DT> narrow(const float* f) {
  Chunk<DT> c;
  if constexpr (DT == kF32) {
#pragma unroll
    for (int e = 0; e < 8; ++e) c.v[e / 4][e % 4] = __float_as_uint(f[e]);
  } else if constexpr (DT == kBf16) {
    c.v[0] = pack8(f);
  } else {
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      // opaque, or the compiler folds the operation before into a mixed-precision one that rounds
      // once where the other kernels round to fp32 first: all of them are to give the same bits
      float lo = f[2 * d], hi = f[2 * d + 1];
      asm("" : "+v"(lo), "+v"(hi));
      c.v[0][d] = f16_bits(lo) | ((uint32_t)f16_bits(hi) << 16);
    }
  }
  return c;
}

// A chunk of a tensor whose element type is a run-time value (weights, read once per workgroup).
__device__ __forceinline__ void ld_weight(const void* p, int dt, int64_t at, int valid, float* f) {
  const char* q = reinterpret_cast<const char*>(p) + at * (dt == kF32 ? 4 : 2);
  if (dt == kBf16) widen<kBf16>(ld_chunk<kBf16>(q, valid), f);
  else if (dt == kF16) widen<kF16>(ld_chunk<kF16>(q, valid), f);
  else widen<kF32>(ld_chunk<kF32>(q, valid), f);
}

// ---------------------------------------------------------------- workgroup barrier
// Waits for this wave's LDS traffic and meets the workgroup; loads from memory stay in flight.  One statement that no
// memory access moves across in either direction.
__device__ __forceinline__ void lds_meet() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// ---------------------------------------------------------------- sums over lanes
// Sum over each group of LANES (16 or 64) consecutive lanes, in every lane: quad and mirror moves of the
// DPP network, then the row swaps, so no LDS round trip.
template <int LANES>
__device__ __forceinline__ float lanes_sum(float v) {
  static_assert(LANES == 16 || LANES == 64, "a DPP row or a wave");
#define LRQ_DPP_ADD(ctrl) v += __uint_as_float(__builtin_amdgcn_update_dpp(0u, __float_as_uint(v), ctrl, 0xf, 0xf, false))
  LRQ_DPP_ADD(0xb1);   // lanes 1 0 3 2 of each quad
  LRQ_DPP_ADD(0x4e);   // lanes 2 3 0 1
  LRQ_DPP_ADD(0x141);  // the other quad of each half row (mirrored: quads are uniform by now)
  LRQ_DPP_ADD(0x140);  // the other half of the row
#undef LRQ_DPP_ADD
  if constexpr (LANES == 64) {
    float a = v, b = v;
    swap16(a, b);
    v = a + b;
    a = v, b = v;
    swap32(a, b);
    v = a + b;
  }
  return v;
}

}  // namespace lrq
