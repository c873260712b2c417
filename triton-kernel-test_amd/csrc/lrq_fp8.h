// 8-bit floating point (OCP e4m3: largest 448, no infinities) with one E8M0 scale 2^(s - 127) for a block of 128 columns
// of a row, or of 128 rows by 128 columns.
//
// Storage: codes [rows, Kp] bytes, Kp = columns rounded up to 128 (two K steps of the 32x32x64 instruction), padding columns
// code 0; scales [rows or ceil(rows / 128), Sp] bytes, Sp = Kp / 128 rounded up to 4, so that four steps' scales of a row
// are one aligned dword.
#pragma once

#include <algorithm>

#include "lrq_elem.h"
#include "lrq_host.h"

namespace lrq {

struct Fp8 {
  uint8_t* codes;
  uint8_t* scales;
  int64_t ldc, lds;  // bytes
  int64_t rows;
  int cols, steps;   // steps of 128 columns
  int shift;         // rows a scale: 1 << shift
};

static inline int validate_fp8(const lrq_fp8* t) {
  if (t == nullptr) return LRQ_ERR_NULL;
  if (t->rows < 0 || t->rows > INT32_MAX || t->cols <= 0 || t->cols > INT32_MAX / 2) return LRQ_ERR_SHAPE;
  if (t->block != 1 && t->block != 128) return LRQ_ERR_UNSUPPORTED;
  const int64_t steps = (t->cols + 127) / 128;
  if (t->ld_codes < 128 * steps || t->ld_scales < (steps + 3) / 4 * 4) return LRQ_ERR_SHAPE;
  if (t->rows > 0 && (t->codes == nullptr || t->scales == nullptr)) return LRQ_ERR_NULL;
  if (!aligned(t->codes, 16) || t->ld_codes % 16 != 0 || !aligned(t->scales, 4) || t->ld_scales % 4 != 0) return LRQ_ERR_ALIGN;
  return LRQ_OK;
}

static inline Fp8 make_fp8(const lrq_fp8* t) {
  return Fp8{(uint8_t*)t->codes, (uint8_t*)t->scales, t->ld_codes, t->ld_scales, t->rows, (int)t->cols,
             (int)((t->cols + 127) / 128), t->block == 128 ? 7 : 0};
}

// A block's scale byte from its largest magnitude's fp32 bits: the smallest power of two that it exceeds at most 448 = 1.75
// * 2^8 times, so that no element rounds past the largest code; 255 (NaN) for a block with an infinity or a NaN, whose codes
// are 0.
__device__ __forceinline__ uint32_t fp8_scale(uint32_t top) {
  const uint32_t e = top >> 23, s = e + ((top & 0x7fffffu) > 0x600000u ? 1u : 0u);
  return e == 255u ? 255u : (s < 8u ? 0u : s - 8u);
}

// x times this is x / 2^(s - 127), exactly (s <= 247; blocks with s = 255 take no codes).
__device__ __forceinline__ float fp8_inverse(uint32_t s) { return __uint_as_float((254u - min(s, 253u)) << 23); }

// 2^(s - 127) as fp32 (2^-127 is subnormal), NaN for 255.
__device__ __forceinline__ float fp8_value_scale(uint32_t s) {
  return __uint_as_float(s == 0u ? 0x00400000u : s == 255u ? 0x7fc00000u : s << 23);
}

// Four elements' codes, already divided by the scale.
__device__ __forceinline__ uint32_t fp8_codes4(float a, float b, float c, float d) {
  const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, lo, true);
}

__device__ __forceinline__ u32x2 fp8_codes8(const float* v, uint32_t s) {
  const float f = fp8_inverse(s);
  const u32x2 c = {fp8_codes4(v[0] * f, v[1] * f, v[2] * f, v[3] * f), fp8_codes4(v[4] * f, v[5] * f, v[6] * f, v[7] * f)};
  return s == 255u ? u32x2{0u, 0u} : c;
}

// Largest magnitude's bits of 8 elements.
__device__ __forceinline__ uint32_t top8(const float* v) {
  uint32_t t = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) t = max(t, __float_as_uint(v[e]) & 0x7fffffffu);
  return t;
}

// The largest over each 16 consecutive lanes, in all of them.
__device__ __forceinline__ uint32_t lanes16_max(uint32_t v) {
#define LRQ_DPP_MAX(ctrl) v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, ctrl, 0xf, 0xf, false))
  LRQ_DPP_MAX(0xb1);   // lanes 1 0 3 2 of each quad
  LRQ_DPP_MAX(0x4e);   // lanes 2 3 0 1
  LRQ_DPP_MAX(0x141);  // the other quad of each half row
  LRQ_DPP_MAX(0x140);  // the other half of the row
#undef LRQ_DPP_MAX
  return v;
}

}  // namespace lrq
