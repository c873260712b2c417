// MXFP4 (OCP Microscaling v1.0): blocks of 32 columns of a row share an E8M0 scale 2^(s - 127), elements are e2m1
// codes (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives).
//
// Storage: codes [rows, Kp / 2] bytes, the even column in the low nibble, and scales [rows, Kp / 32] bytes, Kp =
// columns rounded up to 128 (one K step of the scaled matrix instruction); padding columns have code 0.
#pragma once

#include <algorithm>

#include "lrq_elem.h"
#include "lrq_host.h"

namespace lrq {

struct Mx {
  uint8_t* codes;
  uint8_t* scales;
  int64_t ldc, lds;  // bytes
  int64_t rows;
  int cols, steps;   // steps of 128 columns
};

static inline int validate_mx(const lrq_mxfp4* t) {
  if (t == nullptr) return LRQ_ERR_NULL;
  if (t->rows < 0 || t->rows > INT32_MAX || t->cols <= 0 || t->cols > INT32_MAX / 2) return LRQ_ERR_SHAPE;
  const int64_t steps = (t->cols + 127) / 128;
  if (t->ld_codes < 64 * steps || t->ld_scales < 4 * steps) return LRQ_ERR_SHAPE;
  if (t->rows > 0 && (t->codes == nullptr || t->scales == nullptr)) return LRQ_ERR_NULL;
  if (!aligned(t->codes, 16) || t->ld_codes % 16 != 0 || !aligned(t->scales, 4) || t->ld_scales % 4 != 0) return LRQ_ERR_ALIGN;
  return LRQ_OK;
}

static inline Mx make_mx(const lrq_mxfp4* t) {
  return Mx{(uint8_t*)t->codes, (uint8_t*)t->scales, t->ld_codes, t->ld_scales, t->rows, (int)t->cols,
            (int)((t->cols + 127) / 128)};
}

// Two codes (byte B of w) times the scale whose E8M0 byte is s, as bf16 pair / fp32 pair: exact in bf16 (e2m1 has two
// significant bits).  The conversion takes its scale as the exponent field of an fp32.
__device__ __forceinline__ float e8m0_operand(uint32_t s) { return __uint_as_float(s << 23); }

template <int B>
__device__ __forceinline__ uint32_t fp4_to_bf16x2(uint32_t w, float scale) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, B));
}
template <int B>
__device__ __forceinline__ f32x2_t fp4_to_f32x2(uint32_t w, float scale) {
  return __builtin_bit_cast(f32x2_t, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, B));
}
// The 8 codes of a dword as 8 bf16 (a 16x16x32 operand's 8 consecutive k).
__device__ __forceinline__ u32x4 fp4x8_to_bf16(uint32_t w, float scale) {
  return u32x4{fp4_to_bf16x2<0>(w, scale), fp4_to_bf16x2<1>(w, scale), fp4_to_bf16x2<2>(w, scale),
               fp4_to_bf16x2<3>(w, scale)};
}

}  // namespace lrq
