// MXFP4 quantise and dequantise (format: lrq_mx.h).
#include "lrq_mx.h"

namespace lrq {

// The block's scale byte from its largest magnitude's fp32 bits: floor(log2) - 2 (the format's largest element is
// 1.5 * 2^2), 0 below 2^-124; a block with an infinity or a NaN gets 255 (NaN) and codes of 0.
__device__ __forceinline__ uint32_t mx_scale(uint32_t top) {
  const uint32_t e = top >> 23;
  return e == 255u ? 255u : (e < 2u ? 0u : e - 2u);
}

// The larger of v over the quad's four lanes.
__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0u, v, 0xb1, 0xf, 0xf, false));
  return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0u, v, 0x4e, 0xf, 0xf, false));
}

// Four lanes a block, 8 columns each: 16-byte loads of consecutive lanes, one dword of codes a lane.  HBM-bound: bf16
// [16384, 4096] 27 us with x in the last-level cache and 38 without (4.5 TB/s), and 27 to 29 us (6.0 TB/s) back.
template <int DT>
__global__ __launch_bounds__(256) void k_mx_quantize(const char* x, int64_t ldx, Mx q) {
  constexpr int ES = Elem<DT>::kBytes;
  const int chunks = 16 * q.steps;  // of 8 columns, padding included
  const int64_t total = q.rows * chunks;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / chunks;
    const int c = (int)(i - row * chunks);
    float v[8];
    widen<DT>(ld_chunk<DT>(x + (row * ldx + 8 * (int64_t)c) * ES, min(8, q.cols - 8 * c)), v);
    uint32_t top = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(v[e]) & 0x7fffffffu);
    const uint32_t s = mx_scale(quad_max(top));
    const float sf = e8m0_operand(s);
    uint32_t w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0], v[1], sf, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], sf, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], sf, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], sf, 3);
    st4(q.codes + row * q.ldc + 4 * (int64_t)c, s == 255u ? 0u : w);
    if ((c & 3) == 0) q.scales[row * q.lds + c / 4] = (uint8_t)s;
  }
}

template <int DT>
__global__ __launch_bounds__(256) void k_mx_dequantize(Mx q, char* out, int64_t ldo) {
  constexpr int ES = Elem<DT>::kBytes;
  const int chunks = (q.cols + 7) / 8;
  const int64_t total = q.rows * chunks;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / chunks;
    const int c = (int)(i - row * chunks);
    const uint32_t w = ld4(q.codes + row * q.ldc + 4 * (int64_t)c);
    const float sf = e8m0_operand(q.scales[row * q.lds + c / 4]);
    float v[8];
    const f32x2_t a = fp4_to_f32x2<0>(w, sf), b = fp4_to_f32x2<1>(w, sf), d = fp4_to_f32x2<2>(w, sf),
                  e = fp4_to_f32x2<3>(w, sf);
    v[0] = a[0], v[1] = a[1], v[2] = b[0], v[3] = b[1], v[4] = d[0], v[5] = d[1], v[6] = e[0], v[7] = e[1];
    st_chunk<DT>(out + (row * ldo + 8 * (int64_t)c) * ES, narrow<DT>(v), min(8, q.cols - 8 * c));
  }
}

static dim3 mx_grid(int64_t threads) {
  return dim3((unsigned)std::max<int64_t>(1, std::min<int64_t>((threads + 255) / 256, (int64_t)cu_count() * 64)));
}

}  // namespace lrq

using namespace lrq;

extern "C" int lrq_mxfp4_quantize(const void* x, int64_t ldx, int32_t dtype, const lrq_mxfp4* t, void* stream) {
  LRQ_TRY(validate_mx(t));
  if (dtype < LRQ_BF16 || dtype > LRQ_F32) return LRQ_ERR_UNSUPPORTED;
  if (t->rows == 0) return LRQ_OK;
  if (x == nullptr) return LRQ_ERR_NULL;
  if (ldx < t->cols) return LRQ_ERR_SHAPE;
  if (!aligned(x, dtype == LRQ_F32 ? 4 : 2)) return LRQ_ERR_ALIGN;
  const Mx q = make_mx(t);
  const dim3 grid = mx_grid(q.rows * 16 * q.steps);
  hipStream_t s = (hipStream_t)stream;
  switch (dtype) {
    case LRQ_BF16: return launch(k_mx_quantize<kBf16>, grid, dim3(256), 0, s, (const char*)x, ldx, q);
    case LRQ_F16: return launch(k_mx_quantize<kF16>, grid, dim3(256), 0, s, (const char*)x, ldx, q);
    default: return launch(k_mx_quantize<kF32>, grid, dim3(256), 0, s, (const char*)x, ldx, q);
  }
}

extern "C" int lrq_mxfp4_dequantize(const lrq_mxfp4* t, void* out, int64_t ldo, int32_t dtype, void* stream) {
  LRQ_TRY(validate_mx(t));
  if (dtype < LRQ_BF16 || dtype > LRQ_F32) return LRQ_ERR_UNSUPPORTED;
  if (t->rows == 0) return LRQ_OK;
  if (out == nullptr) return LRQ_ERR_NULL;
  if (ldo < t->cols) return LRQ_ERR_SHAPE;
  if (!aligned(out, dtype == LRQ_F32 ? 4 : 2)) return LRQ_ERR_ALIGN;
  const Mx q = make_mx(t);
  const dim3 grid = mx_grid(q.rows * ((q.cols + 7) / 8));
  hipStream_t s = (hipStream_t)stream;
  switch (dtype) {
    case LRQ_BF16: return launch(k_mx_dequantize<kBf16>, grid, dim3(256), 0, s, q, (char*)out, ldo);
    case LRQ_F16: return launch(k_mx_dequantize<kF16>, grid, dim3(256), 0, s, q, (char*)out, ldo);
    default: return launch(k_mx_dequantize<kF32>, grid, dim3(256), 0, s, q, (char*)out, ldo);
  }
}
