// Products with MXFP4 operands (format: lrq_mx.h), fp32 accumulation:
//
//   lrq_mxfp4_gemm      out[M, N] = A B^T, A [M, K] and B [N, K] both MXFP4 (scaled matrix instructions)
//   lrq_mxfp4_linear    out[M, N] = X W^T, X bf16, W [N, K] MXFP4, widened to bf16 (exactly) on the way
//   lrq_mxfp4_linear_t  out[M, K] = Y W, the gradient of the above for X
#include "lrq_mx.h"

namespace lrq {

typedef int i32x8 __attribute__((ext_vector_type(8)));

// D(16x16) += A(16x128) B(128x16), both e2m1 with E8M0 block scales.  Lane l holds row (column) l % 16, k = 32 (l / 16)
// .. + 31, and its block's scale in the low byte of its scale operand.
__device__ __forceinline__ f32x4 mfma_mx(u32x4 a, u32x4 b, f32x4 c, uint32_t sa, uint32_t sb) {
  const i32x8 a8 = {(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0};
  const i32x8 b8 = {(int)b[0], (int)b[1], (int)b[2], (int)b[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a8, b8, c, 4, 4, 0, (int)sa, 0, (int)sb);
}

template <bool F32>
__device__ __forceinline__ void st_out(void* out, int64_t at, float v) {
  if constexpr (F32) reinterpret_cast<float*>(out)[at] = v;
  else reinterpret_cast<uint16_t*>(out)[at] = (uint16_t)pack_bf16x2(v, 0.f);
}

// Wave: 64 x 64 of the output, operands straight from global memory.  Rows past the operands are read from their last row
// and not stored.
template <bool F32>
__global__ __launch_bounds__(256) void k_mx_gemm(Mx a, Mx b, void* out, int64_t ldo) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, j = lane & 15, g = lane >> 4;
  const int64_t m0 = (int64_t)blockIdx.y * 128 + 64 * (wave >> 1), n0 = (int64_t)blockIdx.x * 128 + 64 * (wave & 1);
  f32x4 acc[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int k = 0; k < 4; ++k) acc[i][k] = zero4();
  const uint8_t *ca[4], *cb[4], *pa[4], *pb[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t ra = min(m0 + 16 * i + j, a.rows - 1), rb = min(n0 + 16 * i + j, b.rows - 1);
    ca[i] = a.codes + ra * a.ldc + 16 * g;
    pa[i] = a.scales + ra * a.lds + g;
    cb[i] = b.codes + rb * b.ldc + 16 * g;
    pb[i] = b.scales + rb * b.lds + g;
  }
  for (int s = 0; s < a.steps; ++s) {
    u32x4 va[4], vb[4];
    uint32_t sa[4], sb[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      va[i] = ld16(ca[i] + 64 * (int64_t)s);
      vb[i] = ld16(cb[i] + 64 * (int64_t)s);
      sa[i] = pa[i][4 * (int64_t)s];
      sb[i] = pb[i][4 * (int64_t)s];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) acc[i][k] = mfma_mx(va[i], vb[k], acc[i][k], sa[i], sb[k]);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const int64_t m = m0 + 16 * i + 4 * g + v, n = n0 + 16 * k + j;
        if (m < a.rows && n < b.rows) st_out<F32>(out, m * ldo + n, acc[i][k][v]);
      }
}

// Workgroup: 16 MT rows of X by 16 rows of W; its 8 waves take every eighth K step of 32 and join in LDS.
template <int MT, bool F32>
__global__ __launch_bounds__(512) void k_mx_linear(const uint16_t* x, int64_t ldx, int64_t rows, Mx w, void* out,
                                                   int64_t ldo) {
  __shared__ float red[8][MT][64][4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, j = lane & 15, g = lane >> 4;
  const int64_t m0 = (int64_t)blockIdx.y * 16 * MT, n0 = (int64_t)blockIdx.x * 16;
  const int64_t rw = min(n0 + j, w.rows - 1);
  const uint8_t* codes = w.codes + rw * w.ldc + 4 * g;
  const uint8_t* scales = w.scales + rw * w.lds;
  const uint16_t* px[MT];
  f32x4 acc[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    px[i] = x + min(m0 + 16 * i + j, rows - 1) * ldx + 8 * g;
    acc[i] = zero4();
  }
  const int steps = (w.cols + 31) / 32;
  for (int s = wave; s < steps; s += 8) {
    const u32x4 b = fp4x8_to_bf16(ld4(codes + 16 * (int64_t)s), e8m0_operand(scales[s]));
    const bool in = 32 * s + 8 * g < w.cols;
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      u32x4 a = u32x4{0u, 0u, 0u, 0u};
      if (in) a = *reinterpret_cast<const u32x4_any*>(px[i] + 32 * (int64_t)s);
      acc[i] = mfma_16x16x32(a, b, acc[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int v = 0; v < 4; ++v) red[wave][i][lane][v] = acc[i][v];
  __syncthreads();
  for (int o = threadIdx.x; o < MT * 256; o += 512) {
    const int i = o >> 8, l = (o >> 2) & 63, v = o & 3;
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) sum += red[k][i][l][v];
    const int64_t m = m0 + 16 * i + 4 * (l >> 4) + v, n = n0 + (l & 15);
    if (m < rows && n < w.rows) st_out<F32>(out, m * ldo + n, sum);
  }
}

// Wave: 16 MT rows of Y by 128 columns of W, summed over the rows of W.  Lane (j, g) widens the 8 x 8 block of
// columns 8j .. 8j + 7 and rows 8g .. 8g + 7 and transposes it in registers: operand c holds column 8j + c, so the
// output of operand c is column 8j + c of the wave's 128.
template <int MT, bool F32>
__global__ __launch_bounds__(256) void k_mx_linear_t(const uint16_t* y, int64_t ldy, int64_t rows, Mx w, void* out,
                                                     int64_t ldo) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, j = lane & 15, g = lane >> 4;
  const int64_t m0 = ((int64_t)blockIdx.y * 4 + wave) * 16 * MT;
  if (m0 >= rows) return;
  const int k0 = blockIdx.x * 128;
  const uint8_t* codes = w.codes + k0 / 2 + 4 * j;
  const uint8_t* scales = w.scales + k0 / 32 + j / 4;
  const uint16_t* py[MT];
  f32x4 acc[MT][8];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    py[i] = y + min(m0 + 16 * i + j, rows - 1) * ldy + 8 * g;
#pragma unroll
    for (int c = 0; c < 8; ++c) acc[i][c] = zero4();
  }
  for (int64_t n = 0; n < w.rows; n += 32) {
    u32x4 r[8];  // row 8g + i, columns 8j .. 8j + 7
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int64_t rw = min(n + 8 * g + i, w.rows - 1);
      r[i] = fp4x8_to_bf16(ld4(codes + rw * w.ldc), e8m0_operand(scales[rw * w.lds]));
    }
    u32x4 a[MT];
    const bool in = n + 8 * g < w.rows;
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      a[i] = u32x4{0u, 0u, 0u, 0u};
      if (in) a[i] = *reinterpret_cast<const u32x4_any*>(py[i] + n);
    }
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      u32x4 b;
#pragma unroll
      for (int p = 0; p < 4; ++p)
        b[p] = __builtin_amdgcn_perm(r[2 * p + 1][c / 2], r[2 * p][c / 2], (c & 1) ? 0x07060302u : 0x05040100u);
#pragma unroll
      for (int i = 0; i < MT; ++i) acc[i][c] = mfma_16x16x32(a[i], b, acc[i][c]);
    }
  }
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const int64_t m = m0 + 16 * i + 4 * g + v;
      const int k = k0 + 8 * j;
      if (m >= rows) continue;
#pragma unroll
      for (int c = 0; c < 8; ++c)
        if (k + c < w.cols) st_out<F32>(out, m * ldo + k + c, acc[i][c][v]);
    }
}

static int validate_out(const void* out, int64_t ldo, int64_t cols, int32_t f32) {
  if (out == nullptr) return LRQ_ERR_NULL;
  if (ldo < cols) return LRQ_ERR_SHAPE;
  return aligned(out, f32 ? 4 : 2) ? LRQ_OK : LRQ_ERR_ALIGN;
}

}  // namespace lrq

using namespace lrq;

extern "C" int lrq_mxfp4_gemm(const lrq_mxfp4* ta, const lrq_mxfp4* tb, void* out, int64_t ldo, int32_t out_fp32,
                              void* stream) {
  LRQ_TRY(validate_mx(ta));
  LRQ_TRY(validate_mx(tb));
  if (ta->cols != tb->cols) return LRQ_ERR_SHAPE;
  if (ta->rows == 0 || tb->rows == 0) return LRQ_OK;
  LRQ_TRY(validate_out(out, ldo, tb->rows, out_fp32));
  const Mx a = make_mx(ta), b = make_mx(tb);
  const int64_t gx = (b.rows + 127) / 128, gy = (a.rows + 127) / 128;
  if (gy > 65535) return LRQ_ERR_SHAPE;
  const dim3 grid((unsigned)gx, (unsigned)gy);
  hipStream_t s = (hipStream_t)stream;
  return out_fp32 ? launch(k_mx_gemm<true>, grid, dim3(256), 0, s, a, b, out, ldo)
                  : launch(k_mx_gemm<false>, grid, dim3(256), 0, s, a, b, out, ldo);
}

extern "C" int lrq_mxfp4_linear(const void* x, int64_t ldx, int64_t rows, const lrq_mxfp4* t, void* out, int64_t ldo,
                                int32_t out_fp32, void* stream) {
  LRQ_TRY(validate_mx(t));
  if (rows < 0 || rows > INT32_MAX) return LRQ_ERR_SHAPE;
  if (rows == 0 || t->rows == 0) return LRQ_OK;
  if (x == nullptr) return LRQ_ERR_NULL;
  if (ldx < (t->cols + 7) / 8 * 8) return LRQ_ERR_SHAPE;
  if (!aligned(x, 2)) return LRQ_ERR_ALIGN;
  LRQ_TRY(validate_out(out, ldo, t->rows, out_fp32));
  const Mx w = make_mx(t);
  hipStream_t s = (hipStream_t)stream;
  const int mt = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
  const dim3 grid((unsigned)((w.rows + 15) / 16), (unsigned)((rows + 16 * mt - 1) / (16 * mt)));
  const uint16_t* px = (const uint16_t*)x;
#define LRQ_GO(MT) return out_fp32 ? launch(k_mx_linear<MT, true>, grid, dim3(512), 0, s, px, ldx, rows, w, out, ldo) \
                                   : launch(k_mx_linear<MT, false>, grid, dim3(512), 0, s, px, ldx, rows, w, out, ldo)
  if (mt == 1) LRQ_GO(1);
  if (mt == 2) LRQ_GO(2);
  LRQ_GO(4);
#undef LRQ_GO
}

extern "C" int lrq_mxfp4_linear_t(const void* y, int64_t ldy, int64_t rows, const lrq_mxfp4* t, void* out, int64_t ldo,
                                  int32_t out_fp32, void* stream) {
  LRQ_TRY(validate_mx(t));
  if (rows < 0 || rows > INT32_MAX) return LRQ_ERR_SHAPE;
  if (rows == 0) return LRQ_OK;
  if (t->rows > 0) {
    if (y == nullptr) return LRQ_ERR_NULL;
    if (ldy < (t->rows + 7) / 8 * 8) return LRQ_ERR_SHAPE;
    if (!aligned(y, 2)) return LRQ_ERR_ALIGN;
  }
  LRQ_TRY(validate_out(out, ldo, t->cols, out_fp32));
  const Mx w = make_mx(t);
  hipStream_t s = (hipStream_t)stream;
  const dim3 grid((unsigned)w.steps, (unsigned)((rows + 127) / 128));
  const uint16_t* py = (const uint16_t*)y;
  return out_fp32 ? launch(k_mx_linear_t<2, true>, grid, dim3(256), 0, s, py, ldy, rows, w, out, ldo)
                  : launch(k_mx_linear_t<2, false>, grid, dim3(256), 0, s, py, ldy, rows, w, out, ldo);
}
