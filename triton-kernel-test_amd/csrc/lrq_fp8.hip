// e4m3 quantise and dequantise (format: lrq_fp8.h).  All are one pass and bound by memory: bf16 [14336, 4096] (176 MB read and
// written) 28.6 us by rows, 27.6 by squares, 29.3 transposed, 27.8 back, 6.0 to 6.4 TB/s; [512, 4096] 3.4 to 4.4, about a launch.
#include "lrq_fp8.h"

namespace lrq {

// Blocks of 128 columns of a row: 16 lanes a block, 8 columns each.
template <int DT>
__global__ __launch_bounds__(256) void k_fp8_rows(const char* x, int64_t ldx, Fp8 q) {
  constexpr int ES = Elem<DT>::kBytes;
  const int chunks = 16 * q.steps;  // of 8 columns, padding included
  const int64_t total = q.rows * chunks;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / chunks;
    const int c = (int)(i - row * chunks);
    float v[8];
    widen<DT>(ld_chunk<DT>(x + (row * ldx + 8 * (int64_t)c) * ES, min(8, q.cols - 8 * c)), v);
    const uint32_t s = fp8_scale(lanes16_max(top8(v)));
    st8(q.codes + row * q.ldc + 8 * (int64_t)c, fp8_codes8(v, s));
    if ((c & 15) == 0) q.scales[row * q.lds + c / 16] = (uint8_t)s;
  }
}

// Blocks of 128 x 128: a workgroup each, 16 lanes a row, every sixteenth row a lane; read once, held as stored.
template <int DT>
__global__ __launch_bounds__(256) void k_fp8_square(const char* x, int64_t ldx, Fp8 q) {
  constexpr int ES = Elem<DT>::kBytes;
  __shared__ uint32_t tops[4];
  const int step = blockIdx.x % q.steps, c = 16 * step + (threadIdx.x & 15), k = min(8, q.cols - 8 * c);
  const int64_t blk = blockIdx.x / q.steps, row0 = 128 * blk + (threadIdx.x >> 4);
  Chunk<DT> in[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t row = row0 + 16 * i;
    in[i] = ld_chunk<DT>(x + (row * ldx + 8 * (int64_t)c) * ES, row < q.rows ? k : 0);
  }
  uint32_t top = 0;
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    widen<DT>(in[i], v);
    top = max(top, top8(v));
  }
  top = lanes16_max(top);
  top = max(top, (uint32_t)__shfl_xor((int)top, 16));
  top = max(top, (uint32_t)__shfl_xor((int)top, 32));
  if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
  __syncthreads();
  const uint32_t s = fp8_scale(max(max(tops[0], tops[1]), max(tops[2], tops[3])));
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t row = row0 + 16 * i;
    widen<DT>(in[i], v);
    if (row < q.rows) st8(q.codes + row * q.ldc + 8 * (int64_t)c, fp8_codes8(v, s));
  }
  if (threadIdx.x == 0) q.scales[blk * q.lds + step] = (uint8_t)s;
}

// Blocks of 128 columns of the transpose's rows: 128 rows by 64 columns of x a workgroup.  Thread (g, c) holds columns 8 c ..
// + 7 of rows 4 g .. + 3: four codes of a column are a dword of the output row, which passes through LDS to leave in
// 16-byte pieces (a plain store would write 4 bytes of a row at a time).  LDS row r (a column of x) keeps its dword d in slot
// d ^ 4 (r / 8): eight lanes of a write, one chunk each, fall in different banks.
template <int DT>
__global__ __launch_bounds__(256) void k_fp8_transpose(const char* x, int64_t ldx, Fp8 q) {
  constexpr int ES = Elem<DT>::kBytes;
  __shared__ uint32_t tops[4][64];
  __shared__ __attribute__((aligned(16))) uint32_t tile[64][32];
  const int c = threadIdx.x & 7, g = threadIdx.x >> 3, wave = threadIdx.x >> 6;
  const int tiles = (int)((q.rows + 63) / 64), step = blockIdx.x / tiles;
  const int64_t col0 = 64 * (int64_t)(blockIdx.x - step * tiles), at = col0 + 8 * c;  // of x
  const int k = (int)min((int64_t)8, q.rows - at);
  Chunk<DT> in[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = 128 * step + 4 * g + i;
    in[i] = ld_chunk<DT>(x + (row * ldx + at) * ES, row < q.cols ? k : 0);
  }
  float v[4][8];
#pragma unroll
  for (int i = 0; i < 4; ++i) widen<DT>(in[i], v[i]);
  uint32_t top[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    top[e] = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) top[e] = max(top[e], __float_as_uint(v[i][e]) & 0x7fffffffu);
#pragma unroll
    for (int d = 8; d < 64; d *= 2) top[e] = max(top[e], (uint32_t)__shfl_xor((int)top[e], d));
  }
  if ((threadIdx.x & 63) < 8) {
#pragma unroll
    for (int e = 0; e < 8; ++e) tops[wave][8 * c + e] = top[e];
  }
  __syncthreads();
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int r = 8 * c + e;
    const uint32_t s = fp8_scale(max(max(tops[0][r], tops[1][r]), max(tops[2][r], tops[3][r])));
    const float f = fp8_inverse(s);
    const uint32_t w = fp8_codes4(v[0][e] * f, v[1][e] * f, v[2][e] * f, v[3][e] * f);
    tile[r][g ^ 4 * c] = s == 255u ? 0u : w;
    if (g == 0 && at + e < q.rows) q.scales[(at + e) * q.lds + step] = (uint8_t)s;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 2; ++i) {  // 8 lanes a row, 16 bytes each
    const int r = 32 * i + (threadIdx.x >> 3), p = threadIdx.x & 7;
    if (col0 + r < q.rows) st16(q.codes + (col0 + r) * q.ldc + 128 * (int64_t)step + 16 * p, ld16(&tile[r][4 * (p ^ (r >> 3))]));
  }
}

// By rows and transposed in one read of x, for a product and its weight's gradient: 128 rows by 128 columns a workgroup.
// Thread (g, c) holds columns 8 c .. + 7 of rows 8 g .. + 7: 16 lanes a row's block, and 8 codes of a column are 8 bytes of the
// transpose, which LDS row r keeps in slot g ^ r / 8 of 16.  bf16 [14336, 4096] 43 us (5.4 TB/s), [2048, 4096] 9.9; in two
// calls 58 and 13.7.
template <int DT>
__global__ __launch_bounds__(256) void k_fp8_both(const char* x, int64_t ldx, Fp8 q, Fp8 t) {
  constexpr int ES = Elem<DT>::kBytes;
  __shared__ uint32_t tops[4][128];
  __shared__ __attribute__((aligned(16))) uint32_t tile[128][32];
  const int c = threadIdx.x & 15, g = threadIdx.x >> 4, wave = threadIdx.x >> 6;
  const int tstep = blockIdx.x / q.steps, step = blockIdx.x - tstep * q.steps, at = 128 * step + 8 * c;
  const int64_t row0 = 128 * (int64_t)tstep + 8 * g;
  const int k = min(8, q.cols - at);
  Chunk<DT> in[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) in[i] = ld_chunk<DT>(x + ((row0 + i) * ldx + at) * ES, row0 + i < q.rows ? k : 0);
  uint32_t top[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) top[e] = 0;
  float v[8][8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    widen<DT>(in[i], v[i]);
    const uint32_t s = fp8_scale(lanes16_max(top8(v[i])));
    if (row0 + i < q.rows) {
      st8(q.codes + (row0 + i) * q.ldc + at, fp8_codes8(v[i], s));
      if (c == 0) q.scales[(row0 + i) * q.lds + step] = (uint8_t)s;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) top[e] = max(top[e], __float_as_uint(v[i][e]) & 0x7fffffffu);
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    top[e] = max(top[e], (uint32_t)__shfl_xor((int)top[e], 16));
    top[e] = max(top[e], (uint32_t)__shfl_xor((int)top[e], 32));
  }
  if ((threadIdx.x & 63) < 16) {
#pragma unroll
    for (int e = 0; e < 8; ++e) tops[wave][8 * c + e] = top[e];
  }
  __syncthreads();
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int r = 8 * c + e;
    const uint32_t s = fp8_scale(max(max(tops[0][r], tops[1][r]), max(tops[2][r], tops[3][r])));
    const float f = fp8_inverse(s);
    const u32x2 w = {fp8_codes4(v[0][e] * f, v[1][e] * f, v[2][e] * f, v[3][e] * f),
                     fp8_codes4(v[4][e] * f, v[5][e] * f, v[6][e] * f, v[7][e] * f)};
    st8(&tile[r][2 * (g ^ c)], s == 255u ? u32x2{0u, 0u} : w);
    if (g == 0 && at + e < q.cols) t.scales[(int64_t)(at + e) * t.lds + tstep] = (uint8_t)s;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) {  // 8 lanes a row, two slots each
    const int r = 32 * i + (threadIdx.x >> 3), p = threadIdx.x & 7, turn = r >> 3;
    const u32x4 w = ld16(&tile[r][4 * (p ^ (turn >> 1))]);
    if (128 * step + r < q.cols)
      st16(t.codes + (128 * (int64_t)step + r) * t.ldc + 128 * (int64_t)tstep + 16 * p,
           (turn & 1) ? u32x4{w[2], w[3], w[0], w[1]} : w);
  }
}

template <int DT>
__global__ __launch_bounds__(256) void k_fp8_dequantize(Fp8 q, char* out, int64_t ldo) {
  constexpr int ES = Elem<DT>::kBytes;
  const int chunks = (q.cols + 7) / 8;
  const int64_t total = q.rows * chunks;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / chunks;
    const int c = (int)(i - row * chunks);
    const u32x2 w = ld8(q.codes + row * q.ldc + 8 * (int64_t)c);
    const float f = fp8_value_scale(q.scales[(row >> q.shift) * q.lds + c / 16]);
    float v[8];
#pragma unroll
    for (int d = 0; d < 2; ++d) {
      const f32x2_t lo = __builtin_bit_cast(f32x2_t, __builtin_amdgcn_cvt_pk_f32_fp8((int)w[d], false));
      const f32x2_t hi = __builtin_bit_cast(f32x2_t, __builtin_amdgcn_cvt_pk_f32_fp8((int)w[d], true));
      v[4 * d] = lo[0] * f, v[4 * d + 1] = lo[1] * f, v[4 * d + 2] = hi[0] * f, v[4 * d + 3] = hi[1] * f;
    }
    st_chunk<DT>(out + (row * ldo + 8 * (int64_t)c) * ES, narrow<DT>(v), min(8, q.cols - 8 * c));
  }
}

static dim3 fp8_grid(int64_t threads) {
  return dim3((unsigned)std::max<int64_t>(1, std::min<int64_t>((threads + 255) / 256, (int64_t)cu_count() * 64)));
}

template <int DT>
static int fp8_quantize(const char* x, int64_t ldx, const Fp8& q, bool transpose, hipStream_t s) {
  if (transpose) {
    const int64_t wgs = (q.rows + 63) / 64 * q.steps;
    if (wgs > INT32_MAX) return LRQ_ERR_SHAPE;
    return launch(k_fp8_transpose<DT>, dim3((unsigned)wgs), dim3(256), 0, s, x, ldx, q);
  }
  if (q.shift == 0) return launch(k_fp8_rows<DT>, fp8_grid(q.rows * 16 * q.steps), dim3(256), 0, s, x, ldx, q);
  const int64_t wgs = (q.rows + 127) / 128 * q.steps;
  if (wgs > INT32_MAX) return LRQ_ERR_SHAPE;
  return launch(k_fp8_square<DT>, dim3((unsigned)wgs), dim3(256), 0, s, x, ldx, q);
}

}  // namespace lrq

using namespace lrq;

extern "C" int lrq_fp8_quantize(const void* x, int64_t ldx, int32_t dtype, const lrq_fp8* t, int32_t transpose, void* stream) {
  LRQ_TRY(validate_fp8(t));
  if (dtype < LRQ_BF16 || dtype > LRQ_F32 || (transpose && t->block != 1)) return LRQ_ERR_UNSUPPORTED;
  if (t->rows == 0) return LRQ_OK;
  if (x == nullptr) return LRQ_ERR_NULL;
  if (ldx < (transpose ? t->rows : t->cols)) return LRQ_ERR_SHAPE;
  if (!aligned(x, dtype == LRQ_F32 ? 4 : 2)) return LRQ_ERR_ALIGN;
  const Fp8 q = make_fp8(t);
  hipStream_t s = (hipStream_t)stream;
  switch (dtype) {
    case LRQ_BF16: return fp8_quantize<kBf16>((const char*)x, ldx, q, transpose != 0, s);
    case LRQ_F16: return fp8_quantize<kF16>((const char*)x, ldx, q, transpose != 0, s);
    default: return fp8_quantize<kF32>((const char*)x, ldx, q, transpose != 0, s);
  }
}

extern "C" int lrq_fp8_quantize_both(const void* x, int64_t ldx, int32_t dtype, const lrq_fp8* t, const lrq_fp8* tt,
                                     void* stream) {
  LRQ_TRY(validate_fp8(t));
  LRQ_TRY(validate_fp8(tt));
  if (dtype < LRQ_BF16 || dtype > LRQ_F32 || t->block != 1 || tt->block != 1) return LRQ_ERR_UNSUPPORTED;
  if (tt->rows != t->cols || tt->cols != t->rows) return LRQ_ERR_SHAPE;
  if (x == nullptr) return LRQ_ERR_NULL;
  if (ldx < t->cols) return LRQ_ERR_SHAPE;
  if (!aligned(x, dtype == LRQ_F32 ? 4 : 2)) return LRQ_ERR_ALIGN;
  const Fp8 q = make_fp8(t), qt = make_fp8(tt);
  const int64_t wgs = (q.rows + 127) / 128 * q.steps;
  if (wgs > INT32_MAX) return LRQ_ERR_SHAPE;
  hipStream_t s = (hipStream_t)stream;
  const auto go = [&](auto kern) { return launch(kern, dim3((unsigned)wgs), dim3(256), 0, s, (const char*)x, ldx, q, qt); };
  switch (dtype) {
    case LRQ_BF16: return go(k_fp8_both<kBf16>);
    case LRQ_F16: return go(k_fp8_both<kF16>);
    default: return go(k_fp8_both<kF32>);
  }
}

extern "C" int lrq_fp8_dequantize(const lrq_fp8* t, void* out, int64_t ldo, int32_t dtype, void* stream) {
  LRQ_TRY(validate_fp8(t));
  if (dtype < LRQ_BF16 || dtype > LRQ_F32) return LRQ_ERR_UNSUPPORTED;
  if (t->rows == 0) return LRQ_OK;
  if (out == nullptr) return LRQ_ERR_NULL;
  if (ldo < t->cols) return LRQ_ERR_SHAPE;
  if (!aligned(out, dtype == LRQ_F32 ? 4 : 2)) return LRQ_ERR_ALIGN;
  const Fp8 q = make_fp8(t);
  const dim3 grid = fp8_grid(q.rows * ((q.cols + 7) / 8));
  hipStream_t s = (hipStream_t)stream;
  switch (dtype) {
    case LRQ_BF16: return launch(k_fp8_dequantize<kBf16>, grid, dim3(256), 0, s, q, (char*)out, ldo);
    case LRQ_F16: return launch(k_fp8_dequantize<kF16>, grid, dim3(256), 0, s, q, (char*)out, ldo);
    default: return launch(k_fp8_dequantize<kF32>, grid, dim3(256), 0, s, q, (char*)out, ldo);
  }
}
