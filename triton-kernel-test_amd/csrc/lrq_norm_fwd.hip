// Layer norm forward (formulas and layout: lrq_norm.h).
#include "lrq_norm.h"

namespace lrq {

// One row's h chunk c (k valid elements): x, dropped, with the residual added, rounded and stored.
template <int DT, bool FUSED>
__device__ __forceinline__ void norm_input(const NormFwd& a, const DropKey& key, int64_t row, int c, int nc, int k,
                                           float* v) {
  constexpr int ES = Elem<DT>::kBytes;
  widen<DT>(ld_chunk<DT>(a.x + (row * a.ldx + 8 * (int64_t)c) * ES, k), v);
  if constexpr (FUSED) {
    if (k > 0) {
      if (a.drop.keep < 65536u) drop_chunk(a.drop, key, (uint64_t)row * nc + c, v);
      if (a.res != nullptr) {
        float q[8];
        widen<DT>(ld_chunk<DT>(a.res + (row * a.ldr + 8 * (int64_t)c) * ES, k), q);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = q[e] + v[e];
      }
      // the statistics are those of h as stored
      const Chunk<DT> hc = narrow<DT>(v);
      st_chunk<DT>(a.h + (row * a.ldh + 8 * (int64_t)c) * ES, hc, k);
      widen<DT>(hc, v);
    }
  }
}

// One pass: a row's chunks are read once.  Each wave reduces its part of the row to (mean, sum of
// squared deviations from it) and the waves' parts are merged (Chan, Golub and LeVeque's update), so a
// row costs one barrier and the variance never comes from a difference of large sums.
template <int DT, int TPR, int C, bool FUSED>
__global__ __launch_bounds__((RowGeom<TPR, C>::kThreads)) void k_norm_fwd(NormFwd a) {
  using G = RowGeom<TPR, C>;
  constexpr int ES = Elem<DT>::kBytes;
  constexpr int L = TPR < 64 ? TPR : 64;
  __shared__ float red[2][G::kGroups][G::kWaves][2], cnts[G::kWaves];
  const int t = threadIdx.x % TPR, grp = threadIdx.x / TPR, wave = t / 64;
  const int n = a.n, nc = (n + 7) / 8;
  int valid[C];
  float wt[C][8], bs[C][8];
  float cnt = 0.f;
#pragma unroll
  for (int j = 0; j < C; ++j) {
    const int c = t + j * TPR;
    valid[j] = c < nc ? min(8, n - 8 * c) : 0;
    cnt += (float)valid[j];
#pragma unroll
    for (int e = 0; e < 8; ++e) wt[j][e] = 1.f, bs[j][e] = 0.f;
    if (a.w != nullptr) ld_weight(a.w, a.wdt, 8 * (int64_t)c, valid[j], wt[j]);
    if (a.b != nullptr) ld_weight(a.b, a.wdt, 8 * (int64_t)c, valid[j], bs[j]);
  }
  cnt = lanes_sum<L>(cnt);  // this wave's columns of a row
  const float rcnt = cnt > 0.f ? 1.f / cnt : 0.f, rn = 1.f / (float)n;
  if constexpr (G::kWaves > 1) {
    if (grp == 0 && (t & 63) == 0) cnts[wave] = cnt;
  }
  DropKey key{};
  if constexpr (FUSED) key = drop_key(a.drop);
  int slot = 0;
  // Every thread takes every step (barriers): a group past the last row works on zeros.
  for (int64_t r0 = (int64_t)blockIdx.x * G::kGroups; r0 < a.rows; r0 += (int64_t)gridDim.x * G::kGroups) {
    const int64_t row = r0 + grp;
    const bool on = row < a.rows;
    float v[C][8];
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < C; ++j) {
      norm_input<DT, FUSED>(a, key, row, t + j * TPR, nc, on ? valid[j] : 0, v[j]);
      if (valid[j] >= 8) {
#pragma unroll
        for (int e = 0; e < 8; ++e) s += v[j][e];
      } else {
#pragma unroll
        for (int e = 0; e < 7; ++e) s += e < valid[j] ? v[j][e] : 0.f;
      }
    }
    float mean = lanes_sum<L>(s) * rcnt, m2 = 0.f;
#pragma unroll
    for (int j = 0; j < C; ++j) {
      if (valid[j] >= 8) {
#pragma unroll
        for (int e = 0; e < 8; ++e) m2 = __builtin_fmaf(v[j][e] - mean, v[j][e] - mean, m2);
      } else {
#pragma unroll
        for (int e = 0; e < 7; ++e) m2 += e < valid[j] ? (v[j][e] - mean) * (v[j][e] - mean) : 0.f;
      }
    }
    m2 = lanes_sum<L>(m2);
    if constexpr (G::kWaves > 1) {
      if ((t & 63) == 0) {
        red[slot][grp][wave][0] = mean;
        red[slot][grp][wave][1] = m2;
      }
      __syncthreads();
      float tm = 0.f;
#pragma unroll
      for (int k = 0; k < G::kWaves; ++k) tm = __builtin_fmaf(red[slot][grp][k][0], cnts[k], tm);
      mean = tm * rn;
      m2 = 0.f;
#pragma unroll
      for (int k = 0; k < G::kWaves; ++k) {
        const float d = red[slot][grp][k][0] - mean;
        m2 += __builtin_fmaf(cnts[k] * d, d, red[slot][grp][k][1]);
      }
      slot ^= 1;  // the next row's parts; this slot is written again only after its barrier
    }
    const float rstd = 1.f / sqrtf(__builtin_fmaf(m2, rn, a.eps));
    if (!on) continue;
    if (t == 0) {
      a.mean[row] = mean;
      a.rstd[row] = rstd;
    }
#pragma unroll
    for (int j = 0; j < C; ++j) {
      float o[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] = __builtin_fmaf((v[j][e] - mean) * rstd, wt[j][e], bs[j][e]);
      st_chunk<DT>(a.y + (row * a.ldy + 8 * (int64_t)(t + j * TPR)) * ES, narrow<DT>(o), valid[j]);
    }
  }
}

// Sum over the workgroup's 16 waves, in every thread (1024 threads).
__device__ __forceinline__ float block_sum1024(float v, float* red) {
  v = lanes_sum<64>(v);
  __syncthreads();  // red may still be read
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  float s = 0.f;
#pragma unroll
  for (int k = 0; k < 16; ++k) s += red[k];
  return s;
}

// Rows wider than the registers hold: one workgroup a row, which is swept three times (the mean, the
// deviations, the output); after the first the row comes from L2.
template <int DT, bool FUSED>
__global__ __launch_bounds__(1024) void k_norm_fwd_wide(NormFwd a) {
  constexpr int ES = Elem<DT>::kBytes;
  __shared__ float red[16];
  const int n = a.n, nc = (n + 7) / 8;
  DropKey key{};
  if constexpr (FUSED) key = drop_key(a.drop);
  const char* src = FUSED ? a.h : a.x;
  const int64_t lds = FUSED ? a.ldh : a.ldx;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    float v[8], s = 0.f;
    for (int c = threadIdx.x; c < nc; c += 1024) {
      const int k = min(8, n - 8 * c);
      norm_input<DT, FUSED>(a, key, row, c, nc, k, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) s += e < k ? v[e] : 0.f;
    }
    const float mean = block_sum1024(s, red) / (float)n;
    float m2 = 0.f;
    for (int c = threadIdx.x; c < nc; c += 1024) {  // each thread re-reads what it wrote
      const int k = min(8, n - 8 * c);
      widen<DT>(ld_chunk<DT>(src + (row * lds + 8 * (int64_t)c) * ES, k), v);
#pragma unroll
      for (int e = 0; e < 8; ++e) m2 += e < k ? (v[e] - mean) * (v[e] - mean) : 0.f;
    }
    const float rstd = 1.f / sqrtf(block_sum1024(m2, red) / (float)n + a.eps);
    if (threadIdx.x == 0) {
      a.mean[row] = mean;
      a.rstd[row] = rstd;
    }
    for (int c = threadIdx.x; c < nc; c += 1024) {
      const int k = min(8, n - 8 * c);
      float w[8], b[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = 1.f, b[e] = 0.f;
      if (a.w != nullptr) ld_weight(a.w, a.wdt, 8 * (int64_t)c, k, w);
      if (a.b != nullptr) ld_weight(a.b, a.wdt, 8 * (int64_t)c, k, b);
      widen<DT>(ld_chunk<DT>(src + (row * lds + 8 * (int64_t)c) * ES, k), v);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = __builtin_fmaf((v[e] - mean) * rstd, w[e], b[e]);
      st_chunk<DT>(a.y + (row * a.ldy + 8 * (int64_t)c) * ES, narrow<DT>(v), k);
    }
  }
}

template <int DT, bool FUSED>
static int norm_fwd(const NormFwd& a, hipStream_t s) {
  const int cus = cu_count();
  if (a.n > kNormMaxWidth)
    return launch((k_norm_fwd_wide<DT, FUSED>), dim3((unsigned)std::min<int64_t>(a.rows, 2 * cus)), dim3(1024), 0, s, a);
  return with_row_geom((a.n + 7) / 8, [&](auto tpr, auto c) {
    using G = RowGeom<tpr(), c()>;
    // as many workgroups as run at once (8 waves per SIMD), each walking rows with the weights held
    const int64_t most = (int64_t)cus * (2048 / G::kThreads);
    const int64_t grid = std::min<int64_t>((a.rows + G::kGroups - 1) / G::kGroups, most);
    return launch((k_norm_fwd<DT, tpr(), c(), FUSED>), dim3((unsigned)grid), dim3(G::kThreads), 0, s, a);
  });
}

}  // namespace lrq

using namespace lrq;

extern "C" int lrq_layer_norm_fwd(const lrq_dropout* drop, const void* x, int64_t ldx, const void* residual,
                                  int64_t ld_residual, int32_t dtype, const void* w, const void* b, int32_t w_dtype,
                                  int64_t rows, int64_t n, float eps, void* h, int64_t ldh, void* y, int64_t ldy,
                                  float* mean, float* rstd, void* stream) {
  const bool fused = h != nullptr;
  if (!fused && (drop != nullptr || residual != nullptr)) return LRQ_ERR_NULL;
  if (dtype < LRQ_BF16 || dtype > LRQ_F32 || w_dtype < LRQ_BF16 || w_dtype > LRQ_F32) return LRQ_ERR_UNSUPPORTED;
  if (rows < 0 || rows > INT32_MAX || n <= 0 || n > INT32_MAX / 2) return LRQ_ERR_SHAPE;
  LRQ_TRY(validate_dropout(drop));
  if (rows == 0) return LRQ_OK;
  if (x == nullptr || y == nullptr || mean == nullptr || rstd == nullptr) return LRQ_ERR_NULL;
  if (ldx < n || ldy < n || (fused && ldh < n) || (residual != nullptr && ld_residual < n)) return LRQ_ERR_SHAPE;
  const int es = dtype == LRQ_F32 ? 4 : 2, ws = w_dtype == LRQ_F32 ? 4 : 2;
  if (!aligned(x, es) || !aligned(y, es) || !aligned(h, es) || !aligned(residual, es) || !aligned(w, ws) ||
      !aligned(b, ws) || !aligned(mean, 4) || !aligned(rstd, 4))
    return LRQ_ERR_ALIGN;
  const NormFwd a{(const char*)x, ldx, (const char*)residual, ld_residual, (char*)h, ldh, (char*)y, ldy, mean, rstd, w, b,
                  w_dtype, rows, (int)n, eps, make_drop(drop)};
  hipStream_t s = (hipStream_t)stream;
  switch (dtype) {
    case LRQ_BF16: return fused ? norm_fwd<kBf16, true>(a, s) : norm_fwd<kBf16, false>(a, s);
    case LRQ_F16: return fused ? norm_fwd<kF16, true>(a, s) : norm_fwd<kF16, false>(a, s);
    default: return fused ? norm_fwd<kF32, true>(a, s) : norm_fwd<kF32, false>(a, s);
  }
}
