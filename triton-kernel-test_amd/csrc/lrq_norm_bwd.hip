// Layer norm backward (formulas and layout: lrq_norm.h).
#include "lrq_norm.h"

namespace lrq {

// dresidual and dx of one chunk from the norm's input gradient dn.
template <int DT, bool FUSED>
__device__ __forceinline__ void norm_outputs(const NormBwd& a, const DropKey& key, int64_t row, int c, int nc, int k,
                                             float* d) {
  constexpr int ES = Elem<DT>::kBytes;
  if (k <= 0) return;
  if constexpr (FUSED) {
    if (a.dh != nullptr) {
      float q[8];
      widen<DT>(ld_chunk<DT>(a.dh + (row * a.lddh + 8 * (int64_t)c) * ES, k), q);
#pragma unroll
      for (int e = 0; e < 8; ++e) d[e] = q[e] + d[e];
    }
    if (a.dres != nullptr) st_chunk<DT>(a.dres + (row * a.lddr + 8 * (int64_t)c) * ES, narrow<DT>(d), k);
    if (a.drop.keep < 65536u) drop_chunk(a.drop, key, (uint64_t)row * nc + c, d);
  }
  if (!FUSED || a.dx != nullptr) st_chunk<DT>(a.dx + (row * a.lddx + 8 * (int64_t)c) * ES, narrow<DT>(d), k);
}

// One pass over dy and h.  A thread owns the same columns in every row of its group, so dy z and dy of the
// weight gradients add up in its registers; the workgroup's groups join them in LDS at the end, and
// k_norm_wgrad adds the workgroups' sums in a fixed order.
template <int DT, int TPR, int C, bool FUSED>
__global__ __launch_bounds__((RowGeom<TPR, C>::kThreads)) void k_norm_bwd(NormBwd a) {
  using G = RowGeom<TPR, C>;
  constexpr int ES = Elem<DT>::kBytes;
  constexpr int L = TPR < 64 ? TPR : 64;
  constexpr int kCols = TPR * 8 * C;
  __shared__ float red[2][G::kGroups][G::kWaves][2];
  extern __shared__ float sums[];  // [groups][kCols], with weight gradients only
  const int t = threadIdx.x % TPR, grp = threadIdx.x / TPR, wave = t / 64;
  const int n = a.n, nc = (n + 7) / 8;
  const float rn = 1.f / (float)n;
  int valid[C];
  float wt[C][8], gw[C][8], gb[C][8];
#pragma unroll
  for (int j = 0; j < C; ++j) {
    const int c = t + j * TPR;
    valid[j] = c < nc ? min(8, n - 8 * c) : 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) wt[j][e] = 1.f, gw[j][e] = 0.f, gb[j][e] = 0.f;
    if (a.w != nullptr) ld_weight(a.w, a.wdt, 8 * (int64_t)c, valid[j], wt[j]);
  }
  DropKey key{};
  if constexpr (FUSED) key = drop_key(a.drop);
  int slot = 0;
  for (int64_t r0 = (int64_t)blockIdx.x * G::kGroups; r0 < a.rows; r0 += (int64_t)gridDim.x * G::kGroups) {
    const int64_t row = r0 + grp;
    const bool on = row < a.rows;
    const float mean = on ? a.mean[row] : 0.f, rstd = on ? a.rstd[row] : 0.f;
    float g[C][8], z[C][8];
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int j = 0; j < C; ++j) {
      const int k = on ? valid[j] : 0;
      const int64_t c8 = 8 * (int64_t)(t + j * TPR);
      // elements past the row are zero in dy, so they add nothing to any sum (z is finite there for
      // finite statistics; a row whose statistics are not finite is lost anyway)
      widen<DT>(ld_chunk<DT>(a.dy + (row * a.lddy + c8) * ES, k), g[j]);
      widen<DT>(ld_chunk<DT>(a.h + (row * a.ldh + c8) * ES, k), z[j]);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        z[j][e] = (z[j][e] - mean) * rstd;
        gw[j][e] = __builtin_fmaf(g[j][e], z[j][e], gw[j][e]);
        gb[j][e] += g[j][e];
        g[j][e] *= wt[j][e];
        s1 += g[j][e];
        s2 = __builtin_fmaf(g[j][e], z[j][e], s2);
      }
    }
    s1 = lanes_sum<L>(s1);
    s2 = lanes_sum<L>(s2);
    if constexpr (G::kWaves > 1) {
      if ((t & 63) == 0) {
        red[slot][grp][wave][0] = s1;
        red[slot][grp][wave][1] = s2;
      }
      __syncthreads();
      s1 = 0.f, s2 = 0.f;
#pragma unroll
      for (int k = 0; k < G::kWaves; ++k) {
        s1 += red[slot][grp][k][0];
        s2 += red[slot][grp][k][1];
      }
      slot ^= 1;
    }
    if (!on) continue;
    s1 *= rn, s2 *= rn;
#pragma unroll
    for (int j = 0; j < C; ++j) {
#pragma unroll
      for (int e = 0; e < 8; ++e) g[j][e] = rstd * (g[j][e] - s1 - z[j][e] * s2);
      norm_outputs<DT, FUSED>(a, key, row, t + j * TPR, nc, valid[j], g[j]);
    }
  }
  if (a.part == nullptr) return;  // uniform
  float* part = a.part + (int64_t)blockIdx.x * 2 * n;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    if (half) __syncthreads();
#pragma unroll
    for (int j = 0; j < C; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) sums[grp * kCols + 8 * (t + j * TPR) + e] = half ? gb[j][e] : gw[j][e];
    __syncthreads();
    for (int c = threadIdx.x; c < n; c += G::kThreads) {
      float s = 0.f;
      for (int k = 0; k < G::kGroups; ++k) s += sums[k * kCols + c];
      part[half * (int64_t)n + c] = s;
    }
  }
}

// Rows wider than the registers hold: one workgroup a row, swept twice; its weight gradients come from
// k_norm_cols.
template <int DT, bool FUSED>
__global__ __launch_bounds__(1024) void k_norm_bwd_wide(NormBwd a) {
  constexpr int ES = Elem<DT>::kBytes;
  __shared__ float red[2][16];
  const int n = a.n, nc = (n + 7) / 8;
  DropKey key{};
  if constexpr (FUSED) key = drop_key(a.drop);
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const float mean = a.mean[row], rstd = a.rstd[row];
    float s1 = 0.f, s2 = 0.f;
    float g[8], z[8], w[8];
    const auto load = [&](int c, int k) {
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = 1.f;
      if (a.w != nullptr) ld_weight(a.w, a.wdt, 8 * (int64_t)c, k, w);
      widen<DT>(ld_chunk<DT>(a.dy + (row * a.lddy + 8 * (int64_t)c) * ES, k), g);
      widen<DT>(ld_chunk<DT>(a.h + (row * a.ldh + 8 * (int64_t)c) * ES, k), z);
#pragma unroll
      for (int e = 0; e < 8; ++e) z[e] = (z[e] - mean) * rstd, g[e] *= w[e];
    };
    for (int c = threadIdx.x; c < nc; c += 1024) {
      load(c, min(8, n - 8 * c));
#pragma unroll
      for (int e = 0; e < 8; ++e) s1 += g[e], s2 = __builtin_fmaf(g[e], z[e], s2);
    }
    s1 = lanes_sum<64>(s1);
    s2 = lanes_sum<64>(s2);
    __syncthreads();  // red may still be read
    if ((threadIdx.x & 63) == 0) red[0][threadIdx.x >> 6] = s1, red[1][threadIdx.x >> 6] = s2;
    __syncthreads();
    s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int k = 0; k < 16; ++k) s1 += red[0][k], s2 += red[1][k];
    s1 /= (float)n, s2 /= (float)n;
    for (int c = threadIdx.x; c < nc; c += 1024) {
      const int k = min(8, n - 8 * c);
      load(c, k);
#pragma unroll
      for (int e = 0; e < 8; ++e) g[e] = rstd * (g[e] - s1 - z[e] * s2);
      norm_outputs<DT, FUSED>(a, key, row, c, nc, k, g);
    }
  }
}

// Sums of dy z and dy over the rows of one slab (blockIdx.y) for wide rows: 64 chunks a workgroup, 4
// waves that take every fourth row.
template <int DT>
__global__ __launch_bounds__(256) void k_norm_cols(NormBwd a) {
  constexpr int ES = Elem<DT>::kBytes;
  __shared__ float sums[4][512];
  const int n = a.n, nc = (n + 7) / 8, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int c = blockIdx.x * 64 + lane, k = c < nc ? min(8, n - 8 * c) : 0;
  float gw[8], gb[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) gw[e] = 0.f, gb[e] = 0.f;
  for (int64_t row = (int64_t)blockIdx.y * 4 + wave; row < a.rows; row += (int64_t)gridDim.y * 4) {
    const float mean = a.mean[row], rstd = a.rstd[row];
    float g[8], z[8];
    widen<DT>(ld_chunk<DT>(a.dy + (row * a.lddy + 8 * (int64_t)c) * ES, k), g);
    widen<DT>(ld_chunk<DT>(a.h + (row * a.ldh + 8 * (int64_t)c) * ES, k), z);
#pragma unroll
    for (int e = 0; e < 8; ++e) gw[e] = __builtin_fmaf(g[e], (z[e] - mean) * rstd, gw[e]), gb[e] += g[e];
  }
  float* part = a.part + (int64_t)blockIdx.y * 2 * n;
  for (int half = 0; half < 2; ++half) {
    if (half) __syncthreads();
#pragma unroll
    for (int e = 0; e < 8; ++e) sums[wave][8 * lane + e] = half ? gb[e] : gw[e];
    __syncthreads();
    for (int i = threadIdx.x; i < 512; i += 256) {
      const int64_t col = (int64_t)blockIdx.x * 512 + i;
      if (col < n) part[half * (int64_t)n + col] = (sums[0][i] + sums[1][i]) + (sums[2][i] + sums[3][i]);
    }
  }
}

// dw (blockIdx.y 0) or db (1): the parts' sums in the order of the parts, 64 columns a workgroup.
__global__ __launch_bounds__(1024) void k_norm_wgrad(const float* part, int parts, int n, void* dw, void* db, int wdt) {
  __shared__ float red[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t col = (int64_t)blockIdx.x * 64 + lane;
  void* out = blockIdx.y ? db : dw;
  float s = 0.f;
  if (col < n) {
#pragma unroll 8
    for (int p = wave; p < parts; p += 16) s += part[((int64_t)p * 2 + blockIdx.y) * n + col];
  }
  red[wave][lane] = s;
  __syncthreads();
  if (wave == 0 && col < n) {
    s = 0.f;
#pragma unroll
    for (int k = 0; k < 16; ++k) s += red[k][lane];
    if (wdt == kF32) reinterpret_cast<float*>(out)[col] = s;
    else if (wdt == kBf16) reinterpret_cast<uint16_t*>(out)[col] = (uint16_t)pack_bf16x2(s, 0.f);
    else reinterpret_cast<uint16_t*>(out)[col] = f16_bits(s);
  }
}

struct BwdPlan {
  int64_t grid;   // workgroups of the row kernel
  int64_t parts;  // sums of the weight gradients
};

static BwdPlan bwd_plan(int64_t rows, int64_t n) {
  constexpr int kCus = 256;  // a fixed count, so that the workspace and the order of the sums depend on the shape alone
  if (n > kNormMaxWidth) return BwdPlan{std::min<int64_t>(rows, 2 * kCus), std::min<int64_t>((rows + 3) / 4, 64)};
  int64_t grid = 0;
  with_row_geom((int)((n + 7) / 8), [&](auto tpr, auto c) {
    using G = RowGeom<tpr(), c()>;
    grid = std::min<int64_t>((rows + G::kGroups - 1) / G::kGroups, (int64_t)kCus * 1024 / G::kThreads);
    return 0;
  });
  return BwdPlan{grid, grid};
}

template <int DT, bool FUSED>
static int norm_bwd(const NormBwd& a, hipStream_t s) {
  const BwdPlan p = bwd_plan(a.rows, a.n);
  if (a.n > kNormMaxWidth) {
    if (a.part != nullptr)
      LRQ_TRY(launch((k_norm_cols<DT>), dim3((unsigned)((a.n + 511) / 512), (unsigned)p.parts), dim3(256), 0, s, a));
    return launch((k_norm_bwd_wide<DT, FUSED>), dim3((unsigned)p.grid), dim3(1024), 0, s, a);
  }
  return with_row_geom((a.n + 7) / 8, [&](auto tpr, auto c) {
    using G = RowGeom<tpr(), c()>;
    const size_t lds = a.part == nullptr ? 0 : sizeof(float) * G::kThreads * 8 * c();
    const void* kern = (const void*)k_norm_bwd<DT, tpr(), c(), FUSED>;
    if (lds >= 64 * 1024) (void)hipFuncSetAttribute(kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    return launch((k_norm_bwd<DT, tpr(), c(), FUSED>), dim3((unsigned)p.grid), dim3(G::kThreads), lds, s, a);
  });
}

}  // namespace lrq

using namespace lrq;

extern "C" int64_t lrq_layer_norm_bwd_workspace(int64_t rows, int64_t n) {
  if (rows < 0 || rows > INT32_MAX || n <= 0 || n > INT32_MAX / 2) return LRQ_ERR_SHAPE;
  return bwd_plan(rows, n).parts * 2 * n * (int64_t)sizeof(float);
}

extern "C" int lrq_layer_norm_bwd(const lrq_dropout* drop, const void* dy, int64_t lddy, const void* dh, int64_t lddh,
                                  const void* h, int64_t ldh, int32_t dtype, const void* w, int32_t w_dtype,
                                  const float* mean, const float* rstd, int64_t rows, int64_t n, void* dx, int64_t lddx,
                                  void* dresidual, int64_t ld_dresidual, void* dw, void* db, void* workspace,
                                  int64_t workspace_bytes, void* stream) {
  if (dtype < LRQ_BF16 || dtype > LRQ_F32 || w_dtype < LRQ_BF16 || w_dtype > LRQ_F32) return LRQ_ERR_UNSUPPORTED;
  if (rows < 0 || rows > INT32_MAX || n <= 0 || n > INT32_MAX / 2) return LRQ_ERR_SHAPE;
  LRQ_TRY(validate_dropout(drop));
  const bool wgrad = dw != nullptr;
  if (wgrad != (db != nullptr)) return LRQ_ERR_NULL;
  const int es = dtype == LRQ_F32 ? 4 : 2, ws = w_dtype == LRQ_F32 ? 4 : 2;
  if (!aligned(dw, ws) || !aligned(db, ws) || !aligned(w, ws)) return LRQ_ERR_ALIGN;
  if (rows > 0) {
    if (dy == nullptr || h == nullptr || mean == nullptr || rstd == nullptr) return LRQ_ERR_NULL;
    if (dx == nullptr && dresidual == nullptr) return LRQ_ERR_NULL;
    if (lddy < n || ldh < n || (dx != nullptr && lddx < n) || (dh != nullptr && lddh < n) ||
        (dresidual != nullptr && ld_dresidual < n))
      return LRQ_ERR_SHAPE;
    if (!aligned(dy, es) || !aligned(dh, es) || !aligned(h, es) || !aligned(dx, es) || !aligned(dresidual, es) ||
        !aligned(mean, 4) || !aligned(rstd, 4))
      return LRQ_ERR_ALIGN;
  }
  if (wgrad && rows > 0) {
    if (workspace == nullptr) return LRQ_ERR_NULL;
    if (!aligned(workspace, 4)) return LRQ_ERR_ALIGN;
    if (workspace_bytes < lrq_layer_norm_bwd_workspace(rows, n)) return LRQ_ERR_WORKSPACE;
  }
  hipStream_t s = (hipStream_t)stream;
  if (rows > 0) {
    const bool fused = drop != nullptr || dh != nullptr || dresidual != nullptr;
    const NormBwd a{(const char*)dy, lddy, (const char*)dh, lddh, (const char*)h, ldh, mean, rstd, w, w_dtype, (char*)dx,
                    lddx, (char*)dresidual, ld_dresidual, wgrad ? (float*)workspace : nullptr, rows, (int)n,
                    make_drop(drop)};
    const auto go = [&] {
      switch (dtype) {
        case LRQ_BF16: return fused ? norm_bwd<kBf16, true>(a, s) : norm_bwd<kBf16, false>(a, s);
        case LRQ_F16: return fused ? norm_bwd<kF16, true>(a, s) : norm_bwd<kF16, false>(a, s);
        default: return fused ? norm_bwd<kF32, true>(a, s) : norm_bwd<kF32, false>(a, s);
      }
    };
    LRQ_TRY(go());
  }
  if (!wgrad) return LRQ_OK;
  const int parts = rows > 0 ? (int)bwd_plan(rows, n).parts : 0;  // no rows: zeros
  return launch(k_norm_wgrad, dim3((unsigned)((n + 63) / 64), 2), dim3(1024), 0, s, (const float*)workspace, parts, (int)n,
                dw, db, w_dtype);
}
