// Layer norm over rows of n elements, forward and backward, alone or behind dropout + residual add.
//
//   h = residual + drop(x)                         (FUSED; else h = x)
//   m = mean(h), r = 1 / sqrt(mean((h - m)^2) + eps), z = (h - m) r, y = z w + b
//   g = dy w,  dn = r (g - mean(g) - z mean(g z)),  dw = sum_rows dy z,  db = sum_rows dy
//   dresidual = dh + dn,  dx = drop(dresidual)
//
// TPR consecutive threads own a row, each with C chunks of 8 columns (chunk t + j TPR), which stay
// in registers between the statistics and the output: one read of the row.  All sums are fp32.
#pragma once

#include "lrq_dropout.h"

#include <algorithm>

namespace lrq {

// A workgroup's row groups walk rows g, g + G, ... (G = groups in the grid).
template <int TPR, int C>
struct RowGeom {
  static constexpr int kThreads = TPR > 256 ? TPR : 256;
  static constexpr int kGroups = kThreads / TPR;          // row groups a workgroup
  static constexpr int kWaves = TPR > 64 ? TPR / 64 : 1;  // waves a row
};

// The widest row of the register-resident kernels; wider rows sweep the row again.
static constexpr int64_t kNormMaxWidth = 1024 * 2 * 8;

struct NormFwd {
  const char* x;
  int64_t ldx;
  const char* res;  // may be NULL (no residual)
  int64_t ldr;
  char* h;          // written when FUSED
  int64_t ldh;
  char* y;
  int64_t ldy;
  float* mean;
  float* rstd;
  const void* w;  // may be NULL: 1
  const void* b;  // may be NULL: 0
  int wdt;
  int64_t rows;
  int n;
  float eps;
  Drop drop;
};

struct NormBwd {
  const char* dy;
  int64_t lddy;
  const char* dh;  // gradient of h from its other uses, may be NULL
  int64_t lddh;
  const char* h;   // the normalised rows (x of the plain layer norm)
  int64_t ldh;
  const float* mean;
  const float* rstd;
  const void* w;
  int wdt;
  char* dx;
  int64_t lddx;
  char* dres;      // FUSED; may be NULL
  int64_t lddr;
  float* part;     // [workgroups][2][n] sums of dy z and dy, or NULL (no weight gradients)
  int64_t rows;
  int n;
  Drop drop;
};

// Picks <TPR, C> for a row of nc chunks: the fewest threads that keep a thread at 4 chunks or fewer;
// f(TPR, C) receives them as integral constants.
template <class F>
static inline int with_row_geom(int nc, F&& f) {
  using std::integral_constant;
#define LRQ_GEOM(T, CC) return f(integral_constant<int, T>{}, integral_constant<int, CC>{})
  if (nc <= 16) LRQ_GEOM(16, 1);
  if (nc <= 64) LRQ_GEOM(64, 1);
  if (nc <= 128) LRQ_GEOM(64, 2);
  if (nc <= 256) LRQ_GEOM(256, 1);
  if (nc <= 512) LRQ_GEOM(256, 2);
  if (nc <= 768) LRQ_GEOM(256, 3);
  if (nc <= 1024) LRQ_GEOM(1024, 1);
  LRQ_GEOM(1024, 2);
#undef LRQ_GEOM
}

}  // namespace lrq
