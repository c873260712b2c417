// Layer norm over rows of n elements, forward and backward, alone or behind dropout + residual add.
//
//   h = residual + drop(x)                         (FUSED; else h = x)
//   m = mean(h), r = 1 / sqrt(mean((h - m)^2) + eps), z = (h - m) r, y = z w + b
//   g = dy w,  dn = r (g - mean(g) - z mean(g z)),  dw = sum_rows dy z,  db = sum_rows dy
//   dresidual = dh + dn,  dx = drop(dresidual)
//
// The threads of a row own C chunks of 8 columns each (thread t chunks t + j * threads), which stay in registers between
// the statistics and the output: one read of the row.  All sums are fp32.
#pragma once

#include "lrq_dropout.h"

#include <algorithm>

namespace lrq {

// Rows of up to 16 chunks take 16 threads, up to 64 chunks a wave, wider ones as many whole waves as they need (LANES 0,
// waves at run time): 5120 columns are five waves of two chunks a thread (forward) or ten of one (backward), with nothing
// idle.  A workgroup's row groups walk rows g, g + G, ... (G = groups in the grid).
struct RowShape {
  int lanes;   // 16, 64, or 0: several waves
  int chunks;  // a thread
  int waves;   // a row
};
// `one`: up to how many chunks a row has one a thread, `more`: how many a thread above that.
static inline RowShape row_shape(int64_t n, int64_t one, int more) {
  const int64_t nc = (n + 7) / 8;
  if (nc <= 16) return RowShape{16, 1, 1};
  if (nc <= 64) return RowShape{64, 1, 1};
  const int c = nc <= one ? 1 : more;
  return RowShape{nc <= 64 * c ? 64 : 0, c, (int)((nc + 64 * c - 1) / (64 * c))};
}

// Row groups of a workgroup of up to `waves` waves: one where the rows are too few for every CU, so that they spread.
static inline int row_groups(const RowShape& r, int64_t rows, int waves) {
  const int64_t most = r.lanes ? 64 * waves / r.lanes : std::max(1, waves / r.waves);
  return (int)std::min<int64_t>(most, std::max<int64_t>(1, r.lanes == 16 ? 4 * ((rows + 1023) / 1024) : (rows + 255) / 256));
}

// The row group of a thread, known to be the wave's where a wave holds one row: its addresses then need one register a
// chunk beside scalar bases.
template <int LANES>
__device__ __forceinline__ int wave_row(int grp) {
  return LANES == 16 ? grp : (int)__builtin_amdgcn_readfirstlane(grp);
}

// The widest row of the register-resident kernels; wider rows sweep the row again.
static constexpr int64_t kNormMaxWidth = 16384;

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
  int waves, groups;  // of a row, of a workgroup
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
  int waves, groups;  // of a row, of a workgroup
  Drop drop;
};

}  // namespace lrq
