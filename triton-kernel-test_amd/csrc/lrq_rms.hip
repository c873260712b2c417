// Root-mean-square norm over rows of n elements, forward and backward, alone or behind a residual add, with an output of the
// row's type or in e4m3 (lrq_fp8.h).
//
//   h = residual + x (or x),  r = 1 / sqrt(mean(h^2) + eps),  z = h r,  y = z w
//   g = dy w,  dx = dh + r (g - z mean(g z)),  dw = sum_rows dy z
//
// Rows are laid over threads as in the layer norm (lrq_norm.h): thread t of a row owns its chunks t + j * threads of 8
// columns, which stay in registers between the sum and the output.  All sums are fp32.
//
// Both directions are bound by memory, every operand is read once and every result written once.  A large copy on this card
// reads and writes 5.1 TB/s.
#include "lrq_fp8.h"
#include "lrq_norm.h"

namespace lrq {

struct RmsFwd {
  const char* x;
  int64_t ldx;
  const char* res;  // may be NULL
  int64_t ldr;
  char* h;          // written when RES
  int64_t ldh;
  char* y;          // or q
  int64_t ldy;
  Fp8 q;
  float* rstd;
  const void* w;    // may be NULL: 1
  int wdt;
  int64_t rows;
  int n;
  int waves, groups;  // of a row, of a workgroup
  float eps;
};

template <int DT>
__device__ __forceinline__ void add_chunks(const Chunk<DT>& x, const Chunk<DT>& r, float* v) {
  float q[8];
  widen<DT>(x, v);
  widen<DT>(r, q);
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = q[e] + v[e];
}

// A chunk of y: stored in the row's type, or quantised with the other 15 lanes' chunks of its block of 128.
template <int DT, bool OUT8>
__device__ __forceinline__ void rms_out(const RmsFwd& a, int64_t row, int c, int valid, const float* o) {
  if constexpr (OUT8) {
    const uint32_t s = fp8_scale(lanes16_max(top8(o)));
    if (c < 16 * a.q.steps) {
      st8(a.q.codes + row * a.q.ldc + 8 * (int64_t)c, fp8_codes8(o, s));
      if ((c & 15) == 0) a.q.scales[row * a.q.lds + c / 16] = (uint8_t)s;
    }
  } else {
    st_chunk<DT>(a.y + row * a.ldy * Elem<DT>::kBytes + 8u * Elem<DT>::kBytes * (uint32_t)c, narrow<DT>(o), valid);
  }
}

// One pass: a row is read once and the next one is on its way while it is reduced and written.  bf16 [16384, 4096]: with
// the residual 90-102 us (5.3-6.0 TB/s over x, residual, h and y), with 8-bit output 88 (5.3), alone 43 (6.3); [8, 4096]: 4.3,
// of which 3.4 are a launch.  The output in 8 bits costs no second pass: 16 lanes hold a block of 128 columns.
template <int DT, int LANES, int C, bool RES, bool OUT8>
__global__ __launch_bounds__(1024) void k_rms_fwd(RmsFwd a) {
  constexpr int ES = Elem<DT>::kBytes, L = LANES == 16 ? 16 : 64;
  __shared__ float red[2][16];
  const int tpr = LANES ? LANES : 64 * a.waves;
  const int grp = wave_row<LANES>(threadIdx.x / tpr), t = threadIdx.x - grp * tpr;
  const int wv = threadIdx.x >> 6, w0 = LANES ? 0 : grp * a.waves;  // this wave, its row's first
  const int n = a.n, nc = (n + 7) / 8;
  const bool odd = n >= 8 && n % 8 != 0;  // rows end inside a chunk, and are as long as one
  int valid[C];
  float wt[C][8];
#pragma unroll
  for (int j = 0; j < C; ++j) {
    const int c = t + j * tpr;
    valid[j] = c < nc ? min(8, n - 8 * c) : 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) wt[j][e] = 1.f;
    if (a.w != nullptr) ld_weight(a.w, a.wdt, 8 * (int64_t)c, valid[j], wt[j]);
  }
  const float rn = 1.f / (float)n;
  struct Row {
    Chunk<DT> x[C], res[RES ? C : 1];
  };
  const auto load = [&](int64_t row) {
    Row r;
    const bool on = row < a.rows;
#pragma unroll
    for (int j = 0; j < C; ++j) {
      const uint32_t at = 8u * ES * (uint32_t)(t + j * tpr);
      const int k = on ? load_size(valid[j], odd && row + 1 < a.rows) : 0;
      r.x[j] = ld_chunk<DT>(a.x + row * a.ldx * ES + at, k);
      if constexpr (RES) r.res[j] = ld_chunk<DT>(a.res + row * a.ldr * ES + at, a.res != nullptr ? k : 0);
    }
    return r;
  };
  int slot = 0;
  const int64_t step = (int64_t)gridDim.x * a.groups;
  Row cur = load((int64_t)blockIdx.x * a.groups + grp);
  // here ahead of the loop, or the wait for it is in the loop, where it meets the next row's loads as well
#pragma unroll
  for (int j = 0; j < C; ++j) {
    pin(cur.x[j]);
    if constexpr (RES) pin(cur.res[j]);
  }
  // every thread takes every step (barriers): a group past the last row works on zeros
  for (int64_t r0 = (int64_t)blockIdx.x * a.groups; r0 < a.rows; r0 += step) {
    const int64_t row = r0 + grp;
    const bool on = row < a.rows;
    if constexpr (C > 1) {  // (the scalar registers do not hold all comparisons over the loop)
#pragma unroll
      for (int j = 0; j < C; ++j) opaque(valid[j]);
    }
    const Row next = load(row + step);
    float v[C][8];
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < C; ++j) {
      mask_chunk<DT>(cur.x[j], valid[j]);
      if constexpr (RES) {
        mask_chunk<DT>(cur.res[j], valid[j]);
        add_chunks<DT>(cur.x[j], cur.res[j], v[j]);
        const Chunk<DT> hc = narrow<DT>(v[j]);  // the norm is that of h as stored
        if (on) st_chunk<DT>(a.h + row * a.ldh * ES + 8u * ES * (uint32_t)(t + j * tpr), hc, valid[j]);
        widen<DT>(hc, v[j]);
      } else {
        widen<DT>(cur.x[j], v[j]);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) s = __builtin_fmaf(v[j][e], v[j][e], s);
    }
    s = lanes_sum<L>(s);
    if constexpr (LANES == 0) {
      if ((threadIdx.x & 63) == 0) red[slot][wv] = s;
      lds_meet();  // (leaves the next row's loads in flight)
      const int k = threadIdx.x & 15;  // each 16 lanes add the waves' sums
      s = lanes_sum<16>(k < a.waves ? red[slot][w0 + k] : 0.f);
      slot ^= 1;  // this slot is written again only after the next row's barrier
    }
    const float rstd = 1.f / sqrtf(__builtin_fmaf(s, rn, a.eps));
    cur = next;
    if (!on) continue;
    if (t == 0) a.rstd[row] = rstd;
#pragma unroll
    for (int j = 0; j < C; ++j) {
      float o[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] = v[j][e] * rstd * wt[j][e];
      rms_out<DT, OUT8>(a, row, t + j * tpr, valid[j], o);
    }
  }
}

// Sum over the workgroup's 16 waves, in every thread (1024 threads).
__device__ __forceinline__ float rms_block_sum(float v, float* red) {
  v = lanes_sum<64>(v);
  __syncthreads();  // red may still be read
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  float s = 0.f;
#pragma unroll
  for (int k = 0; k < 16; ++k) s += red[k];
  return s;
}

// Rows wider than the registers hold: a workgroup a row, swept twice; the second time it comes from L2.  bf16 [2048, 20000]
// with the residual: 67 us, 4.9 TB/s.
template <int DT, bool RES, bool OUT8>
__global__ __launch_bounds__(1024) void k_rms_fwd_wide(RmsFwd a) {
  constexpr int ES = Elem<DT>::kBytes;
  __shared__ float red[16];
  const int n = a.n, nc = (n + 7) / 8, end = OUT8 ? 16 * a.q.steps : nc;
  const char* src = RES ? a.h : a.x;
  const int64_t lds = RES ? a.ldh : a.ldx;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    float v[8], s = 0.f;
    for (int c = threadIdx.x; c < nc; c += 1024) {
      const int k = min(8, n - 8 * c);
      const Chunk<DT> x = ld_chunk<DT>(a.x + (row * a.ldx + 8 * (int64_t)c) * ES, k);
      if constexpr (RES) {
        add_chunks<DT>(x, ld_chunk<DT>(a.res + (row * a.ldr + 8 * (int64_t)c) * ES, a.res != nullptr ? k : 0), v);
        const Chunk<DT> hc = narrow<DT>(v);
        st_chunk<DT>(a.h + (row * a.ldh + 8 * (int64_t)c) * ES, hc, k);
        widen<DT>(hc, v);
      } else {
        widen<DT>(x, v);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) s = __builtin_fmaf(v[e], v[e], s);
    }
    const float rstd = 1.f / sqrtf(rms_block_sum(s, red) / (float)n + a.eps);
    if (threadIdx.x == 0) a.rstd[row] = rstd;
    for (int c = threadIdx.x; c < end; c += 1024) {  // each thread re-reads what it wrote
      const int k = min(8, n - 8 * c);
      float w[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = 1.f;
      if (a.w != nullptr) ld_weight(a.w, a.wdt, 8 * (int64_t)c, k, w);
      widen<DT>(ld_chunk<DT>(src + (row * lds + 8 * (int64_t)c) * ES, k), v);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = v[e] * rstd * w[e];
      rms_out<DT, OUT8>(a, row, c, k, v);
    }
  }
}

// Row groups of a workgroup, `most` at most and `each` workgroups at a time on a CU: the largest number that leaves the CU with
// the most rows as few as any does (1003 rows in groups of three, which a CU takes two rounds of, are up to six a CU; of
// two, four).
template <class F>
static int even_groups(int most, int64_t rows, F each) {
  int best = most;
  int64_t least = INT64_MAX;
  for (int g = most; g >= 1; --g) {
    const int64_t per = (int64_t)each(g) * g, load = (rows + 256 * per - 1) / (256 * per) * per;
    if (load < least) best = g, least = load;
  }
  return best;
}

template <int DT, bool RES, bool OUT8>
static int rms_fwd(RmsFwd a, hipStream_t s) {
  const int cus = cu_count();
  if (a.n > kNormMaxWidth)
    return launch((k_rms_fwd_wide<DT, RES, OUT8>), dim3((unsigned)std::min<int64_t>(a.rows, 2 * cus)), dim3(1024), 0, s, a);
  const RowShape r = row_shape(a.n, 64, 2);
  a.waves = r.waves;
  a.groups = row_groups(r, a.rows, 16);
  if (r.lanes == 0) a.groups = even_groups(a.groups, a.rows, [&](int g) { return 16 / (r.waves * g); });
  const int threads = std::max(64, (r.lanes ? r.lanes : 64 * r.waves) * a.groups);
  // as many workgroups as run at once (4 waves per SIMD), each walking rows with the weights held
  const int64_t grid = std::min<int64_t>((a.rows + a.groups - 1) / a.groups, (int64_t)cus * (1024 / threads));
  const auto go = [&](auto kern) { return launch(kern, dim3((unsigned)grid), dim3(threads), 0, s, a); };
  if (r.lanes == 16) return go(k_rms_fwd<DT, 16, 1, RES, OUT8>);
  if (r.lanes == 64) return r.chunks == 1 ? go(k_rms_fwd<DT, 64, 1, RES, OUT8>) : go(k_rms_fwd<DT, 64, 2, RES, OUT8>);
  return go(k_rms_fwd<DT, 0, 2, RES, OUT8>);
}

struct RmsBwd {
  const char* dy;
  int64_t lddy;
  const char* dh;  // gradient of h from its other uses (DH)
  int64_t lddh;
  const char* h;
  int64_t ldh;
  const float* rstd;
  const void* w;
  int wdt;
  char* dx;
  int64_t lddx;
  float* part;     // [workgroups][n] sums of dy z, or NULL (no weight gradient)
  int64_t rows;
  int n;
  int waves, groups;  // of a row, of a workgroup
};

// One pass over dy, h and dh.  A thread owns the same columns in every row of its group, so dy z of the weight gradient adds
// up in its registers; the workgroup's groups join it in LDS at the end, and k_rms_wgrad adds the workgroups' sums in a
// fixed order.  bf16 [16384, 4096], weight gradient included: 104 us with dh (5.2 TB/s over dy, h, dh and dx), 72-77 without.  The
// next row's loads are ahead only where a thread owns one chunk: with two, the registers do not hold them and it was slower;
// four chunks (rows of 8200 to 16384) read a row when its turn comes, 4.6 TB/s at [4096, 14336].  Rows that end inside a
// chunk: 3.9 TB/s with dh ([8192, 5003]).
template <int DT, int LANES, int C, bool DH>
__global__ __launch_bounds__(C == 4 ? 512 : 1024) void k_rms_bwd(RmsBwd a) {
  constexpr int ES = Elem<DT>::kBytes, L = LANES == 16 ? 16 : 64;
  constexpr bool kPrefetch = C == 1;
  __shared__ float red[2][16];
  extern __shared__ float sums[];  // [groups][threads of a row * 8 C], with a weight gradient only
  const int tpr = LANES ? LANES : 64 * a.waves, kCols = tpr * 8 * C;
  const int grp = wave_row<LANES>(threadIdx.x / tpr), t = threadIdx.x - grp * tpr;
  const int wv = threadIdx.x >> 6, w0 = LANES ? 0 : grp * a.waves;
  const int n = a.n, nc = (n + 7) / 8;
  const bool odd = n >= 8 && n % 8 != 0;
  const float rn = 1.f / (float)n;
  int valid[C];
  float gw[C][8], wt[C][8];
#pragma unroll
  for (int j = 0; j < C; ++j) {
    const int c = t + j * tpr;
    valid[j] = c < nc ? min(8, n - 8 * c) : 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) gw[j][e] = 0.f, wt[j][e] = 1.f;
    if (a.w != nullptr) ld_weight(a.w, a.wdt, 8 * (int64_t)c, valid[j], wt[j]);
  }
  struct Row {
    Chunk<DT> dy[C], h[C], dh[DH ? C : 1];
    float rstd;
  };
  const auto load = [&](int64_t row) {
    Row r;
    const bool on = row < a.rows;
    r.rstd = on ? a.rstd[row] : 0.f;
#pragma unroll
    for (int j = 0; j < C; ++j) {
      const uint32_t at = 8u * ES * (uint32_t)(t + j * tpr);
      const int k = on ? load_size(valid[j], odd && row + 1 < a.rows) : 0;
      r.dy[j] = ld_chunk<DT>(a.dy + row * a.lddy * ES + at, k);
      r.h[j] = ld_chunk<DT>(a.h + row * a.ldh * ES + at, k);
      if constexpr (DH) r.dh[j] = ld_chunk<DT>(a.dh + row * a.lddh * ES + at, k);
    }
    return r;
  };
  int slot = 0;
  const int64_t step = (int64_t)gridDim.x * a.groups, row0 = (int64_t)blockIdx.x * a.groups + grp;
  Row cur;
  if constexpr (kPrefetch) {
    cur = load(row0);
    asm volatile("" : "+v"(cur.rstd));  // ahead of the loop, as in k_rms_fwd
    pin(cur.dy[0]);
    pin(cur.h[0]);
    if constexpr (DH) pin(cur.dh[0]);
  }
  for (int64_t r0 = (int64_t)blockIdx.x * a.groups; r0 < a.rows; r0 += step) {
    const int64_t row = r0 + grp;
    if constexpr (C > 1) {
#pragma unroll
      for (int j = 0; j < C; ++j) opaque(valid[j]);
    }
    Row next;
    if constexpr (kPrefetch) next = load(row + step);
    else cur = load(row);
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < C; ++j) {
      float g[8], z[8];
      mask_chunk<DT>(cur.dy[j], valid[j]);
      mask_chunk<DT>(cur.h[j], valid[j]);
      widen<DT>(cur.dy[j], g);
      widen<DT>(cur.h[j], z);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float zz = z[e] * cur.rstd;
        gw[j][e] = __builtin_fmaf(g[e], zz, gw[j][e]);
        s = __builtin_fmaf(g[e] * wt[j][e], zz, s);
      }
    }
    s = lanes_sum<L>(s);
    if constexpr (LANES == 0) {
      if ((threadIdx.x & 63) == 0) red[slot][wv] = s;
      lds_meet();  // (leaves the next row's loads in flight)
      const int k = threadIdx.x & 15;
      s = lanes_sum<16>(k < a.waves ? red[slot][w0 + k] : 0.f);
      slot ^= 1;
    }
    if (row < a.rows) {
      const float c2 = -(s * rn);
#pragma unroll
      for (int j = 0; j < C; ++j) {
        if constexpr (C > 1) opaque(valid[j]);
        float g[8], z[8];
        widen<DT>(cur.dy[j], g);
        widen<DT>(cur.h[j], z);
#pragma unroll
        for (int e = 0; e < 8; ++e) g[e] = cur.rstd * __builtin_fmaf(z[e] * cur.rstd, c2, g[e] * wt[j][e]);
        if constexpr (DH) {
          float d[8];
          widen<DT>(cur.dh[j], d);
#pragma unroll
          for (int e = 0; e < 8; ++e) g[e] = d[e] + g[e];
        }
        st_chunk<DT>(a.dx + row * a.lddx * ES + 8u * ES * (uint32_t)(t + j * tpr), narrow<DT>(g), valid[j]);
      }
    }
    if constexpr (kPrefetch) cur = next;
  }
  if (a.part == nullptr) return;  // uniform
  float* part = a.part + (int64_t)blockIdx.x * n;
#pragma unroll
  for (int j = 0; j < C; ++j)
#pragma unroll
    for (int e = 0; e < 8; ++e) sums[grp * kCols + 8 * (t + j * tpr) + e] = gw[j][e];
  __syncthreads();
  for (int c = threadIdx.x; c < n; c += blockDim.x) {
    float s = 0.f;
    for (int k = 0; k < a.groups; ++k) s += sums[k * kCols + c];
    part[c] = s;
  }
}

// Rows wider than the registers hold: a workgroup a row, swept twice; its weight gradient comes from k_rms_cols.  bf16
// [2048, 20000]: 72 us with dh, and 27 of k_rms_cols, which reads dy and h again.
template <int DT, bool DH>
__global__ __launch_bounds__(1024) void k_rms_bwd_wide(RmsBwd a) {
  constexpr int ES = Elem<DT>::kBytes;
  __shared__ float red[16];
  const int n = a.n, nc = (n + 7) / 8;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const float rstd = a.rstd[row];
    float g[8], z[8], w[8], s = 0.f;
    const auto load = [&](int c, int k) {
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = 1.f;
      if (a.w != nullptr) ld_weight(a.w, a.wdt, 8 * (int64_t)c, k, w);
      widen<DT>(ld_chunk<DT>(a.dy + (row * a.lddy + 8 * (int64_t)c) * ES, k), g);
      widen<DT>(ld_chunk<DT>(a.h + (row * a.ldh + 8 * (int64_t)c) * ES, k), z);
#pragma unroll
      for (int e = 0; e < 8; ++e) z[e] *= rstd, g[e] *= w[e];
    };
    for (int c = threadIdx.x; c < nc; c += 1024) {
      load(c, min(8, n - 8 * c));
#pragma unroll
      for (int e = 0; e < 8; ++e) s = __builtin_fmaf(g[e], z[e], s);
    }
    s = rms_block_sum(s, red) / (float)n;
    for (int c = threadIdx.x; c < nc; c += 1024) {
      const int k = min(8, n - 8 * c);
      load(c, k);
#pragma unroll
      for (int e = 0; e < 8; ++e) g[e] = rstd * (g[e] - z[e] * s);
      if constexpr (DH) {
        float d[8];
        widen<DT>(ld_chunk<DT>(a.dh + (row * a.lddh + 8 * (int64_t)c) * ES, k), d);
#pragma unroll
        for (int e = 0; e < 8; ++e) g[e] = d[e] + g[e];
      }
      st_chunk<DT>(a.dx + (row * a.lddx + 8 * (int64_t)c) * ES, narrow<DT>(g), k);
    }
  }
}

// Sums of dy z over the rows of one slab (blockIdx.y) for wide rows: 64 chunks a workgroup, 4 waves that take every
// fourth row.
template <int DT>
__global__ __launch_bounds__(256) void k_rms_cols(RmsBwd a) {
  constexpr int ES = Elem<DT>::kBytes;
  __shared__ float sums[4][512];
  const int n = a.n, nc = (n + 7) / 8, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int c = blockIdx.x * 64 + lane, k = c < nc ? min(8, n - 8 * c) : 0;
  float gw[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) gw[e] = 0.f;
  for (int64_t row = (int64_t)blockIdx.y * 4 + wave; row < a.rows; row += (int64_t)gridDim.y * 4) {
    const float rstd = a.rstd[row];
    float g[8], z[8];
    widen<DT>(ld_chunk<DT>(a.dy + (row * a.lddy + 8 * (int64_t)c) * ES, k), g);
    widen<DT>(ld_chunk<DT>(a.h + (row * a.ldh + 8 * (int64_t)c) * ES, k), z);
#pragma unroll
    for (int e = 0; e < 8; ++e) gw[e] = __builtin_fmaf(g[e], z[e] * rstd, gw[e]);
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) sums[wave][8 * lane + e] = gw[e];
  __syncthreads();
  for (int i = threadIdx.x; i < 512; i += 256) {
    const int64_t col = (int64_t)blockIdx.x * 512 + i;
    if (col < n) a.part[(int64_t)blockIdx.y * n + col] = (sums[0][i] + sums[1][i]) + (sums[2][i] + sums[3][i]);
  }
}

// dw: the parts' sums in a fixed order, 32 columns a workgroup: thread (g, c) adds every 32nd part from g on, eight loads in
// flight.  256 parts of 4096 columns (4 MB): 4.6 us, launch included.
__global__ __launch_bounds__(1024) void k_rms_wgrad(const float* part, int parts, int n, void* dw, int wdt) {
  __shared__ float red[32][33];
  const int c = threadIdx.x & 31, g = threadIdx.x >> 5;
  const int64_t col = (int64_t)blockIdx.x * 32 + c;
  float s = 0.f;
  if (col < n) {
#pragma unroll 8
    for (int p = g; p < parts; p += 32) s += part[(int64_t)p * n + col];
  }
  red[g][c] = s;
  __syncthreads();
  if (g == 0 && col < n) {
    s = 0.f;
#pragma unroll
    for (int k = 0; k < 32; ++k) s += red[k][c];
    if (wdt == kF32) reinterpret_cast<float*>(dw)[col] = s;
    else if (wdt == kBf16) reinterpret_cast<uint16_t*>(dw)[col] = (uint16_t)pack_bf16x2(s, 0.f);
    else reinterpret_cast<uint16_t*>(dw)[col] = f16_bits(s);
  }
}

struct RmsPlan {
  RowShape shape;
  int groups;     // rows a workgroup takes at a time
  int64_t grid;   // workgroups of the row kernel
  int64_t parts;  // sums of the weight gradient
};

// Rows the register-resident kernel takes: four fp32 chunks a thread do not fit.
static bool rms_wide(int64_t n, int dt) { return n > (dt == kF32 ? 8192 : kNormMaxWidth); }

static RmsPlan rms_plan(int64_t rows, int64_t n, int dt) {
  constexpr int kCus = 256;  // a fixed count, so that the workspace and the order of the sums depend on the shape alone
  RmsPlan p{row_shape(n, 1024, 4), 1, 0, 0};
  if (rms_wide(n, dt)) {
    p.grid = std::min<int64_t>(rows, 2 * kCus);
    p.parts = std::min<int64_t>((rows + 3) / 4, 64);
    return p;
  }
  p.groups = row_groups(p.shape, rows, p.shape.chunks == 4 ? 8 : 16);
  if (p.shape.lanes == 0) p.groups = even_groups(p.groups, rows, [](int) { return 1; });
  p.grid = p.parts = std::min<int64_t>((rows + p.groups - 1) / p.groups, kCus);
  return p;
}

template <int DT, bool DH>
static int rms_bwd(RmsBwd a, hipStream_t s) {
  const RmsPlan p = rms_plan(a.rows, a.n, DT);
  if (rms_wide(a.n, DT)) {
    if (a.part != nullptr)
      LRQ_TRY(launch((k_rms_cols<DT>), dim3((unsigned)((a.n + 511) / 512), (unsigned)p.parts), dim3(256), 0, s, a));
    return launch((k_rms_bwd_wide<DT, DH>), dim3((unsigned)p.grid), dim3(1024), 0, s, a);
  }
  a.waves = p.shape.waves;
  a.groups = p.groups;
  const int threads = std::max(64, (p.shape.lanes ? p.shape.lanes : 64 * p.shape.waves) * p.groups);
  const size_t lds = a.part == nullptr ? 0 : sizeof(float) * threads * 8 * p.shape.chunks;
  const auto go = [&](auto kern) {
    if (lds >= 64 * 1024) {
      const hipError_t e = hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
      if (e != hipSuccess) return (int)e;
    }
    return launch(kern, dim3((unsigned)p.grid), dim3(threads), lds, s, a);
  };
  if (p.shape.lanes == 16) return go(k_rms_bwd<DT, 16, 1, DH>);
  if (p.shape.lanes == 64) return go(k_rms_bwd<DT, 64, 1, DH>);
  if (p.shape.chunks == 1) return go(k_rms_bwd<DT, 0, 1, DH>);
  if constexpr (DT != kF32) return go(k_rms_bwd<DT, 0, 4, DH>);
  return LRQ_ERR_UNSUPPORTED;  // (not reached: wide)
}

}  // namespace lrq

using namespace lrq;

extern "C" int lrq_rms_norm_fwd(const void* x, int64_t ldx, const void* residual, int64_t ld_residual, int32_t dtype,
                                const void* w, int32_t w_dtype, int64_t rows, int64_t n, float eps, void* h, int64_t ldh,
                                void* y, int64_t ldy, const lrq_fp8* q, float* rstd, void* stream) {
  const bool res = h != nullptr, out8 = q != nullptr;
  if (!res && residual != nullptr) return LRQ_ERR_NULL;
  if (dtype < LRQ_BF16 || dtype > LRQ_F32 || w_dtype < LRQ_BF16 || w_dtype > LRQ_F32) return LRQ_ERR_UNSUPPORTED;
  if (rows < 0 || rows > INT32_MAX || n <= 0 || n > INT32_MAX / 2) return LRQ_ERR_SHAPE;
  if (out8) {
    LRQ_TRY(validate_fp8(q));
    if (y != nullptr || q->block != 1) return LRQ_ERR_UNSUPPORTED;
    if (q->rows != rows || q->cols != n) return LRQ_ERR_SHAPE;
  }
  if (rows == 0) return LRQ_OK;
  if (x == nullptr || (y == nullptr && !out8) || rstd == nullptr) return LRQ_ERR_NULL;
  if (ldx < n || (!out8 && ldy < n) || (res && ldh < n) || (residual != nullptr && ld_residual < n)) return LRQ_ERR_SHAPE;
  const int es = dtype == LRQ_F32 ? 4 : 2, ws = w_dtype == LRQ_F32 ? 4 : 2;
  if (!aligned(x, es) || !aligned(y, es) || !aligned(h, es) || !aligned(residual, es) || !aligned(w, ws) || !aligned(rstd, 4))
    return LRQ_ERR_ALIGN;
  const RmsFwd a{(const char*)x, ldx, (const char*)residual, ld_residual, (char*)h, ldh, (char*)y, ldy,
                 out8 ? make_fp8(q) : Fp8{}, rstd, w, w_dtype, rows, (int)n, 0, 0, eps};
  hipStream_t s = (hipStream_t)stream;
  const auto go = [&](auto dt) {
    if (out8) return res ? rms_fwd<dt(), true, true>(a, s) : rms_fwd<dt(), false, true>(a, s);
    return res ? rms_fwd<dt(), true, false>(a, s) : rms_fwd<dt(), false, false>(a, s);
  };
  switch (dtype) {
    case LRQ_BF16: return go(std::integral_constant<int, kBf16>{});
    case LRQ_F16: return go(std::integral_constant<int, kF16>{});
    default: return go(std::integral_constant<int, kF32>{});
  }
}

extern "C" int64_t lrq_rms_norm_bwd_workspace(int64_t rows, int64_t n) {
  if (rows < 0 || rows > INT32_MAX || n <= 0 || n > INT32_MAX / 2) return LRQ_ERR_SHAPE;
  return std::max(rms_plan(rows, n, kBf16).parts, rms_plan(rows, n, kF32).parts) * n * (int64_t)sizeof(float);
}

extern "C" int lrq_rms_norm_bwd(const void* dy, int64_t lddy, const void* dh, int64_t lddh, const void* h, int64_t ldh,
                                int32_t dtype, const void* w, int32_t w_dtype, const float* rstd, int64_t rows, int64_t n,
                                void* dx, int64_t lddx, void* dw, void* workspace, int64_t workspace_bytes, void* stream) {
  if (dtype < LRQ_BF16 || dtype > LRQ_F32 || w_dtype < LRQ_BF16 || w_dtype > LRQ_F32) return LRQ_ERR_UNSUPPORTED;
  if (rows < 0 || rows > INT32_MAX || n <= 0 || n > INT32_MAX / 2) return LRQ_ERR_SHAPE;
  const int es = dtype == LRQ_F32 ? 4 : 2, ws = w_dtype == LRQ_F32 ? 4 : 2;
  if (!aligned(dw, ws) || !aligned(w, ws)) return LRQ_ERR_ALIGN;
  if (rows > 0) {
    if (dy == nullptr || h == nullptr || rstd == nullptr || dx == nullptr) return LRQ_ERR_NULL;
    if (lddy < n || ldh < n || lddx < n || (dh != nullptr && lddh < n)) return LRQ_ERR_SHAPE;
    if (!aligned(dy, es) || !aligned(dh, es) || !aligned(h, es) || !aligned(dx, es) || !aligned(rstd, 4)) return LRQ_ERR_ALIGN;
  }
  if (dw != nullptr && rows > 0) {
    if (workspace == nullptr) return LRQ_ERR_NULL;
    if (!aligned(workspace, 4)) return LRQ_ERR_ALIGN;
    if (workspace_bytes < lrq_rms_norm_bwd_workspace(rows, n)) return LRQ_ERR_WORKSPACE;
  }
  hipStream_t s = (hipStream_t)stream;
  if (rows > 0) {
    const RmsBwd a{(const char*)dy, lddy, (const char*)dh, lddh, (const char*)h, ldh, rstd, w, w_dtype, (char*)dx, lddx,
                   dw != nullptr ? (float*)workspace : nullptr, rows, (int)n, 0, 0};
    const auto go = [&](auto dt) { return dh != nullptr ? rms_bwd<dt(), true>(a, s) : rms_bwd<dt(), false>(a, s); };
    switch (dtype) {
      case LRQ_BF16: LRQ_TRY(go(std::integral_constant<int, kBf16>{})); break;
      case LRQ_F16: LRQ_TRY(go(std::integral_constant<int, kF16>{})); break;
      default: LRQ_TRY(go(std::integral_constant<int, kF32>{}));
    }
  }
  if (dw == nullptr) return LRQ_OK;
  const int parts = rows > 0 ? (int)rms_plan(rows, n, dtype).parts : 0;  // no rows: zeros
  return launch(k_rms_wgrad, dim3((unsigned)((n + 31) / 32)), dim3(1024), 0, s, (const float*)workspace, parts, (int)n, dw,
                w_dtype);
}
