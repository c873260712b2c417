// Layer norm backward (formulas and layout: lrq_norm.h).
#include "lrq_norm.h"

namespace lrq {

// A chunk of dh (zeros without one).
template <int DT>
__device__ __forceinline__ Chunk<DT> ld_dh(const NormBwd& a, int64_t row, int c, int k) {
  return ld_chunk<DT>(a.dh + row * a.lddh * Elem<DT>::kBytes + 8u * Elem<DT>::kBytes * (uint32_t)c, a.dh != nullptr ? k : 0);
}

// Elements past the row (a chunk holds `valid`) take the row's mean in place of h, so that their z is 0: (0 - mean) rstd may
// overflow where no element of the row does, and their dy of 0 times that is NaN.
__device__ __forceinline__ void fill_mean(float* h, int valid, float mean) {
  if (valid >= 8) return;
#pragma unroll
  for (int e = 0; e < 8; ++e) h[e] = e < valid ? h[e] : mean;
}

// dresidual and dx of one chunk from the norm's input gradient dn, dh (a partial chunk that was not loaded whole: element
// by element here) and the chunk's random numbers.
template <int DT, bool FUSED>
__device__ __forceinline__ void norm_outputs(const NormBwd& a, int64_t row, int c, int k, float* d, const Chunk<DT>& dh,
                                             bool whole, const u32x4& words) {
  constexpr int ES = Elem<DT>::kBytes;
  if (k <= 0) return;
  if constexpr (FUSED) {
    if (a.dh != nullptr) {
      float q[8];
      widen<DT>(dh, q);
#pragma unroll
      for (int e = 0; e < 8; ++e) d[e] = q[e] + d[e];
      if (!whole) {
        const char* p = a.dh + row * a.lddh * ES + 8u * ES * (uint32_t)c;
#pragma unroll
        for (int e = 0; e < 7; ++e)
          if (e < k) d[e] = ld_elem<DT>(p, e) + d[e];
      }
    }
    if (a.dres != nullptr) st_chunk<DT>(a.dres + row * a.lddr * ES + 8u * ES * (uint32_t)c, narrow<DT>(d), k);
    if (a.drop.keep < 65536u) drop_words(a.drop, words, d);
  }
  if (!FUSED || a.dx != nullptr) st_chunk<DT>(a.dx + row * a.lddx * ES + 8u * ES * (uint32_t)c, narrow<DT>(d), k);
}

// One pass over dy and h.  A thread owns the same columns in every row of its group, so dy z and dy of the
// weight gradients add up in its registers; the workgroup's groups join them in LDS at the end, and
// k_norm_wgrad adds the workgroups' sums in a fixed order.  The next row is already on the way while one is reduced and
// written: up to sixteen waves a CU in 128 registers, and few workgroups, whose sums are few.
//
// HBM-bound: bf16 [16384, 4096] 77 to 86 us (4.7 to 5.2 TB/s), with dh, dropout and both outputs 124 to 134 us (5.0 to 5.4
// TB/s); [8192, 5120] 45 and 84 us (ten waves, so one row at a time a CU: 5.0 TB/s).  One chunk a thread: two hold twice the
// weights and sums, 119 registers of 128 at least and spills besides.  Rows above 8192 columns take four and keep nothing
// ahead, [4096, 14336] 84 and 190 us.  No variant may use scratch or spill.
//
// ODD: rows of one chunk a thread, eight elements at least, that end inside a chunk.  Apart from the others, which then have
// whole chunks only (with 128 columns or fewer, or four chunks a thread, partial ones as well): tests of the width at run
// time cost these 2 to 4 %.  [8192, 5003] 55 to 65 and 114 to 118 us, against 103 and 180 with partial chunks loaded by
// elements; fused, dh comes behind the next row's loads.
//
// EARLY: dh comes with its row, where the workgroup has one row at a time ([8192, 5120] 102 -> 86 us; behind the next row's
// loads it waits for them).  With more rows in flight it comes when it is used ([16384, 4096] 130 against 135 us).
enum { kNormPlain = 0, kNormOdd = 1, kNormEarly = 2 };
template <int DT, int LANES, int C, bool FUSED, int MODE>
__global__ __launch_bounds__(C == 4 ? 512 : 1024) void k_norm_bwd(NormBwd a) {
  constexpr bool ODD = MODE == kNormOdd, kDh = MODE == kNormEarly;
  static_assert(C == 1 || MODE == kNormPlain);
  constexpr bool kPart = ODD || C > 1 || LANES == 16;
  constexpr int ES = Elem<DT>::kBytes, L = LANES == 16 ? 16 : 64;
  // (four chunks a thread, or fp32 rows and the generator, leave no registers for a second row or for what is kept)
  constexpr bool kPrefetch = C == 1 && !(FUSED && DT == kF32), kKeep = kPrefetch;
  __shared__ float red[2][16][2];
  extern __shared__ float sums[];  // [groups][threads of a row * 8 C], with weight gradients only
  const int tpr = LANES ? LANES : 64 * a.waves, kCols = tpr * 8 * C;
  const int grp = wave_row<LANES>(threadIdx.x / tpr), t = threadIdx.x - grp * tpr;
  const int wv = threadIdx.x >> 6, w0 = LANES ? 0 : grp * a.waves;
  const int n = a.n, nc = (n + 7) / 8;
  const float rn = 1.f / (float)n;
  int valid[C];
  float gw[C][8], gb[C][8];
#pragma unroll
  for (int j = 0; j < C; ++j) {
    const int c = t + j * tpr;
    valid[j] = c < nc ? (kPart ? min(8, n - 8 * c) : 8) : 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) gw[j][e] = 0.f, gb[j][e] = 0.f;
  }
  // the weights of a thread's columns: held over the rows, or (four chunks a thread and the generator) read again for
  // each use
  constexpr bool kHold = C == 1 || !FUSED;
  const auto weights = [&](int j, float* w) {
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = 1.f;
    if (a.w != nullptr) ld_weight(a.w, a.wdt, 8 * (int64_t)(t + j * tpr), valid[j], w);
  };
  float wt[kHold ? C : 1][8];
  if constexpr (kHold) {
#pragma unroll
    for (int j = 0; j < C; ++j) weights(j, wt[j]);
  }
  DropKey key{};
  if constexpr (FUSED) key = drop_key(a.drop);
  struct Row {
    Chunk<DT> dy[C], h[C], dh;  // (dh: kDh)
    float mean, rstd;
  };
  // a group past the last row works on zeros; elements past the row have a dy and a z of zero and add nothing to any sum (a
  // row whose statistics are not finite is lost anyway)
  int slot = 0;
  const int64_t step = (int64_t)gridDim.x * a.groups, row0 = (int64_t)blockIdx.x * a.groups + grp;
  // the row to load, stepped along (with four chunks a thread computed instead: no registers to spare)
  const char *pdy = a.dy + row0 * a.lddy * ES, *ph = a.h + row0 * a.ldh * ES;
  const int64_t idy = step * a.lddy * ES, ih = step * a.ldh * ES;
  const auto load = [&](int64_t row) {
    Row r;
    const bool on = row < a.rows, more = ODD && row + 1 < a.rows;
    r.mean = on ? a.mean[row] : 0.f;
    r.rstd = on ? a.rstd[row] : 0.f;
    if constexpr (C > 1) pdy = a.dy + row * a.lddy * ES, ph = a.h + row * a.ldh * ES;
#pragma unroll
    for (int j = 0; j < C; ++j) {
      const uint32_t at = 8u * ES * (uint32_t)(t + j * tpr);
      r.dy[j] = ld_chunk<DT>(pdy + at, on ? load_size(valid[j], more) : 0);
      r.h[j] = ld_chunk<DT>(ph + at, on ? load_size(valid[j], more) : 0);
    }
    if constexpr (kDh) r.dh = ld_dh<DT>(a, row, t, on ? valid[0] : 0);
    if constexpr (C == 1) pdy += idy, ph += ih;
    return r;
  };
  Row cur;
  if constexpr (kPrefetch) {
    cur = load(row0);
    // here ahead of the loop, or the wait for it is in the loop, where it meets the next row's loads as well
    asm volatile("" : "+v"(cur.mean), "+v"(cur.rstd));
    pin(cur.dy[0]);
    pin(cur.h[0]);
    if constexpr (kDh) pin(cur.dh);
  }
  for (int64_t r0 = (int64_t)blockIdx.x * a.groups; r0 < a.rows; r0 += step) {
    const int64_t row = r0 + grp;
    const bool on = row < a.rows;
    if constexpr (C > 1 || (FUSED && ODD)) {  // (their scalar registers do not hold them all)
#pragma unroll
      for (int j = 0; j < C; ++j) opaque(valid[j]);
    }
    Row next;
    if constexpr (kPrefetch) next = load(row + step);
    else cur = load(row);
    u32x4 words{};  // drawn now, under the loads, with one chunk a thread
    if constexpr (FUSED && C == 1) {
      if (a.drop.keep < 65536u) words = philox((uint64_t)row * nc + t, key);
    }
    float s1 = 0.f, s2 = 0.f;
    float ge[kKeep ? 8 : 1], ze[kKeep ? 8 : 1];  // dy w and z, kept for the output where registers allow
#pragma unroll
    for (int j = 0; j < C; ++j) {
      float g[8], z[8];
      const int jw = kHold ? j : 0;
      if constexpr (!kHold) weights(j, wt[0]);
      if constexpr (ODD) mask_chunk<DT>(cur.dy[j], valid[j]);
      widen<DT>(cur.dy[j], g);
      widen<DT>(cur.h[j], z);
      fill_mean(z, valid[j], cur.mean);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float zz = (z[e] - cur.mean) * cur.rstd, gg = g[e] * wt[jw][e];
        gw[j][e] = __builtin_fmaf(g[e], zz, gw[j][e]);
        gb[j][e] += g[e];
        s1 += gg;
        s2 = __builtin_fmaf(gg, zz, s2);
        if constexpr (kKeep) ge[e] = gg, ze[e] = zz;
      }
      if constexpr (C > 1) __builtin_amdgcn_sched_barrier(0);
    }
    s1 = lanes_sum<L>(s1);
    s2 = lanes_sum<L>(s2);
    if constexpr (LANES == 0) {
      if ((threadIdx.x & 63) == 0) {
        red[slot][wv][0] = s1;
        red[slot][wv][1] = s2;
      }
      lds_meet();  // (leaves the next row's loads in flight)
      const int k = threadIdx.x & 15;  // each 16 lanes add the waves' sums
      s1 = lanes_sum<16>(k < a.waves ? red[slot][w0 + k][0] : 0.f);
      s2 = lanes_sum<16>(k < a.waves ? red[slot][w0 + k][1] : 0.f);
      slot ^= 1;  // this slot is written again only after the next row's barrier
    }
    if (on) {
      const float c1 = cur.rstd * (s1 * rn), c2 = -cur.rstd * (s2 * rn);
#pragma unroll
      for (int j = 0; j < C; ++j) {
        if constexpr (C > 1) opaque(valid[j]);
        float g[8], z[8];
        if constexpr (kKeep) {
#pragma unroll
          for (int e = 0; e < 8; ++e) g[e] = ge[e], z[e] = ze[e];
        } else {
          // widened again: kept from above, the fp32 values would take twice the registers
#pragma unroll
          for (int k = 0; k < Elem<DT>::kVecs; ++k) pin(cur.dy[j].v[k]), pin(cur.h[j].v[k]);
          const int jw = kHold ? j : 0;
          if constexpr (!kHold) weights(j, wt[0]);
          widen<DT>(cur.dy[j], g);
          widen<DT>(cur.h[j], z);
#pragma unroll
          for (int e = 0; e < 8; ++e) g[e] *= wt[jw][e], z[e] = (z[e] - cur.mean) * cur.rstd;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) g[e] = __builtin_fmaf(z[e], c2, __builtin_fmaf(g[e], cur.rstd, -c1));
        Chunk<DT> dh;
        const bool whole = !ODD || load_size(valid[j], row + 1 < a.rows) >= 8;
        if constexpr (kDh) dh = cur.dh;
        else if constexpr (FUSED) dh = ld_dh<DT>(a, row, t + j * tpr, !ODD ? valid[j] : whole ? 8 : 0);
        if constexpr (FUSED && C > 1) {
          if (a.drop.keep < 65536u) words = philox((uint64_t)row * nc + t + j * tpr, key);
        }
        norm_outputs<DT, FUSED>(a, row, t + j * tpr, valid[j], g, dh, whole, words);
        if constexpr (C > 1) __builtin_amdgcn_sched_barrier(0);  // one chunk's temporaries at a time
      }
    }
    if constexpr (kPrefetch) cur = next;
  }
  if (a.part == nullptr) return;  // uniform
  float* part = a.part + (int64_t)blockIdx.x * 2 * n;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    if (half) __syncthreads();
#pragma unroll
    for (int j = 0; j < C; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) sums[grp * kCols + 8 * (t + j * tpr) + e] = half ? gb[j][e] : gw[j][e];
    __syncthreads();
    for (int c = threadIdx.x; c < n; c += blockDim.x) {
      float s = 0.f;
      for (int k = 0; k < a.groups; ++k) s += sums[k * kCols + c];
      part[half * (int64_t)n + c] = s;
    }
  }
}

// Rows wider than the registers hold: one workgroup a row, swept twice; its weight gradients come from
// k_norm_cols, so dy and h are read three times.  With k_norm_cols (30 us) bf16 [2048, 20000] 90 us, with dh, dropout and both
// outputs 131; fp32 [4096, 14336] 272 (112 of them k_norm_cols) and 365, [2048, 32768] 312 (114) and 413: 2.6 to 2.7 and 3.1 to
// 3.3 TB/s of what has to move once.
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
      fill_mean(z, k, mean);
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
      Chunk<DT> dh;
      u32x4 words{};
      if constexpr (FUSED) {
        dh = ld_dh<DT>(a, row, c, k);
        if (a.drop.keep < 65536u) words = philox((uint64_t)row * nc + c, key);
      }
      norm_outputs<DT, FUSED>(a, row, c, k, g, dh, true, words);
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
  RowShape shape;
  int groups;     // rows a workgroup takes at a time
  int64_t grid;   // workgroups of the row kernel
  int64_t parts;  // sums of the weight gradients
};

// Rows the register-resident kernel takes: four fp32 chunks a thread do not fit.
static bool bwd_wide(int64_t n, int dt) { return n > (dt == kF32 ? 8192 : kNormMaxWidth); }

static BwdPlan bwd_plan(int64_t rows, int64_t n, int dt) {
  constexpr int kCus = 256;  // a fixed count, so that the workspace and the order of the sums depend on the shape alone
  // one chunk a thread as far as 16 waves go (each has 16 sums besides), else four in half as many waves
  BwdPlan p{row_shape(n, 1024, 4), 1, 0, 0};
  if (bwd_wide(n, dt)) {
    p.grid = std::min<int64_t>(rows, 2 * kCus);
    p.parts = std::min<int64_t>((rows + 3) / 4, 64);
    return p;
  }
  p.groups = row_groups(p.shape, rows, p.shape.chunks == 4 ? 8 : 16);
  p.grid = p.parts = std::min<int64_t>((rows + p.groups - 1) / p.groups, kCus);
  return p;
}

template <int DT, bool FUSED>
static int norm_bwd(NormBwd a, hipStream_t s) {
  const BwdPlan p = bwd_plan(a.rows, a.n, DT);
  if (bwd_wide(a.n, DT)) {
    if (a.part != nullptr)
      LRQ_TRY(launch((k_norm_cols<DT>), dim3((unsigned)((a.n + 511) / 512), (unsigned)p.parts), dim3(256), 0, s, a));
    return launch((k_norm_bwd_wide<DT, FUSED>), dim3((unsigned)p.grid), dim3(1024), 0, s, a);
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
  const bool odd = a.n >= 8 && a.n % 8 != 0;
  if (p.shape.lanes == 16) return odd ? go(k_norm_bwd<DT, 16, 1, FUSED, kNormOdd>) : go(k_norm_bwd<DT, 16, 1, FUSED, kNormPlain>);
  if (p.shape.lanes == 64) return odd ? go(k_norm_bwd<DT, 64, 1, FUSED, kNormOdd>) : go(k_norm_bwd<DT, 64, 1, FUSED, kNormPlain>);
  if (p.shape.chunks == 1) {
    if (odd) return go(k_norm_bwd<DT, 0, 1, FUSED, kNormOdd>);
    if constexpr (FUSED && DT != kF32) {
      if (p.groups == 1) return go(k_norm_bwd<DT, 0, 1, FUSED, kNormEarly>);
    }
    return go(k_norm_bwd<DT, 0, 1, FUSED, kNormPlain>);
  }
  if constexpr (DT != kF32) return go(k_norm_bwd<DT, 0, 4, FUSED, kNormPlain>);
  return LRQ_ERR_UNSUPPORTED;  // (not reached: wide)
}

}  // namespace lrq

using namespace lrq;

extern "C" int64_t lrq_layer_norm_bwd_workspace(int64_t rows, int64_t n) {
  if (rows < 0 || rows > INT32_MAX || n <= 0 || n > INT32_MAX / 2) return LRQ_ERR_SHAPE;
  return std::max(bwd_plan(rows, n, kBf16).parts, bwd_plan(rows, n, kF32).parts) * 2 * n * (int64_t)sizeof(float);
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
                    0, 0, make_drop(drop)};
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
  const int parts = rows > 0 ? (int)bwd_plan(rows, n, dtype).parts : 0;  // no rows: zeros
  return launch(k_norm_wgrad, dim3((unsigned)((n + 63) / 64), 2), dim3(1024), 0, s, (const float*)workspace, parts, (int)n,
                dw, db, w_dtype);
}
