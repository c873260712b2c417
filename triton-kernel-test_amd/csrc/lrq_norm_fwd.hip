// Layer norm forward (formulas and layout: lrq_norm.h).
#include "lrq_norm.h"

namespace lrq {

// A chunk of a row's inputs as stored.
template <int DT, bool FUSED>
struct Input {
  Chunk<DT> x, res;
};
template <int DT>
struct Input<DT, false> {
  Chunk<DT> x;
};
template <int DT, bool FUSED>
__device__ __forceinline__ Input<DT, FUSED> ld_input(const NormFwd& a, int64_t row, int c, int k) {
  constexpr int ES = Elem<DT>::kBytes;
  Input<DT, FUSED> in;
  in.x = ld_chunk<DT>(a.x + row * a.ldx * ES + 8u * ES * (uint32_t)c, k);
  if constexpr (FUSED) in.res = ld_chunk<DT>(a.res + row * a.ldr * ES + 8u * ES * (uint32_t)c, a.res != nullptr ? k : 0);
  return in;
}

// h of chunk c (k valid elements): x, dropped, with the residual added, rounded and stored.
template <int DT, bool FUSED>
__device__ __forceinline__ void norm_input(const NormFwd& a, const DropKey& key, const Input<DT, FUSED>& in, int64_t row,
                                           int c, int nc, int k, float* v) {
  widen<DT>(in.x, v);
  if constexpr (FUSED) {
    if (k > 0) {
      if (a.drop.keep < 65536u) drop_chunk(a.drop, key, (uint64_t)row * nc + c, v);
      if (a.res != nullptr) {
        float q[8];
        widen<DT>(in.res, q);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = q[e] + v[e];
      }
      // the statistics are those of h as stored
      const Chunk<DT> hc = narrow<DT>(v);
      st_chunk<DT>(a.h + row * a.ldh * Elem<DT>::kBytes + 8u * Elem<DT>::kBytes * (uint32_t)c, hc, k);
      widen<DT>(hc, v);
    }
  }
}

// One pass: a row's chunks are read once.  Each wave reduces its part of the row to (mean, sum of
// squared deviations from it) and the waves' parts are merged (Chan, Golub and LeVeque's update), so a
// row costs one barrier and the variance never comes from a difference of large sums.
//
// HBM-bound: bf16 [16384, 4096] 46 to 53 us (5.0 to 5.8 TB/s; a copy reaches 5.2), with dropout and the residual 97 to 100 us
// (5.4 TB/s), whose generator runs under the next row's loads.  (Stored past the caches the outputs take 3 and 8 us less,
// and their reader more than that longer: 78 against 75 us with a quantisation of y behind it.)  Two chunks a thread (one
// above 512 columns costs a second row's worth of waves and barriers); [8192, 5120] 29 and 56 to 65 us, [8192, 5003] 33 and 69
// to 73 us (rows that end inside a chunk are read whole; 40 and 86 by elements).  fp32 [1003, 5003]: 13 to 16 us, two rounds of
// rows for a load's latency each.
template <int DT, int LANES, int C, bool FUSED, bool SAME>
__global__ __launch_bounds__(1024) void k_norm_fwd(NormFwd a) {
  constexpr int ES = Elem<DT>::kBytes, L = LANES == 16 ? 16 : 64;
  __shared__ float red[2][16][2], cnts[16];
  const int tpr = LANES ? LANES : 64 * a.waves;
  const int grp = wave_row<LANES>(threadIdx.x / tpr), t = threadIdx.x - grp * tpr;
  const int wv = threadIdx.x >> 6, w0 = LANES ? 0 : grp * a.waves;  // this wave, its row's first
  const int n = a.n, nc = (n + 7) / 8;
  const bool odd = n >= 8 && n % 8 != 0;  // rows end inside a chunk, and are as long as one
  int valid[C];
  float cnt = 0.f;
#pragma unroll
  for (int j = 0; j < C; ++j) {
    const int c = t + j * tpr;
    valid[j] = c < nc ? min(8, n - 8 * c) : 0;
    cnt += (float)valid[j];
  }
  // The weights of a thread's columns, held over the rows: widened, or with dropout and the residual, which leave fewer
  // registers, as stored if both are there in x's type (SAME) and else read again for each row.
  constexpr bool kWide = !FUSED || C == 1, kRaw = !kWide && SAME;
  const auto weights = [&](int j, float* w, float* b) {
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = 1.f, b[e] = 0.f;
    if (a.w != nullptr) ld_weight(a.w, a.wdt, 8 * (int64_t)(t + j * tpr), valid[j], w);
    if (a.b != nullptr) ld_weight(a.b, a.wdt, 8 * (int64_t)(t + j * tpr), valid[j], b);
  };
  float wt[kWide ? C : 1][8], bs[kWide ? C : 1][8];
  Chunk<DT> wr[kRaw ? C : 1], br[kRaw ? C : 1];
#pragma unroll
  for (int j = 0; j < C; ++j) {
    if constexpr (kWide) weights(j, wt[j], bs[j]);
    if constexpr (kRaw) {
      wr[j] = ld_chunk<DT>((const char*)a.w + 8 * ES * (t + j * tpr), valid[j]);
      br[j] = ld_chunk<DT>((const char*)a.b + 8 * ES * (t + j * tpr), valid[j]);
    }
  }
  cnt = lanes_sum<L>(cnt);  // this wave's columns of a row
  const float rcnt = cnt > 0.f ? 1.f / cnt : 0.f, rn = 1.f / (float)n;
  if constexpr (LANES == 0) {
    if ((threadIdx.x & 63) == 0) cnts[wv] = cnt;
  }
  DropKey key{};
  if constexpr (FUSED) key = drop_key(a.drop);
  int slot = 0;
  struct Row {
    Input<DT, FUSED> in[C];
  };
  const auto load = [&](int64_t row) {
    Row r;
#pragma unroll
    for (int j = 0; j < C; ++j)  // (the sums leave out what is past the row)
      r.in[j] = ld_input<DT, FUSED>(a, row, t + j * tpr, row < a.rows ? load_size(valid[j], odd && row + 1 < a.rows) : 0);
    return r;
  };
  const int64_t step = (int64_t)gridDim.x * a.groups;
  constexpr bool kPrefetch = C == 1 || !FUSED || DT != kF32;  // (two fp32 rows of two inputs: too many registers)
  Row cur;
  if constexpr (kPrefetch) {
    cur = load((int64_t)blockIdx.x * a.groups + grp);
    // here ahead of the loop, or the wait for it is in the loop, where it meets the next row's loads as well
#pragma unroll
    for (int j = 0; j < C; ++j) {
      pin(cur.in[j].x);
      if constexpr (FUSED) pin(cur.in[j].res);
    }
  }
  // Every thread takes every step (barriers): a group past the last row works on zeros.  The next row is on its way
  // while this one is reduced and written.
  for (int64_t r0 = (int64_t)blockIdx.x * a.groups; r0 < a.rows; r0 += step) {
    const int64_t row = r0 + grp;
    const bool on = row < a.rows;
    if constexpr (FUSED && C > 1) {  // (its scalar registers do not hold them all)
#pragma unroll
      for (int j = 0; j < C; ++j) opaque(valid[j]);
    }
    Row next;
    if constexpr (kPrefetch) next = load(row + step);
    else cur = load(row);
    float v[C][8];
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < C; ++j) {
      norm_input<DT, FUSED>(a, key, cur.in[j], row, t + j * tpr, nc, on ? valid[j] : 0, v[j]);
      if (valid[j] >= 8) {
#pragma unroll
        for (int e = 0; e < 8; ++e) s += v[j][e];
      } else {
#pragma unroll
        for (int e = 0; e < 7; ++e) s += e < valid[j] ? v[j][e] : 0.f;
      }
      if constexpr (FUSED) __builtin_amdgcn_sched_barrier(0);  // one chunk's generator state at a time
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
    if constexpr (LANES == 0) {
      if ((threadIdx.x & 63) == 0) {
        red[slot][wv][0] = mean;
        red[slot][wv][1] = m2;
      }
      lds_meet();  // (leaves the next row's loads in flight)
      const int k = threadIdx.x & 15;  // each 16 lanes merge the waves' parts
      const bool has = k < a.waves;
      const float pm = has ? red[slot][w0 + k][0] : 0.f, p2 = has ? red[slot][w0 + k][1] : 0.f;
      const float pc = has ? cnts[w0 + k] : 0.f;
      mean = lanes_sum<16>(pm * pc) * rn;
      m2 = lanes_sum<16>(__builtin_fmaf(pc * (pm - mean), pm - mean, p2));
      slot ^= 1;  // the next row's parts; this slot is written again only after its barrier
    }
    const float rstd = 1.f / sqrtf(__builtin_fmaf(m2, rn, a.eps));
    if constexpr (kPrefetch) cur = next;
    if (!on) continue;
    if (t == 0) {
      a.mean[row] = mean;
      a.rstd[row] = rstd;
    }
#pragma unroll
    for (int j = 0; j < C; ++j) {
      const int k = kWide ? j : 0;
      if constexpr (kRaw) {
#pragma unroll
        for (int q = 0; q < Elem<DT>::kVecs; ++q) pin(wr[j].v[q]), pin(br[j].v[q]);
        widen<DT>(wr[j], wt[0]);
        widen<DT>(br[j], bs[0]);
      } else if constexpr (!kWide) {
        weights(j, wt[0], bs[0]);
      }
      float o[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] = __builtin_fmaf((v[j][e] - mean) * rstd, wt[k][e], bs[k][e]);
      st_chunk<DT>(a.y + row * a.ldy * ES + 8u * ES * (uint32_t)(t + j * tpr), narrow<DT>(o), valid[j]);
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
// deviations, the output); after the first the row comes from L2.  bf16 [2048, 20000] 43 us (3.8 TB/s of what it has to
// move), with dropout and the residual 96 (3.4); fp32 [2048, 32768] 167 (3.2) and 265 us (4.1).  Bound by its own waits: a
// sweep's loads have nothing of another row in flight beside them but the CU's second workgroup's.
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
      norm_input<DT, FUSED>(a, key, ld_input<DT, FUSED>(a, row, c, k), row, c, nc, k, v);
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
static int norm_fwd(NormFwd a, hipStream_t s) {
  const int cus = cu_count();
  if (a.n > kNormMaxWidth)
    return launch((k_norm_fwd_wide<DT, FUSED>), dim3((unsigned)std::min<int64_t>(a.rows, 2 * cus)), dim3(1024), 0, s, a);
  const RowShape r = row_shape(a.n, 64, 2);
  a.waves = r.waves;
  a.groups = row_groups(r, a.rows, 16);
  const int threads = std::max(64, (r.lanes ? r.lanes : 64 * r.waves) * a.groups);
  // as many workgroups as run at once (4 waves per SIMD), each walking rows with the weights held
  const int64_t grid = std::min<int64_t>((a.rows + a.groups - 1) / a.groups, (int64_t)cus * (1024 / threads));
  const auto go = [&](auto kern) { return launch(kern, dim3((unsigned)grid), dim3(threads), 0, s, a); };
  if (r.lanes == 16) return go(k_norm_fwd<DT, 16, 1, FUSED, false>);
  if (r.lanes == 64 && r.chunks == 1) return go(k_norm_fwd<DT, 64, 1, FUSED, false>);
  const bool same = FUSED && a.wdt == DT && a.w != nullptr && a.b != nullptr;
  if (r.lanes == 64) return same ? go(k_norm_fwd<DT, 64, 2, FUSED, FUSED>) : go(k_norm_fwd<DT, 64, 2, FUSED, false>);
  return same ? go(k_norm_fwd<DT, 0, 2, FUSED, FUSED>) : go(k_norm_fwd<DT, 0, 2, FUSED, false>);
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
                  w_dtype, rows, (int)n, 0, 0, eps, make_drop(drop)};
  hipStream_t s = (hipStream_t)stream;
  switch (dtype) {
    case LRQ_BF16: return fused ? norm_fwd<kBf16, true>(a, s) : norm_fwd<kBf16, false>(a, s);
    case LRQ_F16: return fused ? norm_fwd<kF16, true>(a, s) : norm_fwd<kF16, false>(a, s);
    default: return fused ? norm_fwd<kF32, true>(a, s) : norm_fwd<kF32, false>(a, s);
  }
}
