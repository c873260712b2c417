// Products with MXFP4 operands (format: lrq_mx.h), fp32 accumulation:
//
//   lrq_mxfp4_gemm      out[M, N] = A B^T, A [M, K] and B [N, K] both MXFP4 (scaled matrix instructions)
//   lrq_mxfp4_linear    out[M, N] = X W^T, X bf16, W [N, K] MXFP4, widened to bf16 (exactly) on the way
//   lrq_mxfp4_linear_t  out[M, K] = Y W, the gradient of the above for X
#include "lrq_mx.h"

namespace lrq {

template <bool F32>
__device__ __forceinline__ void st_out(void* out, int64_t at, float v) {
  if constexpr (F32) reinterpret_cast<float*>(out)[at] = v;
  else reinterpret_cast<uint16_t*>(out)[at] = (uint16_t)pack_bf16x2(v, 0.f);
}

// Columns n and n + 1 of row m (n + 1 only where the output has it).  bf16, always the product itself and never a part that
// is joined, is stored past L2, which holds the operands (4096 rows, both in MXFP4: 148 -> 141 us, and 175 us either way
// with a kernel that reads the output next).
template <bool F32>
__device__ __forceinline__ void st_pair(char* out, int64_t m, int64_t n, int64_t ldo, int64_t cols, float v0, float v1) {
  if (n + 1 < cols) {
    if constexpr (F32) {
      typedef f32x2_t f32x2_any __attribute__((aligned(4)));
      *(f32x2_any*)(out + (m * ldo + n) * 4) = f32x2_t{v0, v1};
    } else {
      typedef uint32_t u32_any __attribute__((aligned(2)));
      __builtin_nontemporal_store(pack_bf16x2(v0, v1), (u32_any*)(out + (m * ldo + n) * 2));
    }
  } else if (n < cols) {
    st_out<F32>(out, m * ldo + n, v0);
  }
}

// 16 zero bytes, read in place of a row's chunks past its end.
__device__ const u32x4 kZeroChunk = u32x4{0u, 0u, 0u, 0u};

template <int BYTES>
__device__ __forceinline__ void ld_to_lds(const void* g, char* lds) {
  const auto l = (__attribute__((address_space(3))) void*)lds;
  if constexpr (BYTES == 16) __builtin_amdgcn_global_load_lds(g, l, 16, 0, 0);
  else __builtin_amdgcn_global_load_lds(g, l, 4, 0, 0);
}

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef u32x4 u32x4_dword __attribute__((aligned(4)));
__device__ __forceinline__ u32x4 ld16_any(const uint8_t* p) { return *reinterpret_cast<const u32x4_dword*>(p); }

__device__ __forceinline__ f32x16 mfma_32x32x16(u32x4 a, u32x4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// D(32x32) += A(32x64) B(64x32), both e2m1 with E8M0 block scales.  Lane l holds row (column) l % 32, k = 32 (l / 32)
// .. + 31, and its block's scale in byte SEL of its scale operand.
typedef int i32x8 __attribute__((ext_vector_type(8)));
template <int SEL>
__device__ __forceinline__ f32x16 mfma_mx(u32x4 a, u32x4 b, f32x16 c, uint32_t sa, uint32_t sb) {
  const i32x8 a8 = {(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0};
  const i32x8 b8 = {(int)b[0], (int)b[1], (int)b[2], (int)b[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a8, b8, c, 4, 4, SEL, (int)sa, SEL, (int)sb);
}

// Workgroup tiles of a product whose contraction may be split: this workgroup's tile and steps.
struct Place {
  int z;
  int64_t m0, n0;
  int first, last;
};
__device__ __forceinline__ Place place(int tiles_m, int tiles_n, int splits, int steps, int bm, int bn) {
  const uint32_t tiles = tiles_m * tiles_n, id = xcd_tile(blockIdx.x, gridDim.x);
  const uint32_t z = __builtin_amdgcn_readfirstlane(id / tiles), tile = id - z * tiles;
  const uint32_t tn = __builtin_amdgcn_readfirstlane(tile / tiles_m), tm = tile - tn * tiles_m;
  return Place{(int)z, (int64_t)tm * bm, (int64_t)tn * bn,
               (int)__builtin_amdgcn_readfirstlane((uint32_t)steps * z / (uint32_t)splits),
               (int)__builtin_amdgcn_readfirstlane((uint32_t)steps * (z + 1) / (uint32_t)splits)};
}

// ---------------------------------------------------------------- both operands in MXFP4
struct GemmArgs {
  Mx a, b;
  void* out;  // [splits][a.rows][ldo] fp32 parts where splits > 1
  int64_t ldo;
  int tiles_m, tiles_n, splits;
};

// Scale bytes come to LDS four steps at a time, 16 bytes a row (one dword a step: a load of a dword a row for each step
// kept the address unit busier than all codes did, 228 against 179 us on [4096, 4096] x [14336, 4096]).  A row holds
// 4 bytes a step, so the last group starts early enough to end with the row; a matrix of fewer than four steps is
// copied by the threads instead.
__device__ __forceinline__ int scale_base(int step, int steps) { return max(0, min(step, steps - 4)); }

__device__ __forceinline__ void short_scales(const uint8_t* row, int steps, char* lds) {
  for (int k = 0; k < steps; ++k) st4(lds + 4 * k, ld4(row + 4 * k));
}

// Workgroup: 64 MT rows of A by 256 rows of B, 8 waves in two rows of four, each 32 MT x 64 of it in 32x32x64 scaled
// instructions, whose operands are the stored codes and scale bytes as they are.  A K step of 128 columns is one scale
// dword a row and 64 code bytes; the codes go straight to LDS, four steps deep, one barrier a step.  Row r's 16-byte
// piece q sits in slot q ^ (r / 4 % 4): 16 lanes of a read cover all banks.  LDS row 64 wn + 32 t + c of B holds row
// 64 wn + 2 c + t, so that a lane's two columns are neighbours in the output.
//
// [4096, 4096] x [14336, 4096]: 146 to 157 us on different cards, 3.1 to 3.3 PFLOP/s.  A step's instructions alone take
// 0.48 us of the matrix unit at 2.1 GHz; a step takes 0.78 us on zeros and 0.9 to 1.1 us on random data, where the card
// lowers its clock for power; 15 us are the output's 117 MB, which no other workgroup's work covers (144 KB of LDS: one
// workgroup a CU).  The last of four rounds of tiles is half empty.
template <int MT>
struct GemmLds {
  static constexpr int kA = 64 * MT * 64, kB = 16384, kStage = kA + kB, kDeep = 4;
  static constexpr int kScales = (64 * MT + 256) * 16, kBytes = kDeep * kStage + 2 * kScales;
};
template <int MT, bool F32>
__global__ __launch_bounds__(512) void k_mx_gemm(GemmArgs p) {
  using G = GemmLds<MT>;
  constexpr int kA = G::kA, kStage = G::kStage, kDeep = G::kDeep, kRing = kDeep * kStage;
  constexpr int kLa = MT >= 2 ? MT / 2 : 1;  // 1 KB loads of A a wave (MT 1: the upper four waves load the same again)
  constexpr int kLoads = kLa + 2;
  extern __shared__ char sm[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave >> 2, wn = wave & 3, c = lane & 31, h = lane >> 5;
  const int steps = p.a.steps;
  const Place at = place(p.tiles_m, p.tiles_n, p.splits, steps, 64 * MT, 256);

  const uint8_t *pa[kLa], *pb[2];
  char *la[kLa], *lb[2];
#pragma unroll
  for (int i = 0; i < kLa; ++i) {
    const int in = MT >= 2 ? kLa * wave + i : wave & 3, r = 16 * in + (lane >> 2);
    pa[i] = p.a.codes + min(at.m0 + r, p.a.rows - 1) * p.a.ldc + 16 * ((lane & 3) ^ (r >> 2 & 3));
    la[i] = sm + 1024 * in;
  }
  const auto b_row = [&](int r) { return min(at.n0 + (r & ~63) + 2 * (r & 31) + (r >> 5 & 1), p.b.rows - 1); };
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = 16 * (2 * wave + i) + (lane >> 2);
    pb[i] = p.b.codes + b_row(r) * p.b.ldc + 16 * ((lane & 3) ^ (r >> 2 & 3));
    lb[i] = sm + kA + 1024 * (2 * wave + i);
  }
  // 64 rows' scales a load: A's rows, then B's (waves past them load the last again)
  const int is = min(wave, MT + 3);
  const uint8_t* ps = is < MT ? p.a.scales + min(at.m0 + 64 * is + lane, p.a.rows - 1) * p.a.lds
                              : p.b.scales + b_row(64 * (is - MT) + lane) * p.b.lds;
  char* ls = sm + kRing + 1024 * is;

  const auto issue_codes = [&](int step, int buf, int i) {
    const int o = buf * kStage;
    if (i < kLa) ld_to_lds<16>(pa[i < kLa ? i : 0] + 64 * (int64_t)step, la[i < kLa ? i : 0] + o);
    else ld_to_lds<16>(pb[i - kLa] + 64 * (int64_t)step, lb[i - kLa] + o);
  };
  const auto issue_scales = [&](int step, int ring) {
    ld_to_lds<16>(ps + 4 * (int64_t)scale_base(step, steps), ls + ring * G::kScales);
  };

  f32x16 acc[MT][2];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int v = 0; v < 16; ++v) acc[i][t][v] = 0.f;

  if (steps >= 4) issue_scales(at.first, 0);
  else short_scales(ps, steps, ls + 16 * lane);
  const auto issue_step = [&](int step, int buf, int k) { issue_codes(min(step, at.last - 1), buf, k); };
  constexpr int kEarly = kLoads / 2;  // loads of a step that are issued in the half step before the others
#pragma unroll
  for (int d = 0; d < kDeep; ++d)
#pragma unroll
    for (int i = 0; i < (d < kDeep - 1 ? kLoads : kEarly); ++i) issue_step(at.first + d, d, i);
  // The operands of instruction column q of a step are read from LDS while the column before runs: those of a step's
  // first column during the last of the step before, so the step's loads are waited for, and the workgroup meets, in the
  // middle of the step before.  Reads and loads go out one at a time between the instructions: a wave that issues them
  // together stands in their queue with the matrix unit idle.
  const int ra = 32 * MT * wm + c, rb = 64 * wn + c, slot = c >> 2 & 3;
  constexpr int kMfma = 2 * MT, kPieces = MT + 2, kPer = (kPieces + kMfma - 1) / kMfma;
  u32x4 va[2][MT], vb[2][2];
  uint32_t sa[MT], sb[2], na[MT], nb[2];
  const auto read = [&](int q, int buf, int j) {
    const char* st = sm + buf * kStage;
    const int o = 16 * ((2 * q + h) ^ slot);
    if (j < 2) vb[q][j < 2 ? j : 0] = ld16(st + kA + 64 * (rb + 32 * j) + o);
    else va[q][j - 2] = ld16(st + 64 * (ra + 32 * (j - 2)) + o);
  };
  const auto read_scales = [&](int step, int phase, int ring) {
    const char* sc = sm + kRing + ring * G::kScales + 4 * min(step - scale_base(step - phase, steps), 3);
#pragma unroll
    for (int i = 0; i < MT; ++i) na[i] = ld4(sc + 16 * (ra + 32 * i));
#pragma unroll
    for (int t = 0; t < 2; ++t) nb[t] = ld4(sc + 1024 * MT + 16 * (rb + 32 * t));
  };
  // Instruction m of a column, then its share of the next column's reads (the first ones' share) and of the loads (the
  // last ones').  The order is held, and there is no branch in a step: the compiler would sink the instructions into
  // the block behind it and issue everything else first.
#define LRQ_COLUMN(Q, SEL, BUF, STEP, TO, FIRST, COUNT)                                                       \
  _Pragma("unroll") for (int m = 0; m < kMfma; ++m) {                                                         \
    acc[m / 2][m % 2] = mfma_mx<SEL>(va[Q][m / 2], vb[Q][m % 2], acc[m / 2][m % 2], sa[m / 2], sb[m % 2]);    \
    __builtin_amdgcn_sched_barrier(0);                                                                        \
    if (Q == 1 && m == 0) read_scales(step + 1, (phase + 1) & 3, ring);                                       \
    _Pragma("unroll") for (int j = m * kPer; j < (m + 1) * kPer; ++j) if (j < kPieces) read(1 - Q, BUF, j);   \
    if (m >= kMfma - (COUNT)) issue_step(STEP, TO, (FIRST) + m - (kMfma - (COUNT)));                          \
    __builtin_amdgcn_sched_barrier(0);                                                                        \
  }
  // the scales' loads are ahead of the codes
  __builtin_amdgcn_s_waitcnt(vmcnt_imm(kLoads * 2 + kEarly));
  lds_meet();
#pragma unroll
  for (int j = 0; j < kPieces; ++j) read(0, 0, j);
  read_scales(at.first, 0, 0);
  int buf = 0, ring = 0;
  for (int step = at.first; step < at.last; ++step) {
    const int phase = (step - at.first) & 3;
    if (phase == 0 && steps >= 4) issue_scales(step + 4, ring ^ 1);
#pragma unroll
    for (int i = 0; i < MT; ++i) sa[i] = na[i] >> (8 * h);
#pragma unroll
    for (int t = 0; t < 2; ++t) sb[t] = nb[t] >> (8 * h);
    __builtin_amdgcn_sched_barrier(0);
    LRQ_COLUMN(0, 0, buf, step + kDeep - 1, (buf + kDeep - 1) & (kDeep - 1), kEarly, kLoads - kEarly)
    // the next step's loads, not those of the two steps after it (the scales are done three steps on, in time)
    __builtin_amdgcn_s_waitcnt(vmcnt_imm(kLoads * (kDeep - 2)));
    lds_meet();  // every wave's are in, and every wave has read all of this step's buffer
    ring ^= (phase + 1) >> 2;
    const int free = buf;
    buf = (buf + 1) & (kDeep - 1);
    __builtin_amdgcn_sched_barrier(0);
    LRQ_COLUMN(1, 2, buf, step + kDeep, free, 0, kEarly)
  }
#undef LRQ_COLUMN
  __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));  // the last loads write LDS: let them end before the workgroup does
  char* out = (char*)p.out + (p.splits > 1 ? (int64_t)at.z * p.a.rows * p.ldo * 4 : 0);
  const int64_t n = at.n0 + 64 * wn + 2 * c;
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int v = 0; v < 16; ++v) {
      const int64_t m = at.m0 + 32 * MT * wm + 32 * i + 8 * (v >> 2) + 4 * h + (v & 3);
      if (m < p.a.rows) st_pair<F32>(out, m, n, p.ldo, p.b.rows, acc[i][0][v], acc[i][1][v]);
    }
}

// ---------------------------------------------------------------- bf16 rows, few of them
// Up to ROWS rows of X (a decoding step) by 16 COLS rows of W a workgroup; each of its WAVES waves takes a run of the K
// steps of 128 and they join in LDS.  Lane (j, g) reads the 16 code bytes of block g of W row j: its k are 32g .. 32g + 31, 8
// of them for each of the step's four matrix instructions, and X is read in the same order.  Everything a wave needs
// for its next D steps is in flight at once: X's columns go to the wave's own part of LDS (16-byte piece i of row r in
// slot i ^ r, so that the 16 rows' reads fall in different banks), the codes and scales to registers.  The time is the
// codes' arrival after a fixed 4 us: one row by [14336, 4096] 8.4 to 9.8 us for 31 MB where they lie in the last-level
// cache and 10.8 to 11.8 from HBM, by [4096, 4096] 4.6 us for 9 MB.  Every workgroup reads all of X through L2, so with
// more than four rows it takes two tiles of W where that leaves 256 workgroups: 16 rows by [14336, 4096] 12.1 us, 12.8 to
// 13.0 from HBM (one tile: 14.8), 5 rows 9.5 (10.4).  A dword of scales a step in place of 16 bytes for four took 10.8 us
// for one row, against 8.4.
template <int ROWS, int WAVES, int COLS, bool F32>
__global__ __launch_bounds__(64 * WAVES) void k_mx_token(const uint16_t* x, int64_t ldx, int rows, Mx w, void* out,
                                                         int64_t ldo) {
  constexpr int D = ROWS > 4 ? 4 : 8, kRow = 256 * D;
  __shared__ __attribute__((aligned(16))) char xs[WAVES][ROWS][kRow];
  __shared__ f32x4 red[WAVES][COLS][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), j = lane & 15, g = lane >> 4;
  const int64_t n0 = (int64_t)blockIdx.x * 16 * COLS;
  const int per = (w.steps + WAVES - 1) / WAVES, first = min(wave * per, w.steps), last = min(first + per, w.steps);
  const uint8_t *codes[COLS], *scales[COLS];
#pragma unroll
  for (int t = 0; t < COLS; ++t) {
    const int64_t rw = min(n0 + 16 * t + j, w.rows - 1);
    codes[t] = w.codes + rw * w.ldc + 16 * g;
    scales[t] = w.scales + rw * w.lds;
  }
  const int row = min(j, rows - 1);  // (lanes past X's rows repeat its last: their rows of the product are not stored)
  f32x4 acc[COLS];
#pragma unroll
  for (int t = 0; t < COLS; ++t) acc[t] = zero4();
  for (int s0 = first; s0 < last; s0 += D) {
    u32x4 c[COLS][D];
    uint32_t sc[COLS][D];
    for (int r = 0; r < rows; ++r)
#pragma unroll
      for (int i = 0; i < kRow / 1024; ++i) {
        const int k = 128 * s0 + 512 * i + 8 * (lane ^ r);
        ld_to_lds<16>(k < w.cols ? (const void*)(x + r * ldx + k) : &kZeroChunk, &xs[wave][r][1024 * i]);
      }
#pragma unroll
    for (int t = 0; t < COLS; ++t)
#pragma unroll
      for (int u = 0; u < D; ++u) c[t][u] = ld16_stream(codes[t] + 64 * (int64_t)min(s0 + u, last - 1));
    if (s0 + D <= w.steps) {  // 16 bytes of scales a load, four steps
#pragma unroll
      for (int t = 0; t < COLS; ++t)
#pragma unroll
        for (int u = 0; u < D; u += 4) {
          const u32x4 v = ld16_any(scales[t] + 4 * (int64_t)(s0 + u));
          sc[t][u] = v[0], sc[t][u + 1] = v[1], sc[t][u + 2] = v[2], sc[t][u + 3] = v[3];
        }
    } else {
#pragma unroll
      for (int t = 0; t < COLS; ++t)
#pragma unroll
        for (int u = 0; u < D; ++u) sc[t][u] = ld4(scales[t] + 4 * (int64_t)min(s0 + u, last - 1));
    }
    __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
    asm volatile("" ::: "memory");
#pragma unroll
    for (int u = 0; u < D; ++u) {
      if (s0 + u >= last) break;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const u32x4 x8 = ld16(&xs[wave][row][16 * ((16 * u + 4 * g + q) ^ row)]);
#pragma unroll
        for (int t = 0; t < COLS; ++t)
          acc[t] = mfma_16x16x32(x8, fp4x8_to_bf16(c[t][u][q], e8m0_operand(sc[t][u] >> (8 * g))), acc[t]);
      }
    }
    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): the reads are done before the next steps' X lands
  }
#pragma unroll
  for (int t = 0; t < COLS; ++t) red[wave][t][lane] = acc[t];
  __syncthreads();
  if (threadIdx.x >= 256) return;
  // 16 columns of an output row to 16 threads
  const int l = (threadIdx.x & 15) + (threadIdx.x >> 2 & 48), v = threadIdx.x >> 4 & 3;
  const int m = 4 * (l >> 4) + v;
#pragma unroll
  for (int t = 0; t < COLS; ++t) {
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < WAVES; ++k) sum += red[k][t][l][v];
    const int64_t n = n0 + 16 * t + (l & 15);
    if (m < rows && n < w.rows) st_out<F32>(out, m * ldo + n, sum);
  }
}

// ---------------------------------------------------------------- bf16 rows, many of them
struct TileArgs {
  const uint16_t* x;  // [rows, contraction]
  int64_t ldx;
  int64_t rows;
  Mx w;
  void* out;          // [splits][rows][ldo] fp32 parts where splits > 1
  int64_t ldo;
  int64_t cols;       // columns of the output
  int tiles_m, tiles_n, splits;
  int steps;          // contraction steps of 128
  int chunks;         // 8-element chunks of a row of x
};

// out = x w^T (TRANS false: the contraction runs along w's columns) or x w (true: along w's rows).
//
// Workgroup: 32 MT rows of x by 256 output columns, 8 waves.  Waves 4 gq .. 4 gq + 3 take the half gq of each contraction
// step of 128, wave 4 gq + wn all its rows and columns 64 wn .. + 63 of it: so W's codes are widened once in a
// workgroup, and two waves a SIMD cover each other's waits.  The halves are added through LDS at the end.  Every
// operand goes straight to LDS, three steps deep, with counted waits: one barrier a step.
//
// 32x32x16 instructions.  Lane (c, h) (c = lane % 32, h = lane / 32) of instruction s < 4 holds contraction indices
// 64 gq + 32 h + 8 s .. + 7 of the step (any order serves that both operands share), and column tile t is columns
// 64 wn + 2 c + t: neighbouring columns end in one lane.
//   TRANS false: those are 32 consecutive k of one W row, so the lane reads 16 code bytes and one scale a step.
//   TRANS true: the lane's two columns are one code byte of each W row.  The transposing LDS read gives it that byte
//   of 8 rows at once; each is widened with its own row's scale and the halves of two rows are paired by v_perm_b32.
//
// 512 rows by [14336, 4096]: 54 to 62 us, and 56 to 63 us and a join of 8 us for the gradient (1.0 to 1.1 PFLOP/s; 42 us
// each at the 1.44 PFLOP/s of a large bf16 product on random data, which power limits: on zeros a step takes 1.27 us, on
// random data 1.4 to 1.7, its instructions alone 0.96 at 2.1 GHz); 4096 rows: 412 to 443 us (1.1 to 1.2).  224 of 256 CUs
// have a tile of 512 rows.
template <bool TRANS, int MT>
struct TileLds {
  static constexpr int kA = 32 * MT * 256, kB = 16384, kS = TRANS ? 3 * 1024 : 0, kStage = kA + kB + kS, kDeep = 3;
  static constexpr int kScales = TRANS ? 0 : 4096, kLoop = kDeep * kStage + 2 * kScales;
  static constexpr int kJoin = (MT >= 2 ? 8 * MT / 2 : 4) * 8192, kBytes = kLoop > kJoin ? kLoop : kJoin;
};
template <bool TRANS, int MT, bool F32>
__global__ __launch_bounds__(512) void k_mx_tile(TileArgs a) {
  using T = TileLds<TRANS, MT>;
  constexpr int kA = T::kA, kB = T::kB, kStage = T::kStage, kRing = T::kDeep * kStage;
  extern __shared__ char sm[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int gq = wave >> 2, wn = wave & 3, c = lane & 31, h = lane >> 5;
  const Place at = place(a.tiles_m, a.tiles_n, a.splits, a.steps, 32 * MT, 256);
  const int64_t m0 = at.m0, n0 = at.n0;
  const int first = at.first, last = at.last;

  // x: instruction i of wave w fills rows 4 (MT w + i) .. + 3 of the tile; chunk q of row r sits in slot q ^ (r % 16)
  const char* px[MT];
  int full[MT];  // this lane's chunk is one of x's in steps below it
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int r = 4 * (MT * wave + i) + (lane >> 4), q = (lane & 15) ^ (r & 15);
    full[i] = (a.chunks - q + 15) >> 4;
    px[i] = (const char*)(a.x + min(m0 + r, a.rows - 1) * a.ldx + 8 * q);
  }
  // codes: TRANS false: 256 rows of 64 bytes, 16-byte piece q of row r in slot q ^ (r / 4 % 4), LDS row 64 wn + 32 t + c
  // holding W row 64 wn + 2 c + t; TRANS true: 128 rows of 128 bytes, piece q of row r in slot q ^ (r / 2 % 4).  Both
  // spread a wave's reads over the banks.
  const auto w_row = [&](int r) { return min(n0 + (r & ~63) + 2 * (r & 31) + (r >> 5 & 1), a.w.rows - 1); };
  const uint8_t* pb[2];
  int rb[2];
  const uint8_t* ps;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int in = 2 * wave + i;
    if constexpr (!TRANS) {
      const int r = 16 * in + (lane >> 2);
      pb[i] = a.w.codes + w_row(r) * a.w.ldc + 16 * ((lane & 3) ^ (r >> 2 & 3));
    } else {
      rb[i] = 8 * in + (lane >> 3);
      pb[i] = a.w.codes + min(n0 / 2 + 16 * ((lane & 7) ^ (rb[i] >> 1 & 3)), 64 * (int64_t)a.w.steps - 16);
    }
  }
  const int rs = TRANS ? (threadIdx.x & 255) >> 1 : 64 * (wave & 3) + lane;
  if constexpr (!TRANS) ps = a.w.scales + w_row(rs) * a.w.lds;
  else ps = a.w.scales + min(n0 / 32 + 4 * (lane & 1), 4 * (int64_t)a.w.steps - 4);

  // part i < 4 of a step's loads (no branch: see the loop)
  const auto issue = [&](int step, int buf, int i) {
    char* st = sm + buf * kStage;
    if (i < MT) {
      const int k = i < MT ? i : 0;
      const char* g = step < full[k] ? px[k] + 256 * (int64_t)step : (const char*)&kZeroChunk;
      ld_to_lds<16>(g, st + 1024 * (MT * wave + i));
    }
    if constexpr (!TRANS) {
      if (i < 2) ld_to_lds<16>(pb[i & 1] + 64 * (int64_t)step, st + kA + 1024 * (2 * wave + i));
    } else {  // rows past W's last: that one (their x is zero)
      const uint32_t r0 = 128 * (uint32_t)step, most = (uint32_t)a.w.rows - 1;
      if (i < 2) ld_to_lds<16>(pb[i & 1] + (int64_t)min(r0 + rb[i & 1], most) * a.w.ldc, st + kA + 1024 * (2 * wave + i));
      if (i == 2 && wave < 4) ld_to_lds<4>(ps + (int64_t)min(r0 + rs, most) * a.w.lds, st + kA + kB + 256 * wave);
    }
  };
  // TRANS false: W's scales, four steps at a time (waves 4 .. 7 load the same again)
  const auto issue_scales = [&](int step, int ring) {
    ld_to_lds<16>(ps + 4 * (int64_t)scale_base(step, a.steps), sm + kRing + ring * T::kScales + 1024 * (wave & 3));
  };

  f32x16 acc[MT][2];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int v = 0; v < 16; ++v) acc[i][t][v] = 0.f;

  if constexpr (!TRANS) {
    if (a.steps >= 4) issue_scales(first, 0);
    else short_scales(ps, a.steps, sm + kRing + 16 * rs);
  }
#pragma unroll
  for (int d = 0; d < 2; ++d)
#pragma unroll
    for (int i = 0; i < 4; ++i) issue(min(first + d, last - 1), d, i);
  issue(min(first + 2, last - 1), 2, 0);

  // TRANS: a step's scales arrive as [row][8]; the four of the thread that loaded them go to [block][row] as bf16, so
  // that half of them are a conversion's scale operand as read.
  const auto turn_scales = [&](int buf) {
    if constexpr (TRANS) {
      if (wave < 4) {
        char* st = sm + buf * kStage + kA + kB;
        const uint32_t s4 = ld4(st + 4 * threadIdx.x);
        uint16_t* to = (uint16_t*)(st + 1024) + 512 * (lane & 1) + rs;
#pragma unroll
        for (int k = 0; k < 4; ++k) to[128 * k] = (uint16_t)((s4 >> (8 * k) & 255u) << 7);
      }
    }
  };
  u32x4 xr[2][MT], b[2][2];
  u32x4 code[2];           // TRANS false: this lane's codes of its two columns, and their scales
  float scale[2];
  u32x2 cols[4];           // TRANS: its code byte of 8 rows, for each instruction, and the rows' scales
  u32x4 rows8[4];
  const auto read_x = [&](int buf, int s, int i) {
    const int r = 32 * i + c;
    xr[s & 1][i] = ld16(sm + buf * kStage + 256 * r + 16 * ((8 * gq + 4 * h + s) ^ (r & 15)));
  };
  const auto read_w = [&](int buf, int step, int phase, int ring) {
    char* st = sm + buf * kStage;
    if constexpr (!TRANS) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int r = 64 * wn + 32 * t + c;
        code[t] = ld16(st + kA + 64 * r + 16 * ((2 * gq + h) ^ (r >> 2 & 3)));
        scale[t] = e8m0_operand((uint8_t)sm[kRing + ring * T::kScales + 16 * r +
                                            4 * min(step - scale_base(step - phase, a.steps), 3) + 2 * gq + h]);
      }
    } else {
      const int r0 = 64 * gq + 32 * h, blk = 2 * wn + (lane >> 4 & 1), r = r0 + (lane >> 1 & 7);
#pragma unroll
      for (int s = 0; s < 4; ++s) rows8[s] = ld16(st + kA + kB + 1024 + 2 * (128 * blk + r0 + 8 * s));
      // by hand, with its wait: for the builtin the compiler first drains the loads to LDS just issued
      const uint32_t p = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)(
          st + kA + 128 * r + 16 * (blk ^ (r >> 1 & 3)) + 8 * (lane & 1));
      asm volatile("ds_read_b64_tr_b8 %0, %4\n\tds_read_b64_tr_b8 %1, %4 offset:1024\n\t"
                   "ds_read_b64_tr_b8 %2, %4 offset:2048\n\tds_read_b64_tr_b8 %3, %4 offset:%5\n\t"
                   "s_waitcnt lgkmcnt(0)"
                   : "=&v"(cols[0]), "=&v"(cols[1]), "=&v"(cols[2]), "=&v"(cols[3])
                   : "v"(p), "n"(3 * 1024)
                   : "memory");
    }
  };
  // W's operand of instruction s
  const auto widen_w = [&](int s) {
    if constexpr (!TRANS) {
#pragma unroll
      for (int t = 0; t < 2; ++t) b[s & 1][t] = fp4x8_to_bf16(code[t][s], scale[t]);
    } else {
      uint32_t e[8];
#pragma unroll
      for (int i = 0; i < 2; ++i) {  // the conversion reads the exponent field alone
        const uint32_t cw = cols[s][i], s01 = rows8[s][2 * i], s23 = rows8[s][2 * i + 1];
        e[4 * i + 0] = fp4_to_bf16x2<0>(cw, __uint_as_float(s01 << 16));
        e[4 * i + 1] = fp4_to_bf16x2<1>(cw, __uint_as_float(s01));
        e[4 * i + 2] = fp4_to_bf16x2<2>(cw, __uint_as_float(s23 << 16));
        e[4 * i + 3] = fp4_to_bf16x2<3>(cw, __uint_as_float(s23));
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        b[s & 1][0][i] = __builtin_amdgcn_perm(e[2 * i + 1], e[2 * i], 0x05040100u);
        b[s & 1][1][i] = __builtin_amdgcn_perm(e[2 * i + 1], e[2 * i], 0x07060302u);
      }
    }
  };

  // the first step's loads (and the scales ahead of them), not those of the next nor the part after it
  __builtin_amdgcn_s_waitcnt(vmcnt_imm(MT + 4));
  turn_scales(0);
  lds_meet();
  int buf = 0, ring = 0;
  read_w(0, first, 0, 0);
#pragma unroll
  for (int i = 0; i < MT; ++i) read_x(0, 0, i);
  widen_w(0);
  // Everything of instruction s + 1 is read and widened while instruction s runs, that of a step's first during the last of
  // the step before, ahead of which the step's loads are waited for and the workgroup meets.  From then on the old step's
  // buffer is free: the loads of three steps on go there, a part with each instruction (at once they would queue up
  // before the first of them).  The order is held, and there is no branch in a step: the compiler would sink the
  // instructions into the block behind it.
  for (int step = first; step < last; ++step) {
    const int phase = (step - first) & 3, ahead = min(step + 2, last - 1), to = buf == 0 ? 2 : buf - 1;
    if constexpr (!TRANS) {
      if (phase == 0 && a.steps >= 4) issue_scales(step + 4, ring ^ 1);
    }
    __builtin_amdgcn_sched_barrier(0);
    int now = buf;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      if (s == 3) {
        // the next step's loads (four steps' scales are in by the time they are read)
        __builtin_amdgcn_s_waitcnt(vmcnt_imm(MT + 2));
        now = buf == 2 ? 0 : buf + 1;
        ring ^= (phase + 1) >> 2;
        turn_scales(now);
        lds_meet();
      }
#pragma unroll
      for (int i = 0; i < MT; ++i) {
#pragma unroll
        for (int t = 0; t < 2; ++t) acc[i][t] = mfma_32x32x16(xr[s & 1][i], b[s & 1][t], acc[i][t]);
        __builtin_amdgcn_sched_barrier(0);
        if (s == 3 && i == MT / 4) read_w(now, step + 1, (phase + 1) & 3, ring);
        // (two at a time: the wait for them is not to meet the last one just issued)
        if (2 * i < MT) read_x(now, (s + 1) & 3, 2 * i);
        if (2 * i + 1 < MT) read_x(now, (s + 1) & 3, 2 * i + 1);
        if (i == MT - 1) {
          if (s < 3) issue(ahead, to, s + 1);
          else issue(min(step + 3, last - 1), buf, 0);
          widen_w((s + 1) & 3);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    buf = now;
  }

  // The two halves' sums meet through LDS: half gq finishes half of the rows (MT 1: half 0 all of them).
  constexpr int kOwn = MT >= 2 ? MT / 2 : 1;
  __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
  __syncthreads();
  f32x4* ex = (f32x4*)sm;
  if (MT >= 2 || gq == 1) {
#pragma unroll
    for (int i = 0; i < kOwn; ++i)
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const f32x16& v = gq ? acc[i][t] : acc[MT - kOwn + i][t];
          ex[(((MT >= 2 ? wave : wn) * kOwn + i) * 8 + 4 * t + q) * 64 + lane] =
              f32x4{v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]};
        }
  }
  __syncthreads();
  if (MT == 1 && gq == 1) return;
  char* out = (char*)a.out + (a.splits > 1 ? (int64_t)at.z * a.rows * a.ldo * 4 : 0);
  const int64_t n = n0 + 64 * wn + 2 * c;
#pragma unroll
  for (int i = 0; i < kOwn; ++i)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      f32x4 v[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const f32x4 o = ex[(((MT >= 2 ? wave ^ 4 : wn) * kOwn + i) * 8 + 4 * t + q) * 64 + lane];
        const f32x16& w = gq ? acc[MT - kOwn + i][t] : acc[i][t];
        v[t] = f32x4{w[4 * q] + o[0], w[4 * q + 1] + o[1], w[4 * q + 2] + o[2], w[4 * q + 3] + o[3]};
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int64_t m = m0 + 32 * (gq * kOwn + i) + 8 * q + 4 * h + k;
        if (m < a.rows) st_pair<F32>(out, m, n, a.ldo, a.cols, v[0][k], v[1][k]);
      }
    }
}

// out[rows, cols] = the splits' sums, in their order; 4 columns a thread.
template <bool F32>
__global__ __launch_bounds__(256) void k_mx_join(const float* part, int splits, int64_t rows, int64_t cols, int64_t ldp,
                                                 void* out, int64_t ldo) {
  const int64_t quads = ldp / 4, total = rows * quads;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t m = i / quads, n = 4 * (i - m * quads);
    f32x4 s = *(const f32x4*)(part + m * ldp + n);
#pragma unroll 4
    for (int z = 1; z < splits; ++z) {
      const f32x4 v = *(const f32x4*)(part + ((int64_t)z * rows + m) * ldp + n);
#pragma unroll
      for (int k = 0; k < 4; ++k) s[k] += v[k];
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (n + k < cols) st_out<F32>(out, m * ldo + n + k, s[k]);
  }
}

struct SplitPlan {
  int mt;  // 32 mt rows a workgroup; 0: the few-row kernel
  int64_t tiles_m, tiles_n;
  int splits, steps;
};

// The tile's height and how often the contraction is split over workgroups: one workgroup runs on a CU at a time, so a
// grid takes ceil(workgroups / CUs) rounds of its steps; every split writes and re-reads fp32 parts.  Times in us, as
// measured (a step of each height; a workgroup's start and end; the join's launch; its bytes at 4 TB/s).  Against every
// height and split forced in turn, over 32 to 4096 rows and five weight shapes, this and the plan below choose one
// within 8 % of the fastest in 101 of 105 cases, and within 26 % in the others.
static SplitPlan split_plan(int64_t rows, const lrq_mxfp4* t, bool trans) {
  constexpr double kSteps[2][3] = {{0.53, 0.72, 1.4}, {0.6, 1.0, 1.6}}, kFixed = 9.0, kJoin = 4.0, kPerByte = 2.0 / 4.0e6;
  const int64_t cols = trans ? t->cols : t->rows, depth = trans ? t->rows : t->cols;
  const int steps = (int)((depth + 127) / 128);
  if (!trans && rows <= 16) return SplitPlan{0, 0, 0, 1, steps};
  SplitPlan best{};
  double least = 0.;
  for (int i = 0; i < 3; ++i) {
    SplitPlan p{1 << i, 0, (cols + 255) / 256, 1, steps};
    p.tiles_m = (rows + 32 * p.mt - 1) / (32 * p.mt);
    for (; p.splits <= 16 && p.splits <= std::max(1, steps / 2); ++p.splits) {
      const double rounds = (double)((p.tiles_m * p.tiles_n * p.splits + 255) / 256);
      const double cost = rounds * ((steps + p.splits - 1) / p.splits * kSteps[trans][i] + kFixed) +
                          (p.splits > 1 ? kJoin + kPerByte * 4. * p.splits * rows * cols : 0.);
      if (best.mt == 0 || cost < least) best = p, least = cost;
    }
  }
  return best;
}

struct GemmPlan {
  int mt;  // 64 mt rows a workgroup
  int64_t tiles_m, tiles_n;
  int splits;
};

// As split_plan; a workgroup's start and end count as three steps.
static GemmPlan gemm_plan(const lrq_mxfp4* a, const lrq_mxfp4* b) {
  constexpr double kStep[3] = {0.35, 0.4, 0.6}, kJoin = 4.0, kPerByte = 2.0 / 4.0e6;
  const int steps = (int)((a->cols + 127) / 128);
  GemmPlan best{};
  double least = 0.;
  for (int i = 0; i < 3; ++i) {
    GemmPlan p{1 << i, 0, (b->rows + 255) / 256, 1};
    p.tiles_m = (a->rows + 64 * p.mt - 1) / (64 * p.mt);
    for (p.splits = 1; p.splits <= 16 && p.splits <= std::max(1, steps / 4); ++p.splits) {
      const double rounds = (double)((p.tiles_m * p.tiles_n * p.splits + 255) / 256);
      const double cost = rounds * ((steps + p.splits - 1) / p.splits + 3) * kStep[i] +
                          (p.splits > 1 ? kJoin + kPerByte * 4. * p.splits * a->rows * b->rows : 0.);
      if (best.mt == 0 || cost < least) best = p, least = cost;
    }
  }
  return best;
}

static int64_t split_bytes(int splits, int64_t rows, int64_t cols) {
  return splits > 1 ? (int64_t)splits * rows * ((cols + 3) / 4 * 4) * 4 : 0;
}

static int validate_workspace(const void* p, int64_t bytes, int64_t need) {
  if (need == 0) return LRQ_OK;
  if (p == nullptr) return LRQ_ERR_NULL;
  if (!aligned(p, 16)) return LRQ_ERR_ALIGN;
  return bytes < need ? LRQ_ERR_WORKSPACE : LRQ_OK;
}

static int join(const float* part, int splits, int64_t rows, int64_t cols, int64_t ldp, void* out, int64_t ldo,
                int32_t out_fp32, hipStream_t s) {
  const dim3 grid((unsigned)std::min<int64_t>((rows * (ldp / 4) + 255) / 256, (int64_t)cu_count() * 32));
  return out_fp32 ? launch(k_mx_join<true>, grid, dim3(256), 0, s, part, splits, rows, cols, ldp, out, ldo)
                  : launch(k_mx_join<false>, grid, dim3(256), 0, s, part, splits, rows, cols, ldp, out, ldo);
}

static int validate_out(const void* out, int64_t ldo, int64_t cols, int32_t f32) {
  if (out == nullptr) return LRQ_ERR_NULL;
  if (ldo < cols) return LRQ_ERR_SHAPE;
  return aligned(out, f32 ? 4 : 2) ? LRQ_OK : LRQ_ERR_ALIGN;
}

}  // namespace lrq

using namespace lrq;

extern "C" int64_t lrq_mxfp4_gemm_workspace(const lrq_mxfp4* ta, const lrq_mxfp4* tb) {
  LRQ_TRY(validate_mx(ta));
  LRQ_TRY(validate_mx(tb));
  if (ta->cols != tb->cols) return LRQ_ERR_SHAPE;
  return split_bytes(gemm_plan(ta, tb).splits, ta->rows, tb->rows);
}

extern "C" int lrq_mxfp4_gemm(const lrq_mxfp4* ta, const lrq_mxfp4* tb, void* out, int64_t ldo, int32_t out_fp32,
                              void* workspace, int64_t workspace_bytes, void* stream) {
  LRQ_TRY(validate_mx(ta));
  LRQ_TRY(validate_mx(tb));
  if (ta->cols != tb->cols) return LRQ_ERR_SHAPE;
  if (ta->rows == 0 || tb->rows == 0) return LRQ_OK;
  LRQ_TRY(validate_out(out, ldo, tb->rows, out_fp32));
  const GemmPlan p = gemm_plan(ta, tb);
  const int64_t need = split_bytes(p.splits, ta->rows, tb->rows), ldp = (tb->rows + 3) / 4 * 4;
  LRQ_TRY(validate_workspace(workspace, workspace_bytes, need));
  const int64_t wgs = p.tiles_m * p.tiles_n * p.splits;
  if (wgs > INT32_MAX) return LRQ_ERR_SHAPE;
  const GemmArgs a{make_mx(ta), make_mx(tb), need ? workspace : out, need ? ldp : ldo, (int)p.tiles_m, (int)p.tiles_n,
                   p.splits};
  hipStream_t s = (hipStream_t)stream;
  const auto go = [&](auto kern) {
    const int lds = p.mt == 4 ? GemmLds<4>::kBytes : p.mt == 2 ? GemmLds<2>::kBytes : GemmLds<1>::kBytes;
    const hipError_t e = hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (e != hipSuccess) return (int)e;
    return launch(kern, dim3((unsigned)wgs), dim3(512), (size_t)lds, s, a);
  };
  const bool f32 = need > 0 || out_fp32;
  if (p.mt == 4) LRQ_TRY(f32 ? go(k_mx_gemm<4, true>) : go(k_mx_gemm<4, false>));
  else if (p.mt == 2) LRQ_TRY(f32 ? go(k_mx_gemm<2, true>) : go(k_mx_gemm<2, false>));
  else LRQ_TRY(f32 ? go(k_mx_gemm<1, true>) : go(k_mx_gemm<1, false>));
  return need ? join((const float*)workspace, p.splits, ta->rows, tb->rows, ldp, out, ldo, out_fp32, s) : LRQ_OK;
}

extern "C" int64_t lrq_mxfp4_linear_workspace(int64_t rows, const lrq_mxfp4* t, int32_t transposed) {
  LRQ_TRY(validate_mx(t));
  if (rows < 0 || rows > INT32_MAX) return LRQ_ERR_SHAPE;
  return split_bytes(split_plan(rows, t, transposed != 0).splits, rows, transposed ? t->cols : t->rows);
}

static int mx_linear(const void* x, int64_t ldx, int64_t rows, const lrq_mxfp4* t, bool trans, void* out, int64_t ldo,
                     int32_t out_fp32, void* workspace, int64_t workspace_bytes, void* stream) {
  LRQ_TRY(validate_mx(t));
  if (rows < 0 || rows > INT32_MAX) return LRQ_ERR_SHAPE;
  const int64_t depth = trans ? t->rows : t->cols, cols = trans ? t->cols : t->rows;
  if (rows == 0 || cols == 0) return LRQ_OK;
  if (depth > 0) {
    if (x == nullptr) return LRQ_ERR_NULL;
    if (ldx < (depth + 7) / 8 * 8) return LRQ_ERR_SHAPE;
    if (!aligned(x, 16) || (ldx % 8) != 0) return LRQ_ERR_ALIGN;
  }
  LRQ_TRY(validate_out(out, ldo, cols, out_fp32));
  if (depth == 0) return LRQ_ERR_SHAPE;  // (a sum over no rows: the caller's zeros)
  const Mx w = make_mx(t);
  hipStream_t s = (hipStream_t)stream;
  const uint16_t* px = (const uint16_t*)x;
  if (!trans && rows <= 16) {
    using std::integral_constant;
    const int64_t tiles = (w.rows + 15) / 16;
    const auto go = [&](auto r, auto waves, auto cols) {
      const dim3 grid((unsigned)((tiles + cols() - 1) / cols()));
      return out_fp32 ? launch((k_mx_token<r(), waves(), cols(), true>), grid, dim3(64 * waves()), 0, s, px, ldx, (int)rows, w, out, ldo)
                      : launch((k_mx_token<r(), waves(), cols(), false>), grid, dim3(64 * waves()), 0, s, px, ldx, (int)rows, w, out, ldo);
    };
    // four waves a workgroup (8 steps each of 4096 columns: one round of loads); eight where workgroups are few and the
    // runs long, 11.3 against 13.3 us on 4096 rows of 14336 columns (but 6.3 against 5.2 us on 4096 of 4096); with 16
    // rows, whose runs are of four steps, there always
#define LRQ_GO(R, W, C) return go(integral_constant<int, R>{}, integral_constant<int, W>{}, integral_constant<int, C>{})
    if (rows <= 4) {
      if (tiles >= 512 || w.steps <= 64) LRQ_GO(4, 4, 1);
      LRQ_GO(4, 8, 1);
    }
    if (tiles >= 512) LRQ_GO(16, 4, 2);
    LRQ_GO(16, 8, 1);
#undef LRQ_GO
  }
  const SplitPlan p = split_plan(rows, t, trans);
  const int64_t need = split_bytes(p.splits, rows, cols);
  LRQ_TRY(validate_workspace(workspace, workspace_bytes, need));
  const int64_t ldp = (cols + 3) / 4 * 4;
  const int64_t wgs = p.tiles_m * p.tiles_n * p.splits;
  if (wgs > INT32_MAX) return LRQ_ERR_SHAPE;
  const TileArgs a{px, ldx, rows, w, need ? workspace : out, need ? ldp : ldo, cols, (int)p.tiles_m, (int)p.tiles_n,
                   p.splits, p.steps, (int)((depth + 7) / 8)};
  const bool f32 = need > 0 || out_fp32;
  const auto go = [&](auto kern, int lds) {
    const hipError_t e = hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (e != hipSuccess) return (int)e;
    return launch(kern, dim3((unsigned)wgs), dim3(512), (size_t)lds, s, a);
  };
  const auto with = [&](auto mt) {
    constexpr int kLds = TileLds<false, mt()>::kBytes, kLdsT = TileLds<true, mt()>::kBytes;
    if (trans) return f32 ? go(k_mx_tile<true, mt(), true>, kLdsT) : go(k_mx_tile<true, mt(), false>, kLdsT);
    return f32 ? go(k_mx_tile<false, mt(), true>, kLds) : go(k_mx_tile<false, mt(), false>, kLds);
  };
  if (p.mt == 4) LRQ_TRY(with(std::integral_constant<int, 4>{}));
  else if (p.mt == 2) LRQ_TRY(with(std::integral_constant<int, 2>{}));
  else LRQ_TRY(with(std::integral_constant<int, 1>{}));
  return need ? join((const float*)workspace, p.splits, rows, cols, ldp, out, ldo, out_fp32, s) : LRQ_OK;
}

extern "C" int lrq_mxfp4_linear(const void* x, int64_t ldx, int64_t rows, const lrq_mxfp4* w, void* out, int64_t ldo,
                                int32_t out_fp32, void* workspace, int64_t workspace_bytes, void* stream) {
  return mx_linear(x, ldx, rows, w, false, out, ldo, out_fp32, workspace, workspace_bytes, stream);
}

extern "C" int lrq_mxfp4_linear_t(const void* y, int64_t ldy, int64_t rows, const lrq_mxfp4* w, void* out, int64_t ldo,
                                  int32_t out_fp32, void* workspace, int64_t workspace_bytes, void* stream) {
  return mx_linear(y, ldy, rows, w, true, out, ldo, out_fp32, workspace, workspace_bytes, stream);
}
