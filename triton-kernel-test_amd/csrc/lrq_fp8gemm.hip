// Products with e4m3 operands (format: lrq_fp8.h) on the scaled matrix instructions, fp32 accumulation:
//
//   lrq_fp8_gemm      out[M, N] = X W^T, X [M, K] and W [N, K]
//   lrq_fp8_gemm_nn   out[M, K] = Y W, the gradient of the above for X
//   lrq_fp8_linear    the first with X quantised on the way, few rows
//   lrq_fp8_quantize_gemm   X quantised, then either
//
// A scale is constant over a K step of 128, a power of two, and the instructions multiply by it: no step's sums pass through
// the vector unit.  The instructions add each eight neighbouring products in a fixed window: bits of a product below 2^-13 of
// the largest one's power of two are lost (measured), so that each eight may lose 7 * 2^-13 of its largest product, in one
// direction where all have one sign; the rest is fp32.  Measured on contractions of 4096 and 14336: normal operands are off by
// 1.5e-5 of the outputs' size in the mean square and by 2e-6 of the sum of their magnitudes at most; positive ones by 4e-7 to
// 5e-7 of it (the library's fp32 products of the same: 0.5e-7 to 4e-7).
#include "lrq_fp8.h"
#include "lrq_fp8plan.h"

namespace lrq {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

// 32 bytes of a row: an instruction's operand of one lane.
struct Frag {
  u32x4 v[2];
};
__device__ __forceinline__ i32x8 operand(const Frag& f) {
  return i32x8{(int)f.v[0][0], (int)f.v[0][1], (int)f.v[0][2], (int)f.v[0][3],
               (int)f.v[1][0], (int)f.v[1][1], (int)f.v[1][2], (int)f.v[1][3]};
}
// D(32x32) += A(32x64) B(64x32), e4m3.  Lane l holds row (column) l % 32, k = 32 (l / 32) .. + 31, and its scale in byte 0.
__device__ __forceinline__ f32x16 mfma8_32(const Frag& a, const Frag& b, f32x16 c, uint32_t sa, uint32_t sb) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(operand(a), operand(b), c, 0, 0, 0, (int)sa, 0, (int)sb);
}
// D(16x16) += A(16x128) B(128x16).  Lane l holds row (column) l % 16, k = 32 (l / 16) .. + 31.
__device__ __forceinline__ f32x4 mfma8_16(const Frag& a, const Frag& b, f32x4 c, uint32_t sa, uint32_t sb) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(operand(a), operand(b), c, 0, 0, 0, (int)sa, 0, (int)sb);
}

__device__ __forceinline__ uint16_t bits16(float v, int dt) {
  return dt == kBf16 ? (uint16_t)pack_bf16x2(v, 0.f) : f16_bits(v);
}
__device__ __forceinline__ uint32_t pack16(float a, float b, int dt) {
  return dt == kBf16 ? pack_bf16x2(a, b) : (uint32_t)f16_bits(a) | (uint32_t)f16_bits(b) << 16;
}

// 64 lanes' 16 (4) bytes at base + off to LDS, lane l's at lds + 16 l (4 l); base and lds are the wave's.  In assembly: the
// compiler does not see the load, which has no output register and whose end is counted by vmcnt as that of any other;
// all waits for it are written out.  (Behind a load to LDS that the compiler knows of, it lets each transposing LDS read wait
// until every load is in; and it takes a 64-bit addition for each address, 2 % of a product.)  m0 has no other use in the
// kernels that call it.
template <int BYTES>
__device__ __forceinline__ void ld_to_lds8(const uint8_t* base, uint32_t off, uint32_t lds) {
  if constexpr (BYTES == 16)
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(lds) : "memory");
  else
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1" ::"v"(off), "s"(base), "s"(lds) : "memory");
}

// ---------------------------------------------------------------- few rows
struct TokenArgs {
  const char* x;  // fp8 codes, or 16-bit elements
  int64_t ldx;    // bytes
  const uint8_t* xs;
  int64_t ldxs;
  int xshift, rows;
  int own;        // rows of W a workgroup
  Fp8 w;
  void* out;
  int64_t ldo;
  int odt;
};

typedef uint32_t u32_byte __attribute__((aligned(1)));

// Up to 16 TM rows of X by `own` rows of W (16 TN at most) a workgroup; its waves take runs of the K steps, D of them with all
// loads in flight at once, and join in LDS.  Bound by W's bytes, which are read once, past the caches: one row by
// [14336, 4096] from memory 13.6 to 15.8 us (4.3 to 3.7 TB/s), by [4096, 4096] 5.2 to 6.8, by [5120, 5120] 8.9 to 10.5;
// 32 rows by the second 9.7.  W is the instruction's first operand, so that a lane ends with four neighbouring outputs of one
// row of X.  Lane (j, g) holds pieces g and g + 4 of row j's 128 bytes (any order of K serves that both operands share): each
// load of W takes 64 neighbouring bytes of 16 rows.
//
// XT kX8: X in e4m3, read as the operand.  kBf16, kF16: four 16-bit rows at most, quantised by every wave for its own steps:
// 16 lanes a row, 8 elements each, then through LDS to the operand's lanes.  (Four rows quantised here: 15.5 us by [14336, 4096],
// as long as by e4m3 rows, and the quantiser's launch is saved; 16 rows took 18.5 to 24 against 16.7 and 2.4 of that launch.)
enum { kX8 = 3 };
template <int XT, int TM, int TN, int WAVES, int D>
__global__ __launch_bounds__(64 * WAVES) void k_fp8_token(TokenArgs a) {
  constexpr bool k8 = XT == kX8;
  static_assert(D <= 4 && (k8 || TM == 1));  // (a dword holds four steps' scales)
  __shared__ f32x4 red[WAVES][TM * TN][64];
  __shared__ __attribute__((aligned(16))) char xq[k8 ? 1 : WAVES][4][128];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), j = lane & 15, g = lane >> 4;
  const int64_t n0 = (int64_t)blockIdx.x * a.own, n1 = min(n0 + a.own, a.w.rows);
  const int steps = a.w.steps, first = steps * wave / WAVES, last = steps * (wave + 1) / WAVES;
  const int sw4 = (steps + 3) / 4 * 4;
  const uint8_t *wp[TN], *wsc[TN];
#pragma unroll
  for (int t = 0; t < TN; ++t) {
    const int64_t r = min(n0 + 16 * t + j, n1 - 1);
    wp[t] = a.w.codes + r * a.w.ldc + 16 * g;
    wsc[t] = a.w.scales + (r >> a.w.shift) * a.w.lds;
  }
  const char* xp[TM];
  const uint8_t* xsc[TM];
#pragma unroll
  for (int i = 0; i < TM; ++i) {  // (lanes past X's rows repeat its last: what they add is not stored)
    const int64_t r = min(16 * i + j, a.rows - 1);
    xp[i] = a.x + r * a.ldx + 16 * g;
    xsc[i] = a.xs + (r >> a.xshift) * a.ldxs;
  }
  f32x4 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int t = 0; t < TN; ++t) acc[i][t] = zero4();
  for (int s0 = first; s0 < last; s0 += D) {
    Frag w[TN][D], x8[k8 ? TM : 1][k8 ? D : 1];
    Chunk<k8 ? kBf16 : XT> x16[k8 ? 1 : D];
    uint32_t sw[TN], sx[TM];
    const int n = min(D, last - s0), base = min(s0, sw4 - 4);
#pragma unroll
    for (int u = 0; u < D; ++u) {
      if (u < n) {
#pragma unroll
        for (int t = 0; t < TN; ++t) {
          w[t][u].v[0] = ld16_stream(wp[t] + 128 * (int64_t)(s0 + u));
          w[t][u].v[1] = ld16_stream(wp[t] + 128 * (int64_t)(s0 + u) + 64);
        }
        if constexpr (k8) {
#pragma unroll
          for (int i = 0; i < TM; ++i) {
            x8[i][u].v[0] = ld16(xp[i] + 128 * (int64_t)(s0 + u));
            x8[i][u].v[1] = ld16(xp[i] + 128 * (int64_t)(s0 + u) + 64);
          }
        } else {
          const int k = 128 * (s0 + u) + 8 * j;
          x16[u] = ld_chunk<XT>(a.x + min(g, a.rows - 1) * a.ldx + 2 * (int64_t)k, k < a.w.cols ? 8 : 0);
        }
      }
    }
#pragma unroll
    for (int t = 0; t < TN; ++t) sw[t] = *reinterpret_cast<const u32_byte*>(wsc[t] + base);
    if constexpr (k8) {
#pragma unroll
      for (int i = 0; i < TM; ++i) sx[i] = *reinterpret_cast<const u32_byte*>(xsc[i] + base);
    }
#pragma unroll
    for (int u = 0; u < D; ++u) {
      if (u >= n) break;
      const int sh = 8 * (s0 + u - base);
      if constexpr (k8) {
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
          for (int t = 0; t < TN; ++t) acc[i][t] = mfma8_16(w[t][u], x8[i][u], acc[i][t], sw[t] >> sh, sx[i] >> sh);
      } else {
        float v[8];
        widen<XT>(x16[u], v);
        const uint32_t mine = fp8_scale(lanes16_max(top8(v)));
        st8(&xq[wave][g][16 * (j / 2 ^ g) + 8 * (j & 1)], fp8_codes8(v, mine));
        const int r = j & 3;  // (rows past four: their products are not stored)
        const uint32_t s = (uint32_t)__shfl((int)mine, 16 * r);
        Frag x;
        asm volatile("" ::: "memory");
        x.v[0] = ld16(&xq[wave][r][16 * (g ^ r)]);
        x.v[1] = ld16(&xq[wave][r][16 * ((g + 4) ^ r)]);
        asm volatile("" ::: "memory");
#pragma unroll
        for (int t = 0; t < TN; ++t) acc[0][t] = mfma8_16(w[t][u], x, acc[0][t], sw[t] >> sh, s);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int t = 0; t < TN; ++t) red[wave][i * TN + t][lane] = acc[i][t];
  __syncthreads();
  for (int p = wave; p < TM * TN; p += WAVES) {
    f32x4 s = red[0][p][lane];
#pragma unroll
    for (int k = 1; k < WAVES; ++k) {
      const f32x4 v = red[k][p][lane];
#pragma unroll
      for (int e = 0; e < 4; ++e) s[e] += v[e];
    }
    const int64_t n = n0 + 16 * (p % TN) + 4 * g, m = 16 * (p / TN) + j;
    if (m >= a.rows) continue;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (n + e >= n1) break;
      if (a.odt == kF32) reinterpret_cast<float*>(a.out)[m * a.ldo + n + e] = s[e];
      else reinterpret_cast<uint16_t*>(a.out)[m * a.ldo + n + e] = bits16(s[e], a.odt);
    }
  }
}

// ---------------------------------------------------------------- many rows
// 16 bytes of an output row, the first `valid` elements of them stored, past L2 where whole.
template <int OT>
struct Out16 {
  u32x4 v;
  __device__ __forceinline__ void store(char* to, int valid) const {
    constexpr int kWide = 16 / Elem<OT>::kBytes;
    if (valid >= kWide) {
      __builtin_nontemporal_store(v, reinterpret_cast<u32x4_any*>(to));
    } else {
#pragma unroll
      for (int e = 0; e < kWide - 1; ++e) {
        if (e < valid) {
          if constexpr (OT == kF32) reinterpret_cast<uint32_t*>(to)[e] = v[e];
          else reinterpret_cast<uint16_t*>(to)[e] = (uint16_t)(v[e / 2] >> (16 * (e & 1)));
        }
      }
    }
  }
};

struct Operand8 {
  const uint8_t *codes, *scales;
  uint32_t ldc, lds, rows;
  int steps, shift;
};
struct Tile8Args {
  Operand8 x, w;
  void* out;      // [splits][x.rows][ldo] fp32 parts where splits > 1
  int64_t ldo;
  int64_t cols;   // of the output
  int odt;
  int tiles_m, tiles_n, splits;
  int steps;      // contraction steps of 128
};

// Workgroup: 64 MT rows of X by 64 NB output columns, four waves in two rows of two, each 32 MT x 32 NB of it in 32x32x64
// instructions: one wave a SIMD, whose sums take half of its registers.  K goes through LDS in steps of 128 bytes a row,
// straight from memory, whole cache lines at a time (with 64 bytes a row the L2s were asked twice as often, 66 % of their
// cycles, and 8192^3 took 480 us).
//
// Bound by power: 8192^3 takes 385 to 400 us (2.8 PFLOP/s), x w^T and dy w alike, with the matrix units busy in 78 % of the
// cycles, at 1.87 GHz; operands of zeros take 300.  Workgroups that walked several tiles, with the next one's loads behind
// the last's steps, filled the gaps between tiles and took as long.  4096 x 14336 x 4096, 896 tiles in four rounds of
// which the last is half empty, 197.
//
// LDS: X and (NN false) W have rows of 128 bytes, row r's 16-byte piece p in slot p ^ (r / 2 % 8): 16 lanes of a read cover
// all banks.  NN: 128 rows of W of 64 NB bytes, piece p of row r in slot p ^ (r % 8) (NB 1, four pieces: p ^ r % 4 ^ r / 4 %
// 2); the transposing read gives a lane its column of 8 rows.
template <int MT, int NB>
struct Tile8Lds {
  static constexpr int kX = 64 * MT * 128, kW = 64 * NB * 128, kStage = kX + kW, kScales = 2048;
  static constexpr int kMost = (160 * 1024 - 2 * kScales) / kStage;
  static constexpr int kDeep = kMost < 4 ? kMost : 4;  // (64 x 128 tiles six deep: 2 to 15 % slower)
  static constexpr int kRing = kDeep * kStage, kLoop = kRing + 2 * kScales;
  static constexpr int kOut = 4 * 32 * (128 + 16);  // of the output, in the ring's place
  static_assert(kLoop <= 160 * 1024 && kOut <= kLoop);
};

template <bool NN, int MT, int NB, int OT>
__global__ __launch_bounds__(256, 1) void k_fp8_tile(Tile8Args a) {
  using T = Tile8Lds<MT, NB>;
  constexpr int kX = T::kX, kStage = T::kStage, kDeep = T::kDeep, kLx = 2 * MT, kLw = 2 * NB, kLoads = kLx + kLw;
  extern __shared__ __attribute__((aligned(16))) char sm[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave >> 1, wn = wave & 1, c = lane & 31, h = lane >> 5;
  const uint32_t tiles = a.tiles_m * a.tiles_n, id = xcd_tile(blockIdx.x, gridDim.x);
  const uint32_t z = __builtin_amdgcn_readfirstlane(id / tiles), tile = id - z * tiles;
  // runs of kBand tiles down, then across: the 32 tiles that an XCD's CUs work on share 8 rows and 4 columns of tiles
  constexpr uint32_t kBand = 8;
  const uint32_t band = __builtin_amdgcn_readfirstlane(tile / (kBand * a.tiles_n)), in = tile - band * kBand * a.tiles_n;
  const uint32_t tall = min(kBand, a.tiles_m - band * kBand);
  const uint32_t tn = __builtin_amdgcn_readfirstlane(in / tall), tm = band * kBand + in - tn * tall;
  const uint32_t m0 = tm * 64 * MT, n0 = tn * 64 * NB;
  // a split's steps: whole groups of four, whose scales come together
  const uint32_t groups = (uint32_t)(a.steps + 3) >> 2;
  const int first = 4 * __builtin_amdgcn_readfirstlane((uint32_t)((uint64_t)groups * z / (uint32_t)a.splits));
  const uint32_t past = __builtin_amdgcn_readfirstlane((uint32_t)((uint64_t)groups * (z + 1) / (uint32_t)a.splits));
  const int last = min(4 * (int)past, a.steps);

  // ---- loads of 1 KB: 8 rows of 128 bytes (NN W: 16 / NB rows of 64 NB), at 32-bit offsets from a tile's first row
  const uint32_t sm0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)sm;
  // NN: row rw + kRows i of a step; its piece depends on the row's last three bits, so on i % 2 at most
  constexpr int kLanes = 4 * NB, kRows = 64 / kLanes, kEven = kRows >= 8 ? 1 : 2;
  const auto turn = [](int r) { return NB == 1 ? (r ^ (r >> 2 & 1)) & 3 : r & 7; };
  const int rw = 32 * wave + lane / kLanes;
  struct {
    const uint8_t *x, *w;
    uint32_t row;
  } to;  // the step that is loaded next (row: NN, of W)
  const auto point = [&](int step) {
    to.row = 128u * (uint32_t)step;
    to.x = a.x.codes + (uint64_t)m0 * a.x.ldc + to.row;
    to.w = NN ? a.w.codes + n0 + (uint64_t)to.row * a.w.ldc : a.w.codes + (uint64_t)n0 * a.w.ldc + to.row;
  };
  uint32_t ox[kLx], ow[NN ? kEven : kLw];
  const uint32_t mx = min(64u * MT, a.x.rows - m0) - 1;
#pragma unroll
  for (int i = 0; i < kLx; ++i) {
    const int r = 8 * (kLx * wave + i) + (lane >> 3);
    ox[i] = min((uint32_t)r, mx) * a.x.ldc + 16 * ((lane & 7) ^ (r >> 1 & 7));
  }
  if constexpr (!NN) {
    const uint32_t mw = min(64u * NB, a.w.rows - n0) - 1;
#pragma unroll
    for (int i = 0; i < kLw; ++i) {
      const int r = 8 * (kLw * wave + i) + (lane >> 3);
      ow[i] = min((uint32_t)r, mw) * a.w.ldc + 16 * ((lane & 7) ^ (r >> 1 & 7));
    }
  } else {
    const uint32_t mw = min(64u * NB, 128u * (uint32_t)a.w.steps - n0) - 16;
#pragma unroll
    for (int i = 0; i < kEven; ++i) ow[i] = min((uint32_t)(16 * ((lane % kLanes) ^ turn(rw + kRows * i))), mw);
  }
  // load i of the step
  const auto issue = [&](int buf, int i) {
    const uint32_t st = sm0 + buf * kStage;
    if (i < kLx) {
      ld_to_lds8<16>(to.x, ox[i < kLx ? i : 0], st + 1024 * (kLx * wave + i));
    } else {
      const int k = i >= kLx ? i - kLx : 0;
      const uint32_t lds = st + kX + 1024 * (kLw * wave + k);
      if constexpr (!NN) {
        ld_to_lds8<16>(to.w, ow[k], lds);
      } else {  // rows past W's last: that one (their x is zero)
        const uint32_t end = a.w.rows - 1 - to.row;
        ld_to_lds8<16>(to.w, min((uint32_t)(rw + kRows * k), end) * a.w.ldc + ow[k % kEven], lds);
      }
    }
  };
  // four steps' scales of 64 rows a load; NN: of the block of 128 columns that this wave's are in, four steps are four rows
  const int is = min(wave, MT - 1), iw = min(wave, NB - 1);
  const int block = min((int)(n0 + 32 * NB * wn) >> 7, a.w.steps - 1);  // NN
  const uint32_t osx = (min(m0 + 64 * is + lane, a.x.rows - 1) >> a.x.shift) * a.x.lds;
  const uint32_t osw = NN ? (uint32_t)(block & ~3) : (min(n0 + 64 * iw + lane, a.w.rows - 1) >> a.w.shift) * a.w.lds;
  const auto issue_scales = [&](int group, int slot) {
    const uint32_t sc = sm0 + T::kRing + slot * T::kScales;
    ld_to_lds8<4>(a.x.scales + 4 * group, osx, sc + 256 * is);
    if constexpr (!NN) ld_to_lds8<4>(a.w.scales + 4 * group, osw, sc + 1024 + 256 * iw);
    else ld_to_lds8<4>(a.w.scales, (uint32_t)min(4 * group + (lane & 3), a.steps - 1) * a.w.lds + osw, sc + 1024 + 256 * wave);
  };

  // ---- operands of half Q of a step (64 of K): piece 4 Q + 2 h + q of a row
  Frag fx[2][MT], fw[2][NB];
  uint32_t sx[MT], sw[NB];
  const auto read_x = [&](int half, int buf, int i, int q) {
    const int r = 32 * MT * wm + 32 * i + c;
    fx[half][i].v[q] = ld16(sm + buf * kStage + 128 * r + 16 * ((4 * half + 2 * h + q) ^ (r >> 1 & 7)));
  };
  const auto read_w = [&](int half, int buf, int t, int q) {
    const char* st = sm + buf * kStage + kX;
    if constexpr (!NN) {
      const int r = 32 * NB * wn + 32 * t + c;
      fw[half][t].v[q] = ld16(st + 128 * r + 16 * ((4 * half + 2 * h + q) ^ (r >> 1 & 7)));
    } else {
      const int r = 64 * half + 32 * h + 16 * q + (lane >> 1 & 7), piece = 2 * NB * wn + 2 * t + (lane >> 4 & 1);
      typedef int i32x2 __attribute__((ext_vector_type(2)));
      const auto p = (__attribute__((address_space(3))) i32x2*)(st + 64 * NB * r + 16 * (piece ^ turn(r)) + 8 * (lane & 1));
      const i32x2 lo = __builtin_amdgcn_ds_read_tr8_b64_v2i32(p), hi = __builtin_amdgcn_ds_read_tr8_b64_v2i32(p + 64 * NB);
      fw[half][t].v[q] = u32x4{(uint32_t)lo[0], (uint32_t)lo[1], (uint32_t)hi[0], (uint32_t)hi[1]};
    }
  };
  const auto read_piece = [&](int half, int buf, int p) {
    if (p < 2 * NB) read_w(half, buf, p >> 1, p & 1);
    else read_x(half, buf, (p - 2 * NB) >> 1, p & 1);
  };
  const auto read_scales = [&](int step, int slot) {
    const char* sc = sm + T::kRing + slot * T::kScales;
    const int sh = 8 * (step & 3);
#pragma unroll
    for (int i = 0; i < MT; ++i) sx[i] = ld4(sc + 4 * (32 * MT * wm + 32 * i + c)) >> sh;
    if constexpr (!NN) {
#pragma unroll
      for (int t = 0; t < NB; ++t) sw[t] = ld4(sc + 1024 + 4 * (32 * NB * wn + 32 * t + c)) >> sh;
    } else {
      sw[0] = ld4(sc + 1024 + 256 * wave + 4 * (step & 3)) >> (8 * (block & 3));
    }
  };

  // Half 1 of a step is read from LDS behind the first instructions of half 0, half 0 of the next step behind those of half 1.
  // The workgroup meets twice in a step: once all of it has been read, whose place the loads of kDeep steps on then take,
  // and before half 1, when the next step's loads are in.  The loads go out evenly over the rest of the step: they are
  // 16 TB/s of the L2s' at full speed, and 1.5 to 2 at a time 8192^3 took 440 us, at 1 behind each instruction of half 1 404,
  // so 395.  The order is held: the compiler would issue all loads first.
  constexpr int kMfma = NB * MT, kHalf = (kMfma + 1) / 2, kPieces = 2 * (MT + NB), kReads = (kPieces + kHalf - 1) / kHalf;
  constexpr int kFirst = 3 * kLoads / 8;  // of a step's loads: behind the second half of half 0's instructions
  // four steps' scales are issued with half 1 of the first step of the four before, and waited for with its last step's loads
  static_assert((kDeep - 2) * kLoads + kFirst <= 3 * kLoads);
  f32x16 acc[MT][NB];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int t = 0; t < NB; ++t) acc[i][t] = f32x16{};
  issue_scales(first >> 2, 0);
#pragma unroll
  for (int d = 0; d < kDeep; ++d) {
    point(min(first + d, last - 1));
#pragma unroll
    for (int i = 0; i < kLoads; ++i) issue(d, i);
  }
  point(first + kDeep);
  __builtin_amdgcn_s_waitcnt(vmcnt_imm((kDeep - 1) * kLoads));
  lds_meet();
#pragma unroll
  for (int p = 0; p < kPieces; ++p) read_piece(0, 0, p);
  read_scales(first, 0);
  // The loads are kDeep steps ahead; the last steps repeat the last's.  A loop for each, so that a step has no branch but
  // that of the scales: the compiler would move the instructions behind it.
  int buf = 0, slot = 0;  // of the step, of its scales
  for (int part = 0, step = first; part < 2; ++part) {
    const int end = part ? last : max(first, last - kDeep);
    const uint64_t ix = part ? 0 : 128, jw = part ? 0 : NN ? 128 * (uint64_t)a.w.ldc : 128;
    if (part) point(last - 1);
    for (; step < end; ++step) {
      const int next = buf + 1 == kDeep ? 0 : buf + 1;
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int m = 0; m < kMfma; ++m) {
        const int i = m / NB, t = m % NB, late = m - kMfma / 2;
        acc[i][t] = mfma8_32(fw[0][t], fx[0][i], acc[i][t], sw[NN ? 0 : t], sx[i]);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int p = kReads * m; p < kReads * (m + 1); ++p)
          if (p < kPieces) read_piece(1, buf, p);
        if (late == 0) lds_meet();
#pragma unroll
        for (int l = 0; l < kFirst; ++l)
          if (l * kHalf / kFirst == late) issue(buf, l);
        __builtin_amdgcn_sched_barrier(0);
      }
      __builtin_amdgcn_s_waitcnt(vmcnt_imm((kDeep - 2) * kLoads + kFirst));
      lds_meet();
      if ((step & 3) == 0 && step + 4 < last) issue_scales((step >> 2) + 1, slot ^ 1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int m = 0; m < kMfma; ++m) {
        const int i = m / NB, t = m % NB;
        acc[i][t] = mfma8_32(fw[1][t], fx[1][i], acc[i][t], sw[NN ? 0 : t], sx[i]);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int l = 0; l < kLoads - kFirst; ++l)
          if (l * kMfma / (kLoads - kFirst) == m) issue(buf, kFirst + l);
#pragma unroll
        for (int p = kReads * m; p < kReads * (m + 1); ++p)
          if (p < kPieces) read_piece(0, next, p);
        __builtin_amdgcn_sched_barrier(0);
      }
      to.x += ix, to.w += jw, to.row += (uint32_t)ix;
      slot ^= (step & 3) == 3 ? 1 : 0;
      read_scales(step + 1, slot);  // (of no use behind the last step)
      buf = next;
    }
  }
  __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));  // the last loads write LDS
  lds_meet();

  // Out through LDS, 32 rows by 128 bytes of the wave's columns at a time: a lane has four neighbouring columns of one row,
  // and leaves with 16 bytes beside its neighbours'.
  constexpr int ES = Elem<OT>::kBytes, kPitch = 128 + 16, kWide = 16 / ES, kTs = NB * ES < 4 ? NB : 4 / ES;
  char* mine = sm + wave * 32 * kPitch;
  char* out = (char*)a.out + (a.splits > 1 ? (int64_t)z * a.x.rows * a.ldo * 4 : 0);
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int64_t m = (int64_t)m0 + 32 * MT * wm + 32 * i + lane / 8;
#pragma unroll
    for (int t0 = 0; t0 < NB; t0 += kTs) {
      const int64_t n = (int64_t)n0 + 32 * NB * wn + 32 * t0 + kWide * (lane % 8);
      const int valid = kWide * (lane % 8) < 32 * kTs ? (int)min((int64_t)kWide, a.cols - n) : 0;
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int t = t0; t < t0 + kTs; ++t) {
        asm volatile("" : "+a"(acc[i][t]));  // not read before: no registers for all of them
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          const f32x4 s = {acc[i][t][4 * v], acc[i][t][4 * v + 1], acc[i][t][4 * v + 2], acc[i][t][4 * v + 3]};
          char* st = mine + c * kPitch + ES * (32 * (t - t0) + 8 * v + 4 * h);
          if constexpr (OT == kF32) st16(st, __builtin_bit_cast(u32x4, s));
          else st8(st, u32x2{pack16(s[0], s[1], OT), pack16(s[2], s[3], OT)});
        }
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      Out16<OT> o[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) o[r].v = ld16(mine + (8 * r + lane / 8) * kPitch + 16 * (lane % 8));
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (m + 8 * r < a.x.rows) o[r].store(out + ((m + 8 * r) * a.ldo + n) * ES, valid);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
  }
}

// out[rows, cols] = the splits' sums, in their order; 4 columns a thread.  4 to 6 us, of which 3 are the launch.
__global__ __launch_bounds__(256) void k_fp8_join(const float* part, int splits, int64_t rows, int64_t cols, int64_t ldp,
                                                  void* out, int64_t ldo, int odt) {
  const int64_t quads = ldp / 4, total = rows * quads;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t m = i / quads, n = 4 * (i - m * quads);
    f32x4 s = *(const f32x4*)(part + m * ldp + n);
#pragma unroll 8
    for (int z = 1; z < splits; ++z) {
      const f32x4 v = *(const f32x4*)(part + ((int64_t)z * rows + m) * ldp + n);
#pragma unroll
      for (int k = 0; k < 4; ++k) s[k] += v[k];
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (n + k >= cols) break;
      if (odt == kF32) reinterpret_cast<float*>(out)[m * ldo + n + k] = s[k];
      else reinterpret_cast<uint16_t*>(out)[m * ldo + n + k] = bits16(s[k], odt);
    }
  }
}

static int64_t parts_bytes(int splits, int64_t rows, int64_t cols) {
  return splits > 1 ? (int64_t)splits * rows * ((cols + 3) / 4 * 4) * 4 : 0;
}

static int validate_out8(const void* out, int64_t ldo, int64_t cols, int32_t dt) {
  if (dt < LRQ_BF16 || dt > LRQ_F32) return LRQ_ERR_UNSUPPORTED;
  if (out == nullptr) return LRQ_ERR_NULL;
  if (ldo < cols) return LRQ_ERR_SHAPE;
  return aligned(out, dt == LRQ_F32 ? 4 : 2) ? LRQ_OK : LRQ_ERR_ALIGN;
}

static int validate_pair(const lrq_fp8* a, const lrq_fp8* b, bool nn) {
  LRQ_TRY(validate_fp8(a));
  LRQ_TRY(validate_fp8(b));
  if (a->cols != (nn ? b->rows : b->cols)) return LRQ_ERR_SHAPE;
  for (const lrq_fp8* t : {a, b}) {  // 32-bit offsets within a tile's codes and from the first scale
    const int64_t tall = (t->rows + t->block - 1) / t->block;
    if (t->ld_codes >= 1 << 24 || t->ld_scales > INT32_MAX) return LRQ_ERR_SHAPE;
    if (tall > 0 && t->ld_scales > UINT32_MAX / tall) return LRQ_ERR_SHAPE;
  }
  return nn && b->block != 128 ? LRQ_ERR_UNSUPPORTED : LRQ_OK;
}

template <int XT, int TM>
static int token(TokenArgs a, hipStream_t s) {
  using std::integral_constant;
  const int64_t n = a.w.rows;
  const auto go = [&](auto tn, auto waves, auto d, int64_t wgs) {
    a.own = (int)std::min<int64_t>(16 * tn(), ((n + wgs - 1) / wgs + 3) / 4 * 4);
    const dim3 grid((unsigned)((n + a.own - 1) / a.own));
    return launch((k_fp8_token<XT, TM, tn(), waves(), d()>), grid, dim3(64 * waves()), 0, s, a);
  };
#define LRQ_GO(TN, WAVES, D, WGS) \
  return go(integral_constant<int, TN>{}, integral_constant<int, WAVES>{}, integral_constant<int, D>{}, WGS)
  // Every CU the same bytes of W, which come to it at about 18 GB/s whatever the others do: a workgroup a CU, of
  // as many rows as that makes ([5120, 5120] by one row 8.9 us; whole tiles of 16 rows, 320 of them: 11.5).  More than 32
  // rows a CU: two workgroups, whose starts and ends overlap ([14336, 4096] 13.7 us against 15.5 with one of 56 rows).
  if constexpr (TM == 1) {
    if (n <= 4096) LRQ_GO(1, 16, 4, 256);
    if (n <= 8192) LRQ_GO(2, 16, 4, 256);
    LRQ_GO(2, 8, 4, 512 * ((n + 16383) / 16384));
  } else {  // (8192 columns at most: few_rows)
    if (n <= 4096) LRQ_GO(1, 16, 2, 256);
    LRQ_GO(2, 16, 2, 256);
  }
#undef LRQ_GO
}

static int fp8_product(const lrq_fp8* ta, const lrq_fp8* tb, bool nn, void* out, int64_t ldo, int32_t odt, void* workspace,
                       int64_t workspace_bytes, hipStream_t s) {
  LRQ_TRY(validate_pair(ta, tb, nn));
  const int64_t rows = ta->rows, cols = nn ? tb->cols : tb->rows;
  if (rows == 0 || cols == 0) return LRQ_OK;
  LRQ_TRY(validate_out8(out, ldo, cols, odt));
  const Plan8 p = plan8(rows, cols, ta->cols, nn);
  const Fp8 x = make_fp8(ta), w = make_fp8(tb);
  if (p.mt == 0) {
    const TokenArgs a{(const char*)x.codes, x.ldc, x.scales, x.lds, x.shift, (int)rows, 0, w, out, ldo, odt};
    return rows <= 16 ? token<kX8, 1>(a, s) : token<kX8, 2>(a, s);
  }
  const int64_t need = parts_bytes(p.splits, rows, cols), ldp = (cols + 3) / 4 * 4;
  if (need > 0) {
    if (workspace == nullptr) return LRQ_ERR_NULL;
    if (!aligned(workspace, 16)) return LRQ_ERR_ALIGN;
    if (workspace_bytes < need) return LRQ_ERR_WORKSPACE;
  }
  const int64_t wgs = p.tiles_m * p.tiles_n * p.splits;
  if (wgs > INT32_MAX) return LRQ_ERR_SHAPE;
  const auto operand = [](const Fp8& t) {
    return Operand8{t.codes, t.scales, (uint32_t)t.ldc, (uint32_t)t.lds, (uint32_t)t.rows, t.steps, t.shift};
  };
  const Tile8Args a{operand(x), operand(w), need ? workspace : out, need ? ldp : ldo, cols, need ? (int)kF32 : odt, (int)p.tiles_m,
                    (int)p.tiles_n, p.splits, p.steps};
  using std::integral_constant;
  const auto with = [&](auto mt, auto nb) {
    const auto go = [&](auto kern) {
      constexpr int kLds = Tile8Lds<mt(), nb()>::kLoop;
      const hipError_t e = hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, kLds);
      if (e != hipSuccess) return (int)e;
      return launch(kern, dim3((unsigned)wgs), dim3(256), (size_t)kLds, s, a);
    };
    const auto typed = [&](auto ot) {
      return nn ? go(k_fp8_tile<true, mt(), nb(), ot()>) : go(k_fp8_tile<false, mt(), nb(), ot()>);
    };
    if (a.odt == kBf16) return typed(integral_constant<int, kBf16>{});
    return a.odt == kF16 ? typed(integral_constant<int, kF16>{}) : typed(integral_constant<int, kF32>{});
  };
  if (p.mt == 4) LRQ_TRY(with(integral_constant<int, 4>{}, integral_constant<int, 4>{}));
  else if (p.mt == 3) LRQ_TRY(with(integral_constant<int, 3>{}, integral_constant<int, 4>{}));
  else if (p.mt == 2 && p.nb == 4) LRQ_TRY(with(integral_constant<int, 2>{}, integral_constant<int, 4>{}));
  else if (p.mt == 2) LRQ_TRY(with(integral_constant<int, 2>{}, integral_constant<int, 2>{}));
  else if (p.nb == 4) LRQ_TRY(with(integral_constant<int, 1>{}, integral_constant<int, 4>{}));
  else if (p.nb == 1) LRQ_TRY(with(integral_constant<int, 1>{}, integral_constant<int, 1>{}));
  else LRQ_TRY(with(integral_constant<int, 1>{}, integral_constant<int, 2>{}));
  if (need == 0) return LRQ_OK;
  const dim3 grid((unsigned)std::min<int64_t>((rows * (ldp / 4) + 255) / 256, (int64_t)cu_count() * 32));
  return launch(k_fp8_join, grid, dim3(256), 0, s, (const float*)workspace, p.splits, rows, cols, ldp, out, ldo, odt);
}

}  // namespace lrq

using namespace lrq;

extern "C" int64_t lrq_fp8_gemm_workspace(const lrq_fp8* a, const lrq_fp8* b, int32_t nn) {
  LRQ_TRY(validate_pair(a, b, nn != 0));
  const int64_t cols = nn ? b->cols : b->rows;
  return parts_bytes(plan8(a->rows, cols, a->cols, nn != 0).splits, a->rows, cols);
}

extern "C" int lrq_fp8_gemm(const lrq_fp8* a, const lrq_fp8* b, void* out, int64_t ldo, int32_t out_dtype, void* workspace,
                            int64_t workspace_bytes, void* stream) {
  return fp8_product(a, b, false, out, ldo, out_dtype, workspace, workspace_bytes, (hipStream_t)stream);
}

extern "C" int lrq_fp8_gemm_nn(const lrq_fp8* a, const lrq_fp8* b, void* out, int64_t ldo, int32_t out_dtype,
                               void* workspace, int64_t workspace_bytes, void* stream) {
  return fp8_product(a, b, true, out, ldo, out_dtype, workspace, workspace_bytes, (hipStream_t)stream);
}

// x quantised, in the part of the workspace behind the split parts.
static lrq_fp8 quantised(void* at, int64_t rows, int64_t cols) {
  const int64_t steps = (cols + 127) / 128;
  return lrq_fp8{at, 128 * steps, (char*)at + rows * 128 * steps, (steps + 3) / 4 * 4, rows, cols, 1};
}

extern "C" int64_t lrq_fp8_quantize_gemm_workspace(int64_t rows, const lrq_fp8* w, int32_t nn) {
  LRQ_TRY(validate_fp8(w));
  alignas(16) static char none[16];  // (its address alone is looked at)
  const lrq_fp8 q = quantised(none, rows, nn ? w->rows : w->cols);
  LRQ_TRY(validate_pair(&q, w, nn != 0));
  const int64_t cols = nn ? w->cols : w->rows;
  return parts_bytes(plan8(rows, cols, q.cols, nn != 0).splits, rows, cols) + rows * (q.ld_codes + q.ld_scales);
}

extern "C" int lrq_fp8_quantize_gemm(const void* x, int64_t ldx, int32_t dtype, int64_t rows, const lrq_fp8* w, int32_t nn,
                                     void* out, int64_t ldo, int32_t out_dtype, void* workspace, int64_t workspace_bytes,
                                     void* stream) {
  const int64_t need = lrq_fp8_quantize_gemm_workspace(rows, w, nn);
  if (need < 0) return (int)need;
  if (dtype < LRQ_BF16 || dtype > LRQ_F32) return LRQ_ERR_UNSUPPORTED;
  const int64_t depth = nn ? w->rows : w->cols, cols = nn ? w->cols : w->rows;
  if (rows == 0 || cols == 0) return LRQ_OK;
  if (x == nullptr || workspace == nullptr) return LRQ_ERR_NULL;
  if (ldx < depth) return LRQ_ERR_SHAPE;
  if (!aligned(x, dtype == LRQ_F32 ? 4 : 2) || !aligned(workspace, 16)) return LRQ_ERR_ALIGN;
  LRQ_TRY(validate_out8(out, ldo, cols, out_dtype));
  if (workspace_bytes < need) return LRQ_ERR_WORKSPACE;
  lrq_fp8 q = quantised(workspace, rows, depth);
  const int64_t parts = need - rows * (q.ld_codes + q.ld_scales);
  q = quantised((char*)workspace + parts, rows, depth);
  LRQ_TRY(lrq_fp8_quantize(x, ldx, dtype, &q, 0, stream));
  return fp8_product(&q, w, nn != 0, out, ldo, out_dtype, workspace, parts, (hipStream_t)stream);
}

extern "C" int lrq_fp8_linear(const void* x, int64_t ldx, int32_t dtype, int64_t rows, const lrq_fp8* t, void* out,
                              int64_t ldo, int32_t out_dtype, void* stream) {
  LRQ_TRY(validate_fp8(t));
  if (dtype != LRQ_BF16 && dtype != LRQ_F16) return LRQ_ERR_UNSUPPORTED;
  if (rows < 0 || rows > LRQ_FP8_LINEAR_ROWS || t->cols % 8 != 0) return LRQ_ERR_SHAPE;
  if (rows == 0 || t->rows == 0) return LRQ_OK;
  if (x == nullptr) return LRQ_ERR_NULL;
  if (ldx < t->cols) return LRQ_ERR_SHAPE;
  if (!aligned(x, 2)) return LRQ_ERR_ALIGN;
  LRQ_TRY(validate_out8(out, ldo, t->rows, out_dtype));
  const TokenArgs a{(const char*)x, 2 * ldx, nullptr, 0, 0, (int)rows, 0, make_fp8(t), out, ldo, out_dtype};
  hipStream_t s = (hipStream_t)stream;
  return dtype == LRQ_BF16 ? token<kBf16, 1>(a, s) : token<kF16, 1>(a, s);
}
