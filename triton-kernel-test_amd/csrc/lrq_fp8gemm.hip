// Products with e4m3 operands (format: lrq_fp8.h) on the scaled matrix instructions, fp32 accumulation:
//
//   lrq_fp8_gemm      out[M, N] = X W^T, X [M, K] and W [N, K]
//   lrq_fp8_gemm_nn   out[M, K] = Y W, the gradient of the above for X
//   lrq_fp8_linear    the first with X quantised on the way, few rows
//
// A scale is constant over a K step of 128, a power of two, and the instructions multiply by it: no step's sums pass through
// the vector unit.
#include "lrq_fp8.h"

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

// 64 lanes' 16 (4) bytes at base + off to LDS, lane l's at lds + 16 l (4 l); base and lds are the wave's.  ASM: the compiler
// does not see the load.  It has no output register; its end is counted by vmcnt as that of any other, and all waits for
// it are written out.  (The transposing LDS reads have no other use: behind a load to LDS that the compiler knows of, it lets
// each of them wait until every load is in.)
template <int BYTES, bool ASM>
__device__ __forceinline__ void ld_to_lds8(const uint8_t* base, uint32_t off, uint32_t lds) {
  if constexpr (!ASM) {
    const auto l = (__attribute__((address_space(3))) void*)(uintptr_t)lds;
    if constexpr (BYTES == 16) __builtin_amdgcn_global_load_lds(base + off, l, 16, 0, 0);
    else __builtin_amdgcn_global_load_lds(base + off, l, 4, 0, 0);
  } else if constexpr (BYTES == 16) {  // (m0 has no other use in these kernels)
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(lds) : "memory");
  } else {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1" ::"v"(off), "s"(base), "s"(lds) : "memory");
  }
}

// The largest of v over the lanes j, j + 16, j + 32, j + 48, in all of them.
__device__ __forceinline__ uint32_t row_top(uint32_t v) {
  const auto a = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  v = max((uint32_t)a[0], (uint32_t)a[1]);
  const auto b = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  return max((uint32_t)b[0], (uint32_t)b[1]);
}

// ---------------------------------------------------------------- few rows
struct TokenArgs {
  const char* x;  // fp8 codes, or 16-bit elements
  int64_t ldx;    // bytes
  const uint8_t* xs;
  int64_t ldxs;
  int xshift, rows;
  Fp8 w;
  void* out;
  int64_t ldo;
  int odt;
};

typedef uint32_t u32_byte __attribute__((aligned(1)));

// Up to 16 TM rows of X by 16 TN rows of W a workgroup; its waves take runs of the K steps and join in LDS.  W is the
// instruction's first operand, so that a lane ends with four neighbouring outputs of one row of X.  XT kX8: X in e4m3; kBf16, kF16: 16-bit
// rows (TM 1), quantised by every workgroup for itself.
enum { kX8 = 3 };
template <int XT, int TM, int TN, int WAVES, int D>
__global__ __launch_bounds__(64 * WAVES) void k_fp8_token(TokenArgs a) {
  static_assert(XT == kX8 || TM == 1);
  __shared__ f32x4 red[WAVES][TM * TN][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), j = lane & 15, g = lane >> 4;
  const int64_t n0 = (int64_t)blockIdx.x * 16 * TN;
  const int steps = a.w.steps, first = steps * wave / WAVES, last = steps * (wave + 1) / WAVES;
  const int sw4 = (steps + 3) / 4 * 4;
  const uint8_t *wp[TN], *wsc[TN], *xsc[TM];
  const char* xp[TM];
#pragma unroll
  for (int t = 0; t < TN; ++t) {
    const int64_t r = min(n0 + 16 * t + j, a.w.rows - 1);
    wp[t] = a.w.codes + r * a.w.ldc + 32 * g;
    wsc[t] = a.w.scales + (r >> a.w.shift) * a.w.lds;
  }
#pragma unroll
  for (int t = 0; t < TM; ++t) {  // (lanes past X's rows repeat its last: what they add is not stored)
    const int64_t r = min(16 * t + j, a.rows - 1);
    xp[t] = a.x + r * a.ldx + (XT == kX8 ? 32 : 64) * g;
    if constexpr (XT == kX8) xsc[t] = a.xs + (r >> a.xshift) * a.ldxs;
  }
  f32x4 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int t = 0; t < TN; ++t) acc[i][t] = zero4();
  constexpr int kXv = XT == kX8 ? 2 : 4;
  struct Group {
    Frag w[TN][D];
    u32x4 x[TM][D][kXv];
    uint32_t sw[TN], sx[TM];
  };
  const auto load = [&](int s0) {
    Group r;
    const int base = min(s0, sw4 - 4);
#pragma unroll
    for (int u = 0; u < D; ++u) {
      const int s = min(s0 + u, last - 1);
#pragma unroll
      for (int t = 0; t < TN; ++t) {
        r.w[t][u].v[0] = ld16_stream(wp[t] + 128 * (int64_t)s);
        r.w[t][u].v[1] = ld16_stream(wp[t] + 128 * (int64_t)s + 16);
      }
#pragma unroll
      for (int t = 0; t < TM; ++t)
#pragma unroll
        for (int q = 0; q < kXv; ++q) {
          if constexpr (XT == kX8) {
            r.x[t][u][q] = ld16(xp[t] + 128 * (int64_t)s + 16 * q);
          } else {
            const int k = 128 * s + 32 * g + 8 * q;
            r.x[t][u][q] = u32x4{0u, 0u, 0u, 0u};
            if (k < a.w.cols) r.x[t][u][q] = *reinterpret_cast<const u32x4_any*>(xp[t] + 256 * (int64_t)s + 16 * q);
          }
        }
    }
#pragma unroll
    for (int t = 0; t < TN; ++t) r.sw[t] = *reinterpret_cast<const u32_byte*>(wsc[t] + base);
#pragma unroll
    for (int t = 0; t < TM; ++t) r.sx[t] = XT == kX8 ? *reinterpret_cast<const u32_byte*>(xsc[t] + base) : 0u;
    return r;
  };
  if (first < last) {
    Group cur = load(first);
    for (int s0 = first; s0 < last; s0 += D) {
      const Group next = load(min(s0 + D, last - 1));
      const int base = min(s0, sw4 - 4);
#pragma unroll
      for (int u = 0; u < D; ++u) {
        if (s0 + u < last) {
          const int sh = 8 * (s0 + u - base);
          Frag x[TM];
          uint32_t sx[TM];
#pragma unroll
          for (int i = 0; i < TM; ++i) {
            if constexpr (XT == kX8) {
              x[i].v[0] = cur.x[i][u][0], x[i].v[1] = cur.x[i][u][1];
              sx[i] = cur.sx[i] >> sh;
            } else {
              float v[4][8];
              uint32_t top = 0;
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                Chunk<XT> c;
                c.v[0] = cur.x[i][u][q];
                widen<XT>(c, v[q]);
                top = max(top, top8(v[q]));
              }
              sx[i] = fp8_scale(row_top(top));
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                const u32x2 c = fp8_codes8(v[q], sx[i]);
                x[i].v[q / 2][2 * (q & 1)] = c[0], x[i].v[q / 2][2 * (q & 1) + 1] = c[1];
              }
            }
          }
#pragma unroll
          for (int t = 0; t < TN; ++t)
#pragma unroll
            for (int i = 0; i < TM; ++i) acc[i][t] = mfma8_16(cur.w[t][u], x[i], acc[i][t], cur.sw[t] >> sh, sx[i]);
        }
      }
      cur = next;
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
    const int m = 16 * (p / TN) + j;
    const int64_t n = n0 + 16 * (p % TN) + 4 * g;
    if (m >= a.rows) continue;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (n + e >= a.w.rows) break;
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

struct Tile8Args {
  Fp8 x, w;
  void* out;      // [splits][x.rows][ldo] fp32 parts where splits > 1
  int64_t ldo;
  int64_t cols;   // of the output
  int odt;
  int tiles_m, tiles_n, splits;
  int steps;      // contraction steps of 128
};

// Workgroup: 64 MT rows of X by 256 output columns, four waves in two rows of two, each 32 MT x 128 of it in 32x32x64
// instructions: one wave a SIMD, whose sums take half of its registers.  K goes through LDS in half steps of 64 bytes a
// row, four deep, straight from memory, one barrier each.
//
// LDS: X and (NN false) W have rows of 64 bytes, row r's 16-byte piece q in slot q ^ (r / 4 % 4): 16 lanes of a read cover
// all banks.  NN: 64 rows of W of 256 bytes, piece q of row r in slot q ^ (r % 8); the transposing read gives a lane its
// column of 8 rows.
template <bool NN, int MT>
struct Tile8Lds {
  static constexpr int kX = 64 * MT * 64, kW = 16384, kStage = kX + kW, kDeep = 4, kRing = kDeep * kStage;
  static constexpr int kScales = 2048, kLoop = kRing + 2 * kScales;
  static constexpr int kPitch = 128 * 4 + 16, kOut = 4 * 32 * kPitch, kBytes = kLoop > kOut ? kLoop : kOut;
};
template <bool NN, int MT, int OT>
__global__ __launch_bounds__(256, 1) void k_fp8_tile(Tile8Args a) {
  using T = Tile8Lds<NN, MT>;
  constexpr int kX = T::kX, kStage = T::kStage, kLoads = MT + 4;
  extern __shared__ __attribute__((aligned(16))) char sm[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave >> 1, wn = wave & 1, c = lane & 31, h = lane >> 5;
  const uint32_t tiles = a.tiles_m * a.tiles_n, id = xcd_tile(blockIdx.x, gridDim.x);
  const uint32_t z = __builtin_amdgcn_readfirstlane(id / tiles), tile = id - z * tiles;
  const uint32_t tn = __builtin_amdgcn_readfirstlane(tile / a.tiles_m), tm = tile - tn * a.tiles_m;
  const int64_t m0 = (int64_t)tm * 64 * MT, n0 = (int64_t)tn * 256;
  const int first = __builtin_amdgcn_readfirstlane((uint32_t)((uint64_t)a.steps * z / (uint32_t)a.splits));
  const int last = __builtin_amdgcn_readfirstlane((uint32_t)((uint64_t)a.steps * (z + 1) / (uint32_t)a.splits));

  // loads of 1 KB: 16 rows of 64 bytes (NN W: 4 rows of 256), at 32-bit offsets from the tile's first row
  const uint32_t sm0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)sm;
  const uint8_t* bx = a.x.codes + m0 * a.x.ldc;
  const uint8_t* bw = NN ? a.w.codes + n0 : a.w.codes + n0 * a.w.ldc;
  uint32_t ox[MT], ow[4];
  int rw[4];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int r = 16 * (MT * wave + i) + (lane >> 2);
    ox[i] = (uint32_t)min((int64_t)r, a.x.rows - 1 - m0) * (uint32_t)a.x.ldc + 16 * ((lane & 3) ^ (r >> 2 & 3));
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (!NN) {
      const int r = 16 * (4 * wave + i) + (lane >> 2);
      ow[i] = (uint32_t)min((int64_t)r, a.w.rows - 1 - n0) * (uint32_t)a.w.ldc + 16 * ((lane & 3) ^ (r >> 2 & 3));
    } else {
      rw[i] = 4 * (4 * wave + i) + (lane >> 4);
      ow[i] = (uint32_t)min((int64_t)16 * ((lane & 15) ^ (rw[i] & 7)), 128 * (int64_t)a.w.steps - 16 - n0);
    }
  }
  // four steps' scales of 64 rows a load; NN: of this wave's 128 columns, four steps are four rows of scales
  const int is = min(wave, MT - 1);
  const uint32_t osx = (uint32_t)(min(m0 + 64 * is + lane, a.x.rows - 1) >> a.x.shift) * (uint32_t)a.x.lds;
  const int kb = (int)min((n0 + 128 * wn) >> 7, (int64_t)a.w.steps - 1);
  const uint32_t osw = NN ? (uint32_t)(kb & ~3) : (uint32_t)(min(n0 + 64 * wave + lane, a.w.rows - 1) >> a.w.shift) * (uint32_t)a.w.lds;
  const int blocks = (int)((a.w.rows + 127) >> 7);

  // load i of half step u (u counts from the contraction's start)
  const auto issue = [&](int u, int buf, int i) {
    const uint32_t st = sm0 + buf * kStage;
    if (i < MT) {
      ld_to_lds8<16, NN>(bx + 64 * (int64_t)u, ox[i < MT ? i : 0], st + 1024 * (MT * wave + i));
    } else {
      const int k = (i - MT) & 3;
      const uint32_t to = st + kX + 1024 * (4 * wave + k);
      if constexpr (!NN) {
        ld_to_lds8<16, NN>(bw + 64 * (int64_t)u, ow[k], to);
      } else {  // rows past W's last: that one (their x is zero)
        const uint32_t end = (uint32_t)a.w.rows - 1, r0 = min(64u * (uint32_t)u, end);
        ld_to_lds8<16, NN>(bw + (int64_t)r0 * a.w.ldc, min((uint32_t)rw[k], end - r0) * (uint32_t)a.w.ldc + ow[k], to);
      }
    }
  };
  const auto issue_scales = [&](int group) {
    const uint32_t sc = sm0 + T::kRing + (group & 1) * T::kScales;
    const int gr = min(group, (a.steps - 1) >> 2);
    ld_to_lds8<4, NN>(a.x.scales + 4 * gr, osx, sc + 256 * is);
    if constexpr (!NN) ld_to_lds8<4, NN>(a.w.scales + 4 * gr, osw, sc + 1024 + 256 * wave);
    else ld_to_lds8<4, NN>(a.w.scales, (uint32_t)min(4 * gr + (lane & 3), blocks - 1) * (uint32_t)a.w.lds + osw, sc + 1024 + 256 * wave);
  };

  Frag fx[2][MT], fw[2][4];
  uint32_t sx[MT], sw[4];
  const auto read_x = [&](int set, int buf, int i, int q) {
    const int r = 32 * MT * wm + 32 * i + c;
    fx[set][i].v[q] = ld16(sm + buf * kStage + 64 * r + 16 * ((2 * h + q) ^ (r >> 2 & 3)));
  };
  const auto read_w = [&](int set, int buf, int t, int q) {
    const char* st = sm + buf * kStage + kX;
    if constexpr (!NN) {
      const int r = 128 * wn + 32 * t + c;
      fw[set][t].v[q] = ld16(st + 64 * r + 16 * ((2 * h + q) ^ (r >> 2 & 3)));
    } else {
      const int r = 32 * h + 16 * q + (lane >> 1 & 7), piece = 8 * wn + 2 * t + (lane >> 4 & 1);
      typedef int i32x2 __attribute__((ext_vector_type(2)));
      const auto p = (__attribute__((address_space(3))) i32x2*)(st + 256 * r + 16 * (piece ^ (r & 7)) + 8 * (lane & 1));
      const i32x2 lo = __builtin_amdgcn_ds_read_tr8_b64_v2i32(p), hi = __builtin_amdgcn_ds_read_tr8_b64_v2i32(p + 8 * 32);
      fw[set][t].v[q] = u32x4{(uint32_t)lo[0], (uint32_t)lo[1], (uint32_t)hi[0], (uint32_t)hi[1]};
    }
  };
  const auto read_scales = [&](int step) {
    const char* sc = sm + T::kRing + (step >> 2 & 1) * T::kScales;
    const int sh = 8 * (step & 3);
#pragma unroll
    for (int i = 0; i < MT; ++i) sx[i] = ld4(sc + 4 * (32 * MT * wm + 32 * i + c)) >> sh;
    if constexpr (!NN) {
#pragma unroll
      for (int t = 0; t < 4; ++t) sw[t] = ld4(sc + 1024 + 4 * (128 * wn + 32 * t + c)) >> sh;
    } else {
      sw[0] = ld4(sc + 1024 + 256 * wave + 4 * (step & 3)) >> (8 * (kb & 3));
    }
  };

  f32x16 acc[MT][4];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int v = 0; v < 16; ++v) acc[i][t][v] = 0.f;

  issue_scales(first >> 2);
  issue_scales((first >> 2) + 1);
  const int end = 2 * last - 1;
#pragma unroll
  for (int d = 0; d < 4; ++d)
#pragma unroll
    for (int i = 0; i < kLoads; ++i) issue(min(2 * first + d, end), d, i);
  __builtin_amdgcn_s_waitcnt(vmcnt_imm(3 * kLoads));
  lds_meet();
#pragma unroll
  for (int q = 0; q < 2; ++q) {
#pragma unroll
    for (int i = 0; i < MT; ++i) read_x(0, 0, i, q);
#pragma unroll
    for (int t = 0; t < 4; ++t) read_w(0, 0, t, q);
  }
  read_scales(first);
  int buf = 0;
  for (int step = first; step < last; ++step) {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      // the next half step's loads are in, not those of the two after it, and every wave has read all of this one's buffer
      __builtin_amdgcn_s_waitcnt(vmcnt_imm(2 * kLoads));
      lds_meet();
      const int u = 2 * step + q, next = (buf + 1) & 3;
      if (q == 0 && (step & 3) == 0 && step > first) issue_scales((step >> 2) + 1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int m = 0; m < 4 * MT; ++m) {
        const int i = m >> 2, t = m & 3;
        acc[i][t] = mfma8_32(fw[q][t], fx[q][i], acc[i][t], sw[NN ? 0 : t], sx[i]);
        __builtin_amdgcn_sched_barrier(0);
        constexpr int kPieces = 2 * (MT + 4), kPer = (kPieces + 4 * MT - 1) / (4 * MT);
#pragma unroll
        for (int p = kPer * m; p < kPer * (m + 1); ++p) {
          if (p < 8) read_w(1 - q, next, p >> 1, p & 1);
          else if (p < kPieces) read_x(1 - q, next, (p - 8) >> 1, p & 1);
        }
        constexpr int kGap = 4 * MT / kLoads > 0 ? 4 * MT / kLoads : 1, kEach = (kLoads + 4 * MT - 1) / (4 * MT);
        if (m % kGap == kGap - 1) {
#pragma unroll
          for (int i2 = kEach * (m / kGap); i2 < kEach * (m / kGap + 1); ++i2)
            if (i2 < kLoads) issue(min(u + 4, end), buf, i2);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      if (q == 1) read_scales(min(step + 1, last - 1));
      buf = next;
    }
  }
  __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));  // the last loads write LDS
  lds_meet();

  // Out through LDS, 32 rows of the wave's 128 columns at a time: a lane has four neighbouring columns of one row, and leaves
  // with 16 bytes beside its neighbours'.
  constexpr int ES = Elem<OT>::kBytes, kPitch = 128 * ES + 16, kWide = 16 / ES, kPer = 128 / kWide;
  char* mine = sm + wave * 32 * kPitch;
  char* out = (char*)a.out + (a.splits > 1 ? (int64_t)z * a.x.rows * a.ldo * 4 : 0);
  const int64_t n = n0 + 128 * wn + kWide * (lane % kPer);
  const int valid = (int)min((int64_t)kWide, a.cols - n);
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int64_t m = m0 + 32 * MT * wm + 32 * i + lane / kPer;
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int t = 0; t < 4; ++t) asm volatile("" : "+a"(acc[i][t]));  // not read before: no registers for all of them
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const f32x4 s = {acc[i][t][4 * v], acc[i][t][4 * v + 1], acc[i][t][4 * v + 2], acc[i][t][4 * v + 3]};
        char* to = mine + c * kPitch + ES * (32 * t + 8 * v + 4 * h);
        if constexpr (OT == kF32) st16(to, __builtin_bit_cast(u32x4, s));
        else st8(to, u32x2{pack16(s[0], s[1], OT), pack16(s[2], s[3], OT)});
      }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll 1
    for (int r = 0; r < 32; r += 64 / kPer) {
      Out16<OT> o{ld16(mine + (r + lane / kPer) * kPitch + 16 * (lane % kPer))};
      if (m + r < a.x.rows) o.store(out + ((m + r) * a.ldo + n) * ES, valid);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }
}

// out[rows, cols] = the splits' sums, in their order; 4 columns a thread.
__global__ __launch_bounds__(256) void k_fp8_join(const float* part, int splits, int64_t rows, int64_t cols, int64_t ldp,
                                                  void* out, int64_t ldo, int odt) {
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
    for (int k = 0; k < 4; ++k) {
      if (n + k >= cols) break;
      if (odt == kF32) reinterpret_cast<float*>(out)[m * ldo + n + k] = s[k];
      else reinterpret_cast<uint16_t*>(out)[m * ldo + n + k] = bits16(s[k], odt);
    }
  }
}

struct Plan8 {
  int mt;  // 64 mt rows a workgroup; 0: the few-row kernel
  int64_t tiles_m, tiles_n;
  int splits, steps;
};

static constexpr int kTokenRows = 64;

// The tile's height and how often the contraction is split over workgroups, by the rounds of workgroups that the grid takes.
static Plan8 plan8(const lrq_fp8* a, const lrq_fp8* b, bool nn) {
  constexpr double kStep[3] = {0.45, 0.6, 1.0}, kFixed = 6.0, kJoin = 4.0, kPerByte = 2.0 / 4.0e6;
  const int64_t rows = a->rows, cols = nn ? b->cols : b->rows;
  const int steps = (int)((a->cols + 127) / 128);
  if (!nn && rows <= kTokenRows) return Plan8{0, 0, 0, 1, steps};
  Plan8 best{};
  double least = 0.;
  for (int i = 0; i < 3; ++i) {
    Plan8 p{1 << i, 0, (cols + 255) / 256, 1, steps};
    p.tiles_m = (rows + 64 * p.mt - 1) / (64 * p.mt);
    for (; p.splits <= 16 && p.splits <= std::max(1, steps / 4); ++p.splits) {
      const double rounds = (double)((p.tiles_m * p.tiles_n * p.splits + 255) / 256);
      const double cost = rounds * ((steps + p.splits - 1) / p.splits * kStep[i] + kFixed) +
                          (p.splits > 1 ? kJoin + kPerByte * 4. * p.splits * rows * cols : 0.);
      if (best.mt == 0 || cost < least) best = p, least = cost;
    }
  }
  return best;
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
    if (t->ld_codes >= 1 << 24 || (tall > 0 && t->ld_scales > UINT32_MAX / tall)) return LRQ_ERR_SHAPE;
  }
  return nn && b->block != 128 ? LRQ_ERR_UNSUPPORTED : LRQ_OK;
}

template <int XT, int TM>
static int token(const TokenArgs& a, hipStream_t s) {
  const int64_t tiles = (a.w.rows + 15) / 16;
  constexpr int D = XT == kX8 ? (TM == 4 ? 1 : 2) : 2;
  // one tile of W a workgroup where that fills the CUs no more than twice
  if (tiles > 1024) return launch((k_fp8_token<XT, TM, 2, 4, D>), dim3((unsigned)((tiles + 1) / 2)), dim3(256), 0, s, a);
  return launch((k_fp8_token<XT, TM, 1, 8, D>), dim3((unsigned)tiles), dim3(512), 0, s, a);
}

static int fp8_product(const lrq_fp8* ta, const lrq_fp8* tb, bool nn, void* out, int64_t ldo, int32_t odt, void* workspace,
                       int64_t workspace_bytes, hipStream_t s) {
  LRQ_TRY(validate_pair(ta, tb, nn));
  const int64_t rows = ta->rows, cols = nn ? tb->cols : tb->rows;
  if (rows == 0 || cols == 0) return LRQ_OK;
  LRQ_TRY(validate_out8(out, ldo, cols, odt));
  const Plan8 p = plan8(ta, tb, nn);
  const Fp8 x = make_fp8(ta), w = make_fp8(tb);
  if (p.mt == 0) {
    const TokenArgs a{(const char*)x.codes, x.ldc, x.scales, x.lds, x.shift, (int)rows, w, out, ldo, odt};
    return rows <= 16 ? token<kX8, 1>(a, s) : rows <= 32 ? token<kX8, 2>(a, s) : token<kX8, 4>(a, s);
  }
  const int64_t need = parts_bytes(p.splits, rows, cols), ldp = (cols + 3) / 4 * 4;
  if (need > 0) {
    if (workspace == nullptr) return LRQ_ERR_NULL;
    if (!aligned(workspace, 16)) return LRQ_ERR_ALIGN;
    if (workspace_bytes < need) return LRQ_ERR_WORKSPACE;
  }
  const int64_t wgs = p.tiles_m * p.tiles_n * p.splits;
  if (wgs > INT32_MAX) return LRQ_ERR_SHAPE;
  const Tile8Args a{x, w, need ? workspace : out, need ? ldp : ldo, cols, need ? (int)kF32 : odt, (int)p.tiles_m, (int)p.tiles_n,
                    p.splits, p.steps};
  const auto go = [&](auto kern, int lds) {
    const hipError_t e = hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (e != hipSuccess) return (int)e;
    return launch(kern, dim3((unsigned)wgs), dim3(256), (size_t)lds, s, a);
  };
  const auto with = [&](auto mt) {
    const auto typed = [&](auto ot) {
      return nn ? go(k_fp8_tile<true, mt(), ot()>, Tile8Lds<true, mt()>::kBytes)
                : go(k_fp8_tile<false, mt(), ot()>, Tile8Lds<false, mt()>::kBytes);
    };
    if (a.odt == kBf16) return typed(std::integral_constant<int, kBf16>{});
    return a.odt == kF16 ? typed(std::integral_constant<int, kF16>{}) : typed(std::integral_constant<int, kF32>{});
  };
  if (p.mt == 4) LRQ_TRY(with(std::integral_constant<int, 4>{}));
  else if (p.mt == 2) LRQ_TRY(with(std::integral_constant<int, 2>{}));
  else LRQ_TRY(with(std::integral_constant<int, 1>{}));
  if (need == 0) return LRQ_OK;
  const dim3 grid((unsigned)std::min<int64_t>((rows * (ldp / 4) + 255) / 256, (int64_t)cu_count() * 32));
  return launch(k_fp8_join, grid, dim3(256), 0, s, (const float*)workspace, p.splits, rows, cols, ldp, out, ldo, odt);
}

}  // namespace lrq

using namespace lrq;

extern "C" int64_t lrq_fp8_gemm_workspace(const lrq_fp8* a, const lrq_fp8* b, int32_t nn) {
  LRQ_TRY(validate_pair(a, b, nn != 0));
  const Plan8 p = plan8(a, b, nn != 0);
  return parts_bytes(p.splits, a->rows, nn ? b->cols : b->rows);
}

extern "C" int lrq_fp8_gemm(const lrq_fp8* a, const lrq_fp8* b, void* out, int64_t ldo, int32_t out_dtype, void* workspace,
                            int64_t workspace_bytes, void* stream) {
  return fp8_product(a, b, false, out, ldo, out_dtype, workspace, workspace_bytes, (hipStream_t)stream);
}

extern "C" int lrq_fp8_gemm_nn(const lrq_fp8* a, const lrq_fp8* b, void* out, int64_t ldo, int32_t out_dtype,
                               void* workspace, int64_t workspace_bytes, void* stream) {
  return fp8_product(a, b, true, out, ldo, out_dtype, workspace, workspace_bytes, (hipStream_t)stream);
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
  const TokenArgs a{(const char*)x, 2 * ldx, nullptr, 0, 0, (int)rows, make_fp8(t), out, ldo, out_dtype};
  hipStream_t s = (hipStream_t)stream;
  return dtype == LRQ_BF16 ? token<kBf16, 1>(a, s) : token<kF16, 1>(a, s);
}
