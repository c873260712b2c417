// Dropout and dropout + residual add: out = residual + (kept ? x * 65536 / keep : 0); the numbers are
// those of lrq_dropout.h.  The same call on the output's gradient is dropout's backward pass.
// HBM-bound by its traffic (x, the residual, out); the generator's ten rounds run under it: bf16 [16384, 4096] 45 us
// (6.0 TB/s), with a residual 61 to 64 us (6.3 to 6.6 TB/s); a copy reaches 5.2.
#include "lrq_dropout.h"

#include <algorithm>

namespace lrq {

struct DropArgs {
  const char* x;
  int64_t ldx;
  const char* res;
  int64_t ldr;
  char* out;
  int64_t ldo;
  int64_t rows;
  int n;
  int tpr;  // threads a row step: a power of two, 1 .. 256
  Drop drop;
};

// A workgroup covers 256 / tpr rows at a time; a thread takes kAhead chunks of its row per step, all loaded before the
// first one's numbers are drawn: the generator's rounds (about 35 us of vector work on [16384, 4096]) run under the loads.
static constexpr int kAhead = 4;
template <int DT, bool RES>
__global__ __launch_bounds__(256) void k_dropout(DropArgs a) {
  constexpr int ES = Elem<DT>::kBytes;
  const DropKey key = drop_key(a.drop);
  const int nc = (a.n + 7) / 8;
  const int rpb = 256 / a.tpr, t = threadIdx.x & (a.tpr - 1), g = threadIdx.x / a.tpr;
  for (int64_t row = (int64_t)blockIdx.x * rpb + g; row < a.rows; row += (int64_t)gridDim.x * rpb) {
    const char* x = a.x + row * a.ldx * ES;
    const char* res = a.res + row * a.ldr * ES;
    char* out = a.out + row * a.ldo * ES;
    const bool more = a.n >= 8 && row + 1 < a.rows;
    for (int c0 = blockIdx.y * a.tpr * kAhead + t; c0 < nc; c0 += a.tpr * kAhead * gridDim.y) {
      Chunk<DT> xc[kAhead], rc[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const int64_t c = c0 + k * a.tpr;
        const int size = load_size((int)(a.n - 8 * c), more);
        xc[k] = ld_chunk<DT, true>(x + 8 * c * ES, size);
        if constexpr (RES) rc[k] = ld_chunk<DT, true>(res + 8 * c * ES, size);
      }
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const int64_t c = c0 + k * a.tpr;
        if (c >= nc) break;
        float v[8], r[8];
        widen<DT>(xc[k], v);
        if (a.drop.keep < 65536u) drop_chunk(a.drop, key, (uint64_t)row * nc + c, v);
        if constexpr (RES) {
          widen<DT>(rc[k], r);
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = r[e] + v[e];
        }
        st_chunk<DT>(out + 8 * c * ES, narrow<DT>(v), (int)(a.n - 8 * c));
      }
    }
  }
}

template <int DT>
static int dropout(const DropArgs& a, dim3 grid, hipStream_t s) {
  return a.res != nullptr ? launch((k_dropout<DT, true>), grid, dim3(256), 0, s, a)
                          : launch((k_dropout<DT, false>), grid, dim3(256), 0, s, a);
}

}  // namespace lrq

using namespace lrq;

extern "C" int lrq_dropout_add(const lrq_dropout* drop, const void* x, int64_t ldx, const void* residual,
                               int64_t ld_residual, int32_t dtype, int64_t rows, int64_t n, void* out, int64_t ldo,
                               void* stream) {
  if (drop == nullptr) return LRQ_ERR_NULL;
  if (dtype < LRQ_BF16 || dtype > LRQ_F32) return LRQ_ERR_UNSUPPORTED;
  if (rows < 0 || rows > INT32_MAX || n < 0 || n > INT32_MAX / 2) return LRQ_ERR_SHAPE;
  LRQ_TRY(validate_dropout(drop));
  if (rows == 0 || n == 0) return LRQ_OK;
  if (x == nullptr || out == nullptr) return LRQ_ERR_NULL;
  if (ldx < n || ldo < n || (residual != nullptr && ld_residual < n)) return LRQ_ERR_SHAPE;
  const int es = dtype == LRQ_F32 ? 4 : 2;
  if (!aligned(x, es) || !aligned(residual, es) || !aligned(out, es)) return LRQ_ERR_ALIGN;
  const int nc = (int)((n + 7) / 8);
  int tpr = 1;
  while (tpr < 256 && tpr * kAhead < nc) tpr *= 2;
  const DropArgs a{(const char*)x, ldx, (const char*)residual, ld_residual, (char*)out, ldo, rows, (int)n, tpr,
                   make_drop(drop)};
  const int64_t gx = std::min<int64_t>((rows + 256 / tpr - 1) / (256 / tpr), 1 << 20);
  const dim3 grid((unsigned)gx, (unsigned)std::min<int64_t>((nc + tpr * kAhead - 1) / (tpr * kAhead), 1024));
  hipStream_t s = (hipStream_t)stream;
  switch (dtype) {
    case LRQ_BF16: return dropout<kBf16>(a, grid, s);
    case LRQ_F16: return dropout<kF16>(a, grid, s);
    default: return dropout<kF32>(a, grid, s);
  }
}
