// How an 8-bit product is laid over the card: the tile, and the splits of its contraction.  Host code that needs no HIP, so that
// a test can compile it by itself.
#pragma once

#include <stdint.h>

#include <algorithm>

namespace lrq {

struct Plan8 {
  int mt, nb;  // 64 mt rows by 64 nb columns a workgroup; 0: the few-row kernel
  int64_t tiles_m, tiles_n;
  int splits, steps;
};

// Rows that the few-row kernel takes: 16, and up to 32 by a W that is neither tall nor wide, of which no workgroup has much
// to read while it reads X again (from memory, 32 rows by [4096, 4096] 9.9 us against 11.8 in tiles, by [5120, 5120] 14.2 and
// 14.3, but by [4096, 8192] 17.0 and 14.2, by [14336, 4096] 20.1 and 17.5; 16 rows by that 17.3 and 17.4).
static bool few_rows(int64_t rows, int64_t cols, int steps) { return rows <= 16 || (rows <= 32 && steps <= 40 && cols <= 8192); }

// out[rows, cols] with a contraction of `depth` (nn: dy w): the tile and how often the contraction is split over workgroups.
// One workgroup runs on a CU at a time, so a grid takes rounds of its longest split's steps, and every split writes and
// re-reads fp32 parts.  Times in us, fitted to 380 products measured with every tile and split by weights that came from
// memory: a step of each tile; a workgroup's start and end; the share of a full round that a nearly empty one takes, which
// runs at higher clocks; what a step waits longer for W where few rows of tiles share it; the join's launch, and its time
// for each element of a part, longer past what the L2s hold.  The plan taken is within 5 % of the best one in 347 of them
// (1.1 % longer on average).  Small tiles are for what does not fill the card with larger ones: 64 rows by [4096, 4096] 12.5
// us in tiles of 64 x 64, 14.1 of 64 x 128 and 16.2 of 64 x 256, 256 rows 14.7, 16.9 and 20.7 (19.2 of 128 x 128), 1024 rows
// 22.8 of 128 x 128 against 30.9 of 128 x 256; they read their operands from the L2s more often, 8192^3 takes 540 us in
// tiles of 128 x 128.
static Plan8 plan8(int64_t rows, int64_t cols, int64_t depth, bool nn) {
  struct Kind {
    int mt, nb;
    double step, fixed, empty;
  };
  constexpr Kind kKinds[] = {{1, 1, 0.26, 0.9, 0.76}, {1, 2, 0.47, 2.0, 0.58}, {1, 4, 0.71, 3.4, 0.45}, {2, 2, 0.56, 3.1, 0.61},
                             {2, 4, 0.90, 4.8, 0.56}, {3, 4, 1.18, 7.3, 0.52}, {4, 4, 1.36, 10.5, 0.46}};
  constexpr double kHalves = 0.07;  // longer is a step of dy w by 64 columns, which reads half cache lines of W
  constexpr double kAlone = 0.19, kJoin = 3.1, kPart = 0.9e-6, kSpilt = 0.8e-6, kHeld = 4e6;
  constexpr int kCus = 256;  // a fixed count, so that the workspace and the order of the sums depend on the shape alone
  const int steps = (int)((depth + 127) / 128);
  if (!nn && few_rows(rows, cols, steps)) return Plan8{0, 0, 0, 0, 1, steps};
  Plan8 best{};
  double least = 0.;
  for (const Kind& k : kKinds) {
    if (k.mt > 1 && 64 * (k.mt - 1) >= rows) continue;  // part of the tile without a row
    Plan8 p{k.mt, k.nb, (rows + 64 * k.mt - 1) / (64 * k.mt), (cols + 64 * k.nb - 1) / (64 * k.nb), 1, steps};
    for (; p.splits <= 16 && p.splits <= std::max(1, steps / 6); ++p.splits) {
      const int64_t wgs = p.tiles_m * p.tiles_n * p.splits, over = wgs % kCus;
      const double rounds = (double)(wgs / kCus) + (over == 0 ? 0. : k.empty + (1. - k.empty) * (double)over / kCus);
      const int run = std::min(steps, 4 * (((steps + 3) / 4 + p.splits - 1) / p.splits));
      const double sums = (double)p.splits * rows * cols;
      const double step = k.step + kAlone * k.nb / p.tiles_m + (nn && k.nb == 1 ? kHalves : 0.);
      const double cost = rounds * (run * step + k.fixed) +
                          (p.splits > 1 ? kJoin + kPart * sums + kSpilt * std::max(0., sums - kHeld) : 0.);
      if (best.mt == 0 || cost < least) best = p, least = cost;
    }
  }
  return best;
}

}  // namespace lrq
