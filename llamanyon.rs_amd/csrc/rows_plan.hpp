// rows_plan.hpp -- how swamp_gemm_rows_i8 cuts a call into workgroups: which kernel, which
// tiles, how many pieces of the sums.  Host-only arithmetic on sizes, so that it can be checked
// without a GPU.
#pragma once
#include <cstdint>

namespace swamp_rows {

// Which tiles, and in how many pieces the sums: of every choice its time by a model, whose
// numbers are fitted to 148 sizes (48 to 2048 rows of x, 640 to 28672 of w, 512 to 14336
// columns), each measured in up to 25 ways.  A round of tiles costs a tile's filling and
// storing and its steps, a last one that does not fill the CUs 0.73 of that and the rest by
// its share; pieces cost their sums' writing and reading.  The choice is 1.6% slower than the
// fastest on average, 33% at worst (192 x 16384 x 512, 13 us for 10), then 26% (160 rows of
// the same, 65 x 1024 x 1024), 24% (640 x 4096 x 14336, 75 us for 61) and 17%.
struct Tiles {
  int tm, tn;
  double step, fixed;  // us
  int threads;
};
constexpr Tiles kTiles[] = {
    {64, 128, 0.205, 5.9, 256},  {128, 128, 0.24, 9.0, 512}, {256, 128, 0.468, 7.0, 512},
    {128, 256, 0.516, 6.4, 512}, {256, 256, 0.86, 13.6, 512}};
// A launch holds less threads than this.  256 x 256 tiles stay below it for every call of less
// than 2^38 products.
constexpr int64_t kMostThreads = int64_t(1) << 32;

struct Plan {
  int shape;  // of kTiles; -1: few_kernel, of `tiles_n` tiles of 16 rows a workgroup
  int tiles_m, tiles_n, pieces, steps;
};

inline Plan plan_of(int m, int n, int k, int cus) {
  const int KT = (k + 63) / 64;
  Plan best{-1, 1, 1, 1, KT};
  // Up to 64 rows, where one round of few_kernel's workgroups takes all of w: the smallest of
  // them that do (one row of 6144 x 4096: 7.6 us with two tiles of 16 a workgroup, 9.5 with
  // one, 10.6 with four).  The limits are where tiles overtake it, us here and there:
  //   m      n x k          here  tiles        n x k          here  tiles
  //   16     16384 x 4096   16.4  18.4         28672 x 4096   29.5  27.1
  //   16     28672 x 1024    8.6  10.5         28672 x 2048   15.2  15.3
  //   32     8192 x 6144    14.5  18.1         8192 x 8192    21.0  19.3
  //   32     16384 x 2048   10.0  14.1         16384 x 5120   22.3  22.0
  //   64     4096 x 4096    11.9  15.0         4096 x 8192    21.2  17.0
  //   64     8192 x 4096    15.5  16.8         8192 x 6144    21.3  20.1
  const int wide = (n + 15) / 16 <= cus ? 1
                   : (n + 31) / 32 <= cus ? 2
                   : (n + 63) / 64 <= cus || k <= 2048 ? 4 : 0;
  if (wide && (m <= 16 || (n + 63) / 64 <= cus) &&
      (m <= 16 || (m <= 32 && k <= (wide <= 2 ? 8192 : 4096)) ||
       (m <= 64 && wide <= 2 && k <= 4096))) {
    best.tiles_n = wide;
    return best;
  }
  double least = 0;
  for (int i = 0; i < int(sizeof(kTiles) / sizeof(kTiles[0])); i++) {
    const Tiles &t = kTiles[i];
    Plan p;
    p.shape = i;
    p.tiles_m = (m + t.tm - 1) / t.tm;
    p.tiles_n = (n + t.tn - 1) / t.tn;
    const int64_t tiles = int64_t(p.tiles_m) * p.tiles_n;
    if (tiles * t.threads >= kMostThreads) continue;
    for (int pieces = 1; pieces <= 8 && (pieces == 1 || (KT / pieces >= 4 && tiles * pieces <= 3 * cus));
         pieces++) {
      p.steps = ((KT + pieces - 1) / pieces + 1) / 2 * 2;  // whole pairs
      p.pieces = (KT + p.steps - 1) / p.steps;
      const int64_t units = tiles * p.pieces, rem = units % cus;
      const double round = t.fixed + p.steps * t.step;
      double us = double(units / cus) * round;
      if (rem) us += round * (0.73 + 0.27 * double(rem) / cus);
      if (p.pieces > 1) us += 0.9 + p.pieces * (double(m) * n * 8.0 / 3.6e6);
      if (best.shape < 0 || us < least) {
        least = us;
        best = p;
      }
    }
  }
  return best;
}

}  // namespace swamp_rows
