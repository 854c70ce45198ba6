// How the products with 4-bit weights of many rows are shared out (linear_4bit_tile.cu), and what they take, which the host weighs against the kernel
// for few rows (plain C++: both include it).
#pragma once
#include <cstdint>

namespace castle {

struct TilePlan {
  int bn, ks;   // rows of x in a tile; CTAs of a cluster, which share K out
  double us;
};
// A tile takes some 2.5 us and 0.027 a row of x around its steps of 128 k, a step 0.41 us (the unpacking) or 0.0021 a row of x (the products); a cluster's sum of its
// CTAs' shares 1.5 us and 0.06 for each of a CTA's rows of it.  As many tiles as there are SMs (clusters of 4: 36, of 8: 15) work at a time.  us with one
// CTA a tile / the plan's clusters, bf16, groups of 64: 40 x 4096 -> 4096 16.6 / 9.8, 64 x 4096 -> 4096 17.0 / 10.6, 128 x 4096 -> 4096 16.6 / 13.1, 48 x 16384 -> 512
// 53.5 / 11.8, 100 x 8192 -> 1024 28.3 / 10.8, 500 x 8000 -> 200 30.6 / 10.9, 500 x 8000 -> 1000 32.5 / 18.1; from a tile for every SM on one CTA is the faster:
// 300 x 2048 -> 2048 10.6, with two 11.4, 2000 x 8192 -> 1024 33.3, with two 38.8.
inline TilePlan linear_4bit_tile_plan(int64_t rows, int64_t K, int64_t N) {
  const int64_t steps = (K + 127) / 128, n_tiles = (N + 127) / 128;
  TilePlan best = {256, 1, 0.0};
  for (int ks = 1; ks <= 8 && ks <= steps; ks *= 2) {
    const int64_t at_once = ks == 8 ? 15 : ks == 4 ? 36 : 148 / ks;
    for (int bn = 256; bn >= 32; bn -= 16) {
      const int64_t r_tiles = (rows + bn - 1) / bn, waves = (r_tiles * n_tiles + at_once - 1) / at_once;
      if (r_tiles > 65535) break;
      const double step = 0.0021 * bn > 0.41 ? 0.0021 * bn : 0.41;
      const double us = (double)waves * (2.5 + 0.027 * bn + step * (double)((steps + ks - 1) / ks) + (ks > 1 ? 1.5 + 0.06 * bn / ks : 0.0));
      if (best.us == 0.0 || us < best.us) best = {bn, ks, us};
    }
  }
  return best;
}

}  // namespace castle
