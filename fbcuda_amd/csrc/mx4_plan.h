// Which kernel a product with 4-bit rows takes (mx4.hip).  Arithmetic only, which a host compiler runs, too.
#pragma once

#include "linear_step.h"

#include <algorithm>
#include <cstddef>

namespace fbfft_amd {
namespace {

// The kernel of a product: its tile, or its fragments of x and w, and the ranges that k is cut into.
struct Mx4Plan {
  enum Kind { Way, Few, Tiles };
  int kind, rows, cols;  // Way, Few: RB and NB; Tiles: of a tile
  long ranges, range;    // blocks
};

constexpr size_t kWayMost = 64 << 10;  // of LDS, for x that a workgroup quantises
// of x in LDS: rows of codes 16 bytes apart, and their scales
inline size_t fewBytes(long M, long blocks) { return std::min(M, 16l) * 17 * (blocks + 1); }

// The kernel with the least expected time, in us.  Few rows: a base, for each block of k and workgroup the numbers below in ns,
// but no less than 230 workgroups' (fewer leave compute units idle), and as much again for the results of every workgroup after
// those.  Tiles: a base, and for each round of workgroups its steps of eight blocks and its results.  (`way`: whether the
// workgroups may quantise x, which rows one by one are read for: 0.07 ns of a block at one row, 0.144 at 16.)
// Measured on rows from 1 to 6476 and weights of 256 x 256 to 32000 x 4096, each kernel with each number of ranges, x quantised
// by the workgroups or in front: 1 x 2048 x 8192 5.5 us on the way and 7.2 in two launches, 128 x 1151 x 1000 6.0 and 7.0,
// tiles 11.6; 32 x 8192 x 8192 21.8 and tiles in four ranges 19.6; 8192 x 8192 x 8192 in tiles of 256 282, of 128 377.
// x quantised already: 64 x 4096 x 4096 9.8 by few rows, 13.0 in tiles; 256 x 1152 x 4608 10.0 and 7.9; 6476 x 96 x 4576, most
// of it results, 70 and 24.
inline Mx4Plan planOf(long M, long blocks, long N, bool way, int units) {
  if (blocks == 0) return {Mx4Plan::Few, 1, 1, 1, 0};
  Mx4Plan best{};
  double least = 0;
  auto offer = [&](const Mx4Plan& plan, double time) {
    if (least == 0 || time < least) least = time, best = plan;
  };
  const double x = (double)std::min(M, 16l);
  auto few = [&](int kind, int rows, int cols, double base, double each, double results) {
    const double groups = (double)ceilDivLong(M, 16 * rows) * ceilDivLong(N, 16 * cols), many = std::max(groups, 230.0);
    offer({kind, rows, cols, 1, blocks}, base + (many * blocks * each + (many - 230) * results * x / 16) / 1e3);
  };
  if (way && fewBytes(M, blocks) <= kWayMost) {
    few(Mx4Plan::Way, 1, 1, 3.3, 0.068 + 0.0047 * x, 0.6);
    few(Mx4Plan::Way, 1, 2, 3.3, 0.15 + 0.0046 * x, 1.5);
  }
  static const double each[3][2] = {{0.106, 0.157}, {0.157, 0.226}, {0.32, 0.42}}, results[3][2] = {{0.6, 1.5}, {0.8, 3.5}, {1.4, 10.8}};
  for (int r = 0; r < 3; ++r)
    for (int c = 0; c < 2; ++c) few(Mx4Plan::Few, 1 << r, 1 << c, 5.7, each[r][c], results[r][c]);
  struct Option {
    int side, together;  // together: workgroups that share a compute unit
    double alone, last, shared, results;  // 256 k and the results: of a lone workgroup, of one among many
  };
  static const Option options[] = {{128, 2, 0.9, 2, 1.34, 4.4}, {256, 1, 1.9, 4.9, 1.9, 8}};
  for (const Option& a : options) {
    const long tiles = ceilDivLong(M, a.side) * ceilDivLong(N, a.side);
    for (long ranges = 1; ranges <= 32; ranges *= 2) {
      const long range = ceilDivLong(ceilDivLong(blocks, ranges), 8) * 8, used = ceilDivLong(blocks, range);
      if (ranges > 1 && range < 16) break;
      const long groups = tiles * used, slots = (long)units * a.together;
      const bool lone = groups <= units;
      const double rounds = groups <= slots ? 1.0 : std::max((double)groups / slots, groups < 4 * slots ? (double)ceilDivLong(groups, slots) : 1.0);
      double time = 6.5 + rounds * (range / 8 * (lone ? a.alone : a.shared) + (lone ? a.last : a.results));
      if (used > 1) time += 2.5 + (double)M * N * used * 4 / 4e6;
      offer({Mx4Plan::Tiles, a.side, a.side, used, range}, time);
    }
  }
  return best;
}

}  // namespace
}  // namespace fbfft_amd
