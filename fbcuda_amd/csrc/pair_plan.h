// Which kernels Newton-Schulz products take (orthogonalize.hip).  Arithmetic only, which a host compiler runs, too.
#pragma once

#include "linear_step.h"

#include <algorithm>
#include <cmath>

namespace fbfft_amd {
namespace {

inline long padded(long n) { return (n + 31) / 32 * 32; }

// ---- small matrices: all steps in one launch ----

constexpr int kWholeSteps = 3;          // of 32 rows of X, at most
constexpr int kWholeLarge = 156 << 10;  // bytes of LDS

inline long wholeBytes(long P, long Q) { return P * (4 * Q + 16) + 2 * P * (4 * P + 16); }
inline bool inOneLaunch(long P, long Q) { return P <= 32 * kWholeSteps && wholeBytes(P, Q) <= kWholeLarge; }

// ---- products ----

// The kernel of a product, and the ranges that its k is cut into.
enum PairKind { Small16, Small32, Deep64, Wide64, Deep128, Wide128, Wide256 };
struct PairPlan {
  int kind, side;  // side: of a tile
  long tiles, ranges, range;
};

// The kernel with the least expected time, in us, from what each takes for a step of 32 k: `alone` where workgroups have compute
// units to themselves, else `each` for every one that a compute unit gets (in whole rounds where few fit it), and besides for
// results, more of them where they are left both ways round.  Ranges add a launch, and their sums' way to memory and back.
// Measured in every kernel on products from 64 x 64 x 64 to 2048 x 8192 x 8192: 1024 x 1024 x 1024 with half of it a mirror
// image: Deep64 11.4, Wide64 18.4, Wide128 28; 2048 x 2048 x 2048 so: Wide64 40, Deep128 42, Wide128 in three ranges 44;
// 2048 x 8192 x 2048: Wide256 167, Wide128 189, Wide64 240; 256 x 256 x 8192: Small32 in one range 58, in eight 17; 256 x 256 x
// 6432: Small32 in nine 20, Deep64 in eight 13.
inline PairPlan planOf(bool symmetric, long batch, long M, long N, long K, double units) {
  struct Option {
    int kind, side, most;  // most: ranges
    double alone, each;
    bool whole;
    double results;
  };
  static const Option options[] = {
      {Small16, 16, 1, 0.136, 0.148, false, 3}, {Small32, 32, 16, 0.24, 0.42, false, 3}, {Deep64, 64, 8, 0.18, 0.24, true, 4},
      {Wide64, 64, 8, 0.4, 0.25, false, 5},     {Deep128, 128, 8, 0.56, 0.68, true, 6},   {Wide128, 128, 8, 0.62, 0.63, true, 6},
      {Wide256, 256, 8, 1.8, 2.4, true, 10}};
  PairPlan best{};
  double least = 0;
  const long steps = K / 32;
  for (const Option& o : options) {
    const long down = ceilDivLong(M, o.side), across = ceilDivLong(N, o.side);
    const long tiles = symmetric ? down * (down + 1) / 2 : down * across;
    // (B X has at least as many columns as rows, and its k are its rows: where ranges of 256 k could be cut, tiles fill the chip)
    for (long ranges = 1; ranges <= (symmetric ? o.most : 1); ranges += ranges < 4 ? 1 : ranges < 8 ? 2 : 4) {
      const long range = ceilDivLong(steps, ranges), used = ceilDivLong(steps, range);
      if (ranges > 1 && range < 8) break;
      const double share = (double)batch * tiles * used / units, rounds = o.whole && share < 8 ? std::ceil(share) : share;
      double time = o.results + (symmetric ? 0 : 2) + range * (share <= 0.75 ? o.alone : std::max(o.alone, rounds * o.each));
      if (used > 1) time += 4.5 + (double)batch * tiles * used * o.side * o.side * 8 / 4e6;
      if (least == 0 || time < least) {
        least = time;
        best = PairPlan{o.kind, o.side, tiles < 8 ? tiles : (tiles + 7) / 8 * 8, used, 32 * range};
      }
    }
  }
  return best;
}

}  // namespace
}  // namespace fbfft_amd
