// Host-side check of what products of 16-bit operands read straight into LDS (fbcuda_amd/csrc/linear_step.h): every
// word of every thread's loads, over ragged rows and k, both layouts, lines with and without gaps, and ranges of k.
//   * a word that is read holds eight elements of the operand, inside its rows and the range of k
//   * every element of the tile's step is read, once, and lies in LDS where the fragments are read from
//   * nothing is read for the steps behind the last one, which are requested, too
// Prints OK and returns 0 when all of it holds.
#include <algorithm>
#include <cstdio>
#include <vector>

#include "../../fbcuda_amd/csrc/linear_step.h"

using namespace fbfft_amd;

static int failures = 0;

template <int ROWS, int DEEP, bool KC>
static void check(long rows, long K, long step, long range) {
  constexpr int THREADS = 512;
  typedef StepWords<ROWS, DEEP, KC, THREADS / 64> S;
  auto fail = [&](const char* what, long row, long k) {
    if (++failures <= 20)
      std::printf("FAIL %s: row %ld k %ld, %s of %ld x %ld, lines %ld apart, tile %d x %d, ranges of %ld\n", what, row, k,
                  KC ? "rows" : "columns", rows, K, step, ROWS, DEEP, range);
  };
  for (long first = 0; first < K; first += range)
    for (long m0 = 0; m0 < rows; m0 += ROWS) {
      const long end = std::min(first + range, K), inside = std::min(rows - m0, (long)ROWS);
      long base = KC ? m0 * step + first : first * step + m0;  // elements
      long left = end - first;
      for (int ahead = 0; ahead < 4; left -= DEEP, base += KC ? DEEP : DEEP * step) {
        if (left <= 0) ++ahead;
        std::vector<char> seen(ROWS * DEEP, 0);
        for (int t = 0; t < THREADS; ++t)
          for (int i = 0; i < S::loads; ++i) {
            const unsigned place = S::placeOf(S::wordOf(t, i, step, inside), (int)left);
            if (place >= (unsigned)kReach) continue;
            const int lds = (t / 64 * S::loads + i) * 1024 + t % 64 * 16;
            for (int j = 0; j < 8; ++j) {
              const long at = base + place / 2 + j, line = at / step, in = at % step;
              const long row = KC ? line : in, k = KC ? in : line;
              if (row >= rows || k >= end) {
                fail("outside the operand", row, k);
                continue;
              }
              const long r = row - m0, q = k - (end - left);
              if (r < 0 || r >= ROWS || q < 0 || q >= DEEP) {
                fail("outside the step", row, k);
                continue;
              }
              if (seen[r * DEEP + q]++) fail("read twice", row, k);
              const int l = (int)(KC ? r : q), e = (int)(KC ? q : r);
              if (lds + 2 * j != l * S::perLine * 16 + S::permuted(l, e / 8) * 16 + e % 8 * 2) fail("elsewhere in LDS", row, k);
            }
          }
        for (long r = 0; r < inside; ++r)
          for (long q = 0; q < std::min(left, (long)DEEP); ++q)
            if (!seen[r * DEEP + q]) fail("left out", m0 + r, end - left + q);
      }
    }
}

template <int ROWS, int DEEP, bool KC>
static void sweep() {
  const long whole[] = {8, 16, 24, 32, 40, 56, 64, 72, 120, 128, 136, 192, 200, 264, 1000};
  const long any[] = {1, 2, 7, 31, 32, 33, 63, 64, 65, 100, 127, 129, 200, 300};
  for (long line : whole)
    for (long other : any)
      for (long gap : {0, 8, 64})
        for (long range : {1L << 20, 2L * DEEP}) {
          const long rows = KC ? other : line, K = KC ? line : other;
          check<ROWS, DEEP, KC>(rows, K, line + gap, range);
        }
}

int main() {
  sweep<256, 64, true>();
  sweep<128, 64, true>();
  sweep<256, 32, true>();
  sweep<128, 32, true>();
  sweep<256, 32, false>();
  sweep<128, 32, false>();
  if (failures) {
    std::printf("%d failures\n", failures);
    return 1;
  }
  std::printf("OK\n");
  return 0;
}
