// Host-side: the kernels that products of given sizes take on 256 compute units (fbcuda_amd/csrc/mx4_plan.h, pair_plan.h).  Reads
// lines of sizes, and writes a line for each:
//   mx4 M K N way     way R C (x quantised by the workgroups) | few R C | tiles SIDE RANGES BLOCKS (of a range)
//   orth BATCH R C    whole BYTES | KIND SIDE RANGES K (of a range) for X X^T, A A and B X
#include <cstdio>
#include <cstring>

#include "../../fbcuda_amd/csrc/mx4_plan.h"
#include "../../fbcuda_amd/csrc/pair_plan.h"

using namespace fbfft_amd;

int main() {
  char what[16];
  long a, b, c;
  while (std::scanf("%15s %ld %ld %ld", what, &a, &b, &c) == 4) {
    if (!std::strcmp(what, "mx4")) {
      int way;
      if (std::scanf("%d", &way) != 1) return 1;
      const Mx4Plan p = planOf(a, ceilDivLong(b, 32), c, way != 0, 256);
      if (p.kind == Mx4Plan::Tiles)
        std::printf("tiles %d %ld %ld\n", p.rows, p.ranges, p.range);
      else
        std::printf("%s %d %d\n", p.kind == Mx4Plan::Way ? "way" : "few", p.rows, p.cols);
    } else {
      const long P = padded(std::min(b, c)), Q = padded(std::max(b, c));
      if (inOneLaunch(P, Q)) {
        std::printf("whole %ld\n", wholeBytes(P, Q));
        continue;
      }
      static const char* const names[] = {"small16", "small32", "deep64", "wide64", "deep128", "wide128", "wide256"};
      const PairPlan plans[] = {planOf(true, a, P, P, Q, 256), planOf(true, a, P, P, P, 256), planOf(false, a, P, Q, P, 256)};
      for (const PairPlan& p : plans) std::printf("%s %d %ld %ld ", names[p.kind], p.side, p.ranges, p.range);
      std::printf("\n");
    }
  }
  return 0;
}
