// Host driver for the lines of the tiling rule with weights in 4 bits
// (rows8_rule.h): reads "line rows copies N K cus" lines, line 0 NT of 8-bit
// rows, 1 FC1, 2 NT of 4-bit rows, K in columns, and prints the tile height
// taken for each (384: 256 and 128).  Built and run by tests/test_rows4.py with the host compiler.
#include <cstdio>

#include "rows8_rule.h"

int main() {
  int line;
  long long rows, copies, N, K, cus;
  while (std::scanf("%d %lld %lld %lld %lld %lld", &line, &rows, &copies, &N, &K, &cus) == 6)
    std::printf("%d\n", line < 2 && pmx::rows8_rests_apart(pmx::kRows8x4Lines[line], rows, copies, N, K, cus) ? 384
                        : line < 2 ? pmx::rows8_tiling(pmx::kRows8x4Lines[line], rows, copies, N, K, cus)
                                 : pmx::rows8_tiling(pmx::kRows4x4Lines[0], rows, copies, N, K / 2, cus));
  return 0;
}
