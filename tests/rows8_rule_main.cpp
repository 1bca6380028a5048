// Host driver for the rule that picks the tiles of a grouped GEMM over 8-bit
// rows (rows8_rule.h): reads "kind rows copies N K cus" lines and prints the
// tile height taken for each.  Built and run by tests/test_rows8.py with the
// host compiler.
#include <cstdio>

#include "rows8_rule.h"

int main() {
  int kind;
  long long rows, copies, N, K, cus;
  while (std::scanf("%d %lld %lld %lld %lld %lld", &kind, &rows, &copies, &N, &K, &cus) == 6)
    std::printf("%d\n", pmx::rows8_tiling(kind, rows, copies, N, K, cus));
  return 0;
}
