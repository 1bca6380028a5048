// Prints what gated_rule.h decides: "tiling kind rows N K", "few T H I N" or "wgrad K M N" per line of input.
#include <cstdio>
#include <cstring>

#include "../placemoe_amd/csrc/gated_rule.h"

int main() {
  char what[16];
  long long a, b, c, d;
  while (std::scanf("%15s %lld %lld %lld %lld", what, &a, &b, &c, &d) == 5) {
    if (!std::strcmp(what, "tiling")) {
      std::printf("%d\n", pmx::gated_tiling((int)a, b, c, d, 256));
    } else if (!std::strcmp(what, "few")) {
      std::printf("%d\n", pmx::gated_few(a, b, c, d, 256) ? 1 : 0);
    } else {
      const pmx::GatedWgrad w = pmx::gated_wgrad(a, b, c, 256);
      std::printf("%d %d %lld\n", w.small ? 1 : 0, w.splits, (long long)pmx::gated_chunk(a, w.splits));
    }
  }
  return 0;
}
