// Which tiles a grouped GEMM over 8-bit rows runs on.
//
// The host knows the rows and the copies, not the counts.  Four tilings:
//   32 x 64, two waves per block, three blocks per CU: where they are all there at
//     once (one token), and for copies with few rows where their rounds are shorter
//     (8 tokens, 8 each, through 160 copies of 1536 x 2048 and back: 75 -> 70 us);
//   32 x 256, one block per CU, three stages: copies with few rows otherwise, where
//     the call reads every copy's weights once and the matrix cores idle;
//   128 x 128, two blocks per CU: one block's epilogue, tile switch and loads run
//     behind the other's products;
//   256 x 256, one block per CU: half the operand bytes per product.
// Measured (us, 32 x 64 / 32 x 256 / 128 / 256; log-normal counts with sigma 0.4; N x K):
//   copies rows   N     K     NT                       fc1 (N = 2 I)
//   16     1      7168  2048   10.8/ 14.0/ 14.9/ 27.7   14.4/ 17.1/ 20.8/ 47.2
//   8      256    1536  2048   11.9/ 13.9/ 15.2/ 27.9   17.3/ 17.9/ 21.6/ 48.3
//   160    640    1536  2048    89 /  90 /  97 / 111     92 /  92 / 117 / 187
//   16     256    4096  7168    92 /  84 /  86 /  95     96 /  85 /  96 / 156
//   160    2560   1536  2048   100 /  94 / 100 / 113    102 /  94 / 120 / 190
//   160    5120   1536  2048   114 / 106 / 102 / 115    124 / 111 / 124 / 193
//   160    41k    1536  2048   424 / 373 / 204 / 186    589 / 459 / 284 / 299
//   160    96k    1536  2048     -    -  / 420 / 341      -    -  / 624 / 549
//   16     16k    4096  7168     -    -  / 524 / 468      -    -  / 826 / 822
// Between the 32-row tilings the rounds of tiles decide, each at the rows of A
// and B that it reads: a copy's rows are read again for every tile across N.
// Past the few-rows line a round costs its K-tiles
// and a fixed part (epilogue and tile switch), both fitted to such calls.  Over
// 239 calls of each kind (8 to 256 copies, 0.1 to 2000 rows per copy, 12 layers)
// the choice takes 1.015 (NT) and 1.011 (fc1) of the best tiling's time in geometric
// mean, 1.33 at worst (a row each for 96 copies of 1040 x 528: 14.9 us for 11.2).
//
// A result's bits do not depend on the choice: every tiling adds up K in the same
// steps.
//
// Plain C++, so that the rule is unit-tested on the host.
#pragma once

#include <stdint.h>

namespace pmx {

// Rows per copy (with rows) up to which the 32-row tiles run: NT, FC1.
constexpr int64_t kRows8Few[2] = {16, 32};
// A round's cost in us: per K-tile of 128, and beside them.
constexpr double kRows8Round128[2][2] = {{1.25, 2.0}, {1.7, 2.0}};
constexpr double kRows8Round256[2][2] = {{1.5, 5.0}, {2.7, 8.0}};

// The m-tile height, 32 (0: 32 x 64 tiles), 128 or 256, for `rows` rows over `copies` copies, N rows of a
// copy's B (fc1: 2 I), K deep, on `cus` CUs.  kind: 0 NT, 1 FC1.
inline int rows8_tiling(int kind, int64_t rows, int64_t copies, int64_t N, int64_t K, int64_t cus) {
  const auto div_up = [](int64_t a, int64_t b) { return (a + b - 1) / b; };
  const int64_t active = rows < copies ? rows : copies, nk = div_up(K, 128);
  const int64_t mtiles = active > rows / 32 + active / 2 ? active : rows / 32 + active / 2;
  if (mtiles * div_up(N, 64) <= 3 * cus) return 0;
  // a round reads, per CU, 3 x 64 rows of B or 256, and with each tile a copy's rows of A, rows / active
  if (rows <= kRows8Few[kind] * active)
    return div_up(mtiles * div_up(N, 64), 3 * cus) * 3 * (64 * active + rows) <
                   div_up(mtiles * div_up(N, 256), cus) * (256 * active + rows)
               ? 0 : 32;
  // a copy's last tile half full on average; an eighth of the copies past their first tile
  const auto cost = [&](int64_t tile, int64_t blocks, const double (&round)[2]) {
    const int64_t spread = active + active / 8, even = rows / tile + active / 2;
    const int64_t rounds = div_up((spread > even ? spread : even) * div_up(N, tile), blocks);
    return (double)rounds * (round[0] * (double)nk + round[1]);
  };
  return cost(256, cus, kRows8Round256[kind]) < cost(128, 2 * cus, kRows8Round128[kind]) ? 256 : 128;
}

}  // namespace pmx
