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
//   16     1      7168  2048   11.5/ 13.7/ 14.7/ 27.5   14.3/ 17.4/ 21.2/ 48.5
//   8      256    1536  2048   11.9/ 14.3/ 15.3/ 28.2   17.7/ 18.2/ 22.3/ 49.7
//   160    640    1536  2048    90 /  90 /  98 / 112     94 /  94 / 119 / 193
//   16     256    4096  7168    93 /  84 /  86 /  95     98 /  85 /  97 / 159
//   160    2560   1536  2048    99 /  93 /  99 / 115    103 /  95 / 122 / 193
//   160    5120   1536  2048   115 / 106 / 102 / 116    125 / 111 / 122 / 199
//   160    41k    1536  2048   424 / 373 / 204 / 186    589 / 459 / 284 / 299
//   160    96k    1536  2048     -    -  / 420 / 341      -    -  / 624 / 549
//   16     16k    4096  7168     -    -  / 524 / 468      -    -  / 826 / 822
// Past the few-rows line the rounds of tiles decide: a round costs its K-tiles
// and a fixed part (epilogue and tile switch), both fitted to such calls.  Over
// 150 calls of each kind (8 to 256 copies, 0.1 to 2000 rows per copy, 10 layers)
// the choice takes 1.015 (NT) and 1.01 (fc1) of the best tiling's time in geometric
// mean, 1.33 at worst (a copy whose count straddles a tile's height).
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
  if ((active > rows / 32 + active / 2 ? active : rows / 32 + active / 2) * div_up(N, 64) <= 3 * cus) return 0;
  // a round of either takes as long as its weights: 3 x 64 rows of B per CU, or 256
  if (rows <= kRows8Few[kind] * active)
    return 3 * div_up(active * div_up(N, 64), 3 * cus) < 4 * div_up(active * div_up(N, 256), cus) ? 0 : 32;
  // a copy's last tile half full on average; an eighth of the copies past their first tile
  const auto cost = [&](int64_t tile, int64_t blocks, const double (&round)[2]) {
    const int64_t spread = active + active / 8, even = rows / tile + active / 2;
    const int64_t rounds = div_up((spread > even ? spread : even) * div_up(N, tile), blocks);
    return (double)rounds * (round[0] * (double)nk + round[1]);
  };
  return cost(256, cus, kRows8Round256[kind]) < cost(128, 2 * cus, kRows8Round128[kind]) ? 256 : 128;
}

}  // namespace pmx
