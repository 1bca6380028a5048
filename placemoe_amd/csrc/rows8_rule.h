// Which tiles a grouped GEMM over 8-bit rows runs on.
//
// The host knows the rows and the copies, not the counts.  Four tilings:
//   32 x 64, a wave per block, three blocks per CU: so few tiles that wider ones
//     would leave CUs idle (one token);
//   32 x 256, one block per CU, three stages: copies with few rows, where the
//     call reads every copy's weights once and the matrix cores idle;
//   128 x 128, two blocks per CU: one block's epilogue, tile switch and loads run
//     behind the other's products;
//   256 x 256, one block per CU: half the operand bytes per product.
// Measured (us, 32 / 128 / 256; log-normal counts with sigma 0.4; N x K):
//   copies rows   N     K     NT                 fc1 (N = 2 I)
//   160    4      1536  2048   92 /  98 / 119     95 / 119 / 196
//   160    32     1536  2048  107 / 103 / 120    114 / 125 / 193
//   160    64     1536  2048  148 / 108 / 121    171 / 131 / 205
//   160    256    1536  2048  397 / 210 / 197    501 / 299 / 330
//   160    600    1536  2048  857 / 435 / 361   1146 / 653 / 606
//   16     400    7168  2048  254 / 114 / 119    346 / 195 / 212
//   16     2000   4096  7168    - /1069 / 868      - /1722 /1502
//   12     192    1000  1104   20 /  13 /  21      -
// 32 x 64 against 32 x 256 (weights not in a cache; NT, fc1): 8 rows over 160 copies of
// 1536 x 2048 20 / 23, 22 / 26; 64 over 128 63 / 70, 65 / 74; 768 over 160 149 / 152,
// 152 / 152; 2400 over 160 163 / 153, 166 / 154.
// Past the few-rows line the rounds of tiles decide: a round costs its K-tiles
// and a fixed part (epilogue and tile switch), both fitted to such calls.  Over
// 150 calls (8 to 256 copies, 0.1 to 2000 rows per copy, 10 layers) the choice takes
// 1.02 of the best tiling's time in geometric mean, 1.33 at worst (a copy whose count
// straddles a tile's height).
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
constexpr double kRows8Round128[2][2] = {{1.25, 2.0}, {1.9, 2.5}};
constexpr double kRows8Round256[2][2] = {{1.7, 6.0}, {2.9, 10.0}};

// The m-tile height, 32 (0: 32 x 64 tiles), 128 or 256, for `rows` rows over `copies` copies, N rows of a
// copy's B (fc1: 2 I), K deep, on `cus` CUs.  kind: 0 NT, 1 FC1.
inline int rows8_tiling(int kind, int64_t rows, int64_t copies, int64_t N, int64_t K, int64_t cus) {
  const auto div_up = [](int64_t a, int64_t b) { return (a + b - 1) / b; };
  const int64_t active = rows < copies ? rows : copies, nk = div_up(K, 128);
  if (rows <= kRows8Few[kind] * active) return active * div_up(N, 256) <= 2 * cus ? 0 : 32;
  // a copy's last tile half full on average; an eighth of the copies past their first tile
  const auto cost = [&](int64_t tile, int64_t blocks, const double (&round)[2]) {
    const int64_t spread = active + active / 8, even = rows / tile + active / 2;
    const int64_t rounds = div_up((spread > even ? spread : even) * div_up(N, tile), blocks);
    return (double)rounds * (round[0] * (double)nk + round[1]);
  };
  return cost(256, cus, kRows8Round256[kind]) < cost(128, 2 * cus, kRows8Round128[kind]) ? 256 : 128;
}

}  // namespace pmx
