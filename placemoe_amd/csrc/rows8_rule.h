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
// With weights in 4 bits the lines lie elsewhere: half the weights' bytes, more stages of them on
// their way, and rows in 4 bits at twice the depth per K-tile (K there: A's bytes per row).  Over 183 calls of each
// kind (10 layers, 0.05 to 2000 rows per copy) the choice takes 1.009 (8-bit rows), 1.012 (4-bit rows) and
// 1.007 (fc1) of the best tiling's time, 1.27 at worst (768 rows of 16 copies of 4096 x 7168: 70 us for 55; with
// the lines of 8-bit weights 1.027, 1.015 and 1.010, 1.42 at worst).  us, as above:
//   copies rows   N     K     NT, rows in 8 bits       NT, rows in 4            fc1
//   160    64     1536  2048    20/  23/  26/  50        18/  20/  21/  34        30/  32/  39/  88
//   160    640    1536  2048    45/  44/  58/  95        40/  42/  45/  64        67/  59/ 103/ 170
//   160    1600   1536  2048    46/  46/  60/  95        41/  42/  46/  64        68/  59/ 103/ 171
//   160    5120   1536  2048    67/  62/  64/  97        46/  50/  47/  66        97/  84/ 105/ 172
//   160    20480  1536  2048   192/ 162/ 101/ 115       112/ 104/  64/  81       284/ 228/ 162/ 194
//   160    81920  1536  2048   684/ 559/ 296/ 280       392/ 354/ 192/ 188      1035/ 811/ 516/ 505
//   16     1      4096  7168    20/  26/  30/  70        12/  18/  20/  42        31/  42/  52/ 132
//   16     256    4096  7168    44/  38/  46/  74        39/  38/  39/  46        61/  46/  88/ 139
//   16     16000  4096  7168   996/ 830/ 436/ 409       550/ 490/ 275/ 253      1603/1276/ 820/ 763
//
// A result's bits do not depend on the choice: every tiling adds up K in the same
// steps.
//
// Plain C++, so that the rule is unit-tested on the host.
#pragma once

#include <stdint.h>

namespace pmx {

struct Rows8Lines {
  int64_t few;         // rows per copy (with rows) up to which the 32-row tiles run
  double narrow;       // a 32 x 64 round beside a 32 x 256 one that reads as much
  double round128[2];  // a round's cost in us: per K-tile of 128, and beside them
  double round256[2];
};
// NT, FC1
constexpr Rows8Lines kRows8Lines[2] = {{16, 1.0, {1.25, 2.0}, {1.5, 5.0}}, {32, 1.0, {1.7, 2.0}, {2.7, 8.0}}};
constexpr Rows8Lines kRows8x4Lines[2] = {{24, 1.05, {0.9, 3.0}, {1.5, 5.0}}, {48, 1.05, {0.9, 3.0}, {1.5, 5.0}}};
constexpr Rows8Lines kRows4x4Lines[1] = {{12, 1.0, {1.0, 3.0}, {1.5, 6.0}}};

// A call in tiles of one height: a copy's last tile half full on average; an eighth of the copies past their first tile.
inline double rows8_cost(int64_t tile, int64_t blocks, const double (&round)[2], int64_t rows, int64_t active, int64_t N, int64_t nk) {
  const int64_t spread = active + active / 8, even = rows / tile + active / 2;
  const int64_t tiles = (spread > even ? spread : even) * ((N + tile - 1) / tile);
  return (double)((tiles + blocks - 1) / blocks) * (round[0] * (double)nk + round[1]);
}

// The m-tile height, 32 (0: 32 x 64 tiles), 128 or 256, for `rows` rows over `copies` copies, N rows of a
// copy's B (fc1: 2 I), K deep, on `cus` CUs.
inline int rows8_tiling(const Rows8Lines& line, int64_t rows, int64_t copies, int64_t N, int64_t K, int64_t cus) {
  const auto div_up = [](int64_t a, int64_t b) { return (a + b - 1) / b; };
  const int64_t active = rows < copies ? rows : copies, nk = div_up(K, 128);
  const int64_t mtiles = active > rows / 32 + active / 2 ? active : rows / 32 + active / 2;
  if (mtiles * div_up(N, 64) <= 3 * cus) return 0;
  // a round reads, per CU, 3 x 64 rows of B or 256, and with each tile a copy's rows of A, rows / active
  if (rows <= line.few * active)
    return line.narrow * (double)(div_up(mtiles * div_up(N, 64), 3 * cus) * 3 * (64 * active + rows)) <
                   (double)(div_up(mtiles * div_up(N, 256), cus) * (256 * active + rows))
               ? 0 : 32;
  return rows8_cost(256, cus, line.round256, rows, active, N, nk) < rows8_cost(128, 2 * cus, line.round128, rows, active, N, nk) ? 256 : 128;
}

// Rows in 8 bits with weights in 4, past the few-rows line: whether a copy's rows past its whole 256s, where they are
// 128 or fewer (half of the copies), run on 128-row tiles in a launch of their own, and the other rows on 256-row
// tiles.  That saves half a 256-row tile per copy and costs half a 128-row one, a quarter of a round more for each
// launch's last, and the launch.  Over 110 (NT) and 97 (fc1) calls of 10 layers, 100 to 4000 rows per copy, it takes 30 of
// each, to 0.962 and 0.942 of the better tiling's time, 1.08 at worst; at 160 copies (us, 128 / 256 / so):
//   rows   N     K     NT                 fc1
//   41k    1536  2048  164 / 175 / 152    307 / 294 / 261
//   82k    1536  2048  313 / 284 / 270    536 / 486 / 466
//   82k    2048  768   167 / 172 / 154    313 / 285 / 261
// (Rows in 4 bits gain nothing: 0.87 to 1.07 of the better one's in such calls, 0.99 on average.)
inline bool rows8_rests_apart(const Rows8Lines& line, int64_t rows, int64_t copies, int64_t N, int64_t K, int64_t cus) {
  if (rows < 256 * copies || rows <= line.few * copies) return false;
  const int64_t nk = (K + 127) / 128;
  const auto rounds = [&](double mtiles, int64_t tile, int64_t blocks) { return mtiles * (double)((N + tile - 1) / tile) / (double)blocks + 0.25; };
  const double apart = rounds((double)(rows / 256), 256, cus) * (line.round256[0] * (double)nk + line.round256[1]) +
                       rounds((double)(copies + 1) / 2, 128, 2 * cus) * (line.round128[0] * (double)nk + line.round128[1]) + 12.0;
  return apart < rows8_cost(256, cus, line.round256, rows, copies, N, nk) &&
         apart < rows8_cost(128, 2 * cus, line.round128, rows, copies, N, nk);
}
// With weights in 8 bits; kind: 0 NT, 1 FC1.
inline int rows8_tiling(int kind, int64_t rows, int64_t copies, int64_t N, int64_t K, int64_t cus) {
  return rows8_tiling(kRows8Lines[kind], rows, copies, N, K, cus);
}

}  // namespace pmx
