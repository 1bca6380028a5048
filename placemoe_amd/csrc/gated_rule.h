// Which kernels the dense gated block's products run on.
//
// Plain C++, so that the rules are unit-tested on the host.
#pragma once

#include <stdint.h>

namespace pmx {

// The products of rows run on 64 x 128 tiles (two blocks per CU), 128 x 256 ones
// or 256 x 256 ones.  A call takes as long as its rounds of tiles, each its K-tiles
// of 64 and a fixed part (epilogue, tile switch), in us; a CU with one 64 x 128
// tile is faster through it than one with two.  Fitted to 105 calls of each kind
// (7 layers from 512 x 264 to 7168 x 2048, 17 to 8192 rows), of which the tiling
// that this rule takes is within 0.3% of the best one's time in geometric mean, 1.20
// at worst.  (Single times lie further from the formula: a round of 256-row tiles of fc2's dgrad over 2048 columns counts as
// 65, and is 80-85 at 8192 rows, 88 at 16384, whose sums are more bytes.)  Measured, operands at hand (64 / 128 / 256):
//   rows   H     I      fc1                fc2                fc1 dgrad          fc2 dgrad
//   256    2048  768     17 /  30 /  52      9 /  15 /  20     14 /  24 /  34     19 /  37 /  72
//   2048   2048  768     27 /  35 /  58     15 /  18 /  29     23 /  27 /  45     22 /  41 /  74
//   8192   2048  768     87 /  70 /  63     49 /  37 /  30     79 /  57 /  48     51 /  46 /  80
//   1024   7168  2048    76 /  91 / 164     50 /  35 /  57     86 /  60 / 105     56 /  92 / 172
//   8192   7168  2048   622 / 410 / 363    308 / 216 / 210    589 / 404 / 392    330 / 243 / 220
struct GatedRound {
  double ktile, fixed;
};
constexpr double kGated64[4][4] = {  // K-tile with two blocks on a CU, with one, fixed, of the call
    {0.63, 0.342, 5.04, 0.2}, {0.645, 0.328, 3.78, 1.6}, {0.624, 0.344, 4.45, 1.0}, {0.662, 0.349, 7.44, 0.0}};
constexpr GatedRound kGated128[4] = {{0.711, 7.44}, {0.636, 7.49}, {0.656, 7.85}, {0.725, 12.4}};
constexpr GatedRound kGated256[4] = {{1.196, 13.8}, {1.056, 9.6}, {1.109, 9.5}, {1.371, 20.9}};
// 256 x 256 tiles whose depth is not a multiple of 64: fc2 and fc1's dgrad, on the kernel whose loads are masked.  (fc1 and
// fc2's dgrad: at 1.45 times the figures above, twice as many 128-row tiles take less at every depth.)
constexpr double kGatedMasked = 1.45;

// The m-tile height of a product of `rows` rows, N columns (fc1: 2 I) and depth K on `cus` CUs.
// kind: 0 fc1, 1 fc2, 2 fc1 dgrad, 3 fc2 dgrad.
struct GatedTiling {
  int height;
  double us;
};
inline GatedTiling gated_fastest(int kind, int64_t rows, int64_t N, int64_t K, int64_t cus) {
  const auto div_up = [](int64_t a, int64_t b) { return (a + b - 1) / b; };
  const double nk = (double)div_up(K, 64);
  const int64_t per_cu = div_up(div_up(rows, 64) * div_up(N, 128), cus);
  const double* c = kGated64[kind];
  const double t64 = ((double)(per_cu / 2) * c[0] + (double)(per_cu % 2) * c[1]) * nk + (double)div_up(per_cu, 2) * c[2] + c[3];
  const auto rounds = [&](int64_t height, const GatedRound& r) {
    return (double)div_up(div_up(rows, height) * div_up(N, 256), cus) * (nk * r.ktile + r.fixed);
  };
  const double t128 = rounds(128, kGated128[kind]), t256 = rounds(256, kGated256[kind]) * (K % 64 ? kGatedMasked : 1.0);
  if (K % 64 && (kind == 0 || kind == 3)) return t64 <= t128 ? GatedTiling{64, t64} : GatedTiling{128, t128};
  if (t64 <= t128 && t64 <= t256) return {64, t64};
  return t128 <= t256 ? GatedTiling{128, t128} : GatedTiling{256, t256};
}
inline int gated_tiling(int kind, int64_t rows, int64_t N, int64_t K, int64_t cus) { return gated_fastest(kind, rows, N, K, cus).height; }

// Whether the forward of T tokens runs on the kernels that give every wave a share of the
// weights' columns (gated_ffn.hip): up to 64 tokens, where reading the weights once, at 4.3 TB/s, and the tokens for each
// 8 columns of act and 16 of out, at 8.4 TB/s from the L2s, takes less than the tiles of rows and the weights' way from
// memory (the times above are of weights at hand; 5 layers, 1 to 64 tokens, weights from memory: 7168 x 2048, 64 tokens
// 66 us for 80; 4096 x 11008, 32 tokens 123 for 129, 48 159 for 135).
inline bool gated_few(int64_t T, int64_t H, int64_t I, int64_t N, int64_t cus) {
  if (T <= 16) return true;  // these keep act in two values (by the figures below within 1% of the faster ones in the largest layers)
  if (T > 64) return false;
  const double weights = 2.0 * ((double)(2 * I) * (double)H + (double)N * (double)I);
  const double tokens = (double)T * ((double)(I / 8) * (double)H + (double)(N / 16) * (double)I) * 2.0;
  return 5.0 + weights / 4.3e6 + tokens / 8.4e6 <=
         gated_fastest(0, T, 2 * I, H, cus).us + gated_fastest(1, T, N, I, cus).us + weights / 5.5e6;
}

// A weight gradient [M, N] over K rows on `cus` CUs: 128 x 128 tiles, or 256 x 256 ones
// over `splits` chunks of the rows, so that they fill the chip where one
// gradient's own do not; the chunks' fp32 sums are then added by a kernel more.
// The small tiles come in two kernels: four blocks per CU that load a K-tile and
// multiply it in turn, or two that load the next one meanwhile, where there are no
// more.  Costs in us fitted to 110 calls of each (512 x 264 to 7168 x 2048, 17 to 16384 rows;
// four blocks / two / 256 x 256 / in chunks and their sum):
//   rows    M     N
//   64      2000  1416     6 /   7 /  12 /   -
//   1531    2000  1416    33 /  24 /  41 /  22 + 13 (5)
//   1024    2816  4096    29 /  36 /  32 /   -
//   16384   1536  2048   294 / 182 / 308 /  89 + 14 (5)
//   16384   2048  768    274 / 183 / 302 /  53 + 14 (10)
//   8192    4096  7168   604 / 599 / 361 /   -
inline bool gated_wgrad_two(int64_t blocks, int64_t K, int64_t cus) { return blocks <= 2 * cus && K > 256; }
struct GatedWgrad {
  bool small;  // 128 x 128 tiles
  int32_t splits;
};
inline GatedWgrad gated_wgrad(int64_t K, int64_t M, int64_t N, int64_t cus) {
  const auto div_up = [](int64_t a, int64_t b) { return (a + b - 1) / b; };
  const int64_t tiles = div_up(M, 256) * div_up(N, 256), nk = div_up(K, 64);
  const int64_t blocks = div_up(M, 128) * div_up(N, 128);
  const double per_cu = (double)div_up(blocks, cus);
  const double ktile = 0.46 * per_cu > 1.03 ? 0.46 * per_cu : 1.03;
  GatedWgrad best = {true, 1};
  double least = gated_wgrad_two(blocks, K, cus) ? (double)nk * 0.72 + 5.0 : (double)nk * ktile + 3.0 + 1.07 * per_cu;
  for (int64_t s = 1; s <= 32 && s <= nk; ++s) {
    const double sums = s > 1 ? (double)s * (double)M * (double)N * 4e-6 : 0.0;  // MB
    const double rounds = (double)div_up(tiles * s, cus);
    const double cost = rounds * ((double)div_up(nk, s) * 1.30 + 1.6) + 7.7 + sums * 0.15 + (s > 1 ? 4.5 + sums / 7.0 : 0.0);
    if (cost < least) least = cost, best = {false, (int32_t)s};
  }
  return best;
}

// Rows of a chunk, whole K-tiles; the number of chunks is what they make.
inline int64_t gated_chunk(int64_t K, int32_t splits) {
  const int64_t nk = (K + 63) / 64;
  return (nk + splits - 1) / splits * 64;
}

}  // namespace pmx
