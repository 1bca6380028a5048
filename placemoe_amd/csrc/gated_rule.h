// Which kernels the dense gated block's products run on.
//
// Plain C++, so that the rules are unit-tested on the host.
#pragma once

#include <stdint.h>

namespace pmx {

// Tokens up to which the forward runs on the kernels that give every wave a
// share of the weights' columns (gated_ffn.hip).
constexpr int64_t kGatedFewTokens = 16;

// The m-tile height, 64 (64 x 128 tiles), 128 (128 x 256) or 256 (256 x 256), of a product of `rows` rows, N
// columns (fc1: 2 I) and depth K on `cus` CUs.  kind: 0 fc1, 1 fc2, 2 fc1 dgrad, 3 fc2 dgrad.
inline int gated_tiling(int kind, int64_t rows, int64_t N, int64_t K, int64_t cus) {
  (void)kind, (void)K, (void)cus, (void)N;
  return rows <= 64 ? 64 : 256;
}

// Chunks of the K rows of a weight gradient [M, N] on `cus` CUs: their 256 x 256 tiles fill the chip where one
// gradient's own do not.
inline int32_t gated_splits(int64_t K, int64_t M, int64_t N, int64_t cus) {
  const auto div_up = [](int64_t a, int64_t b) { return (a + b - 1) / b; };
  const int64_t tiles = div_up(M, 256) * div_up(N, 256), nk = div_up(K, 64);
  double best = 0;
  int32_t splits = 1;
  for (int32_t s = 1; s <= 64 && s <= nk; ++s) {
    // us: a K-tile, a tile's epilogue and switch; the chunks' sums are written and read again
    const double cost = (double)div_up(tiles * s, cus) * ((double)div_up(nk, s) * 1.7 + 5.0) +
                        (s > 1 ? 4.0 + (double)s * (double)M * (double)N * 8.0 / 4.0e6 : 0.0);
    if (s == 1 || cost < best) best = cost, splits = s;
  }
  return splits;
}

// Rows of a chunk, whole K-tiles; the number of chunks is what they make.
inline int64_t gated_chunk(int64_t K, int32_t splits) {
  const int64_t nk = (K + 63) / 64;
  return (nk + splits - 1) / splits * 64;
}

}  // namespace pmx
