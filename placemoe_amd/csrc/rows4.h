// Rows in 4 bits: what their kernels share.
//
// As rows in 8 bits (rows8.h), with e2m1 values: 0, 0.5, 1, 1.5, 2, 3, 4, 6 and
// a sign.  With `most` a block's largest magnitude,
//   e    = the smallest integer with most < 7 * 2^e, within [-127, 127]; 0 for a block of zeros
//   code = x / 2^e rounded to the nearest value, ties to the even code
// What lies between 6 and 7 rounds to 6 as it would if the values went on (to
// 8), so that nothing is off by more than the rounding's half step: 2^-2 of a
// value, down to 2^e.  (Of random rows the root mean square error is 0.112 of their values,
// with 6 in the place of 7 0.115, and with 8, where the top quarter of the
// range is cut to 6, 0.115.)  The values have no infinity and no NaN: a block
// that holds one takes the exponent byte 255, which stands for NaN in all 32 columns.
//
// codes:  [.., R, ceil(N / 2)], column 2 j in the low half of byte j (the half
//   past an odd row's end: 0).
// scales: as of rows in 8 bits.
#pragma once

#include "rows8.h"

// Between the sources of the layer, not part of the C ABI (as in rows8.h).
__attribute__((visibility("hidden"))) int pmx_rows4_layer_check(int64_t T, int32_t K, int64_t H, int64_t I, int32_t C);
__attribute__((visibility("hidden"))) int pmx_rows4_group_gemm_nt_f24(const void* a, const void* a_scales, const void* b,
                                                                      const void* b_scales, const int32_t* offsets, int32_t G,
                                                                      int64_t M, int64_t N, int64_t K, void* y_high, void* y_low,
                                                                      pmx_stream_t stream);

namespace {

constexpr uint32_t kScaleNaN = 255;

// The exponent byte of a block whose largest magnitude, finite, has the fp32 bits `most`: 7 = 1.75 * 2^2.
__device__ __forceinline__ uint32_t scale_byte4(uint32_t most) {
  const int b = (int)(most >> 23) - 2 + ((most & 0x7fffffu) >= 0x600000u ? 1 : 0);
  return most == 0 ? 127u : (uint32_t)(b < 0 ? 0 : b);
}

}  // namespace
