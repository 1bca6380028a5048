// Rows in 8 bits: what their kernels share.
//
// Blocks of 32 neighbouring columns of a row share a power of two; each value
// is held beside it as an e4m3 float or as an int8.  With `most` the block's
// largest finite magnitude and room = 448 (e4m3's largest) or 127,
//   e    = the smallest integer with most <= room * 2^e, within [-127, 127]; 0 for a block of zeros
//   code = x / 2^e rounded to nearest even
// so nothing saturates, and both the division and, in fp32 and bf16, the value
// code * 2^e that is read back are exact; the rounding to 8 bits is the only
// one.  (The floor of log2(most), as the microscaling formats' usual recipe
// has it, would cut the top eighth of a block's range to 448.)  A code that is
// not finite stands for NaN: e4m3's NaN, -128 for int8; infinities become NaN.
//
// codes:  [.., R, N] one byte each, row-major.
// scales: [.., B, R, 16] with B = ceil(N / 512), byte [b, r, j] = e + 127 of
//   row r's columns 512 b + 32 j .. + 31 (127 past the last column).  The
//   16 bytes of 512 columns lie together and those of neighbouring rows next to
//   each other, so that a GEMM brings in the exponents of four K-tiles of 64
//   rows with one 1 KB load.
#pragma once

#include "common.h"

// Threads of a block of the sum over a token's rows; a block per token.
inline unsigned rows8_sum_threads(int64_t H) {
  const int64_t waves = (H / 8 + 63) / 64;
  return (unsigned)(waves < 4 ? waves : 4) * 64;
}

// Between the sources of the layer, not part of the C ABI.
__attribute__((visibility("hidden"))) int pmx_rows8_layer_check(int64_t T, int32_t K, int64_t H, int64_t I, int32_t C);
// The grouped product as rows of 24-bit floats (below): y_high [M, N] 16 bits, y_low [M, N] 8; N a multiple of 16.
__attribute__((visibility("hidden"))) int pmx_rows8_group_gemm_nt_f24(const void* a, const void* a_scales, const void* b,
                                                                      const void* b_scales, const int32_t* offsets, int32_t G,
                                                                      int64_t M, int64_t N, int64_t K, void* y_high, void* y_low,
                                                                      pmx_stream_t stream);
// out[t] = sum of the rows pos[t, k] of y, in k order, rounded once to bf16 or fp16.
__attribute__((visibility("hidden"))) int pmx_rows8_sum_f24(const void* y_high, const void* y_low, const int32_t* pos, int64_t T,
                                                            int32_t K, int64_t H, bool f16, void* out, pmx_stream_t stream);

namespace {

constexpr int kFmtE4M3 = 0, kFmtInt8 = 1;
constexpr int kScaleBlock = 32, kScaleGroup = 512, kScaleBytes = 16;

// The exponent byte of a block whose largest finite magnitude has the fp32
// bits `most`: 448 = 1.75 * 2^8 and 127 = 1.984375 * 2^6.  (A subnormal fp32
// has exponent field 0 and ends at the lower clamp with the small normals.)
template <int FMT>
__device__ __forceinline__ uint32_t scale_byte(uint32_t most) {
  const int e = (int)(most >> 23);
  const uint32_t m = most & 0x7fffffu;
  const int b = FMT == kFmtE4M3 ? e - 8 + (m > 0x600000u ? 1 : 0) : e - 6 + (m > 0x7e0000u ? 1 : 0);
  return most == 0 ? 127u : (uint32_t)(b < 0 ? 0 : b);
}
// 2^(127 - b), b <= 249 (a block of int8 at the top of bf16): a normal fp32.
__device__ __forceinline__ float inv_scale(uint32_t b) { return __uint_as_float((254u - b) << 23); }
// 2^(b - 127); 2^-127 is subnormal.
__device__ __forceinline__ float scale_of(uint32_t b) { return __uint_as_float(b == 0 ? 0x400000u : b << 23); }

// Four values (already divided by the block's power of two) -> four codes.
template <int FMT>
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d) {
  if constexpr (FMT == kFmtE4M3) {
    // infinities come out as NaN
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
    return (uint32_t)w;
  } else {
    const auto one = [](float v) -> uint32_t {
      return __builtin_fabsf(v) <= 127.0f ? (uint32_t)(int)__builtin_rintf(v) & 0xffu : 0x80u;  // NaN: false
    };
    return one(a) | one(b) << 8 | one(c) << 16 | one(d) << 24;
  }
}

// fc2's rows between the product and the sum over a token's experts: the upper
// 24 bits of an fp32, rounded to nearest, in two planes: sign, exponent and 7
// bits (a truncated bf16), and 8 bits more.  A value is off by at most 2^-16 of
// itself, so that the rounding of the sum is the only one that counts.  bf16
// rows are off by up to 2^-9 of themselves, as much as that rounding (the layer
// was 0.0024 from its definition in 64 bits, with these rows 0.0017); 16-bit
// integers beside a power of two per 32 columns are off by a share of the
// block's largest value (columns beside one 1000 times as loud were 0.013
// off, beside one 8000 times as loud 0.11).
constexpr int kF24 = 24;
struct EltF24 {
  static constexpr int kCode = kF24;
};
// Two values' upper halves, four values' next bytes; `u` holds fp32 bits to which half a step, 0x80, has been added.
__device__ __forceinline__ uint32_t f24_high2(const uint32_t* u) { return __builtin_amdgcn_perm(u[1], u[0], 0x07060302u); }
__device__ __forceinline__ uint32_t f24_low4(const uint32_t* u) {
  const uint32_t lo = __builtin_amdgcn_perm(u[1], u[0], 0x0c0c0501u), hi = __builtin_amdgcn_perm(u[3], u[2], 0x05010c0cu);
  return lo | hi;
}
// Eight values from both planes.
__device__ __forceinline__ void f24_values8(const uint4 high, const uint2 low, float* f) {
  const uint32_t h[4] = {high.x, high.y, high.z, high.w}, l[2] = {low.x, low.y};
  constexpr uint32_t kPick[4] = {0x0504000cu, 0x0706010cu, 0x0504020cu, 0x0706030cu};
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] = __uint_as_float(__builtin_amdgcn_perm(h[j / 2], l[j / 4], kPick[j % 4]));
}

// Four codes -> the values that they stand for beside 2^0 (exact).
template <int FMT>
__device__ __forceinline__ void values4(uint32_t w, float* v) {
  if constexpr (FMT == kFmtE4M3) {
    const f32x2_t lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    v[0] = lo[0], v[1] = lo[1], v[2] = hi[0], v[3] = hi[1];
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c = (int)(w << (24 - 8 * j)) >> 24;
      v[j] = c == -128 ? __uint_as_float(0x7fc00000u) : (float)c;
    }
  }
}

}  // namespace
