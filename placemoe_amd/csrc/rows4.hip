// Rows in 4 bits (rows4.h): writing them and reading them back.
//
// Both are bound by HBM: 2 bytes per value on the 16-bit side, half a byte and
// 1/32 on the other.  16 x 4096 x 7168, written in 194-214 us, 5.6-6.1 TB/s, read
// back, four bytes of five of that being stores, in 271-285, 4.2-4.4 (a large copy
// 4.8).  1531 rows of 1000 (2.8 + 2.8 us) are a round of blocks.

#include "rows4.h"
#include "rows_io.h"

namespace {

typedef uint32_t u32_any __attribute__((aligned(1)));

// Bytes b .. b+3 of a row of `bytes`, b < bytes (past the row: zero, as in load8).
__device__ __forceinline__ uint32_t load4(const uint8_t* row, int64_t b, int64_t bytes) {
  uint32_t w = 0;
  if (bytes < 4) {
    for (int j = 0; b + j < bytes; ++j) w |= (uint32_t)row[b + j] << (8 * j);
  } else {
    const int64_t at = b + 4 <= bytes ? b : bytes - 4;
    w = __builtin_nontemporal_load(reinterpret_cast<const u32_any*>(row + at)) >> (8 * (int)(b - at));
  }
  return w;
}

// Whichever of them the row has.
__device__ __forceinline__ void store4(uint8_t* row, int64_t b, int64_t bytes, uint32_t w) {
  uint8_t* p = row + b;
  if (b + 4 <= bytes) {
    *reinterpret_cast<u32_any*>(p) = w;
    return;
  }
  const int n = (int)(bytes - b);
  if (n & 2) *reinterpret_cast<u16_a1*>(p) = (uint16_t)w, p += 2, w >>= 16;
  if (n & 1) *p = (uint8_t)w;
}

// The largest of 8 magnitudes (16-bit patterns compare as integers; infinities and NaN are the largest).
__device__ __forceinline__ uint32_t most8(const uint4 v) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  uint32_t most = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) most = max(most, max(w[j] & 0x7fffu, (w[j] >> 16) & 0x7fffu));
  return most;
}

// Eight values beside a power of two -> eight codes.
template <class E>
__device__ __forceinline__ uint32_t codes8(const uint4 v, float scale) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  uint32_t c = 0;
  if constexpr (E::kCode == EltF16::kCode) {
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, __builtin_bit_cast(f16x2_t, w[0]), scale, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, __builtin_bit_cast(f16x2_t, w[1]), scale, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, __builtin_bit_cast(f16x2_t, w[2]), scale, 2);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, __builtin_bit_cast(f16x2_t, w[3]), scale, 3);
  } else {
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2_t, w[0]), scale, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2_t, w[1]), scale, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2_t, w[2]), scale, 2);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2_t, w[3]), scale, 3);
  }
  return c;
}

// A block: 4 * PER rows x 512 columns of one group, PER rows per wave, all in
// flight together; a lane's 8 columns are one 16-byte load and one 4-byte
// store, a block of 32 columns four lanes.  PER = 2 where 8 would be fewer
// blocks than CUs have room for.
template <class E, int PER>
__global__ __launch_bounds__(256) void quantize_rows4_kernel(const bf16_t* __restrict__ x, int64_t ldx, int64_t gsx, int64_t R,
                                                             int64_t N, int64_t row_tiles, uint8_t* __restrict__ codes,
                                                             uint8_t* __restrict__ scales) {
  constexpr int kTileRows = 4 * PER;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t B = (N + kScaleGroup - 1) / kScaleGroup, bytes = (N + 1) / 2;
  const uint32_t rest = blockIdx.x / (uint32_t)B, g = rest / (uint32_t)row_tiles;
  const int64_t b = blockIdx.x % (uint32_t)B, r0 = (int64_t)(rest % (uint32_t)row_tiles) * kTileRows;
  const int64_t c = b * kScaleGroup + lane * 8;
  const bf16_t* xg = x + g * gsx;
  uint8_t* cg = codes + g * R * bytes;
  uint8_t* sg = scales + (g * B + b) * R * kScaleBytes;
  uint4 v[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int64_t r = r0 + i * 4 + wave;
    v[i] = r < R && c < N ? load8(xg + r * ldx, c, N) : make_uint4(0, 0, 0, 0);
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    constexpr uint32_t kInf = E::kCode == EltF16::kCode ? 0x7c00u : 0x7f80u;
    const int64_t r = r0 + i * 4 + wave;
    uint32_t most = most8(v[i]);
    most = max(most, (uint32_t)__shfl_xor((int)most, 1, 64));
    most = max(most, (uint32_t)__shfl_xor((int)most, 2, 64));
    const bool nan = most >= kInf;
    const uint32_t byte = nan ? kScaleNaN : scale_byte4(__float_as_uint(E::to_f32(most)));
    if (r >= R) continue;
    // The conversion divides by the power of two whose exponent field `scale` has.  (A block that is NaN: 6
    // throughout.)  Past an odd row's end the columns are zeros.
    uint32_t w = nan ? 0x77777777u : codes8<E>(v[i], __uint_as_float(byte << 23));
    if (nan && N - c < 8) w &= (1u << (4 * (int)(N - c < 0 ? 0 : N - c))) - 1u;
    if (c < N) store4(cg + r * bytes, c / 2, bytes, w);
    if ((lane & 3) == 0) sg[r * kScaleBytes + (lane >> 2)] = (uint8_t)byte;
  }
}

// A wave: 512 columns of PER rows.
template <class E, int PER>
__global__ __launch_bounds__(256) void dequantize_rows4_kernel(const uint8_t* __restrict__ codes,
                                                               const uint8_t* __restrict__ scales, int64_t R, int64_t N,
                                                               int64_t row_tiles, bf16_t* __restrict__ out) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t B = (N + kScaleGroup - 1) / kScaleGroup, bytes = (N + 1) / 2;
  const uint32_t rest = blockIdx.x / (uint32_t)B, g = rest / (uint32_t)row_tiles;
  const int64_t b = blockIdx.x % (uint32_t)B, r0 = (int64_t)(rest % (uint32_t)row_tiles) * (4 * PER);
  const int64_t c = b * kScaleGroup + lane * 8;
  if (c >= N) return;
  const uint8_t* cg = codes + g * R * bytes;
  const uint8_t* sg = scales + (g * B + b) * R * kScaleBytes;
  bf16_t* og = out + g * R * N;
  uint32_t v[PER], s[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int64_t r = r0 + i * 4 + wave;
    if (r < R) {
      v[i] = load4(cg + r * bytes, c / 2, bytes);
      s[i] = sg[r * kScaleBytes + (lane >> 2)];
    }
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int64_t r = r0 + i * 4 + wave;
    if (r >= R) continue;
    const f32x2_t f2[4] = {__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(v[i], 1.0f, 0), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(v[i], 1.0f, 1),
                           __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(v[i], 1.0f, 2), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(v[i], 1.0f, 3)};
    const float scale = s[i] == kScaleNaN ? __uint_as_float(0x7fc00000u) : scale_of(s[i]);
    float f[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = to_range<E>(f2[j / 2][j % 2] * scale);
    store8(og + r * N, c, N, pack8e<E>(f));
  }
}

// Blocks of eight rows per wave that fill the chip (two per CU).
constexpr int64_t kManyBlocks = 512;

// a * b, or -1 where it passes 2^62 (a, b >= 0).
int64_t product(int64_t a, int64_t b) { return a != 0 && b > (((int64_t)1 << 62) / a) ? -1 : a * b; }

// The grid over G groups of R rows, per rows to a wave: blocks, or 0 where a launch does not hold them.
int64_t grid_of(int64_t G, int64_t R, int64_t N, int64_t& tiles, bool& many) {
  const int64_t B = (N + kScaleGroup - 1) / kScaleGroup;
  if (product(G, R) < 0 || product(G * R, N) < 0 || product(G * R, B) < 0) return 0;
  const auto blocks = [&](int64_t rows) { return G * ((R + rows - 1) / rows) * B; };
  many = blocks(32) >= kManyBlocks;
  const int64_t rows = many ? 32 : 8;
  tiles = (R + rows - 1) / rows;
  return grid_fits(blocks(rows), 256) ? blocks(rows) : 0;
}

template <class E>
int quantize_t(const void* x, int64_t ldx, int64_t gsx, int64_t G, int64_t R, int64_t N, void* codes, void* scales,
               pmx_stream_t stream) {
  if (G < 0 || R < 0 || N < 0 || ldx < N) return PMX_ERR_ARG;
  if (G == 0 || R == 0 || N == 0) return PMX_OK;
  if (!x || !codes || !scales) return PMX_ERR_ARG;
  int64_t tiles = 0;
  bool many = false;
  const int64_t grid = grid_of(G, R, N, tiles, many);
  if (grid == 0 || product(G * R, ldx) < 0) return PMX_ERR_SHAPE;
  const auto run = [&](auto kernel) {
    kernel<<<(unsigned)grid, 256, 0, stream>>>((const bf16_t*)x, ldx, gsx, R, N, tiles, (uint8_t*)codes, (uint8_t*)scales);
  };
  if (many) run(quantize_rows4_kernel<E, 8>);
  else run(quantize_rows4_kernel<E, 2>);
  PMX_LAUNCH_CHECK();
  return PMX_OK;
}

template <class E>
int dequantize_t(const void* codes, const void* scales, int64_t G, int64_t R, int64_t N, void* out, pmx_stream_t stream) {
  if (G < 0 || R < 0 || N < 0) return PMX_ERR_ARG;
  if (G == 0 || R == 0 || N == 0) return PMX_OK;
  if (!codes || !scales || !out) return PMX_ERR_ARG;
  int64_t tiles = 0;
  bool many = false;
  const int64_t grid = grid_of(G, R, N, tiles, many);
  if (grid == 0) return PMX_ERR_SHAPE;
  const auto run = [&](auto kernel) {
    kernel<<<(unsigned)grid, 256, 0, stream>>>((const uint8_t*)codes, (const uint8_t*)scales, R, N, tiles, (bf16_t*)out);
  };
  if (many) run(dequantize_rows4_kernel<E, 8>);
  else run(dequantize_rows4_kernel<E, 2>);
  PMX_LAUNCH_CHECK();
  return PMX_OK;
}

}  // namespace

extern "C" {

#define PMX_ROWS4_ENTRIES(SUFFIX, E)                                                                                      \
  int pmx_rows4_quantize##SUFFIX(const void* x, int64_t ldx, int64_t gsx, int64_t G, int64_t R, int64_t N, void* codes,   \
                                 void* scales, pmx_stream_t stream) {                                                     \
    return quantize_t<E>(x, ldx, gsx, G, R, N, codes, scales, stream);                                                    \
  }                                                                                                                       \
  int pmx_rows4_dequantize##SUFFIX(const void* codes, const void* scales, int64_t G, int64_t R, int64_t N, void* out,     \
                                   pmx_stream_t stream) {                                                                 \
    return dequantize_t<E>(codes, scales, G, R, N, out, stream);                                                          \
  }

PMX_ROWS4_ENTRIES(, EltBF16)
PMX_ROWS4_ENTRIES(_f16, EltF16)

}  // extern "C"
