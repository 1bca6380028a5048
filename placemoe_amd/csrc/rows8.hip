// Rows in 8 bits (rows8.h): writing them, reading them back (in order or into
// the rows of the expert copies), and the SwiGLU backward from 8-bit gate and
// up rows.  An activation checkpoint of the expert layer is such a pair: its
// hidden states and its gate/up rows, 2I + H / K bytes per row of the copies
// (K experts per token) where the layer otherwise keeps 6I + 4H, or 6I + 2H with
// the router weights on fc2's input; the SwiGLU activations are recomputed.
//
// All are bound by HBM: 3 bytes per value written, 1 + 2K per value read back
// into K rows, 10 per activation of the SwiGLU backward, each with 1/32 of a
// byte per value for the exponents.  Measured: 16384 rows of 2048 written in 21 us
// (4.7 TB/s; 65536 of 4096: 5.8), read back into 8 rows each in 108 (5.3), the
// SwiGLU backward of 65536 rows of 2048 in 250 (5.4; a large copy: 4.8).
//
// Rows need no alignment: a lane's 8 columns are one load wherever they
// start (gfx950 takes unaligned vector accesses); a row's last, partial 8 are
// shifted out of the 8 that end with it.

#include "rows8.h"
#include "rows_io.h"

namespace {

// fp32 bits of the largest finite magnitude among 8 elements (16-bit
// magnitudes compare as integers; infinities and NaN count as zero).
template <class E>
__device__ __forceinline__ uint32_t most_finite8(const uint4 v) {
  constexpr uint32_t kInf = E::kCode == EltF16::kCode ? 0x7c00u : 0x7f80u;
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  uint32_t most = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t lo = w[j] & 0x7fffu, hi = (w[j] >> 16) & 0x7fffu;
    most = max(most, lo < kInf ? lo : 0u);
    most = max(most, hi < kInf ? hi : 0u);
  }
  return most;
}

// ---------------------------------------------------------------------------
// Writing
// ---------------------------------------------------------------------------

// What a routed call adds: row pos[t,k] of the copies' rows holds token t and
// its weight w[t,k].
struct RowMap {
  const int32_t* pos;  // [T, K], null: none
  const bf16_t* w;     // [T, K]
  int32_t K;
  int32_t* row_token;  // [T * K]
  bf16_t* row_w;       // [T * K]
};

// A block: 4 * PER rows x 512 columns of one group, PER rows per wave, a lane's
// 8 columns in one 16-byte load; all of a wave's rows are in flight
// together.  PER = 8: the 32 rows' exponents are 512 contiguous bytes that
// one XCD's L2 collects.  PER = 2, where that would be fewer blocks than CUs
// have room for: more of them.  A block of 32 columns is four lanes.
template <class E, int FMT, int PER>
__global__ __launch_bounds__(256) void quantize_rows_kernel(const bf16_t* __restrict__ x, int64_t ldx, int64_t gsx,
                                                            int64_t R, int64_t N, int64_t row_tiles, RowMap map,
                                                            uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
  constexpr int kTileRows = 4 * PER;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t B = (N + kScaleGroup - 1) / kScaleGroup;
  // column groups fastest: a row's blocks run side by side
  // (32-bit divisions: a 64-bit one takes longer than the rows of a small call)
  const uint32_t rest = blockIdx.x / (uint32_t)B, g = rest / (uint32_t)row_tiles;
  const int64_t b = blockIdx.x % (uint32_t)B, r0 = (int64_t)(rest % (uint32_t)row_tiles) * kTileRows;
  const int64_t c = b * kScaleGroup + lane * 8;
  const bf16_t* xg = x + g * gsx;
  uint8_t* cg = codes + g * R * N;
  uint8_t* sg = scales + (g * B + b) * R * kScaleBytes;
  uint4 v[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int64_t r = r0 + i * 4 + wave;
    v[i] = r < R && c < N ? load8(xg + r * ldx, c, N) : make_uint4(0, 0, 0, 0);
  }
  if (map.pos != nullptr && b == 0) {
    const int32_t rows = (int32_t)(R - r0 < kTileRows ? R - r0 : kTileRows), A = (int32_t)R * map.K;  // T * K fits
    for (int32_t i = threadIdx.x; i < rows * map.K; i += 256) {
      const int32_t a = (int32_t)r0 * map.K + i, p = map.pos[a];
      if (p >= 0 && p < A) {
        map.row_token[p] = (int32_t)((uint32_t)a / (uint32_t)map.K);
        map.row_w[p] = map.w[a];
      }
    }
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int64_t r = r0 + i * 4 + wave;
    uint32_t most = most_finite8<E>(v[i]);
    most = max(most, (uint32_t)__shfl_xor((int)most, 1, 64));
    most = max(most, (uint32_t)__shfl_xor((int)most, 2, 64));
    const uint32_t byte = scale_byte<FMT>(__float_as_uint(E::to_f32(most)));
    const float inv = inv_scale(byte);
    float f[8];
    unpack8e<E>(v[i], f);
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] *= inv;
    if (r < R) {
      if (c < N) store8(cg + r * N, c, N, make_uint2(codes4<FMT>(f[0], f[1], f[2], f[3]), codes4<FMT>(f[4], f[5], f[6], f[7])));
      if ((lane & 3) == 0) sg[r * kScaleBytes + (lane >> 2)] = (uint8_t)byte;
    }
  }
}

// ---------------------------------------------------------------------------
// Reading back
// ---------------------------------------------------------------------------

// A wave: 512 columns of PER rows; row r goes to out[r], or with pos [R, K] to
// out[pos[r, k]] for every k (rows outside the output are not written).
template <class E, int FMT, int PER>
__global__ __launch_bounds__(256) void dequantize_rows_kernel(const uint8_t* __restrict__ codes,
                                                              const uint8_t* __restrict__ scales,
                                                              const int32_t* __restrict__ pos, int64_t R, int32_t K,
                                                              int64_t N, bf16_t* __restrict__ out) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t B = (N + kScaleGroup - 1) / kScaleGroup;
  const int64_t b = blockIdx.x % (uint32_t)B, r0 = (int64_t)(blockIdx.x / (uint32_t)B) * (4 * PER);
  const int64_t c = b * kScaleGroup + lane * 8;
  if (c >= N) return;
  uint2 v[PER];
  uint32_t s[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int64_t r = r0 + i * 4 + wave;
    if (r < R) {
      v[i] = load8(codes + r * N, c, N);
      s[i] = scales[(b * R + r) * kScaleBytes + (lane >> 2)];
    }
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int64_t r = r0 + i * 4 + wave;
    if (r >= R) continue;
    float f[8];
    values4<FMT>(v[i].x, f);
    values4<FMT>(v[i].y, f + 4);
    const float scale = scale_of(s[i]);
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = to_range<E>(f[j] * scale);
    const uint4 w = pack8e<E>(f);
    if (pos == nullptr) {
      store8(out + r * N, c, N, w);
    } else {
      for (int k = 0; k < K; ++k) {
        const int64_t p = pos[r * K + k];
        if (p >= 0 && p < R * K) store8(out + p * N, c, N, w);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// SwiGLU backward
// ---------------------------------------------------------------------------

// Gate or up columns c .. c+7 (of I from column `first` of the row): values.
template <int FMT, bool WHOLE>
__device__ __forceinline__ void gate_up8(const uint8_t* row, const uint8_t* scales, int64_t sstep, int64_t first, int64_t c,
                                         int64_t I, float* f) {
  const uint2 v = load8(row + first, c, I);
  const int64_t q = (first + c) / kScaleBlock;
  const auto byte = [&](int64_t q) { return (uint32_t)scales[(q >> 4) * sstep + (q & 15)]; };
  values4<FMT>(v.x, f);
  values4<FMT>(v.y, f + 4);
  const float s0 = scale_of(byte(q));
  if constexpr (WHOLE) {
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] *= s0;
  } else {
    // the 8 columns may lie in two blocks: the first n in block q
    const int n = kScaleBlock - (int)((first + c) % kScaleBlock);
    const float s1 = n < 8 && c + n < I ? scale_of(byte(q + 1)) : s0;
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] *= j < n ? s0 : s1;
  }
}

// One wave per row r, all in fp32 and rounded once at the end:
//   s = g sigmoid(g), dact = d w
//   dG1[r] = (dact u (sigmoid(g) + s (1 - sigmoid(g))), dact s)
//   act_w[r] = w s u,  dw[row_src[r]] = sum_j d_j s_j u_j
// (row_w null: w = 1; dw null: not wanted; a row_src outside [0, A) is not
// written).  WHOLE: I a multiple of 8, so that 8 columns lie in one block.
template <class E, int FMT, bool WHOLE>
__global__ __launch_bounds__(256) void swiglu_bwd_rows8_kernel(const bf16_t* __restrict__ d, const uint8_t* __restrict__ codes,
                                                               const uint8_t* __restrict__ scales,
                                                               const bf16_t* __restrict__ row_w,
                                                               const int32_t* __restrict__ row_src, int64_t R, int64_t I,
                                                               int64_t A, bf16_t* __restrict__ dg1,
                                                               bf16_t* __restrict__ act_w, bf16_t* __restrict__ dw) {
  const int lane = threadIdx.x & 63;
  const int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (r >= R) return;
  const float w = row_w != nullptr ? E::to_f32(row_w[r]) : 1.0f;
  const int64_t sstep = R * kScaleBytes;
  const uint8_t* srow = scales + r * kScaleBytes;
  const uint8_t* crow = codes + r * 2 * I;
  float part = 0.f;
  for (int64_t c = lane * 8; c < I; c += 512) {
    float dv[8], g[8], u[8], a[8], dg[8], du[8];
    const uint4 dv8 = load8(d + r * I, c, I);
    gate_up8<FMT, WHOLE>(crow, srow, sstep, 0, c, I, g);
    gate_up8<FMT, WHOLE>(crow, srow, sstep, I, c, I, u);
    unpack8e<E>(dv8, dv);
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float sig = sigmoid_f32(g[j]), s = g[j] * sig, dact = dv[j] * w;
      const float act = s * u[j];
      dg[j] = dact * u[j] * __builtin_fmaf(s, 1.0f - sig, sig);
      du[j] = dact * s;
      a[j] = act * w;
      if (WHOLE || c + j < I) sum = __builtin_fmaf(dv[j], act, sum);
    }
    part += sum;
    store8(dg1 + r * 2 * I, c, I, pack8e<E>(dg));
    store8(dg1 + r * 2 * I + I, c, I, pack8e<E>(du));
    store8(act_w + r * I, c, I, pack8e<E>(a));
  }
  if (dw == nullptr) return;
  part = wave_sum(part);
  if (lane == 0) {
    const int64_t k = row_src[r];
    if (k >= 0 && k < A) dw[k] = (bf16_t)E::from_f32(part);
  }
}

// ---------------------------------------------------------------------------
// A token's rows, summed
// ---------------------------------------------------------------------------

// out[t] = sum_k of row pos[t, k] of y, in k order, in fp32 with one rounding.
// A block per token, 8 columns per thread; KC > 0: K == KC, whose loads go out
// together.  Bound by HBM: 3 K + 2 bytes per value; 8192 tokens of 2048 from 8
// rows each 75 us, 5.8 TB/s.
template <class E, int KC>
__global__ __launch_bounds__(256) void sum_f24_kernel(const uint16_t* __restrict__ y_high, const uint8_t* __restrict__ y_low,
                                                      const int32_t* __restrict__ pos, int64_t A, int32_t K, int64_t H,
                                                      bf16_t* __restrict__ out) {
  constexpr int N = KC > 0 ? KC : 1;
  const int64_t t = blockIdx.x;
  const int32_t* p = pos + t * K;
  for (int64_t c = (int64_t)threadIdx.x * 8; c < H; c += (int64_t)blockDim.x * 8) {
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (int k0 = 0; k0 < K; k0 += N) {
      uint4 high[N];
      uint2 low[N];
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const int64_t r = p[k0 + k];
        const bool in = r >= 0 && r < A;
        high[k] = in ? ld_stream(y_high + r * H + c) : make_uint4(0, 0, 0, 0);
        low[k] = in ? ld8(y_low + r * H + c) : make_uint2(0, 0);
      }
#pragma unroll
      for (int k = 0; k < N; ++k) {
        float f[8];
        f24_values8(high[k], low[k], f);
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[j] += f[j];
      }
    }
    *reinterpret_cast<uint4*>(out + t * H + c) = pack8e<E>(acc);
  }
}

template <class E>
int sum_f24_t(const void* y_high, const void* y_low, const int32_t* pos, int64_t T, int32_t K, int64_t H, void* out,
              pmx_stream_t stream) {
  const unsigned threads = rows8_sum_threads(H);
  const auto run = [&](auto kernel) {
    kernel<<<(unsigned)T, threads, 0, stream>>>((const uint16_t*)y_high, (const uint8_t*)y_low, pos, T * K, K, H, (bf16_t*)out);
  };
  switch (K) {
    case 2: run(sum_f24_kernel<E, 2>); break;
    case 4: run(sum_f24_kernel<E, 4>); break;
    case 6: run(sum_f24_kernel<E, 6>); break;
    case 8: run(sum_f24_kernel<E, 8>); break;
    default: run(sum_f24_kernel<E, 0>);
  }
  PMX_LAUNCH_CHECK();
  return PMX_OK;
}

// ---------------------------------------------------------------------------
// Launches
// ---------------------------------------------------------------------------

// Blocks of eight rows per wave that fill the chip (two per CU).
constexpr int64_t kManyBlocks = 512;

// a * b, or -1 where it passes 2^62 (a, b >= 0).
int64_t product(int64_t a, int64_t b) { return a != 0 && b > (((int64_t)1 << 62) / a) ? -1 : a * b; }

template <class E>
int quantize_t(const void* x, int64_t ldx, int64_t gsx, int64_t G, int64_t R, int64_t N, int32_t format, RowMap map,
               void* codes, void* scales, pmx_stream_t stream) {
  if (G < 0 || R < 0 || N < 0 || ldx < N || (format != kFmtE4M3 && format != kFmtInt8)) return PMX_ERR_ARG;
  if (G == 0 || R == 0 || N == 0) return PMX_OK;
  if (!x || !codes || !scales) return PMX_ERR_ARG;
  const int64_t B = (N + kScaleGroup - 1) / kScaleGroup;
  if (product(G, R) < 0 || product(G * R, ldx) < 0 || product(G * R, B) < 0) return PMX_ERR_SHAPE;
  const auto blocks = [&](int64_t rows) { return G * ((R + rows - 1) / rows) * B; };
  const int per = blocks(32) >= kManyBlocks ? 8 : 2;
  const int64_t grid = blocks(4 * per), tiles = (R + 4 * per - 1) / (4 * per);
  if (!grid_fits(grid, 256)) return PMX_ERR_SHAPE;
  const auto run = [&](auto kernel) {
    kernel<<<(unsigned)grid, 256, 0, stream>>>((const bf16_t*)x, ldx, gsx, R, N, tiles, map, (uint8_t*)codes, (uint8_t*)scales);
  };
  if (format == kFmtE4M3) {
    if (per == 8) run(quantize_rows_kernel<E, kFmtE4M3, 8>);
    else run(quantize_rows_kernel<E, kFmtE4M3, 2>);
  } else {
    if (per == 8) run(quantize_rows_kernel<E, kFmtInt8, 8>);
    else run(quantize_rows_kernel<E, kFmtInt8, 2>);
  }
  PMX_LAUNCH_CHECK();
  return PMX_OK;
}

template <class E>
int quantize_routed_t(const void* x, const int32_t* pos, const void* w, int64_t T, int32_t K, int64_t H, void* codes,
                      void* scales, int32_t* row_token, void* row_w, pmx_stream_t stream) {
  if (T < 0 || K <= 0 || H < 0) return PMX_ERR_ARG;
  if (T > INT32_MAX / K) return PMX_ERR_SHAPE;
  if (T == 0) return PMX_OK;
  if (H == 0) return PMX_ERR_SHAPE;
  if (!pos || !w || !row_token || !row_w) return PMX_ERR_ARG;
  RowMap map = {pos, (const bf16_t*)w, K, row_token, (bf16_t*)row_w};
  return quantize_t<E>(x, H, 0, 1, T, H, kFmtE4M3, map, codes, scales, stream);
}

template <class E>
int dequantize_t(const void* codes, const void* scales, const int32_t* pos, int64_t R, int32_t K, int64_t N, int32_t format,
                 void* out, pmx_stream_t stream) {
  if (R < 0 || K < 0 || N < 0 || (pos != nullptr && K == 0) || (format != kFmtE4M3 && format != kFmtInt8)) return PMX_ERR_ARG;
  if (R == 0 || N == 0) return PMX_OK;
  if (!codes || !scales || !out) return PMX_ERR_ARG;
  if (pos != nullptr && R > INT32_MAX / K) return PMX_ERR_SHAPE;  // positions are int32
  const int64_t B = (N + kScaleGroup - 1) / kScaleGroup;
  if (product(R, N) < 0 || product(R, B) < 0) return PMX_ERR_SHAPE;
  const auto blocks = [&](int64_t rows) { return (R + rows - 1) / rows * B; };
  const int per = blocks(16) >= kManyBlocks ? 4 : 1;
  if (!grid_fits(blocks(4 * per), 256)) return PMX_ERR_SHAPE;
  const auto run = [&](auto kernel) {
    kernel<<<(unsigned)blocks(4 * per), 256, 0, stream>>>((const uint8_t*)codes, (const uint8_t*)scales, pos, R, K, N,
                                                          (bf16_t*)out);
  };
  if (format == kFmtE4M3) {
    if (per == 4) run(dequantize_rows_kernel<E, kFmtE4M3, 4>);
    else run(dequantize_rows_kernel<E, kFmtE4M3, 1>);
  } else {
    if (per == 4) run(dequantize_rows_kernel<E, kFmtInt8, 4>);
    else run(dequantize_rows_kernel<E, kFmtInt8, 1>);
  }
  PMX_LAUNCH_CHECK();
  return PMX_OK;
}

template <class E>
int swiglu_bwd_t(const void* d, const void* codes, const void* scales, const void* row_w, const int32_t* row_src, int64_t R,
                 int64_t I, int64_t A, int32_t format, void* dG1, void* act_w, void* dw, pmx_stream_t stream) {
  if (R < 0 || I < 0 || A < 0 || (format != kFmtE4M3 && format != kFmtInt8)) return PMX_ERR_ARG;
  if ((dw == nullptr) != (row_src == nullptr)) return PMX_ERR_ARG;
  if (R == 0 || I == 0) return PMX_OK;
  if (!d || !codes || !scales || !dG1 || !act_w) return PMX_ERR_ARG;
  if (product(R, I) < 0 || product(R, 2 * I) < 0 || !grid_fits((R + 3) / 4, 256)) return PMX_ERR_SHAPE;
  const auto run = [&](auto kernel) {
    kernel<<<(unsigned)((R + 3) / 4), 256, 0, stream>>>((const bf16_t*)d, (const uint8_t*)codes, (const uint8_t*)scales,
                                                        (const bf16_t*)row_w, row_src, R, I, A, (bf16_t*)dG1,
                                                        (bf16_t*)act_w, (bf16_t*)dw);
  };
  const bool whole = I % 8 == 0;
  if (format == kFmtE4M3) {
    if (whole) run(swiglu_bwd_rows8_kernel<E, kFmtE4M3, true>);
    else run(swiglu_bwd_rows8_kernel<E, kFmtE4M3, false>);
  } else {
    if (whole) run(swiglu_bwd_rows8_kernel<E, kFmtInt8, true>);
    else run(swiglu_bwd_rows8_kernel<E, kFmtInt8, false>);
  }
  PMX_LAUNCH_CHECK();
  return PMX_OK;
}

}  // namespace

// The layer has checked T (with its grid), K and H (a multiple of 16), and the pointers.
int pmx_rows8_sum_f24(const void* y_high, const void* y_low, const int32_t* pos, int64_t T, int32_t K, int64_t H, bool f16,
                      void* out, pmx_stream_t stream) {
  if (T == 0) return PMX_OK;
  return f16 ? sum_f24_t<EltF16>(y_high, y_low, pos, T, K, H, out, stream)
             : sum_f24_t<EltBF16>(y_high, y_low, pos, T, K, H, out, stream);
}

extern "C" {

#define PMX_ROWS8_ENTRIES(SUFFIX, E)                                                                                      \
  int pmx_rows8_quantize##SUFFIX(const void* x, int64_t ldx, int64_t gsx, int64_t G, int64_t R, int64_t N, int32_t format, \
                                 void* codes, void* scales, pmx_stream_t stream) {                                        \
    return quantize_t<E>(x, ldx, gsx, G, R, N, format, RowMap{}, codes, scales, stream);                                  \
  }                                                                                                                       \
  int pmx_rows8_quantize_routed##SUFFIX(const void* x, const int32_t* pos, const void* w, int64_t T, int32_t K, int64_t H, \
                                        void* codes, void* scales, int32_t* row_token, void* row_w,                       \
                                        pmx_stream_t stream) {                                                            \
    return quantize_routed_t<E>(x, pos, w, T, K, H, codes, scales, row_token, row_w, stream);                             \
  }                                                                                                                       \
  int pmx_rows8_dequantize##SUFFIX(const void* codes, const void* scales, const int32_t* pos, int64_t R, int32_t K,       \
                                   int64_t N, int32_t format, void* out, pmx_stream_t stream) {                           \
    return dequantize_t<E>(codes, scales, pos, R, K, N, format, out, stream);                                             \
  }                                                                                                                       \
  int pmx_rows8_swiglu_bwd##SUFFIX(const void* d_act, const void* codes, const void* scales, const void* row_w,           \
                                   const int32_t* row_src, int64_t R, int64_t I, int64_t A, int32_t format, void* dG1,    \
                                   void* act_w, void* dw, pmx_stream_t stream) {                                          \
    return swiglu_bwd_t<E>(d_act, codes, scales, row_w, row_src, R, I, A, format, dG1, act_w, dw, stream);                \
  }

PMX_ROWS8_ENTRIES(, EltBF16)
PMX_ROWS8_ENTRIES(_f16, EltF16)

}  // extern "C"
