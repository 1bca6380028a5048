// Grouped GEMM over ragged row groups, both operands rows in 8 bits (rows8.h,
// e4m3):
//   NT   C[rows of g] = A[rows of g] B[g]^T                          (bf16 or fp16)
//   FC1  (gate | up) = A[rows of g] B[g]^T, act = silu(gate) * up * row_w, written
//        as rows in 8 bits again, ready to be fc2's A
// A row map lets A's rows come from anywhere: fc1 reads each token's row where
// it lies, once per copy it is routed to, and the permuted copy of the hidden
// states is never made.
//
// NT multiplies on v_mfma_scale_f32_32x32x64_f8f6f4, which takes the two
// operands' powers of two per 32 columns with the codes, at twice the rate of
// bf16.  It adds products in eights of neighbouring columns, each cut (towards
// zero) below 2^-13 of the power of two of the largest of its eight; the sums of
// the eights, and the instructions', are added in fp32.  So a result is off by
// less than 7 * 2^-13 of the largest product of each eight; of random values by
// 1.5e-5 of itself, a hundredth of the half step to which bf16 rounds it (fp16:
// a tenth).  FC1's results are rounded to 8
// bits, and there an error of 1e-5 moves one code in some thousands across a
// border, by a whole step: of the layer's output that is 0.002, more than its
// rounding to bf16 (0.0017).  So FC1 converts the codes, with their powers of
// two, to bf16 in registers (v_cvt_scalef32_pk_bf16_fp8, exact) and multiplies
// on v_mfma_f32_32x32x16_bf16, whose sums are good to fp32; it reads as few bytes.
//
// Bound: MFMA from some hundred rows per group on, the weights' bytes below.
// Measured: NT 65536 x 4096 x 7168 over 16 groups 1.57-1.71 ms, 2.25-2.45 PFLOP/s at
// the power limit (torch's 8-bit product of 8192^3 in one process with it: 2.50
// against 2.46); FC1 of 65536 rows of 160 copies of 1536 x 2048 0.42-0.53 ms, 0.8-1.0
// PFLOP/s (bf16 products of 8192^3: 1.28); 768 rows of those copies 89 (NT) and 91 us,
// 5.6 TB/s of weights.
//
// Tiles of BM x BN, K in steps of 128 through a ring of NST stages filled by
// buffer->LDS loads; 128-byte rows with 16-byte chunk c at c ^ ((row >> 1) & 7),
// as in the bf16 kernels, whose K-tiles are as many bytes.  The exponents of
// four K-tiles are 16 bytes per row (rows8.h): they come with the first of the
// four, 64 rows per load, into a ring of their own, and each wave picks a
// K-tile's word per row from there.

#include <atomic>

#include "gemm_util.h"
#include "rows8.h"
#include "rows8_rule.h"

namespace {

typedef int32_t i32x8_t __attribute__((ext_vector_type(8)));
typedef int32_t i32x4_t __attribute__((ext_vector_type(4)));

constexpr int kMaxGroups = 2048;  // groups (their m-tiles' prefix in LDS)
constexpr int KT = 128;           // depth of a K-tile
constexpr int kStreaming = 2;     // cache policy of stores that this kernel does not read back
constexpr int kScaleTiles = kScaleGroup / KT;

enum Kind8 { NT8 = 0, FC18 = 1 };

struct Params8 {
  const uint8_t *a, *as;     // A's codes [a_rows, K] and exponents
  const int32_t* row_token;  // row r of the groups is row row_token[r] of A; null: row r
  int64_t a_rows;
  const uint8_t *b, *bs;     // [G, N, K]
  const int32_t* offsets;    // [G + 1]
  int32_t G;
  int64_t M, N, K;           // M rows over all groups; N: rows of a B[g] (FC1: 2 I)
  int64_t I;
  bf16_t* c;                 // NT: [M, N]
  uint8_t* c_low;            // NT in 24 bits: the low bytes [M, N] of c
  uint8_t *q, *qs;           // FC1: act's codes [M, I] and exponents
  const bf16_t* row_w;       // FC1: [M], null: 1
};

// WM x WN waves, each FM x FN tiles of 32 x 32; NST stages; BPC blocks per CU.
template <int WM_, int WN_, int FM_, int FN_, int NST_, int BPC_>
struct Cfg8 {
  static constexpr int WM = WM_, WN = WN_, FM = FM_, FN = FN_, NST = NST_, BPC = BPC_;
  static constexpr int NW = WM * WN, NTH = 64 * NW;
  static constexpr int BM = WM * FM * 32, BN = WN * FN * 32;
  static constexpr int A_BYTES = BM * KT, STAGE = (BM + BN) * KT;
  static constexpr int QA = BM / 8 / NW, QB = BN / 8 / NW;  // 1 KB loads (8 rows) of one wave per K-tile
  static constexpr int SA = (BM + 63) / 64, SB = BN / 64;   // 1 KB loads of exponents (64 rows), all waves
  static constexpr int QS = (SA + SB + NW - 1) / NW;
  static constexpr int SLOT = (SA + SB) * 1024;
  static constexpr int LDS = NST * (STAGE + SLOT);
  static_assert(BM / 8 % NW == 0 && BN / 8 % NW == 0 && BN % 64 == 0, "whole loads per wave");
  static_assert(FN % 2 == 0 || (FN == 1 && WN == 2), "a wave, or the two of a block, has 32 gate columns and their up columns");
  static_assert(NST >= 2 && (NST - 1) * (QA + QB) <= 63, "vmcnt is 6 bits");
};

// Where one output tile lies.
struct Place {
  int32_t g, ntile, row0, row_end;
};

// The issue cursor's loads for one output tile.
template <class CF>
struct Loads {
  __amdgpu_buffer_rsrc_t a, b, as, bs;
  uint32_t off[CF::QA + CF::QB];  // a lane's byte offset (kOOB: outside of the operand)
  uint32_t soff[CF::QS];
  uint32_t past;                  // bit j: load j's lane lies past K in the last K-tile
};

// Row of B for the tile's virtual row: FC1 alternates 32 gate rows and the
// matching 32 up rows; 16 and 16 where a wave has one column tile.
template <int KIND, class CF>
__device__ __forceinline__ int32_t b_row(const Params8& P, int32_t ntile, int row) {
  if constexpr (KIND == FC18) {
    constexpr int W = CF::FN == 1 ? 16 : 32;
    const int32_t I = (int32_t)P.I, j = ntile * (CF::BN / 2) + row / (2 * W) * W + row % W;
    return j < I ? (row & W ? I : 0) + j : -1;
  } else {
    const int32_t j = ntile * CF::BN + row;
    return j < (int32_t)P.N ? j : -1;
  }
}

template <int KIND, class CF>
__device__ __forceinline__ void setup(const Params8& P, const Place& at, Loads<CF>& ld, int wave, int lane) {
  asm volatile("" : "+v"(lane));  // keep the per-lane arithmetic here
  const int krem = (int)(P.K - (P.K - 1) / KT * KT);
  const int64_t kgroups = (P.K + kScaleGroup - 1) / kScaleGroup;
  const bool mapped = KIND == FC18 && P.row_token != nullptr;
  const int64_t base = mapped ? 0 : at.row0;
  const int32_t rows = at.row_end - at.row0;  // some
  const auto load_row = [&](int j) { return (j * CF::NW + wave) * 8 + lane / 8; };
  const auto scale_row = [&](int j) { return (j * CF::NW + wave) * 64 + lane; };
  // A's row behind each load, relative to `base`; -1: none.  The tokens' loads all at once: one behind
  // the other they took 2 us of a call for one token.
  int32_t a_row[CF::QA], as_row[CF::QS];
  const auto held = [&](int row) { return row < rows ? row : rows - 1; };
  if (mapped) {
    const int32_t* tokens = P.row_token + at.row0;
#pragma unroll
    for (int j = 0; j < CF::QA; ++j) a_row[j] = tokens[held(load_row(j))];
#pragma unroll
    for (int j = 0; j < CF::QS; ++j) as_row[j] = tokens[held(scale_row(j))];
  } else {
#pragma unroll
    for (int j = 0; j < CF::QA; ++j) a_row[j] = load_row(j);
#pragma unroll
    for (int j = 0; j < CF::QS; ++j) as_row[j] = scale_row(j);
  }
  const auto of_a = [&](int row, int32_t r) { return row < rows && r < (int32_t)P.a_rows ? r : -1; };
  const uint32_t K = (uint32_t)P.K;
  ld.a = make_rsrc(P.a + base * P.K, (uint64_t)(P.a_rows - base) * P.K);
  ld.b = make_rsrc(P.b + (int64_t)at.g * P.N * P.K, (uint64_t)P.N * P.K);
  ld.as = make_rsrc(P.as + base * kScaleBytes, (uint64_t)(kgroups * P.a_rows - base) * kScaleBytes);
  ld.bs = make_rsrc(P.bs + (int64_t)at.g * kgroups * P.N * kScaleBytes, (uint64_t)kgroups * P.N * kScaleBytes);
  ld.past = 0;
#pragma unroll
  for (int i = 0; i < CF::QA + CF::QB; ++i) {
    const int j = i < CF::QB ? CF::QA + i : i - CF::QB;  // B's first: A's wait for their tokens
    const bool is_a = j < CF::QA;
    const int row = load_row(is_a ? j : j - CF::QA);
    const int c = (lane % 8) ^ kc_swz(row);
    const int32_t r = is_a ? of_a(row, a_row[is_a ? j : 0]) : b_row<KIND, CF>(P, at.ntile, row);
    ld.off[j] = r >= 0 ? (uint32_t)r * K + (uint32_t)c * 16u : kOOB;
    ld.past |= (c * 16 < krem ? 0u : 1u) << j;
    asm volatile("" : "+v"(ld.off[j]));  // one register, worked out here
  }
#pragma unroll
  for (int j = 0; j < CF::QS; ++j) {
    const int s = j * CF::NW + wave;
    const int row = (s < CF::SA ? s : s - CF::SA) * 64 + lane;
    const int32_t r = s < CF::SA ? (row < CF::BM ? of_a(row, as_row[j]) : -1) : b_row<KIND, CF>(P, at.ntile, row);
    ld.soff[j] = r >= 0 ? (uint32_t)r * kScaleBytes : kOOB;
    asm volatile("" : "+v"(ld.soff[j]));
  }
}

// FC1: codes of a 32-deep quarter (16 per lane), the K-tile's exponents of the
// lane's rows (byte q: quarter q), and the values of half a quarter.
template <class CF>
struct Codes8 {
  i32x4_t v[CF::FM + CF::FN];
};
template <class CF>
struct Words8 {
  uint32_t v[CF::FM + CF::FN];
};
template <class CF>
struct Values8 {
  bf16x8_t v[CF::FM + CF::FN];
};

// The I-th fragment in the order the (m-major) MFMAs use them: A0, B0 ..
// B(FN-1), A1 .. ; ids count A's first, then B's.
template <class CF>
constexpr int order8(int i) { return i == 0 ? 0 : i <= CF::FN ? CF::FM + i - 1 : i - CF::FN; }

// Exchanges the upper half-wave's `lo` with the lower half-wave's `hi`.
__device__ __forceinline__ void swap_halves(uint32_t& lo, uint32_t& hi) {
  const auto v = __builtin_amdgcn_permlane32_swap(lo, hi, false, false);
  lo = v[0];
  hi = v[1];
}

// The largest finite magnitude among the N values of this lane and the one 32 lanes on; `finite`: no lane of the
// wave holds another kind.  (Maxima that pass NaN on, two values to an instruction.)
template <int N>
__device__ __forceinline__ float most_finite(const float* f, bool& finite) {
  const auto halves = [](float m) __attribute__((always_inline)) {
    const auto v = __builtin_amdgcn_permlane32_swap(__float_as_uint(m), __float_as_uint(m), false, false);
    return __builtin_elementwise_maximum(__uint_as_float(v[0]), __uint_as_float(v[1]));
  };
  float most = 0.f;
#pragma unroll
  for (int i = 0; i < N; i += 2)
    most = __builtin_elementwise_maximum(__builtin_elementwise_maximum(most, __builtin_fabsf(f[i])), __builtin_fabsf(f[i + 1]));
  most = halves(most);
  finite = __ballot(!(most < __builtin_inff())) == 0;
  if (!finite) {
    most = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float a = __builtin_fabsf(f[i]);
      most = a > most && a < __builtin_inff() ? a : most;
    }
    most = halves(most);
  }
  return most;
}

// An accumulator holds its 32 x 32 output tile transposed (B is the MFMA's
// first operand): lane l has row l%32, columns 8*(i/4) + 4*(l/32) + i%4.
template <class E, int KIND, class CF>
__device__ __forceinline__ void epilogue(const Params8& P, const Place& at, int wm, int wn, int wave, int lane,
                                         [[maybe_unused]] char* stage, [[maybe_unused]] float* shared,
                                         f32x16_t (&acc)[CF::FM][CF::FN]) {
  // Each accumulator leaves the accumulation registers where it is used: read
  // right behind their last MFMAs, they would need as many vector registers.
  const auto here = [](f32x16_t& v) __attribute__((always_inline)) { asm volatile("" : "+a"(v)); };
  asm volatile("" : "+v"(lane));
  const int h = lane >> 5;
  // NT: the output from the tile's first row to the group's end (what lies behind fails the range check); the
  // lane's place in a store of whole row segments.
  const uint32_t ldc = (uint32_t)P.N * 2;
  [[maybe_unused]] const __amdgpu_buffer_rsrc_t out =
      make_rsrc(P.c + (int64_t)at.row0 * P.N, (uint64_t)(at.row_end - at.row0) * ldc);
  const int32_t col = at.ntile * CF::BN + wn * CF::FN * 32 + lane % (CF::FN * 4) * 8;
  [[maybe_unused]] const uint32_t voff =
      col < (int32_t)P.N ? (uint32_t)(lane / (CF::FN * 4)) * ldc + (uint32_t)col * 2 : kOOB;
  // NT in 24 bits: the same for the plane of low bytes, 16 columns per lane.
  const int32_t col_low = at.ntile * CF::BN + wn * CF::FN * 32 + lane % (CF::FN * 2) * 16;
  [[maybe_unused]] const __amdgpu_buffer_rsrc_t out_low =
      make_rsrc(P.c_low + (int64_t)at.row0 * P.N, (uint64_t)(at.row_end - at.row0) * P.N);
  [[maybe_unused]] const uint32_t voff_low =
      col_low < (int32_t)P.N ? (uint32_t)(lane / (CF::FN * 2)) * (uint32_t)P.N + (uint32_t)col_low : kOOB;
#pragma unroll
  for (int m = 0; m < CF::FM; ++m) {
    const int64_t r = (int64_t)at.row0 + (wm * CF::FM + m) * 32 + (lane & 31);
    const bool in = r < at.row_end;
    if constexpr (KIND == NT8) {
      // 32 rows of CPR 16-byte chunks pass through the wave's own 1 KB pieces
      // of the stage just freed (those that its loads fill, so that no other
      // wave touches them) and leave as whole row segments: straight from the
      // registers a store would have 32 bytes of each of 32 rows, four times
      // the requests to the L2.  Chunk c of row r at c ^ r (mod CPR), so that
      // neither side has bank conflicts.
      // (24 bits: the low bytes likewise through the next pieces, rows of LCPR chunks.)
      constexpr int CPR = CF::FN * 4, RPP = 64 / CPR;  // chunks of a row, rows of a piece (and of a store)
      constexpr int LCPR = CF::FN * 2, LRPP = 64 / LCPR;
      static_assert(32 / RPP + 32 / LRPP <= CF::QA + CF::QB, "enough pieces");
      const auto place = [&](int row, int c) {
        const int sw = CPR == 16 ? row & 15 : CPR == 8 ? kc_swz(row) : row >> 2 & 3;
        return stage + ((row / RPP) * CF::NW + wave) * 1024 + (row % RPP) * (CPR * 16) + ((c ^ sw) << 4);
      };
      [[maybe_unused]] const auto place_low = [&](int row, int c) {
        const int sw = LCPR == 8 ? kc_swz(row) : LCPR == 4 ? row >> 2 & 3 : row >> 3 & 1;
        return stage + ((32 / RPP + row / LRPP) * CF::NW + wave) * 1024 + (row % LRPP) * (LCPR * 16) + ((c ^ sw) << 4);
      };
#pragma unroll
      for (int n = 0; n < CF::FN; ++n) {
        here(acc[m][n]);
        const f32x16_t& v = acc[m][n];
        uint32_t w[8];  // pairs of columns 8 (i/2) + 4 h + 2 (i%2)
        if constexpr (E::kCode == kF24) {
          uint32_t u[16], low[4];
          float nan = 0.f;  // NaN if one of the values is (two values to an instruction)
#pragma unroll
          for (int i = 0; i < 16; i += 2) {
            nan = __builtin_elementwise_maximum(__builtin_elementwise_maximum(nan, v[i]), v[i + 1]);
            u[i] = __float_as_uint(v[i]) + 0x80u;  // infinities stay: the low byte is dropped
            u[i + 1] = __float_as_uint(v[i + 1]) + 0x80u;
          }
          if (__ballot(nan != nan)) {  // a NaN of ones throughout would become a zero
#pragma unroll
            for (int i = 0; i < 16; ++i) u[i] = v[i] != v[i] ? 0x7fc00000u : u[i];
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) w[i] = f24_high2(u + 2 * i);
#pragma unroll
          for (int i = 0; i < 4; ++i) low[i] = f24_low4(u + 4 * i);
#pragma unroll
          for (int p = 0; p < 2; ++p) {
            swap_halves(low[2 * p], low[2 * p + 1]);
            *reinterpret_cast<uint2*>(place_low(lane & 31, n * 2 + p) + h * 8) = make_uint2(low[2 * p], low[2 * p + 1]);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) w[i] = E::pack2(v[2 * i], v[2 * i + 1]);
        }
#pragma unroll
        for (int p = 0; p < 2; ++p) {  // 16 columns: the half-waves exchange, and each lane has 8 of them
          swap_halves(w[4 * p], w[4 * p + 2]);
          swap_halves(w[4 * p + 1], w[4 * p + 3]);
          *reinterpret_cast<uint4*>(place(lane & 31, n * 4 + p * 2 + h)) =
              make_uint4(w[4 * p], w[4 * p + 1], w[4 * p + 2], w[4 * p + 3]);
        }
      }
      wait_lds();
#pragma unroll
      for (int q = 0; q < 32 / RPP; ++q) {
        const int row = q * RPP + lane / CPR;
        const u32x4_t v = *reinterpret_cast<const u32x4_t*>(place(row, lane % CPR));
        __builtin_amdgcn_raw_buffer_store_b128(v, out, voff + (uint32_t)((wm * CF::FM + m) * 32 + q * RPP) * ldc, 0, kStreaming);
      }
      if constexpr (E::kCode == kF24) {
#pragma unroll
        for (int q = 0; q < 32 / LRPP; ++q) {
          const u32x4_t v = *reinterpret_cast<const u32x4_t*>(place_low(q * LRPP + lane / LCPR, lane % LCPR));
          __builtin_amdgcn_raw_buffer_store_b128(v, out_low, voff_low + (uint32_t)((wm * CF::FM + m) * 32 + q * LRPP) * (uint32_t)P.N,
                                                 0, kStreaming);
        }
      }
      __builtin_amdgcn_sched_barrier(0);  // one tile's registers at a time
    } else {
      const float w = in && P.row_w != nullptr ? E::to_f32(P.row_w[r]) : 1.0f;
      // The group's blocks past I that no tile covers: 2^0, like those of zeros (fc2's last K-tiles take them along).
      if (in && h == 0 && wn == CF::WN - 1 && (int64_t)(at.ntile + 1) * (CF::BN / 2) >= P.I) {
        const int64_t end = (P.I + kScaleGroup - 1) / kScaleGroup * kScaleGroup;
        for (int64_t j = (int64_t)(at.ntile + 1) * (CF::BN / 2); j < end;) {
          uint8_t* const byte = P.qs + (j / kScaleGroup * P.M + r) * kScaleBytes + j / kScaleBlock % 16;
          if (j % KT == 0) *reinterpret_cast<uint32_t*>(byte) = 0x7f7f7f7fu, j += KT;
          else *byte = 127, j += kScaleBlock;
        }
      }
      // A block's exponent and codes: `f` holds the lane's N values, columns 8 (i/4) + 4 h + i%4 of the block or,
      // one column tile per wave, of the wave's half of it.
      const auto weigh = [&](float gate, float up) { return silu_f32(gate) * up * w; };
      const auto code = [](const float* f, float inv) {
        return codes4<kFmtE4M3>(f[0] * inv, f[1] * inv, f[2] * inv, f[3] * inv);
      };
      const auto put_scale = [&](int64_t j, uint32_t byte) {
        P.qs[(j / kScaleGroup * P.M + r) * kScaleBytes + j / kScaleBlock % 16] = (uint8_t)byte;
      };
      if constexpr (CF::FN == 1) {
        here(acc[m][0]);
        float f[8];
        bool finite;
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = weigh(acc[m][0][i], acc[m][0][i + 8]);
        const float most = most_finite<8>(f, finite);
        // `shared`: [2][32]; a K-tile's barrier before it is used again
        if (h == 0) shared[wn * 32 + lane] = most;
        wait_lds();
        block_barrier();
        const uint32_t byte = scale_byte<kFmtE4M3>(__float_as_uint(fmaxf(most, shared[(1 - wn) * 32 + (lane & 31)])));
        const float inv = inv_scale(byte);
        uint32_t c0 = code(f, inv), c1 = code(f + 4, inv);
        swap_halves(c0, c1);  // columns 8 h .. + 7 of the wave's 16
        const int64_t j = (int64_t)at.ntile * 32 + wn * 16;
        if (in) {
          if (j < P.I) *reinterpret_cast<uint2*>(P.q + r * P.I + j + h * 8) = make_uint2(c0, c1);
          if (h == 0 && wn == 0) put_scale(j, byte);
        }
      } else {
#pragma unroll
        for (int n = 0; n < CF::FN; n += 2) {
          here(acc[m][n]);
          here(acc[m][n + 1]);
          float f[16];
          bool finite;
#pragma unroll
          for (int i = 0; i < 16; ++i) f[i] = weigh(acc[m][n][i], acc[m][n + 1][i]);
          const float most = most_finite<16>(f, finite);
          const uint32_t byte = scale_byte<kFmtE4M3>(__float_as_uint(most));
          const float inv = inv_scale(byte);
          uint32_t c[4];  // columns 8 i + 4 h .. + 3
#pragma unroll
          for (int i = 0; i < 4; ++i) c[i] = code(f + 4 * i, inv);
          // ... and after the exchange each lane has columns 16 h .. + 15
          swap_halves(c[0], c[2]);
          swap_halves(c[1], c[3]);
          const int64_t j = (int64_t)at.ntile * (CF::BN / 2) + (wn * CF::FN + n) * 16;
          if (in) {
            if (j + h * 16 < P.I)
              *reinterpret_cast<uint4*>(P.q + r * P.I + j + h * 16) = make_uint4(c[0], c[2], c[1], c[3]);
            if (h == 0) put_scale(j, byte);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
  }
}

// Sum over the wave's lanes up to and with this one: shifts within rows of 16 lanes, then the rows' last lanes.
__device__ __forceinline__ int32_t wave_scan(int32_t v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // row_shr:1
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast:15 into rows 1 and 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // row_bcast:31 into rows 2 and 3
  return v;
}

template <class E, int KIND, class CF>
__global__ __launch_bounds__(CF::NTH, CF::NW * CF::BPC / 4) void rows8_grouped_gemm_kernel(Params8 P) {
  constexpr int NW = CF::NW, L = CF::QA + CF::QB;
  __shared__ __attribute__((aligned(1024))) char lds[CF::LDS];
  __shared__ int32_t tend[kMaxGroups];  // m-tiles of the groups up to and with g
  char* const slots = lds + CF::NST * CF::STAGE;
  float* shared = nullptr;  // what FC1's two waves of one column tile each exchange
  if constexpr (KIND == FC18 && CF::FN == 1) {
    __shared__ float exchange[64];
    shared = exchange;
  }
  const int t = threadIdx.x;
  const int lane = t & 63;
  const int wave = uni(t >> 6);
  const int wm = wave / CF::WN, wn = wave % CF::WN;
  const int G = P.G;
  // offsets as they are used: within [0, M], whatever the tensor holds
  const auto offset = [&](int g) {
    const int32_t o = P.offsets[g];
    return o < 0 ? 0 : o > P.M ? (int32_t)P.M : o;
  };

  // Prefix of the groups' m-tiles, a group per thread at a time: a scan within each wave, then over the waves.
  // Four groups' loads of a thread go out together.
  {
    int32_t* const wsum = reinterpret_cast<int32_t*>(lds);  // two turns' worth, a wave's sum each
    int32_t before = 0;
    bool bad = false;  // offsets that descend are not row groups: nothing to do
    for (int32_t base = 0; base < G; base += 4 * CF::NTH) {
      int32_t o[4][2];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) o[i][e] = offset(base + i * CF::NTH + t + e < G ? base + i * CF::NTH + t + e : G);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int32_t g = base + i * CF::NTH + t;
        if (base + i * CF::NTH >= G) break;
        const int32_t inc = wave_scan((o[i][1] - o[i][0] + CF::BM - 1) / CF::BM);  // past the last group: none
        const bool descends = __ballot(o[i][1] < o[i][0]) != 0;
        int32_t sum = __builtin_amdgcn_readlane(inc, 63), lower = 0;
        bad |= descends;
        if constexpr (NW > 1) {
          int32_t* const turn_sums = wsum + i % 2 * NW;
          if (lane == 0) turn_sums[wave] = descends ? -1 : sum;
          __syncthreads();
          sum = 0;
          for (int w = 0; w < NW; ++w) {
            const int32_t v = uni(turn_sums[w]);
            bad |= v < 0;
            lower += w < wave ? v : 0;
            sum += v;
          }
        }
        if (g < G) tend[g] = before + lower + inc;
        before += sum;
      }
    }
    if (bad) return;
    __syncthreads();
  }
  const int32_t ntn = (int32_t)(KIND == FC18 ? (P.I + CF::BN / 2 - 1) / (CF::BN / 2) : (P.N + CF::BN - 1) / CF::BN);
  const int32_t total = uni(tend[G - 1]) * ntn;  // the host has checked that it fits
  // The main loops.  Whole: one row tile per wave, K-tiles in pairs; halves: NT otherwise, a tile's first and
  // last K-tiles are two.  What that adds past K is zeros.
  constexpr bool kWhole = CF::FM == 1, kHalves = KIND == NT8 && !kWhole;
  const int32_t ktiles = (int32_t)((P.K + KT - 1) / KT);
  const int32_t nk = kWhole ? ktiles + ktiles % 2 : kHalves && ktiles < 2 ? 2 : ktiles;
  // Blocks go round-robin over the XCDs: each XCD walks its own eighth of the
  // tile list, its blocks round-robin within it.
  int32_t first = blockIdx.x, step = gridDim.x, end = total;
  if (gridDim.x % kNumXcd == 0) {
    const int32_t x = blockIdx.x % kNumXcd;
    step = gridDim.x / kNumXcd;
    end = (int32_t)((int64_t)total * (x + 1) / kNumXcd);
    first = (int32_t)((int64_t)total * x / kNumXcd) + blockIdx.x / kNumXcd;
  }
  if (first >= end) return;

  // Tile order: group by group, in bands of 8 m-tiles walked n-tile by n-tile:
  // neighbouring tiles share a strip of B, and a band of A.  The group: 64
  // equal parts of the prefix at once, then the entries of the one.
  const int32_t part = (G + 63) / 64;
  auto decode = [&](int32_t tile, Place& at) __attribute__((always_inline)) {
    constexpr uint32_t kBand = 8;
    const int32_t m = (int32_t)((uint32_t)tile / (uint32_t)ntn);
    const auto first_past = [&](int32_t v) { return uni(__builtin_ctzll(__ballot(v > m))); };  // some entry is: m < tend[G-1]
    const int32_t hi = (lane + 1) * part < G ? (lane + 1) * part : G;
    int32_t g = first_past(tend[hi - 1]) * part;
    if (part > 1) g += first_past(tend[g + lane < G && lane < part ? g + lane : G - 1]);
    const int32_t m0 = g > 0 ? uni(tend[g - 1]) : 0, gm = uni(tend[g]) - m0;
    const uint32_t local = (uint32_t)(tile - m0 * ntn);
    const uint32_t band = local / (kBand * ntn) * kBand;
    const uint32_t rest = local - band * ntn;
    const uint32_t high = gm - band < kBand ? gm - band : kBand;
    at.g = g;
    at.ntile = (int32_t)(rest / high);
    at.row0 = uni(offset(g)) + (int32_t)(band + rest % high) * CF::BM;
    at.row_end = uni(offset(g + 1));
  };

  // Issue cursor, running ahead of the K-tile being multiplied.
  Loads<CF> ld;
  int32_t i_tile = first;
  int32_t i_kt = 0, i_stage = 0, i_slot = 0;
  bool i_live = true;
  // kOOB's bit on top of the offsets that lie past K: in the last K-tile, and all of those behind it.  (Done once,
  // here: a wave issues an instruction in 5 cycles, and a select per load was a sixth of those of a one-wave tile.)
  auto past_k = [&]() __attribute__((always_inline)) {
    const uint32_t past = i_kt == ktiles - 1 ? ld.past : ~0u;
#pragma unroll
    for (int q = 0; q < L; ++q) ld.off[q] |= (past >> q) << 31;
  };
  auto set_tile = [&]() __attribute__((always_inline)) {
    Place at;
    decode(i_tile, at);
    setup<KIND, CF>(P, at, ld, wave, lane);
    if (ktiles == 1) past_k();
  };
  set_tile();
  // The K-tile's exponents, where it is the first of four; ahead of its other
  // loads, so that whoever waits for those has these too.
  auto issue_scales = [&]() __attribute__((always_inline)) {
    if (i_kt % kScaleTiles != 0 || !i_live) return;
    const uint32_t kg = (uint32_t)(i_kt / kScaleTiles);
#pragma unroll
    for (int j = 0; j < CF::QS; ++j) {
      const int s = j * NW + wave;
      if (s >= CF::SA + CF::SB) continue;
      char* dst = slots + i_slot * CF::SLOT + s * 1024;
      if (s < CF::SA) dma16(ld.as, dst, ld.soff[j], kg * (uint32_t)(P.a_rows * kScaleBytes));
      else dma16(ld.bs, dst, ld.soff[j], kg * (uint32_t)(P.N * kScaleBytes));
    }
  };
  auto issue = [&](auto jj) __attribute__((always_inline)) {
    constexpr int J = decltype(jj)::value;
    char* stage = lds + i_stage * CF::STAGE;
    if constexpr (J < CF::QA) dma16(ld.a, stage + (J * NW + wave) * 1024, ld.off[J], (uint32_t)i_kt * KT);
    else dma16(ld.b, stage + CF::A_BYTES + ((J - CF::QA) * NW + wave) * 1024, ld.off[J], (uint32_t)i_kt * KT);
  };
  auto advance_issue = [&]() __attribute__((always_inline)) {
    i_stage = i_stage + 1 == CF::NST ? 0 : i_stage + 1;
    if (!i_live) return;
    ++i_kt;
    if (i_kt < nk) {
      if (i_kt % kScaleTiles == 0) i_slot = i_slot + 1 == CF::NST ? 0 : i_slot + 1;
      if (i_kt >= ktiles - 1) past_k();
      return;
    }
    i_kt = 0;
    i_slot = i_slot + 1 == CF::NST ? 0 : i_slot + 1;
    i_tile += step;
    if (i_tile < end) {
      set_tile();
    } else {
      // past the block's last K-tile: loads out of range, so that every K-tile issues the same number
      i_live = false;
#pragma unroll
      for (int q = 0; q < L; ++q) ld.off[q] = kOOB;
    }
  };
  // All stages are in flight before the first K-tile is multiplied: a stage is refilled once its K-tile is in
  // registers.
#pragma unroll
  for (int s = 0; s < CF::NST; ++s) {
    issue_scales();
    static_for<0, L>(issue);
    advance_issue();
  }
  wait_loads<(CF::NST - 1) * L>();
  block_barrier();

  const int h = lane >> 5, r32 = lane & 31;
  const int32_t arow = wm * CF::FM * 32, brow = wn * CF::FN * 32;
  // Fragment J's first row, within A's or B's rows of a stage, and its place there.
  const auto row_of = [&](int J) __attribute__((always_inline)) { return J < CF::FM ? arow + J * 32 : brow + (J - CF::FM) * 32; };
  const auto in_stage = [&](int J) __attribute__((always_inline)) { return (J < CF::FM ? 0 : CF::A_BYTES) + row_of(J) * KT; };
  const auto in_slot = [&](int J) __attribute__((always_inline)) {
    return (J < CF::FM ? 0 : CF::SA * 1024) + (row_of(J) + r32) * kScaleBytes;
  };
  constexpr int NM = CF::FM * CF::FN, NR = CF::FM + CF::FN;
  f32x16_t acc[CF::FM][CF::FN];
  int c_stage = 0, c_slot = 0;
  const auto next_stage = [&]() { c_stage = c_stage + 1 == CF::NST ? 0 : c_stage + 1; };
  const auto next_slot = [&]() { c_slot = c_slot + 1 == CF::NST ? 0 : c_slot + 1; };
  // The end of a K-tile: the next one has landed (at most the loads of the
  // NST - 2 K-tiles issued after it are outstanding), and every wave has read
  // this one.
  auto turn = [&]() __attribute__((always_inline)) {
    wait_loads_lds<(CF::NST - 2) * L>();
    block_barrier();
  };

  if constexpr (kHalves) {
    // In half ks of the K-tile lane l holds row l%32, columns 16 h .. + 15 and
    // 32 + 16 h .. + 15 of the half's 64 (h = l/32), and the exponent of its
    // block h.
    //
    // A K-tile is multiplied in four steps: the first half of the tile's rows in
    // its two halves of K, then the second.  Each operand register is read
    // again in the step behind its last use, so that one set of them does, and
    // a stage is read within three steps: from the step before its K-tile's
    // first to its second.  Its refill then has five steps to land; with the
    // K halves outermost (all rows in each) it had four (65536 rows over 16
    // groups of 4096 x 7168, operands of zeros, so that power does not limit the
    // clock: 1533 -> 1418 us; with values 1710 and 1741, at 1.7 GHz).
    constexpr int HM = CF::FM / 2, HN = HM * CF::FN, HL = L / 2;
    int32_t at[2][2];
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
      for (int e = 0; e < 2; ++e) at[ks][e] = r32 * KT + (((ks * 4 + e * 2 + h) ^ kc_swz(r32)) << 4);
    const uint32_t pick = 0x06040200u + 0x01010101u * h;  // bytes h and 2 + h of two words
    i32x8_t fa[2][CF::FM], fb[2][CF::FN];
    // the lane's exponents, two fragments to a word: byte 2 (f & 1) + ks is fragment f's in half ks of the K-tile
    int32_t sa[HM], sb[CF::FN / 2];
    Words8<CF> words;
    // Fragment J (A's first, then B's) of half ks.
    auto read = [&](auto jj, auto kk, const char* stage) __attribute__((always_inline)) {
      constexpr int J = decltype(jj)::value, ks = decltype(kk)::value;
      const char* p = stage + in_stage(J);
      const i32x4_t lo = *reinterpret_cast<const i32x4_t*>(p + at[ks][0]);
      const i32x4_t hi = *reinterpret_cast<const i32x4_t*>(p + at[ks][1]);
      const i32x8_t v = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
      if constexpr (J < CF::FM) fa[ks][J] = v;
      else fb[ks][J - CF::FM] = v;
    };
    auto read_words = [&](const char* slot) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < NR; ++j) words.v[j] = *reinterpret_cast<const uint32_t*>(slot + in_slot(j));
    };
    auto pack_words = [&]() __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < HM; ++j) sa[j] = (int32_t)__builtin_amdgcn_perm(words.v[2 * j + 1], words.v[2 * j], pick);
#pragma unroll
      for (int j = 0; j < CF::FN / 2; ++j)
        sb[j] = (int32_t)__builtin_amdgcn_perm(words.v[CF::FM + 2 * j + 1], words.v[CF::FM + 2 * j], pick);
    };
    // The MFMAs of row half mh in half ks, one per group, `work(group)` behind each.
    auto step4 = [&](auto zero, auto mm, auto kk, auto work) __attribute__((always_inline)) {
      static_for<0, HN>([&](auto xx) __attribute__((always_inline)) {
        constexpr int x = decltype(xx)::value, m = decltype(mm)::value * HM + x / CF::FN, n = x % CF::FN;
        constexpr int ks = decltype(kk)::value;
        acc[m][n] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(
            fb[ks][n], fa[ks][m], decltype(zero)::value ? f32x16_t{} : acc[m][n], 0, 0, n % 2 * 2 + ks, sb[n / 2],
            m % 2 * 2 + ks, sa[m / 2]);
        work(xx);
        __builtin_amdgcn_sched_barrier(0);
      });
    };
    // The MFMAs stay in front of this: left alone, the compiler sinks them past the branches of the
    // issue cursor, behind everything that they are to hide.
    auto hold = [&]() __attribute__((always_inline)) {
#pragma unroll
      for (int m = 0; m < CF::FM; ++m)
#pragma unroll
        for (int n = 0; n < CF::FN; ++n) {
          f32x16_t& v = acc[m][n];
          asm volatile("" : "+a"(v));
        }
    };
    // The fragments that a step reads, C of them over its groups: id(i) is the i-th.
    auto reads = [&](auto xx, auto cc, auto kk, const char* stage, auto id) __attribute__((always_inline)) {
      constexpr int x = decltype(xx)::value, C = decltype(cc)::value, G2 = (HN + 1) / 2;  // in the step's first half
      if constexpr (x < G2)
        static_for<x * C / G2, (x + 1) * C / G2>([&](auto i) __attribute__((always_inline)) {
          read(Int<decltype(id)::at(decltype(i)::value)>{}, kk, stage);
        });
    };
    struct RowsLow { static constexpr int at(int i) { return i; } };                                    // A, first row half
    struct RowsHigh { static constexpr int at(int i) { return HM + i; } };                              // A, second
    struct ColsAndLow { static constexpr int at(int i) { return i < CF::FN ? CF::FM + i : i - CF::FN; } };  // B, then A's first
    constexpr int kBoth = CF::FN + HM;
    // `end_` (the tile's last K-tile): its stage serves the epilogue before it is refilled.  A constant: the
    // compiler would sink the MFMAs past branches between them.
    auto ktile = [&](auto zero, auto end_, int32_t kt) __attribute__((always_inline)) {
      constexpr bool last = decltype(end_)::value;
      const char* stage = lds + c_stage * CF::STAGE;
      step4(zero, Int<0>{}, Int<0>{}, [&](auto x) __attribute__((always_inline)) { reads(x, Int<kBoth>{}, Int<1>{}, stage, ColsAndLow{}); });
      step4(Int<0>{}, Int<0>{}, Int<1>{}, [&](auto x) __attribute__((always_inline)) {
        reads(x, Int<HM>{}, Int<0>{}, stage, RowsHigh{});
        reads(x, Int<HM>{}, Int<1>{}, stage, RowsHigh{});
      });
      wait_lds();  // every wave has read this stage
      block_barrier();
      next_stage();
      const int32_t k4 = last ? 0 : (kt + 1) % kScaleTiles;
      if (k4 == 0) next_slot();
      step4(zero, Int<1>{}, Int<0>{}, [&](auto x) __attribute__((always_inline)) {
        constexpr int j = decltype(x)::value;
        if constexpr (!last) static_for<j * HL / HN, (j + 1) * HL / HN>(issue);
      });
      // the next K-tile has landed: what is outstanding was issued behind it
      if constexpr (last) wait_loads<(CF::NST - 2) * L>();
      else wait_loads<(CF::NST - 2) * L + HL>();
      block_barrier();
      const char* ahead = lds + c_stage * CF::STAGE;
      read_words(slots + c_slot * CF::SLOT + k4 * 4);
      step4(Int<0>{}, Int<1>{}, Int<1>{}, [&](auto x) __attribute__((always_inline)) {
        constexpr int j = decltype(x)::value;
        reads(x, Int<kBoth>{}, Int<0>{}, ahead, ColsAndLow{});
        if constexpr (!last) static_for<HL + j * (L - HL) / HN, HL + (j + 1) * (L - HL) / HN>(issue);
      });
      pack_words();
      hold();
      if constexpr (!last) {
        issue_scales();
        advance_issue();
      }
    };

    read_words(slots);
    static_for<0, kBoth>([&](auto i) __attribute__((always_inline)) { read(Int<ColsAndLow::at(decltype(i)::value)>{}, Int<0>{}, lds); });
    pack_words();
    for (int32_t tile = first; tile < end; tile += step) {
      ktile(Int<1>{}, Int<0>{}, 0);
      for (int32_t kt = 1; kt < nk - 1; ++kt) ktile(Int<0>{}, Int<0>{}, kt);
      ktile(Int<0>{}, Int<1>{}, nk - 1);
      char* free_stage = lds + (c_stage == 0 ? CF::NST - 1 : c_stage - 1) * CF::STAGE;  // the tile's last K-tile's
      Place place;
      decode(tile, place);
      epilogue<E, KIND, CF>(P, place, wm, wn, wave, lane, free_stage, nullptr, acc);
      issue_scales();
      static_for<0, L>(issue);
      advance_issue();
    }
  } else if constexpr (kWhole) {
    // One row tile per wave: few rows.  The weights' bytes bound a call with many copies.  With a few (one
    // token) a wave's way through its instructions does, one in 5 to 6 cycles: the next K-tile is read whole while
    // this one is multiplied, so that no wave waits for LDS, and a 32 x 64 tile is two waves' (fc1, per K-tile
    // of a token's 16: 0.74 us with one wave that reads a quarter ahead, 0.61 so, 0.50 with two waves).
    constexpr bool kNT = KIND == NT8;
    const uint32_t pick = 0x06040200u + 0x01010101u * h;  // bytes h and 2 + h of two words
    int32_t at[4];  // the lane's 16-byte chunk of each quarter: two make one of NT's operands
#pragma unroll
    for (int q = 0; q < 4; ++q) at[q] = r32 * KT + (((q * 2 + h) ^ kc_swz(r32)) << 4);
    struct KTile {
      i32x4_t v[4][NR];
      uint32_t words[NR];
    };
    KTile t0, t1;
    auto read = [&](KTile& to, const char* stage, const char* slot) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < NR; ++j) to.v[i][j] = *reinterpret_cast<const i32x4_t*>(stage + in_stage(j) + at[i]);
#pragma unroll
      for (int j = 0; j < NR; ++j) to.words[j] = *reinterpret_cast<const uint32_t*>(slot + in_slot(j));
    };
    // FC1: fragment J's values of half hh of the K-tile's eight
    Values8<CF> c0, c1;
    auto convert = [&](auto jj, auto hh, const KTile& from, Values8<CF>& to) __attribute__((always_inline)) {
      constexpr int J = decltype(jj)::value, q = decltype(hh)::value / 2, s = decltype(hh)::value % 2;
      const float scale = __uint_as_float(q < 3 ? from.words[J] << (q < 3 ? 23 - 8 * q : 0) : from.words[J] >> 1);
#pragma unroll
      for (int pair = 0; pair < 4; pair += 2) {
        const uint32_t four = (uint32_t)from.v[q][J][2 * s + pair / 2];
        const bf16x2_t lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(four, scale, false);
        const bf16x2_t hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(four, scale, true);
        to.v[J][2 * pair] = lo[0], to.v[J][2 * pair + 1] = lo[1];
        to.v[J][2 * pair + 2] = hi[0], to.v[J][2 * pair + 3] = hi[1];
      }
    };
    // K-tile kt from `cur`; `end_`: the tile's last, whose stage serves the epilogue before it is refilled.
    auto ktile = [&](auto zero, auto end_, int32_t kt, KTile& cur, KTile& next) __attribute__((always_inline)) {
      constexpr bool last = kNT && decltype(end_)::value;
      turn();
      next_stage();
      const int32_t k4 = kt + 1 < nk ? (kt + 1) % kScaleTiles : 0;
      if (k4 == 0) next_slot();
      if constexpr (!last) issue_scales();
      // the MFMAs of a step, one per column tile, and behind each what it hides
      constexpr int STEPS = kNT ? 2 : 8, MM = STEPS * CF::FN;
      static_for<0, MM>([&](auto xx) __attribute__((always_inline)) {
        constexpr int x = decltype(xx)::value, step_ = x / CF::FN, n = x % CF::FN;
        if constexpr (kNT) {
          const auto both = [&](int j) __attribute__((always_inline)) {
            const i32x4_t lo = cur.v[2 * step_][j], hi = cur.v[2 * step_ + 1][j];
            return i32x8_t{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
          };
          const int32_t sa = (int32_t)__builtin_amdgcn_perm(cur.words[0], cur.words[0], pick);
          const int32_t sb = (int32_t)__builtin_amdgcn_perm(cur.words[(n | 1) < CF::FN ? 1 + (n | 1) : 1 + n], cur.words[1 + (n & ~1)], pick);
          acc[0][n] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(
              both(1 + n), both(0), decltype(zero)::value && step_ == 0 ? f32x16_t{} : acc[0][n], 0, 0, n % 2 * 2 + step_, sb,
              step_, sa);
        } else {
          const Values8<CF>& now = step_ % 2 ? c1 : c0;
          acc[0][n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
              now.v[1 + n], now.v[0], decltype(zero)::value && step_ == 0 ? f32x16_t{} : acc[0][n], 0, 0, 0);
        }
        if constexpr (x == 0) read(next, lds + c_stage * CF::STAGE, slots + c_slot * CF::SLOT + k4 * 4);
        if constexpr (!last) static_for<x * L / MM, (x + 1) * L / MM>(issue);
        if constexpr (!kNT)
          static_for<n * NR / CF::FN, (n + 1) * NR / CF::FN>([&](auto j) __attribute__((always_inline)) {
            convert(j, Int<(step_ + 1) % 8>{}, step_ < 7 ? cur : next, step_ % 2 ? c0 : c1);
          });
        __builtin_amdgcn_sched_barrier(0);
      });
#pragma unroll
      for (int n = 0; n < CF::FN; ++n) {
        f32x16_t& v = acc[0][n];
        asm volatile("" : "+a"(v));  // the MFMAs stay in front of the branches
      }
      if constexpr (!last) advance_issue();
    };

    read(t0, lds, slots);
    if constexpr (!kNT) static_for<0, NR>([&](auto j) __attribute__((always_inline)) { convert(j, Int<0>{}, t0, c0); });
    for (int32_t tile = first; tile < end; tile += step) {
      ktile(Int<1>{}, Int<0>{}, 0, t0, t1);
      for (int32_t kt = 1; kt < nk - 1; kt += 2) {
        ktile(Int<0>{}, Int<0>{}, kt, t1, t0);
        ktile(Int<0>{}, Int<0>{}, kt + 1, t0, t1);
      }
      ktile(Int<0>{}, Int<1>{}, nk - 1, t1, t0);
      char* free_stage = lds + (c_stage == 0 ? CF::NST - 1 : c_stage - 1) * CF::STAGE;  // the tile's last K-tile's
      Place place;
      decode(tile, place);
      epilogue<E, KIND, CF>(P, place, wm, wn, wave, lane, free_stage, shared, acc);
      if constexpr (kNT) {
        issue_scales();
        static_for<0, L>(issue);
        advance_issue();
      }
    }
  } else {
    // In quarter q of the K-tile lane l holds row l%32, columns 16 h .. + 15 of
    // the quarter's 32: eight of them each for two bf16 MFMAs.
    int32_t at[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) at[q] = r32 * KT + (((q * 2 + h) ^ kc_swz(r32)) << 4);
    Codes8<CF> r0, r1;
    Words8<CF> words, upcoming;
    Values8<CF> c0, c1;
    auto read = [&](auto jj, auto qq, const char* stage, const char* slot, Codes8<CF>& to, Words8<CF>& w)
        __attribute__((always_inline)) {
      constexpr int J = decltype(jj)::value, q = decltype(qq)::value;
      to.v[J] = *reinterpret_cast<const i32x4_t*>(stage + in_stage(J) + at[q]);
      if constexpr (q == 0) w.v[J] = *reinterpret_cast<const uint32_t*>(slot + in_slot(J));
    };
    // Two values, Y of the 4 * NR pairs of half s of quarter q; the conversion takes the exponent field alone.
    auto convert = [&](auto yy, auto qq, auto ss, const Codes8<CF>& from, const Words8<CF>& w, Values8<CF>& to)
        __attribute__((always_inline)) {
      constexpr int J = order8<CF>(decltype(yy)::value / 4), pair = decltype(yy)::value % 4;
      constexpr int q = decltype(qq)::value, s = decltype(ss)::value;
      const float scale = __uint_as_float(q < 3 ? w.v[J] << (q < 3 ? 23 - 8 * q : 0) : w.v[J] >> 1);
      const bf16x2_t v =
          __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((uint32_t)from.v[J][2 * s + pair / 2], scale, pair % 2 == 1);
      to.v[J][2 * pair] = v[0];
      to.v[J][2 * pair + 1] = v[1];
    };
    // The MFMAs of half s of a quarter from `now`; meanwhile the next half's
    // values are converted, the codes after them read (s = 0) and the freed
    // stage refilled (loads).
    auto half = [&](auto zero, auto ss, const Values8<CF>& now, auto work) __attribute__((always_inline)) {
      static_for<0, NM>([&](auto xx) __attribute__((always_inline)) {
        constexpr int x = decltype(xx)::value, m = x / CF::FN, n = x % CF::FN;
        acc[m][n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(now.v[CF::FM + n], now.v[m],
                                                            decltype(zero)::value ? f32x16_t{} : acc[m][n], 0, 0, 0);
        work(xx);
        __builtin_amdgcn_sched_barrier(0);
      });
    };
    // Quarter q: its codes in `cur`, the first half's values in c0 when it
    // begins.  q = 3 reads the next K-tile, the next tile's first one behind the
    // tile's last (behind the block's last, zeros that nothing uses), and
    // refills the stage that this one has left.
    auto quarter = [&](auto zero, auto qq, const char* stage, const char* slot, const Codes8<CF>& cur, Codes8<CF>& next)
        __attribute__((always_inline)) {
      constexpr int q = decltype(qq)::value, NC = 4 * NR, qn = (q + 1) % 4;
      Words8<CF>& w = q == 3 ? upcoming : words;
      if constexpr (q == 3) issue_scales();
      half(zero, Int<0>{}, c0, [&](auto xx) __attribute__((always_inline)) {
        constexpr int x = decltype(xx)::value;
        static_for<x * NR / NM, (x + 1) * NR / NM>(
            [&](auto j) __attribute__((always_inline)) { read(Int<order8<CF>(decltype(j)::value)>{}, Int<qn>{}, stage, slot, next, w); });
        if constexpr (q == 3) static_for<x * L / NM, (x + 1) * L / NM>(issue);
        static_for<x * NC / NM, (x + 1) * NC / NM>(
            [&](auto y) __attribute__((always_inline)) { convert(y, qq, Int<1>{}, cur, words, c1); });
      });
      half(Int<0>{}, Int<1>{}, c1, [&](auto xx) __attribute__((always_inline)) {
        constexpr int x = decltype(xx)::value;
        static_for<x * NC / NM, (x + 1) * NC / NM>(
            [&](auto y) __attribute__((always_inline)) { convert(y, Int<qn>{}, Int<0>{}, next, w, c0); });
      });
      if constexpr (q == 3) words = upcoming;
    };
    auto ktile = [&](auto zero, int32_t kt) __attribute__((always_inline)) {
      const char* stage = lds + c_stage * CF::STAGE;
      quarter(zero, Int<0>{}, stage, nullptr, r0, r1);
      quarter(Int<0>{}, Int<1>{}, stage, nullptr, r1, r0);
      quarter(Int<0>{}, Int<2>{}, stage, nullptr, r0, r1);
      turn();
      next_stage();
      const int32_t k4 = kt + 1 < nk ? (kt + 1) % kScaleTiles : 0;
      if (k4 == 0) next_slot();
      quarter(Int<0>{}, Int<3>{}, lds + c_stage * CF::STAGE, slots + c_slot * CF::SLOT + k4 * 4, r1, r0);
      advance_issue();
    };

    static_for<0, NR>([&](auto j) __attribute__((always_inline)) { read(j, Int<0>{}, lds, slots, r0, words); });
    static_for<0, 4 * NR>([&](auto y) __attribute__((always_inline)) { convert(y, Int<0>{}, Int<0>{}, r0, words, c0); });
    for (int32_t tile = first; tile < end; tile += step) {
      ktile(Int<1>{}, 0);
      for (int32_t kt = 1; kt < nk; ++kt) ktile(Int<0>{}, kt);
      Place place;
      decode(tile, place);
      epilogue<E, KIND, CF>(P, place, wm, wn, wave, lane, nullptr, nullptr, acc);
    }
  }
  wait_loads<0>();
}

// ---------------------------------------------------------------------------
// Launches
// ---------------------------------------------------------------------------

int cu_count() {
  static std::atomic<int> cached{0};
  int cus = cached.load(std::memory_order_relaxed);
  if (cus == 0) {
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess) return -1;
    if (hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || cus <= 0) return -1;
    cached.store(cus, std::memory_order_relaxed);
  }
  return cus;
}

// The tilings of rows8_rule.h.
using Narrow32 = Cfg8<1, 2, 1, 1, 3, 3>;  // 32 x 64, a wave per 32 x 32
using Rows32 = Cfg8<1, 4, 1, 2, 3, 1>;    // 32 x 256, one wave per 32 x 64
using Rows128 = Cfg8<2, 2, 2, 2, 2, 2>;  // 128 x 128, 64 x 64
using Rows256 = Cfg8<2, 2, 4, 4, 2, 1>;  // 256 x 256, 128 x 128

// Tiles, and the cursor's step past the last one, are counted in 32 bits.
template <int KIND, class CF>
bool tiles_fit(const Params8& P, int cus) {
  const int64_t ntn = KIND == FC18 ? (P.I + CF::BN / 2 - 1) / (CF::BN / 2) : (P.N + CF::BN - 1) / CF::BN;
  return (P.M / CF::BM + P.G) * ntn <= INT32_MAX - cus * CF::BPC;
}

template <class E, int KIND, class CF>
int launch_cfg(const Params8& P, int cus, pmx_stream_t stream) {
  if (!tiles_fit<KIND, CF>(P, cus)) return PMX_ERR_SHAPE;
  rows8_grouped_gemm_kernel<E, KIND, CF><<<cus * CF::BPC, CF::NTH, 0, stream>>>(P);
  PMX_LAUNCH_CHECK();
  return PMX_OK;
}

template <class E, int KIND>
int launch(const Params8& P, pmx_stream_t stream) {
  const int cus = cu_count();
  if (cus <= 0) return PMX_ERR_HIP;
  switch (pmx::rows8_tiling(KIND, P.M, P.G, P.N, P.K, cus)) {
    case 0: return launch_cfg<E, KIND, Narrow32>(P, cus, stream);
    case Rows32::BM: return launch_cfg<E, KIND, Rows32>(P, cus, stream);
    case Rows128::BM: return launch_cfg<E, KIND, Rows128>(P, cus, stream);
    default: return launch_cfg<E, KIND, Rows256>(P, cus, stream);
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// What one buffer descriptor covers: offsets are 32 bits, the top one marks
// what lies outside.
bool one_window(int64_t rows, int64_t bytes) { return rows <= (int64_t)0x7fffffff / bytes; }

// The checks that both kinds share; PMX_OK to go on.
int check(const Params8& P) {
  if (P.G <= 0 || P.G > kMaxGroups || P.M < 0 || P.N <= 0 || P.K <= 0 || P.a_rows < 0) return PMX_ERR_ARG;
  if (P.K % 16 || P.M > INT32_MAX - 256 || P.a_rows > INT32_MAX) return PMX_ERR_SHAPE;
  const int64_t kgroups = (P.K + kScaleGroup - 1) / kScaleGroup;
  if (!one_window(P.N, P.K) || !one_window(P.N, kgroups * kScaleBytes) || !one_window(P.a_rows, kgroups * kScaleBytes) ||
      !one_window(P.row_token != nullptr ? P.a_rows : 256, P.K) || !one_window(256, 2 * P.N))
    return PMX_ERR_SHAPE;
  return PMX_OK;
}

template <int KIND>
bool any_tiles_fit(const Params8& P) {
  return tiles_fit<KIND, Narrow32>(P, 1024);  // the most tiles, and more CUs than there are
}

template <class E>
int nt_t(const void* a, const void* as, const void* b, const void* bs, const int32_t* offsets, int32_t G, int64_t M, int64_t N,
         int64_t K, void* c, void* c_low, pmx_stream_t stream) {
  Params8 P = {};
  P.a = (const uint8_t*)a, P.as = (const uint8_t*)as, P.a_rows = M;
  P.b = (const uint8_t*)b, P.bs = (const uint8_t*)bs;
  P.offsets = offsets, P.G = G, P.M = M, P.N = N, P.K = K, P.c = (bf16_t*)c, P.c_low = (uint8_t*)c_low;
  if (const int rc = check(P)) return rc;
  if (N % (E::kCode == kF24 ? 16 : 8)) return PMX_ERR_SHAPE;
  if (M == 0) return PMX_OK;
  if (!a || !as || !b || !bs || !offsets || !c || (E::kCode == kF24 && !c_low)) return PMX_ERR_ARG;
  if (!aligned16(a) || !aligned16(as) || !aligned16(b) || !aligned16(bs) || !aligned16(c) || !aligned16(c_low)) return PMX_ERR_SHAPE;
  return launch<E, NT8>(P, stream);
}

template <class E>
int fc1_t(const void* x, const void* xs, int64_t T, const int32_t* row_token, const void* w, const void* ws,
          const int32_t* offsets, int32_t G, int64_t A, int64_t H, int64_t I, const void* row_w, void* act, void* act_s,
          pmx_stream_t stream) {
  if (I <= 0 || I > INT32_MAX / 2) return PMX_ERR_ARG;
  Params8 P = {};
  P.a = (const uint8_t*)x, P.as = (const uint8_t*)xs, P.a_rows = T, P.row_token = row_token;
  P.b = (const uint8_t*)w, P.bs = (const uint8_t*)ws;
  P.offsets = offsets, P.G = G, P.M = A, P.N = 2 * I, P.K = H, P.I = I;
  P.q = (uint8_t*)act, P.qs = (uint8_t*)act_s, P.row_w = (const bf16_t*)row_w;
  if (const int rc = check(P)) return rc;
  if (I % 16) return PMX_ERR_SHAPE;
  if (A == 0) return PMX_OK;
  if (!x || !xs || !w || !ws || !offsets || !act || !act_s || (row_token == nullptr && T != A)) return PMX_ERR_ARG;
  if (!aligned16(x) || !aligned16(xs) || !aligned16(w) || !aligned16(ws) || !aligned16(act) || !aligned16(act_s))
    return PMX_ERR_SHAPE;
  return launch<E, FC18>(P, stream);
}

}  // namespace

// Whether a layer of T tokens, K copies each, fits both products and the sum (rows8_layer.hip asks before it launches anything).
int pmx_rows8_layer_check(int64_t T, int32_t K, int64_t H, int64_t I, int32_t C) {
  if (T < 0 || K <= 0 || H <= 0 || I <= 0 || C <= 0) return PMX_ERR_ARG;
  if (H % 16 || I % 16 || I > INT32_MAX / 2 || T > INT32_MAX / K || !grid_fits(T, rows8_sum_threads(H))) return PMX_ERR_SHAPE;
  static const int32_t some_map = 0;
  Params8 P = {};
  P.G = C, P.M = T * K;
  P.a_rows = T, P.row_token = &some_map, P.N = 2 * I, P.K = H, P.I = I;
  if (const int rc = check(P)) return rc;
  if (!any_tiles_fit<FC18>(P)) return PMX_ERR_SHAPE;
  P.a_rows = P.M, P.row_token = nullptr, P.N = H, P.K = I;
  if (const int rc = check(P)) return rc;
  return any_tiles_fit<NT8>(P) ? PMX_OK : PMX_ERR_SHAPE;
}

int pmx_rows8_group_gemm_nt_f24(const void* a, const void* a_scales, const void* b, const void* b_scales, const int32_t* offsets,
                                int32_t G, int64_t M, int64_t N, int64_t K, void* y_high, void* y_low, pmx_stream_t stream) {
  return nt_t<EltF24>(a, a_scales, b, b_scales, offsets, G, M, N, K, y_high, y_low, stream);
}

extern "C" {

#define PMX_ROWS8_GEMM_ENTRIES(SUFFIX, E)                                                                                   \
  int pmx_rows8_group_gemm_nt##SUFFIX(const void* a, const void* a_scales, const void* b, const void* b_scales,             \
                                      const int32_t* offsets, int32_t G, int64_t M, int64_t N, int64_t K, void* c,          \
                                      pmx_stream_t stream) {                                                                \
    return nt_t<E>(a, a_scales, b, b_scales, offsets, G, M, N, K, c, nullptr, stream);                                      \
  }                                                                                                                         \
  int pmx_rows8_gemm_fc1_swiglu##SUFFIX(const void* x, const void* x_scales, int64_t T, const int32_t* row_token,           \
                                        const void* w, const void* w_scales, const int32_t* offsets, int32_t G, int64_t A,  \
                                        int64_t H, int64_t I, const void* row_w, void* act, void* act_scales,               \
                                        pmx_stream_t stream) {                                                              \
    return fc1_t<E>(x, x_scales, T, row_token, w, w_scales, offsets, G, A, H, I, row_w, act, act_scales, stream);           \
  }

PMX_ROWS8_GEMM_ENTRIES(, EltBF16)
PMX_ROWS8_GEMM_ENTRIES(_f16, EltF16)

}  // extern "C"
