// The dense gated block: out = (gate(x Wg^T) * (x Wu^T)) Wd^T, forward and
// backward, with Wg and Wu the two halves of one matrix.
//
// Many tokens: the grouped GEMM's kernels, built for one group that is the whole
// call (gated_gemm.h):
//   forward   act = fc1 (both projections, gate and product in its epilogue);  out = act Wd^T
//   backward  dgu = the gate's gradients of (dout Wd), in its epilogue;  dWd = dout^T act;
//             dW = dgu^T x;  dx = dgu W
// act and dgu are rounded to 16 bits, being operands of 16-bit products: each
// such rounding is as large as the outputs' own, so that every output is 1.4 times as
// far from the definition in 64 bits as one rounded once is.  The gate and up
// sums between the forward and the backward are kept in fp32: in 16 bits, as dout Wd
// staged in 16, they made dx and dW twice as far (0.0034, rounded once 0.0017, now 0.0023, in bf16).  As the
// accumulators hold them they go to memory and back without a turn through LDS: 8192
// tokens of 7168 x 2048, forward and backward, 1883 -> 1777 us.
// A weight gradient's tiles are few where
// the weights are small: its rows are cut into chunks whose fp32 sums are then
// added in order (sum_parts_kernel).
//
// Few tokens: a call reads every weight once, and what counts is how many bytes
// are on their way.  256 x 256 tiles would put 16 of them on the whole chip.
// Here a block has 16 rows of the weights (fc1: 8 gate rows and their 8 up rows)
// for all tokens, its waves a share of the columns each, straight from memory to
// the matrix instruction (16 weight rows x 16 tokens, 32 columns); their sums
// meet in LDS.  Bound: HBM; from some tens of tokens on, their being read again by
// every block.  One token through 7168 x 2048: 22.9 us, 3.8 TB/s of weights (a large
// copy: 4.8), on 64 x 128 tiles 72; 64 tokens 66 and 80.  (32 weight rows per block:
// as fast for few, 30% slower where that leaves less than a block per CU.)

#include "gated.h"
#include "gated_rule.h"

namespace {

constexpr int kFewWaves = 8;  // (4 or 16, and 4 to 16 steps on their way: within 5%)

template <class E>
__device__ __forceinline__ f32x4_t mfma16(const uint4& w, const uint4& x, const f32x4_t& c) {
  if constexpr (E::kCode == EltF16::kCode) {
    typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, w), __builtin_bit_cast(f16x8_t, x), c, 0, 0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, w), __builtin_bit_cast(bf16x8_t, x), c, 0, 0, 0);
  }
}

// The sums of 16 weight rows (wrow: the lane's, that of row lane % 16) with
// tokens 0 .. 16 FT - 1 of x [T, K]: red[wave][weight row][token], after a barrier.
// K a multiple of 8.  Lanes past K, and past T, multiply zeros.  A wave has
// kSteps steps of 32 columns on their way; a token's sum is the same however many there are.
// PLANES 2: x [2, T, K], whose two planes add up to the tokens, summed apart: of an infinite weight the second,
// of either sign, is left out.
template <class E, int FT, int PLANES>
__device__ __forceinline__ void few_products(const bf16_t* wrow, const bf16_t* x, int64_t T, int64_t K, int lane, int wave,
                                             float (*red)[16][16 * FT]) {
  constexpr int kSteps = FT == 1 ? 8 : FT == 2 ? 6 : 4;
  const int t = lane & 15, quarter = lane >> 4;
  bool token[FT];
  const bf16_t* xrow[FT];
#pragma unroll
  for (int f = 0; f < FT; ++f) {
    token[f] = f * 16 + t < T;
    xrow[f] = x + (token[f] ? f * 16 + t : 0) * K;
  }
  const int64_t chunks = K / 8;
  f32x4_t acc[PLANES][FT] = {};
  for (int64_t c0 = (int64_t)wave * 4; c0 < chunks; c0 += 4 * kFewWaves * kSteps) {
    uint4 w[kSteps], v[kSteps][PLANES][FT];
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const int64_t c = c0 + s * (4 * kFewWaves) + quarter;
      const bool in = c < chunks;
      w[s] = in ? ld_stream(wrow + c * 8) : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int p = 0; p < PLANES; ++p)
#pragma unroll
        for (int f = 0; f < FT; ++f)
          v[s][p][f] = in && token[f] ? *reinterpret_cast<const uint4*>(xrow[f] + p * T * K + c * 8) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
#pragma unroll
      for (int p = 0; p < PLANES; ++p)
#pragma unroll
        for (int f = 0; f < FT; ++f) acc[p][f] = mfma16<E>(w[s], v[s][p][f], acc[p][f]);
  }
  // lane: token lane % 16, weight rows 4 (lane / 16) .. + 3
#pragma unroll
  for (int f = 0; f < FT; ++f)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float sum = acc[0][f][e];
      if constexpr (PLANES == 2) sum += __builtin_isfinite(sum) ? acc[1][f][e] : 0.f;
      red[wave][quarter * 4 + e][f * 16 + t] = sum;
    }
  __syncthreads();
}

// act among up to 16 tokens: rounded, and what that leaves kept behind it for fc2.  There one rounded value may be most
// of an output (two fp16 tokens of 280 x 64: out 0.00037 from 64 bits; so 0.00021, as rounded once).  One token
// through 7168 x 2048 takes 0.6 us more, 16 tokens 33.4 for 29.7; 64 would take 81 for 64.
// The weights' gradients of so few tokens are sums of as few products: they read act and dgu so too, each as twice
// the rows, beside two copies of the tokens' other rows.
constexpr int64_t kTwoValues = 16;
template <int FT>
constexpr int act_planes() { return FT * 16 <= kTwoValues ? 2 : 1; }

// fc1: eight columns of act (and gates) per block.
template <class E, int FT>
__global__ __launch_bounds__(64 * kFewWaves) void gated_few_fc1_kernel(const bf16_t* __restrict__ x, const bf16_t* __restrict__ w,
                                                                       int64_t T, int64_t H, int64_t I, Gate gate,
                                                                       float* __restrict__ gates, bf16_t* __restrict__ act) {
  __shared__ float red[kFewWaves][16][16 * FT];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t j0 = (int64_t)blockIdx.x * 8;
  const int r = lane & 15;
  few_products<E, FT, 1>(w + ((r < 8 ? 0 : I) + j0 + r % 8) * H, x, T, H, lane, wave, red);
  const int j = threadIdx.x & 7;
  for (int64_t t = threadIdx.x >> 3; t < T && t < 16 * FT; t += 8 * kFewWaves) {
    float g = 0.f, u = 0.f;
#pragma unroll
    for (int i = 0; i < kFewWaves; ++i) g += red[i][j][t], u += red[i][8 + j][t];
    if (gates != nullptr) {  // four columns' gates, then their ups
      float* const to = gates + (t * I + j0 + (j & 4)) * 2 + (j & 3);
      to[0] = g, to[4] = u;
    }
    const float v = gate.value(g) * u;
    const bf16_t high = (bf16_t)E::from_f32(v);
    [[maybe_unused]] const float left = v - E::to_f32(high);
    act[t * I + j0 + j] = high;
    if constexpr (act_planes<FT>() == 2) act[(T + t) * I + j0 + j] = __builtin_isfinite(left) ? (bf16_t)E::from_f32(left) : (bf16_t)0;
  }
}

// fc2: 16 columns of out per block.
template <class E, int FT>
__global__ __launch_bounds__(64 * kFewWaves) void gated_few_fc2_kernel(const bf16_t* __restrict__ act, const bf16_t* __restrict__ w,
                                                                       int64_t T, int64_t N, int64_t I, bf16_t* __restrict__ out) {
  __shared__ float red[kFewWaves][16][16 * FT];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t n0 = (int64_t)blockIdx.x * 16;
  const int64_t n = n0 + (lane & 15);
  few_products<E, FT, act_planes<FT>()>(w + (n < N ? n : N - 1) * I, act, T, I, lane, wave, red);
  const int j = threadIdx.x & 15;
  if (n0 + j >= N) return;
  for (int64_t t = threadIdx.x >> 4; t < T && t < 16 * FT; t += 4 * kFewWaves) {
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < kFewWaves; ++i) sum += red[i][j][t];
    out[t * N + n0 + j] = (bf16_t)E::from_f32(sum);
  }
}

template <class E, int FT>
int few_forward(const void* x, const void* gate_up, const void* down, int64_t T, int64_t H, int64_t I, int64_t N, const Gate& gate,
                float* gates, void* act, void* out, pmx_stream_t stream) {
  gated_few_fc1_kernel<E, FT><<<(unsigned)(I / 8), 64 * kFewWaves, 0, stream>>>((const bf16_t*)x, (const bf16_t*)gate_up, T, H, I, gate,
                                                                                gates, (bf16_t*)act);
  PMX_LAUNCH_CHECK();
  gated_few_fc2_kernel<E, FT><<<(unsigned)((N + 15) / 16), 64 * kFewWaves, 0, stream>>>((const bf16_t*)act, (const bf16_t*)down, T, N, I,
                                                                                        (bf16_t*)out);
  PMX_LAUNCH_CHECK();
  return PMX_OK;
}

// The chunks' sums, in order: a thread per four neighbouring elements.
template <class E>
__global__ __launch_bounds__(256) void sum_parts_kernel(const float* __restrict__ parts, int32_t splits, int64_t size,
                                                        bf16_t* __restrict__ out) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= size) return;  // a multiple of 8
  f32x4_t sum = *reinterpret_cast<const f32x4_t*>(parts + i);
  for (int32_t s = 1; s < splits; ++s) sum += *reinterpret_cast<const f32x4_t*>(parts + s * size + i);
  *reinterpret_cast<uint2*>(out + i) = make_uint2(E::pack2(sum[0], sum[1]), E::pack2(sum[2], sum[3]));
}

// Eight values, zeros in the place of infinities and NaN.
template <class E>
__device__ __forceinline__ uint4 finite8(const uint4 v) {
  constexpr uint32_t kInf = E::kCode == EltF16::kCode ? 0x7c00u : 0x7f80u;
  const auto two = [](uint32_t w) {
    return ((w & kInf) == kInf ? 0u : w & 0xffffu) | ((w >> 16 & kInf) == kInf ? 0u : w & 0xffff0000u);
  };
  return make_uint4(two(v.x), two(v.y), two(v.z), two(v.w));
}

// Two copies, one behind the other, of a (na chunks of 16 bytes) and of b: the second is multiplied with what a
// rounding left, of either sign, and has what is finite alone.
template <class E>
__global__ __launch_bounds__(256) void two_copies_kernel(const uint4* __restrict__ a, int64_t na, uint4* __restrict__ a2,
                                                         const uint4* __restrict__ b, int64_t nb, uint4* __restrict__ b2) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i < na) {
    a2[i] = a[i], a2[na + i] = finite8<E>(a[i]);
  } else if (i - na < nb) {
    b2[i - na] = b[i - na], b2[nb + i - na] = finite8<E>(b[i - na]);
  }
}

bool gate_of(int32_t gate, Gate& g) {
  constexpr float kGelu = 1.5957691216057308f;  // 2 sqrt(2 / pi)
  switch (gate) {
    case PMX_GATE_SILU: g = {1.0f, 0.0f}; return true;
    case PMX_GATE_GELU_TANH: g = {kGelu, kGelu * 0.044715f}; return true;
    case PMX_GATE_QUICK_GELU: g = {1.702f, 0.0f}; return true;
    default: return false;
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// One descriptor holds offsets below 2^31 bytes.
bool one_window(int64_t rows, int64_t cols) { return rows < (int64_t)0x7fffffff / 2 / cols; }

// Sizes that every product of the block takes; PMX_OK to go on.
int check(int64_t T, int64_t H, int64_t I, int64_t N) {
  if (T < 0 || H <= 0 || I <= 0 || N <= 0) return PMX_ERR_ARG;
  if (H % 8 || I % 8 || N % 8 || T > INT32_MAX - 256 || I > INT32_MAX / 2) return PMX_ERR_SHAPE;
  const int64_t I2 = 2 * I;
  // whole weights through one descriptor, 256 rows of every operand
  if (!one_window(I2, H) || !one_window(N, I) || !one_window(256, I2) || !one_window(256, H) || !one_window(256, N)) return PMX_ERR_SHAPE;
  return PMX_OK;
}

constexpr int64_t kCus = 256;  // of the rules here: the same for the workspace and the call

// How a weight gradient [M, N] over K rows runs; on small tiles where the operands pass what one descriptor holds (a
// chunk's kernel has one for each).
struct Wgrad {
  bool small;
  int64_t chunk;
  int32_t splits;
};
Wgrad wgrad_of(int64_t K, int64_t M, int64_t N) {
  const pmx::GatedWgrad w = pmx::gated_wgrad(K, M, N, kCus);
  if (!one_window(K, M) || !one_window(K, N) || !one_window(2 * M, N)) return {w.small, pmx::gated_chunk(K, 1), 1};
  const int64_t chunk = pmx::gated_chunk(K, w.splits);
  return {w.small, chunk, (int32_t)((K + chunk - 1) / chunk)};
}

// The backward's workspace: dgu (up to kTwoValues tokens: and what its rounding left), two copies of dout and of x
// there, then the fp32 sums of one weight gradient's chunks.
int64_t wgrad_rows(int64_t T) { return T <= kTwoValues ? 2 * T : T; }
size_t dgu_bytes(int64_t T, int64_t I) { return ((size_t)wgrad_rows(T) * 2 * I * 2 + 255) / 256 * 256; }
size_t copies_bytes(int64_t T, int64_t cols) { return T <= kTwoValues ? ((size_t)2 * T * cols * 2 + 255) / 256 * 256 : 0; }
size_t parts_bytes(int64_t K, int64_t M, int64_t N) {
  const Wgrad w = wgrad_of(K, M, N);
  return w.splits > 1 ? (size_t)w.splits * M * N * 4 : 0;
}

template <class E>
struct Gemms;
template <>
struct Gemms<EltBF16> {
  static constexpr auto fc1 = pmx_gated_fc1;
  static constexpr auto nt = pmx_gated_nt, nn = pmx_gated_nn;
  static constexpr auto dgate = pmx_gated_dgate;
  static constexpr auto tn = pmx_gated_tn;
  static constexpr auto tn_small = pmx_gated_tn_small;
};
template <>
struct Gemms<EltF16> {
  static constexpr auto fc1 = pmx_gated_fc1_f16;
  static constexpr auto nt = pmx_gated_nt_f16, nn = pmx_gated_nn_f16;
  static constexpr auto dgate = pmx_gated_dgate_f16;
  static constexpr auto tn = pmx_gated_tn_f16;
  static constexpr auto tn_small = pmx_gated_tn_small_f16;
};

template <class E>
int forward_t(const void* x, const void* gate_up, const void* down, int64_t T, int64_t H, int64_t I, int64_t N, int32_t kind,
              float* gates, void* act, void* out, pmx_stream_t stream) {
  Gate gate;
  if (!gate_of(kind, gate)) return PMX_ERR_ARG;
  if (const int rc = check(T, H, I, N)) return rc;
  if (T == 0) return PMX_OK;
  if (!x || !gate_up || !down || !act || !out) return PMX_ERR_ARG;
  if (!aligned16(x) || !aligned16(gate_up) || !aligned16(down) || !aligned16(gates) || !aligned16(act) || !aligned16(out)) return PMX_ERR_SHAPE;
  if (pmx::gated_few(T, H, I, N, kCus)) {
    if (T <= 16) return few_forward<E, 1>(x, gate_up, down, T, H, I, N, gate, gates, act, out, stream);
    if (T <= 32) return few_forward<E, 2>(x, gate_up, down, T, H, I, N, gate, gates, act, out, stream);
    return few_forward<E, 4>(x, gate_up, down, T, H, I, N, gate, gates, act, out, stream);
  }
  // The sizes have been checked: what fails from here on is a launch.
  if (Gemms<E>::fc1(x, gate_up, T, H, I, gate.a, gate.b, gates, act, stream) != PMX_OK) return PMX_ERR_HIP;
  return Gemms<E>::nt(act, down, T, N, I, out, stream) != PMX_OK ? PMX_ERR_HIP : PMX_OK;
}

// The gradients `w`, one or two, over K rows: those on small tiles in one launch.
template <class E>
int weight_gradients(GatedWgradCall* w, int n, int64_t K, float* parts, pmx_stream_t stream) {
  GatedWgradCall small[2];
  int few = 0;
  for (int i = 0; i < n; ++i) {
    const Wgrad how = wgrad_of(K, w[i].M, w[i].N);
    w[i].chunk = how.chunk, w[i].splits = how.splits, w[i].parts = parts;
    if (how.small) {
      small[few++] = w[i];
      continue;
    }
    if (Gemms<E>::tn(w[i], K, stream) != PMX_OK) return PMX_ERR_HIP;
    if (how.splits > 1) {
      const int64_t size = w[i].M * w[i].N;
      sum_parts_kernel<E><<<(unsigned)((size / 4 + 255) / 256), 256, 0, stream>>>(parts, how.splits, size, (bf16_t*)w[i].c);
      PMX_LAUNCH_CHECK();
    }
  }
  return few > 0 ? Gemms<E>::tn_small(small, few, K, stream) : PMX_OK;
}

template <class E>
int backward_t(const void* dout, const void* x, const void* gate_up, const void* down, const float* gates, const void* act, int64_t T,
               int64_t H, int64_t I, int64_t N, int32_t kind, void* dx, void* dgate_up, void* ddown, void* workspace,
               size_t workspace_bytes, pmx_stream_t stream) {
  Gate gate;
  if (!gate_of(kind, gate)) return PMX_ERR_ARG;
  if (const int rc = check(T, H, I, N)) return rc;
  if (T == 0) return PMX_OK;
  if (!dout || (!dx && !dgate_up && !ddown)) return PMX_ERR_ARG;
  if (((dx || dgate_up) && (!down || !gates)) || (dgate_up && !x) || (dx && !gate_up) || (ddown && !act)) return PMX_ERR_ARG;
  const void* all[] = {dout, x, gate_up, down, gates, act, dx, dgate_up, ddown, workspace};
  for (const void* p : all)
    if (!aligned16(p)) return PMX_ERR_SHAPE;
  if (!workspace || workspace_bytes < pmx_gated_ffn_workspace_bytes(T, H, I, N)) return PMX_ERR_ARG;
  void* dgu = workspace;
  char* at = static_cast<char*>(workspace) + dgu_bytes(T, I);
  char* const dout2 = at;
  char* const x2 = at += copies_bytes(T, N);
  float* parts = reinterpret_cast<float*>(at += copies_bytes(T, H));
  const bool two = T <= kTwoValues;
  if (two && (ddown || dgate_up)) {
    const int64_t na = ddown ? T * N / 8 : 0, nb = dgate_up ? T * H / 8 : 0;
    two_copies_kernel<E><<<(unsigned)((na + nb + 255) / 256), 256, 0, stream>>>((const uint4*)dout, na, (uint4*)dout2, (const uint4*)x,
                                                                               nb, (uint4*)x2);
    PMX_LAUNCH_CHECK();
  }
  int rc = PMX_OK;
  if (dx || dgate_up)
    rc = Gemms<E>::dgate(dout, down, gates, T, N, I, gate.a, gate.b, dgu, two ? (bf16_t*)dgu + T * 2 * I : nullptr, stream);
  GatedWgradCall w[2];
  int n = 0;
  if (ddown) w[n++] = {two ? dout2 : dout, act, N, I, 0, 0, ddown, nullptr};
  if (dgate_up) w[n++] = {dgu, two ? x2 : x, 2 * I, H, 0, 0, dgate_up, nullptr};
  if (rc == PMX_OK) rc = weight_gradients<E>(w, n, wgrad_rows(T), parts, stream);
  if (rc == PMX_OK && dx) rc = Gemms<E>::nn(dgu, gate_up, T, H, 2 * I, dx, stream);
  return rc != PMX_OK ? PMX_ERR_HIP : PMX_OK;
}

}  // namespace

extern "C" {

size_t pmx_gated_ffn_workspace_bytes(int64_t T, int64_t H, int64_t I, int64_t N) {
  if (check(T, H, I, N) != PMX_OK || T == 0) return 0;
  const size_t a = parts_bytes(wgrad_rows(T), N, I), b = parts_bytes(wgrad_rows(T), 2 * I, H);
  return dgu_bytes(T, I) + copies_bytes(T, N) + copies_bytes(T, H) + (a > b ? a : b);
}

#define PMX_GATED_FFN(SUFFIX, E)                                                                                            \
  int pmx_gated_ffn_fwd##SUFFIX(const void* x, const void* gate_up, const void* down, int64_t T, int64_t H, int64_t I,      \
                                int64_t N, int32_t gate, float* gates, void* act, void* out, pmx_stream_t stream) {         \
    return forward_t<E>(x, gate_up, down, T, H, I, N, gate, gates, act, out, stream);                                       \
  }                                                                                                                         \
  int pmx_gated_ffn_bwd##SUFFIX(const void* dout, const void* x, const void* gate_up, const void* down, const float* gates, \
                                const void* act, int64_t T, int64_t H, int64_t I, int64_t N, int32_t gate, void* dx,        \
                                void* dgate_up, void* ddown, void* workspace, size_t workspace_bytes, pmx_stream_t stream) { \
    return backward_t<E>(dout, x, gate_up, down, gates, act, T, H, I, N, gate, dx, dgate_up, ddown, workspace,              \
                         workspace_bytes, stream);                                                                          \
  }

PMX_GATED_FFN(, EltBF16)
PMX_GATED_FFN(_f16, EltF16)

}  // extern "C"
