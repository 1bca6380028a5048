// The dense gated block's products: host side of the build of grouped_gemm.hip
// with -DPMX_GATED.
#include "gated.h"
#include "gated_rule.h"

namespace {

template <int KIND>
int launch_rows(const GemmParams& P, hipStream_t stream) {
  const int64_t ntn = KIND == KIND_FC1 ? (P.I + 127) / 128 : (P.N + BN - 1) / BN;
  if (ntn >= (int64_t)1 << 19) return PMX_ERR_SHAPE;  // the LDS tile table keeps an n-tile index in 19 bits
  const int grid = grid_size();
  if (grid <= 0) return PMX_ERR_HIP;
  const int tiling = P.left != nullptr ? Few64::BM : pmx::gated_tiling(KIND, P.M, P.N, P.K, grid);
  if (tiling == Few64::BM) return launch_few<KIND, Few64>(P, grid, stream);
  if (tiling == Few128::BM) return launch_few<KIND, Few128>(P, grid, stream);
  const bool fast = P.K % BK == 0;
  if constexpr (KIND == KIND_FC1 || KIND == KIND_NNS) {  // whole K-tiles: the rule takes smaller tiles otherwise
    w4::grouped_gemm_w4_kernel<KIND><<<grid, w4::NT, 0, stream>>>(P);
  } else if (!fast) {
    grouped_gemm_kernel<KIND, kBM><<<grid, NTHREADS, 0, stream>>>(P);
  } else if constexpr (KIND == KIND_NT) {  // the kernels of few copies with many rows, as in grouped_gemm.hip
    grouped_gemm_kernel<KIND, kBM, false, true, true><<<grid, NTHREADS, 0, stream>>>(P);
  } else {
    grouped_gemm_kernel<KIND, kBM, false, true><<<grid, NTHREADS, 0, stream>>>(P);
  }
  PMX_LAUNCH_CHECK();
  return PMX_OK;
}

GemmParams dense(const void* a, const void* b, int64_t M, int64_t N, int64_t K, int64_t ldb) {
  GemmParams P = {};
  P.a = one(a, 0, K);
  P.b = one(b, 0, ldb);
  P.G = 1, P.chunk = P.rows = (uint32_t)M;
  P.M = M, P.N = N, P.K = K;
  P.ldc = N;
  return P;
}

}  // namespace

int PMX_GEMM_FN(pmx_gated_fc1)(const void* x, const void* w, int64_t T, int64_t H, int64_t I, float a, float b, float* gates,
                               void* act, pmx_stream_t stream) {
  if (!fits_rsrc(I, H) || !fits_rsrc(kBM, H)) return PMX_ERR_SHAPE;
  GemmParams P = dense(x, w, T, 2 * I, H, H);
  P.b.p1 = P.b.p0 + I * H;
  P.b.split = I;
  P.I = I;
  P.gates = gates;
  P.act = static_cast<bf16_t*>(act);
  P.gate = {a, b};
  return launch_rows<KIND_FC1>(P, stream);
}

int PMX_GEMM_FN(pmx_gated_nt)(const void* a, const void* b, int64_t M, int64_t N, int64_t K, void* c, pmx_stream_t stream) {
  if (!fits_rsrc(N, K) || !fits_rsrc(kBM, K)) return PMX_ERR_SHAPE;
  GemmParams P = dense(a, b, M, N, K, K);
  P.c0 = static_cast<bf16_t*>(c);
  return launch_rows<KIND_NT>(P, stream);
}

int PMX_GEMM_FN(pmx_gated_nn)(const void* a, const void* b, int64_t M, int64_t N, int64_t K, void* c, pmx_stream_t stream) {
  if (!fits_rsrc(K, N) || !fits_rsrc(kBM, K)) return PMX_ERR_SHAPE;
  GemmParams P = dense(a, b, M, N, K, N);
  P.c0 = static_cast<bf16_t*>(c);
  return launch_rows<KIND_NN>(P, stream);
}

int PMX_GEMM_FN(pmx_gated_dgate)(const void* dout, const void* w, const float* gates, int64_t T, int64_t N, int64_t I, float a,
                                 float b, void* dgu, void* left, pmx_stream_t stream) {
  if (!fits_rsrc(N, I) || !fits_rsrc(kBM, N)) return PMX_ERR_SHAPE;
  GemmParams P = dense(dout, w, T, I, N, I);
  P.I = I;
  P.c0 = static_cast<bf16_t*>(dgu);
  P.left = static_cast<bf16_t*>(left);
  P.ldc = 2 * I;
  P.gates = const_cast<float*>(gates);
  P.gate = {a, b};
  return launch_rows<KIND_NNS>(P, stream);
}

namespace {
GemmParams wgrad(const GatedWgradCall& w, int64_t K) {
  GemmParams P = {};
  P.a = one(w.a, 0, w.M);
  P.b = one(w.b, 0, w.N);
  P.G = w.splits, P.chunk = (uint32_t)w.chunk, P.rows = (uint32_t)K;
  P.K = K, P.M = w.M, P.N = w.N;
  P.c0 = P.c1 = static_cast<bf16_t*>(w.c);
  P.parts = w.splits > 1 ? w.parts : nullptr;
  P.cgs = w.splits > 1 ? w.M * w.N : 0;
  P.ldc = w.N;
  P.csplit = INT64_MAX;
  return P;
}
}  // namespace

int PMX_GEMM_FN(pmx_gated_tn)(const GatedWgradCall& w, int64_t K, pmx_stream_t stream) {
  if (!fits_rsrc(BK, w.M) || !fits_rsrc(BK, w.N)) return PMX_ERR_SHAPE;
  const int grid = grid_size();
  if (grid <= 0) return PMX_ERR_HIP;
  const GemmParams P = wgrad(w, K);
  // the four-wave kernel: every row of the operands, and the gradient, within 31-bit offsets
  if (fits_rsrc(K, w.M) && fits_rsrc(K, w.N) && fits_rsrc(2 * w.M, w.N)) {
    w4::grouped_gemm_w4_kernel<KIND_TN><<<grid, w4::NT, 0, stream>>>(P);
  } else if (w.splits > 1) {
    return PMX_ERR_SHAPE;
  } else {
    grouped_gemm_kernel<KIND_TN, kBM><<<grid, NTHREADS, 0, stream>>>(P);
  }
  PMX_LAUNCH_CHECK();
  return PMX_OK;
}

int PMX_GEMM_FN(pmx_gated_tn_small)(const GatedWgradCall* w, int32_t n, int64_t K, pmx_stream_t stream) {
  fr::Two two = {};
  int64_t first = 0, blocks = 0;
  for (int32_t i = 0; i < n; ++i) {
    if (!fits_rsrc(BK, w[i].M) || !fits_rsrc(BK, w[i].N)) return PMX_ERR_SHAPE;
    two.p[i] = wgrad(w[i], K);
    const int64_t tiles = ((w[i].M + fr::kWgT - 1) / fr::kWgT) * ((w[i].N + fr::kWgT - 1) / fr::kWgT);
    blocks += (tiles + kNumXcd - 1) / kNumXcd * kNumXcd;
    if (i == 0) first = blocks;
  }
  if (blocks >= (int64_t)1 << 24) return PMX_ERR_SHAPE;
  const int grid = grid_size();
  if (grid <= 0) return PMX_ERR_HIP;
  if (pmx::gated_wgrad_two(blocks, K, grid)) fr::wgrad_grouped_gemm_kernel<2><<<(unsigned)blocks, fr::kWgNT, 0, stream>>>(two, (uint32_t)first);
  else fr::wgrad_grouped_gemm_kernel<1><<<(unsigned)blocks, fr::kWgNT, 0, stream>>>(two, (uint32_t)first);
  PMX_LAUNCH_CHECK();
  return PMX_OK;
}
