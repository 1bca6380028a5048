// The grouped products (rows8_gemm.h) with weights in 4 bits: of rows in 8 bits
// (fc1 with SwiGLU, fc2 and plain products), and of rows in 4.

#include "rows4.h"
#include "rows8_gemm.h"

namespace {
using Rows8x4 = Fmt<8, 4>;
using Rows4x4 = Fmt<4, 4>;
}  // namespace

// rows8_layer.hip asks before it launches anything.
int pmx_rows4_layer_check(int64_t T, int32_t K, int64_t H, int64_t I, int32_t C) { return layer_check<Rows8x4>(T, K, H, I, C); }

int pmx_rows4_group_gemm_nt_f24(const void* a, const void* a_scales, const void* b, const void* b_scales, const int32_t* offsets,
                                int32_t G, int64_t M, int64_t N, int64_t K, void* y_high, void* y_low, pmx_stream_t stream) {
  return nt_t<EltF24, Rows8x4>(a, a_scales, b, b_scales, offsets, G, M, N, K, y_high, y_low, stream);
}

extern "C" {

#define PMX_ROWS4_GEMM_ENTRIES(SUFFIX, E)                                                                                   \
  int pmx_rows4_group_gemm_nt##SUFFIX(const void* a, const void* a_scales, int32_t a_bits, const void* b,                   \
                                      const void* b_scales, const int32_t* offsets, int32_t G, int64_t M, int64_t N,        \
                                      int64_t K, void* c, pmx_stream_t stream) {                                            \
    if (a_bits == 8) return nt_t<E, Rows8x4>(a, a_scales, b, b_scales, offsets, G, M, N, K, c, nullptr, stream);            \
    if (a_bits == 4) return nt_t<E, Rows4x4>(a, a_scales, b, b_scales, offsets, G, M, N, K, c, nullptr, stream);            \
    return PMX_ERR_ARG;                                                                                                     \
  }                                                                                                                         \
  int pmx_rows4_gemm_fc1_swiglu##SUFFIX(const void* x, const void* x_scales, int64_t T, const int32_t* row_token,           \
                                        const void* w, const void* w_scales, const int32_t* offsets, int32_t G, int64_t A,  \
                                        int64_t H, int64_t I, const void* row_w, void* act, void* act_scales,               \
                                        pmx_stream_t stream) {                                                              \
    return fc1_t<E, Rows8x4>(x, x_scales, T, row_token, w, w_scales, offsets, G, A, H, I, row_w, act, act_scales, stream);  \
  }

PMX_ROWS4_GEMM_ENTRIES(, EltBF16)
PMX_ROWS4_GEMM_ENTRIES(_f16, EltF16)

}  // extern "C"
