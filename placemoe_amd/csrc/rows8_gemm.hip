// The grouped products (rows8_gemm.h) of 8-bit rows with 8-bit weights.

#include "rows8_gemm.h"

namespace {
using Rows8x8 = Fmt<8, 8>;
}

// rows8_layer.hip asks before it launches anything.
int pmx_rows8_layer_check(int64_t T, int32_t K, int64_t H, int64_t I, int32_t C) { return layer_check<Rows8x8>(T, K, H, I, C); }

int pmx_rows8_group_gemm_nt_f24(const void* a, const void* a_scales, const void* b, const void* b_scales, const int32_t* offsets,
                                int32_t G, int64_t M, int64_t N, int64_t K, void* y_high, void* y_low, pmx_stream_t stream) {
  return nt_t<EltF24, Rows8x8>(a, a_scales, b, b_scales, offsets, G, M, N, K, y_high, y_low, stream);
}

extern "C" {

#define PMX_ROWS8_GEMM_ENTRIES(SUFFIX, E)                                                                                   \
  int pmx_rows8_group_gemm_nt##SUFFIX(const void* a, const void* a_scales, const void* b, const void* b_scales,             \
                                      const int32_t* offsets, int32_t G, int64_t M, int64_t N, int64_t K, void* c,          \
                                      pmx_stream_t stream) {                                                                \
    return nt_t<E, Rows8x8>(a, a_scales, b, b_scales, offsets, G, M, N, K, c, nullptr, stream);                                      \
  }                                                                                                                         \
  int pmx_rows8_gemm_fc1_swiglu##SUFFIX(const void* x, const void* x_scales, int64_t T, const int32_t* row_token,           \
                                        const void* w, const void* w_scales, const int32_t* offsets, int32_t G, int64_t A,  \
                                        int64_t H, int64_t I, const void* row_w, void* act, void* act_scales,               \
                                        pmx_stream_t stream) {                                                              \
    return fc1_t<E, Rows8x8>(x, x_scales, T, row_token, w, w_scales, offsets, G, A, H, I, row_w, act, act_scales, stream);           \
  }

PMX_ROWS8_GEMM_ENTRIES(, EltBF16)
PMX_ROWS8_GEMM_ENTRIES(_f16, EltF16)

}  // extern "C"
