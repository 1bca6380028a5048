// The dense gated block: what its sources share, not part of the C ABI.
#pragma once

#include "gate.h"

// A weight gradient c [M, N] = a [K, M]^T b [K, N]; splits > 1: the K rows in chunks, their fp32 sums in parts.
struct GatedWgradCall {
  const void *a, *b;
  int64_t M, N, chunk;
  int32_t splits;
  void* c;
  float* parts;
};

// The block's products on the grouped GEMM's kernels (a build of
// grouped_gemm.hip of their own; _f16: fp16 tensors).  Checked by the caller.
#define PMX_GATED_GEMMS(SUFFIX)                                                                                              \
  /* act [T, I] (and, unless null, gates [T, I / 4, 2, 4] in fp32) of x [T, H], w [2I, H] */                                 \
  __attribute__((visibility("hidden"))) int pmx_gated_fc1##SUFFIX(const void* x, const void* w, int64_t T, int64_t H,        \
                                                                  int64_t I, float a, float b, float* gates, void* act,      \
                                                                  pmx_stream_t stream);                                      \
  /* c [M, N] = a [M, K] b [N, K]^T */                                                                                       \
  __attribute__((visibility("hidden"))) int pmx_gated_nt##SUFFIX(const void* a, const void* b, int64_t M, int64_t N,         \
                                                                 int64_t K, void* c, pmx_stream_t stream);                   \
  /* c [M, N] = a [M, K] b [K, N] */                                                                                         \
  __attribute__((visibility("hidden"))) int pmx_gated_nn##SUFFIX(const void* a, const void* b, int64_t M, int64_t N,         \
                                                                 int64_t K, void* c, pmx_stream_t stream);                   \
  /* dgu [T, 2I] from dout [T, N], w [N, I] and gates; left: null, or up to 64 rows, what dgu's rounding leaves */           \
  __attribute__((visibility("hidden"))) int pmx_gated_dgate##SUFFIX(const void* dout, const void* w, const float* gates,     \
                                                                    int64_t T, int64_t N, int64_t I, float a, float b,       \
                                                                    void* dgu, void* left, pmx_stream_t stream);             \
  /* a gradient on 256 x 256 tiles */                                                                                        \
  __attribute__((visibility("hidden"))) int pmx_gated_tn##SUFFIX(const GatedWgradCall& w, int64_t K, pmx_stream_t stream);   \
  /* one or two on 128 x 128 tiles, whole */                                                                                 \
  __attribute__((visibility("hidden"))) int pmx_gated_tn_small##SUFFIX(const GatedWgradCall* w, int32_t n, int64_t K,        \
                                                                       pmx_stream_t stream);
PMX_GATED_GEMMS()
PMX_GATED_GEMMS(_f16)
