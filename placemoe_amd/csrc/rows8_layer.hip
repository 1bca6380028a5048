// The expert layer over 8-bit weights in one call: its five steps enqueued one
// behind the other over one workspace.  A decode step's kernels are a few
// microseconds each; made from Python one by one, the calls took longer than
// the kernels (one token through 8 of 160 copies of 2048 x 768: 72 us against
// 42 us of kernels).

#include "rows8.h"

namespace {

// Where the workspace's parts begin (bytes, multiples of 256).  The routing's
// own workspace is first: its status word is the workspace's.
struct Parts {
  size_t route, phys, pos, counts, offsets, row_token, row_w, x, xs, act, acts, y_high, y_low, total;
};

// false: more than a size_t holds (or no such layer).
bool parts_of(int64_t T, int32_t K, int64_t H, int64_t I, int32_t C, Parts& p) {
  if (pmx_rows8_layer_check(T, K, H, I, C) != PMX_OK) return false;
  const uint64_t A = (uint64_t)T * K, t = (uint64_t)T, h = (uint64_t)H, i = (uint64_t)I;
  const uint64_t gh = (h + kScaleGroup - 1) / kScaleGroup, gi = (i + kScaleGroup - 1) / kScaleGroup;
  uint64_t at = 0;
  const auto take = [&](uint64_t bytes) {
    const uint64_t here = at;
    at += (bytes + 255) / 256 * 256;
    return (size_t)here;
  };
  // within 2^31 rows of 2^31 bytes each by the check: no sum here wraps
  p.route = take(pmx_route_workspace_bytes((int64_t)A, C));
  p.phys = take(A * 4);
  p.pos = take(A * 4);
  p.counts = take((uint64_t)C * 4);
  p.offsets = take(((uint64_t)C + 1) * 4);
  p.row_token = take(A * 4);
  p.row_w = take(A * 2);
  p.x = take(t * h);
  p.xs = take(gh * t * kScaleBytes);
  p.act = take(A * i);
  p.acts = take(gi * A * kScaleBytes);
  p.y_high = take(A * h * 2);
  p.y_low = take(A * h);
  p.total = at;
  return true;
}

template <class E>
int layer_t(const void* hidden, const void* w, const int64_t* sel, const int64_t* M, const int64_t* src, int32_t src_const,
            int32_t S, int32_t E_, const void* gate_up, const void* gate_up_scales, const void* down, const void* down_scales,
            int64_t T, int32_t K, int64_t H, int64_t I, int32_t C, void* out, int32_t* counts, void* workspace,
            size_t workspace_bytes, int32_t* status_host, pmx_stream_t stream) {
  constexpr bool f16 = E::kCode == EltF16::kCode;
  if (const int rc = pmx_rows8_layer_check(T, K, H, I, C)) return rc;
  Parts p;
  if (!parts_of(T, K, H, I, C, p)) return PMX_ERR_SHAPE;
  if (T > 0 && (!hidden || !w || !out || !gate_up || !gate_up_scales || !down || !down_scales)) return PMX_ERR_ARG;
  if (!workspace || workspace_bytes < p.total) return PMX_ERR_ARG;
  const auto aligned = [](const void* q) { return (reinterpret_cast<uintptr_t>(q) & 15u) == 0; };
  if (!aligned(workspace) || !aligned(gate_up) || !aligned(gate_up_scales) || !aligned(down) || !aligned(down_scales) ||
      !aligned(out))
    return PMX_ERR_SHAPE;
  char* ws = static_cast<char*>(workspace);
  int32_t* pos = reinterpret_cast<int32_t*>(ws + p.pos);
  int32_t* offsets = reinterpret_cast<int32_t*>(ws + p.offsets);
  int32_t* row_token = reinterpret_cast<int32_t*>(ws + p.row_token);
  int32_t* n = counts != nullptr ? counts : reinterpret_cast<int32_t*>(ws + p.counts);
  const size_t route_bytes = pmx_route_workspace_bytes(T * K, C);
  int rc = pmx_route_reported(sel, M, src, src_const, S, E_, T, K, C, reinterpret_cast<int32_t*>(ws + p.phys), n, offsets, pos,
                              ws + p.route, route_bytes, status_host, stream);
  if (rc != PMX_OK || T == 0) return rc;
  rc = (f16 ? pmx_rows8_quantize_routed_f16 : pmx_rows8_quantize_routed)(hidden, pos, w, T, K, H, ws + p.x, ws + p.xs,
                                                                          row_token, ws + p.row_w, stream);
  if (rc != PMX_OK) return PMX_ERR_HIP;  // the sizes have been checked: a launch failed
  rc = (f16 ? pmx_rows8_gemm_fc1_swiglu_f16 : pmx_rows8_gemm_fc1_swiglu)(ws + p.x, ws + p.xs, T, row_token, gate_up,
                                                                          gate_up_scales, offsets, C, T * K, H, I, ws + p.row_w,
                                                                          ws + p.act, ws + p.acts, stream);
  if (rc != PMX_OK) return PMX_ERR_HIP;
  rc = pmx_rows8_group_gemm_nt_f24(ws + p.act, ws + p.acts, down, down_scales, offsets, C, T * K, H, I, ws + p.y_high,
                                   ws + p.y_low, stream);
  if (rc != PMX_OK) return PMX_ERR_HIP;
  rc = pmx_rows8_sum_f24(ws + p.y_high, ws + p.y_low, pos, T, K, H, f16, out, stream);
  return rc != PMX_OK ? PMX_ERR_HIP : PMX_OK;
}

}  // namespace

extern "C" {

size_t pmx_rows8_layer_workspace_bytes(int64_t T, int32_t K, int64_t H, int64_t I, int32_t C) {
  Parts p;
  return parts_of(T, K, H, I, C, p) ? p.total : 0;
}

#define PMX_ROWS8_LAYER(SUFFIX, ELT)                                                                                      \
  int pmx_rows8_layer##SUFFIX(const void* hidden, const void* w, const int64_t* sel, const int64_t* M, const int64_t* src, \
                              int32_t src_const, int32_t S, int32_t E, const void* gate_up, const void* gate_up_scales,    \
                              const void* down, const void* down_scales, int64_t T, int32_t K, int64_t H, int64_t I,       \
                              int32_t C, void* out, int32_t* counts, void* workspace, size_t workspace_bytes,              \
                              int32_t* status_host, pmx_stream_t stream) {                                                 \
    return layer_t<ELT>(hidden, w, sel, M, src, src_const, S, E, gate_up, gate_up_scales, down, down_scales, T, K, H, I, C, \
                        out, counts, workspace, workspace_bytes, status_host, stream);                                     \
  }

PMX_ROWS8_LAYER(, EltBF16)
PMX_ROWS8_LAYER(_f16, EltF16)

}  // extern "C"
