// The gates of the dense gated block: x sigmoid(x (a + b x^2)).
//   silu        a = 1,                b = 0
//   gelu, tanh  a = 2 sqrt(2 / pi),   b = 0.044715 a      (tanh(z) = 2 sigmoid(2 z) - 1)
//   quick gelu  a = 1.702,            b = 0
// One formula with two numbers, so that a kernel has no branch on the gate.
#pragma once

#include "common.h"

namespace {

struct Gate {
  float a, b;

  // (x^2 only where it cannot overflow: far before 2^40 the sigmoid is 0 or 1, and
  // its slope 0, which times an infinite square would be NaN.)
  __device__ __forceinline__ float square(float x) const {
    const float c = __builtin_amdgcn_fmed3f(x, -0x1p40f, 0x1p40f);
    return c * c;
  }
  __device__ __forceinline__ float sigmoid(float x, float square) const { return sigmoid_f32(x * __builtin_fmaf(b, square, a)); }
  __device__ __forceinline__ float value(float x) const { return x * sigmoid(x, square(x)); }

  // Of value(g) * u, from its gradient d: with s the sigmoid, value' = s + g s (1 - s) (a + 3 b g^2).
  __device__ __forceinline__ void gradients(float d, float g, float u, float& dg, float& du) const {
    const float q = square(g), s = sigmoid(g, q), v = g * s;
    dg = d * u * __builtin_fmaf(v * (1.0f - s), __builtin_fmaf(3.0f * b, q, a), s);
    du = d * v;
  }
};

}  // namespace
