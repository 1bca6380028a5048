// Loads and stores of a lane's 8 neighbouring columns of a row, wherever the row
// starts and ends; what the kernels that write rows in 8 or 4 bits and read them
// back share.
#pragma once

#include "common.h"

namespace {

typedef uint32_t u32x4_a2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x2_a1 __attribute__((ext_vector_type(2), aligned(1)));

__device__ __forceinline__ uint4 ld16(const bf16_t* p) {
  const u32x4_a2 v = __builtin_nontemporal_load(reinterpret_cast<const u32x4_a2*>(p));
  return make_uint4(v.x, v.y, v.z, v.w);
}
__device__ __forceinline__ void st16(bf16_t* p, const uint4 v) {
  *reinterpret_cast<u32x4_a2*>(p) = u32x4_a2{v.x, v.y, v.z, v.w};
}
__device__ __forceinline__ uint2 ld8(const uint8_t* p) {
  const u32x2_a1 v = __builtin_nontemporal_load(reinterpret_cast<const u32x2_a1*>(p));
  return make_uint2(v.x, v.y);
}
__device__ __forceinline__ void st8(uint8_t* p, const uint2 v) {
  *reinterpret_cast<u32x2_a1*>(p) = u32x2_a1{v.x, v.y};
}

// The row's last chunk, where fewer than 8 columns are left: the 8 columns that
// end with the row, shifted, so that every lane makes the same load (element by
// element the one lane held up its wave: 1531 rows of 1412 columns took 11.3 us
// to write, of 1408 columns 7.1); its stores go out as 4, 2 and 1 elements.

// Columns c .. c+7 of a row of N, c < N (elements past the row: zero).
__device__ __forceinline__ uint4 load8(const bf16_t* row, int64_t c, int64_t N) {
  if (N < 8) {
    uint64_t w[2] = {0, 0};
    for (int j = 0; c + j < N; ++j) w[j / 4] |= (uint64_t)row[c + j] << (16 * (j & 3));
    return make_uint4((uint32_t)w[0], (uint32_t)(w[0] >> 32), (uint32_t)w[1], (uint32_t)(w[1] >> 32));
  }
  const int64_t at = c + 8 <= N ? c : N - 8;
  const uint4 v = ld16(row + at);
  const int s = 16 * (int)(c - at);
  if (s == 0) return v;
  uint64_t lo = (uint64_t)v.y << 32 | v.x, hi = (uint64_t)v.w << 32 | v.z;
  lo = s < 64 ? lo >> s | hi << (64 - s) : hi >> (s - 64);
  hi = s < 64 ? hi >> s : 0;
  return make_uint4((uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32));
}
__device__ __forceinline__ uint2 load8(const uint8_t* row, int64_t c, int64_t N) {
  uint64_t w = 0;
  if (N < 8) {
    for (int j = 0; c + j < N; ++j) w |= (uint64_t)row[c + j] << (8 * j);
  } else {
    const int64_t at = c + 8 <= N ? c : N - 8;
    const uint2 v = ld8(row + at);
    w = ((uint64_t)v.y << 32 | v.x) >> (8 * (int)(c - at));
  }
  return make_uint2((uint32_t)w, (uint32_t)(w >> 32));
}

typedef uint64_t u64_a1 __attribute__((aligned(1)));
typedef uint32_t u32_a1 __attribute__((aligned(1)));
typedef uint16_t u16_a1 __attribute__((aligned(1)));

__device__ __forceinline__ void store8(bf16_t* row, int64_t c, int64_t N, const uint4 v) {
  bf16_t* p = row + c;
  if (c + 8 <= N) {
    st16(p, v);
    return;
  }
  const int n = (int)(N - c);
  uint64_t w = (uint64_t)v.y << 32 | v.x;
  if (n & 4) *reinterpret_cast<u64_a1*>(p) = w, p += 4, w = (uint64_t)v.w << 32 | v.z;
  if (n & 2) *reinterpret_cast<u32_a1*>(p) = (uint32_t)w, p += 2, w >>= 32;
  if (n & 1) *p = (bf16_t)w;
}
__device__ __forceinline__ void store8(uint8_t* row, int64_t c, int64_t N, const uint2 v) {
  uint8_t* p = row + c;
  if (c + 8 <= N) {
    st8(p, v);
    return;
  }
  const int n = (int)(N - c);
  uint32_t w = v.x;
  if (n & 4) *reinterpret_cast<u32_a1*>(p) = w, p += 4, w = v.y;
  if (n & 2) *reinterpret_cast<u16_a1*>(p) = (uint16_t)w, p += 2, w >>= 16;
  if (n & 1) *p = (uint8_t)w;
}

// Values beyond the type's range (a fp16 block whose largest value rounded up
// past 65504, or the top binade of bf16) become its largest finite value.
template <class E>
__device__ __forceinline__ float to_range(float v) {
  const float most = E::kCode == EltF16::kCode ? 65504.0f : __uint_as_float(0x7f7f0000u);
  return __builtin_fabsf(v) > most ? __builtin_copysignf(most, v) : v;  // NaN compares false
}

}  // namespace
