// What the grouped GEMM kernels share: buffer descriptors, buffer->LDS loads
// counted by hand, the block barrier, wave-uniform values, compile-time loops.
#pragma once

#include "common.h"

namespace {

constexpr uint32_t kOOB = 0x80000000u;  // buffer offset that always fails the range check
constexpr uint32_t kRsrcWord3 = 0x00020000u;

constexpr int kNumXcd = 8;  // compute dies, each with an L2; blocks go round-robin over them

#define LDS_PTR(p) ((__attribute__((address_space(3))) void*)(p))

__device__ __forceinline__ __amdgpu_buffer_rsrc_t make_rsrc(const void* base, uint64_t bytes) {
  const uint32_t n = bytes > 0x7fffffffull ? 0x7fffffffu : (uint32_t)bytes;
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), (short)0, (int)n, (int)kRsrcWord3);
}

// 16-byte chunk swizzle of the 128-byte rows of K-contiguous tiles: 16
// consecutive rows read at one logical chunk hit 16 distinct (row parity,
// chunk) bank groups.
__device__ __forceinline__ int kc_swz(int row) { return (row >> 1) & 7; }

// Wave-uniform copies (SGPRs) of values every lane holds alike: tile
// bookkeeping read from LDS or memory would otherwise stay in VGPRs, and
// descriptor selections on it would become branches around each load.
__device__ __forceinline__ int32_t uni(int32_t v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ int64_t uni64(int64_t v) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)((uint64_t)v >> 32));
  return (int64_t)(((uint64_t)hi << 32) | lo);
}

// One buffer->LDS instruction: 64 lanes x 16 bytes land contiguously at `dst`
// (M0 holds the wave's LDS address).  Written as inline asm so that the
// compiler does not track it: its own LDS-DMA bookkeeping cannot tell the
// pipeline stages apart and would wait for younger stages before every LDS
// read.  Completion is tracked by hand (wait_loads) and published to the
// other waves by block_barrier, both of which clobber memory; this asm does
// not, so LDS reads of other stages may be scheduled across it.
__device__ __forceinline__ void dma16(__amdgpu_buffer_rsrc_t r, char* dst, uint32_t voff, uint32_t soff) {
  const uint32_t m0 = (uint32_t)(uintptr_t)LDS_PTR(dst);
  asm volatile("buffer_load_dwordx4 %0, %1, %2 offen lds" ::"v"(voff), "s"(r), "s"(soff), "{m0}"(m0));
}

// Compile-time loop: f(Int<I>{}) for I = B .. E-1, so that accumulator
// indices stay constants however large the unrolled body grows.
template <int V>
struct Int {
  static constexpr int value = V;
};
template <int B, int E, typename F>
__device__ __forceinline__ void static_for(F&& f) {
  if constexpr (B < E) {
    f(Int<B>{});
    static_for<B + 1, E>(f);
  }
}

// Wait until at most PENDING of this wave's vector memory operations (its
// buffer->LDS loads, and any stores since) are in flight.
template <int PENDING>
__device__ __forceinline__ void wait_loads() {
  static_assert(PENDING >= 0 && PENDING <= 63, "vmcnt is 6 bits");
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(PENDING) : "memory");
}

// Same, and this wave's LDS reads and writes have completed.
template <int PENDING>
__device__ __forceinline__ void wait_loads_lds() {
  static_assert(PENDING >= 0 && PENDING <= 63, "vmcnt is 6 bits");
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(PENDING) : "memory");
}

// Wait until this wave's LDS reads and writes have completed.
__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// Workgroup barrier that neither the compiler's memory model nor its
// scheduler moves anything across: memory operations stay on their side (the
// asm clobbers memory), and so do the MFMAs, so that every LDS read consumed
// before the barrier has returned by the time the wave reaches it.
__device__ __forceinline__ void block_barrier() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

}  // namespace
