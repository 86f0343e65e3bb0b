// Device helpers of the kernels that stage tiles in LDS by
// global_load_lds_dwordx4 and pipeline their loops by hand.
#pragma once

#include "qdec_common.h"

namespace qdec {

__device__ __forceinline__ uint4 ld16(const uint16_t *p) { return *reinterpret_cast<const uint4 *>(p); }

// 16 bytes per lane from global memory into LDS at byte address lds_addr +
// 16 * lane (global_load_lds_dwordx4; M0 holds the wave's LDS address).
// Issued from inline assembly so the compiler does not make every later LDS
// read wait for all of these loads; the caller waits (vmcnt) and
// synchronises the workgroup itself.
// M0 is saved and restored around the load.
__device__ __forceinline__ void dma16(const void *g, uint32_t lds_addr) {
  uint32_t saved;
  asm volatile(
      "s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off\n\ts_mov_b32 m0, %0"
      : "=&s"(saved)
      : "v"(g), "s"(__builtin_amdgcn_readfirstlane(lds_addr))
      : "memory");
}
// The same from a wave-uniform base and a lane offset, without saving M0
// (for kernels none of whose other instructions read it).
__device__ __forceinline__ void dma16s(const char *base, uint32_t lane_off, uint32_t lds_addr) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
               :: "v"(lane_off), "s"(base), "s"(lds_addr)
               : "memory");
}
// ... and saving M0.
__device__ __forceinline__ void dma16u(const void *base, uint32_t lane_off, uint32_t lds_addr) {
  uint32_t saved;
  asm volatile(
      "s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2\n\ts_mov_b32 m0, %0"
      : "=&s"(saved)
      : "v"(lane_off), "s"(base), "s"(lds_addr)
      : "memory");
}
__device__ __forceinline__ uint32_t lds_addr(const void *p) { return (uint32_t)reinterpret_cast<uintptr_t>(p); }

// Keeps the computation of v where it stands among other pins and volatile
// assembly (the compiler moves plain arithmetic and MFMAs past scheduling
// barriers before it schedules).
template <class V>
__device__ __forceinline__ void pin(V &v) {
  asm volatile("" : "+v"(v));
}

// Maximum of v over the lane pairs (l, l ^ 16) and then (l, l ^ 32), with
// gfx950's row swaps instead of LDS permutes: after v_permlane16_swap the two
// outputs hold the odd / even 16-lane rows exchanged, after
// v_permlane32_swap the two halves, so the maximum of both outputs is the
// pairwise maximum in every lane.
__device__ __forceinline__ float max_xor16_32(float v) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// s_waitcnt encodings (gfx9 family): vmcnt in bits 3:0 and 15:14, expcnt
// 6:4, lgkmcnt 11:8; the other counters at their maximum (no wait).
constexpr int vmcnt_enc(int n) { return (n & 15) | ((n >> 4) << 14) | (7 << 4) | (15 << 8); }
constexpr int kVmcnt0 = vmcnt_enc(0);

template <int V>
struct Int {
  static constexpr int value = V;
};

}  // namespace qdec
