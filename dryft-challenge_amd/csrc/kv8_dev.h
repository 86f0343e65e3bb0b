// Arithmetic of the 8-bit KV cache, shared by its kernels.
//
// A row x of D channels is held as q = round(127 x / top), top = max|x|, ties to
// even, and scale = top / 127; it stands for q * scale, off by half a step or
// less.  (One scale for each token and head: a scale over several tokens would
// have to grow as louder ones arrive, rounding what is there a second time, and
// a row's bits would depend on how many rows its pass had.)  127 x of a bf16 x has 15
// bits, so in fp32 it is exact and only the division rounds: quotients that
// are halves, as of x = top / 2, come out as such, and no other quotient of two
// bf16 numbers is nearer to one than 2^-16 of itself (127 * 254 / 255 = 126.502), 2^7
// times what the refined quotient below can be off by.  A row with an infinity or
// a NaN gets the scale NaN, one with top below 2^-100, whose reciprocals would
// leave fp32's range, the scale 0.
#pragma once

#include "qdec_common.h"

namespace qdec {

constexpr float kKv8Tiny = 7.8886090522101180541e-31f;  // 2^-100

typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));

__device__ __forceinline__ float kv8_scale(float top, bool finite) {
  return finite ? (top < kKv8Tiny ? 0.f : top / 127.f) : __builtin_nanf("");
}
// The low bytes of four words.
__device__ __forceinline__ uint32_t low_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __builtin_amdgcn_perm(b, a, 0x0c0c0400u) | __builtin_amdgcn_perm(d, c, 0x04000c0cu);
}

// Rounding of a row's values.  127 x / top as (127 / 256) x / (top / 256), which keeps
// 127 x in range; the quotient by one step of refinement, within 2^-23 of itself, which leaves a
// quotient that fp32 can hold as it is; rounded by adding 1.5 * 2^23, whose sum's low bits are
// the whole number.  A row held as zeros (and inf * 0 = NaN) has the reciprocal 0.
struct Kv8Div {
  float div, rcp;
  __device__ __forceinline__ Kv8Div() {}
  __device__ __forceinline__ Kv8Div(float top, bool finite) {
    const bool held = finite && top >= kKv8Tiny;
    div = held ? top * 0.00390625f : 0.f;
    rcp = held ? __builtin_amdgcn_rcpf(div) : 0.f;
    rcp = __builtin_fmaf(__builtin_fmaf(-div, rcp, 1.f), rcp, rcp);
  }
  // An int8 in the low byte.
  __device__ __forceinline__ uint32_t one(float x) const {
    const float a = 0.49609375f * x, q = a * rcp;
    return __float_as_uint(__builtin_fmaf(__builtin_fmaf(-q, div, a), rcp, q) + 12582912.f);
  }
  __device__ __forceinline__ uint32_t four(float x0, float x1, float x2, float x3) const {
    return low_bytes(one(x0), one(x1), one(x2), one(x3));
  }
  // Lane I's of this lane's 16-lane row.
  template <int I>
  __device__ __forceinline__ Kv8Div at() const {
    Kv8Div r;
    r.div = dpp_f<0x150 + I>(div);
    r.rcp = dpp_f<0x150 + I>(rcp);
    return r;
  }
};

}  // namespace qdec
