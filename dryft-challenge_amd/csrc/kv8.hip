// The 8-bit KV cache written from a bf16 slab (kv8_store) and read back into one
// (kv8_load).  Both are copies: what bounds them is the bytes they move, 3 per
// element.
#include "kv8_dev.h"
#include "qdec_kernels.h"

namespace qdec {

namespace {

constexpr int kGroup = 16;  // slots of one wave: a 16-slot group of the V layout
constexpr int kWaves = 4;

__device__ __forceinline__ float bf_at(const uint4 &v, int i) {
  const uint32_t w = i < 2 ? v.x : i < 4 ? v.y : i < 6 ? v.z : v.w;
  return (i & 1) ? hi16(w) : lo16(w);
}

// One wave per 16-slot group: keys 8 channels to a lane (16 / 8 lanes to a row),
// values 8 slots of a channel to a lane, as both slabs have them.
template <int D>
__global__ void __launch_bounds__(64 * kWaves) kv8_store_kernel(const Kv8CopyParams p) {
  const int lane = threadIdx.x & 63;
  const int64_t unit = (int64_t)blockIdx.x * kWaves + (threadIdx.x >> 6);
  const int g0 = p.pos0 / kGroup;
  const int64_t cell = unit / p.groups;  // b * nkv + kvh
  if (cell >= p.cells) return;
  const int s0 = (g0 + (int)(unit - cell * p.groups)) * kGroup, s1 = p.pos0 + p.n;

  // ---- keys
  constexpr int LPR = D / 8, RPW = 64 / LPR;
  const uint16_t *ks = p.k_slab + (size_t)cell * p.slab_cap * D;
  int8_t *k8 = p.k8 + (size_t)cell * p.cap * D;
  float *kscale = p.k_scale + (size_t)cell * p.cap;
#pragma unroll
  for (int i = 0; i < kGroup / RPW; ++i) {
    const int slot = s0 + i * RPW + lane / LPR, ch = lane % LPR * 8;
    const bool in = slot >= p.pos0 && slot < s1;
    const uint4 raw = in ? *reinterpret_cast<const uint4 *>(ks + (size_t)slot * D + ch) : zero4();
    float x[8];
    unpack8(raw, x);
    float top = 0.f;
    bool fin = true;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      top = fmaxf(top, fabsf(x[e]));
      fin &= finite_f(x[e]);
    }
    top = fmaxf(top, dpp_f<0xB1>(top));
    top = fmaxf(top, dpp_f<0x4E>(top));
    top = fmaxf(top, dpp_f<0x141>(top));
    if constexpr (LPR == 16) top = fmaxf(top, dpp_f<0x140>(top));
    const uint64_t bad = __ballot(!fin) >> (lane & ~(LPR - 1));
    fin = (bad & ((1ull << LPR) - 1)) == 0;
    const Kv8Div div(top, fin);
    const uint2 q = make_uint2(div.four(x[0], x[1], x[2], x[3]), div.four(x[4], x[5], x[6], x[7]));
    if (in) {
      *reinterpret_cast<uint2 *>(k8 + (size_t)slot * D + ch) = q;
      if (lane % LPR == 0) kscale[slot] = kv8_scale(top, fin);
    }
  }

  // ---- values: lane takes channels lane + 64 j, slots s0 .. s0 + 15
  constexpr int CPL = D / 64;
  const uint16_t *vs = p.v_slab + (size_t)cell * p.slab_cap * D;
  int8_t *v8 = p.v8 + (size_t)cell * p.cap * D;
  float *vscale = p.v_scale + (size_t)cell * p.cap;
  uint4 raw[CPL][2];
#pragma unroll
  for (int j = 0; j < CPL; ++j)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int s = s0 + 8 * h;  // 8 slots of the slab, which has whole groups of 8
      raw[j][h] = s < p.slab_cap ? *reinterpret_cast<const uint4 *>(vs + ((size_t)(s >> 3) * D + lane + 64 * j) * 8) : zero4();
    }
  uint32_t q[CPL][4] = {};
#pragma unroll
  for (int i = 0; i < kGroup; ++i) {
    float x[CPL], top = 0.f;
    bool fin = true;
#pragma unroll
    for (int j = 0; j < CPL; ++j) {
      x[j] = bf_at(raw[j][i >> 3], i & 7);
      top = fmaxf(top, fabsf(x[j]));
      fin &= finite_f(x[j]);
    }
    top = wave_max(top);
    fin = __all(fin);
    const Kv8Div div(top, fin);
#pragma unroll
    for (int j = 0; j < CPL; ++j) q[j][i >> 2] |= (div.one(x[j]) & 0xffu) << (8 * (i & 3));
    const int slot = s0 + i;
    if (lane == 0 && slot >= p.pos0 && slot < s1) vscale[slot] = kv8_scale(top, fin);
  }
  const bool whole = s0 >= p.pos0 && s0 + kGroup <= s1;
#pragma unroll
  for (int j = 0; j < CPL; ++j) {
    int8_t *dst = v8 + ((size_t)(s0 >> 4) * D + lane + 64 * j) * kGroup;
    if (whole)
      *reinterpret_cast<uint4 *>(dst) = make_uint4(q[j][0], q[j][1], q[j][2], q[j][3]);
    else
#pragma unroll
      for (int i = 0; i < kGroup; ++i)
        if (s0 + i >= p.pos0 && s0 + i < s1) dst[i] = (int8_t)(q[j][i >> 2] >> (8 * (i & 3)));
  }
}

__device__ __forceinline__ float s8f(uint32_t w, int i) { return (float)(int8_t)(w >> (8 * i)); }

// One wave per 16 slots of the slab.  The run begins at any slot of the 8-bit
// cache, so a lane's 8 values of a channel may lie across two 8-byte halves of
// its groups.
template <int D>
__global__ void __launch_bounds__(64 * kWaves) kv8_load_kernel(const Kv8CopyParams p) {
  const int lane = threadIdx.x & 63;
  const int64_t unit = (int64_t)blockIdx.x * kWaves + (threadIdx.x >> 6);
  const int64_t cell = unit / p.groups;
  if (cell >= p.cells) return;
  const int i0 = (int)(unit - cell * p.groups) * kGroup;
  const int64_t s0 = p.starts ? p.starts[cell / p.nkv] : 0;
  const int64_t cap = p.cap;

  // ---- keys
  constexpr int LPR = D / 8, RPW = 64 / LPR;
  uint16_t *ks = p.k_slab + (size_t)cell * p.slab_cap * D;
  const int8_t *k8 = p.k8 + (size_t)cell * p.cap * D;
  const float *kscale = p.k_scale + (size_t)cell * p.cap;
#pragma unroll
  for (int i = 0; i < kGroup / RPW; ++i) {
    const int r = i0 + i * RPW + lane / LPR, ch = lane % LPR * 8;
    if (r >= p.n) continue;
    const int64_t slot = s0 + r;
    uint4 o = make_uint4(0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u);
    if (slot >= 0 && slot < cap) {
      const uint2 w = *reinterpret_cast<const uint2 *>(k8 + (size_t)slot * D + ch);
      const float s = kscale[slot];
      float x[8];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[e] = s8f(w.x, e) * s;
        x[4 + e] = s8f(w.y, e) * s;
      }
      o = pack8(x);
    }
    *reinterpret_cast<uint4 *>(ks + (size_t)r * D + ch) = o;
  }

  // ---- values
  uint16_t *vs = p.v_slab + (size_t)cell * p.slab_cap * D;
  const int8_t *v8 = p.v8 + (size_t)cell * p.cap * D;
  const float *vscale = p.v_scale + (size_t)cell * p.cap;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = i0 + 8 * h;
    if (r >= p.n) break;
    const int64_t s = s0 + r;
    float sc[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) sc[e] = s + e >= 0 && s + e < cap ? vscale[s + e] : __builtin_nanf("");
    const int64_t a = s & ~7ll;  // the two halves that hold slots s .. s + 7
    const int sh = (int)(s - a) * 8;
#pragma unroll
    for (int j = 0; j < D / 64; ++j) {
      const int ch = lane + 64 * j;
      auto half = [&](int64_t at) -> uint64_t {
        return at >= 0 && at < cap ? *reinterpret_cast<const uint64_t *>(v8 + ((size_t)(at >> 4) * D + ch) * 16 + (at & 8)) : 0ull;
      };
      uint64_t w = half(a) >> sh;
      if (sh) w |= half(a + 8) << (64 - sh);
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = s8f((uint32_t)(w >> (e < 4 ? 0 : 32)), e & 3) * sc[e];
      const uint4 o = pack8(x);
      uint16_t *dst = vs + ((size_t)(r >> 3) * D + ch) * 8;
      if (r + 8 <= p.n) {
        *reinterpret_cast<uint4 *>(dst) = o;
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (r + e < p.n) dst[e] = (uint16_t)f2bf(x[e]);
      }
    }
  }
}

}  // namespace

hipError_t launch_kv8_store(const Kv8CopyParams &p, hipStream_t s) {
  const dim3 grid((unsigned)((p.cells * p.groups + kWaves - 1) / kWaves)), block(64 * kWaves);
  if (p.head_dim == 128) hipLaunchKernelGGL((kv8_store_kernel<128>), grid, block, 0, s, p);
  else hipLaunchKernelGGL((kv8_store_kernel<64>), grid, block, 0, s, p);
  return hipSuccess;
}

hipError_t launch_kv8_load(const Kv8CopyParams &p, hipStream_t s) {
  const dim3 grid((unsigned)((p.cells * p.groups + kWaves - 1) / kWaves)), block(64 * kWaves);
  if (p.head_dim == 128) hipLaunchKernelGGL((kv8_load_kernel<128>), grid, block, 0, s, p);
  else hipLaunchKernelGGL((kv8_load_kernel<64>), grid, block, 0, s, p);
  return hipSuccess;
}

}  // namespace qdec
