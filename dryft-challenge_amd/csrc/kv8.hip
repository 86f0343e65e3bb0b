// The 8-bit KV cache written from a bf16 slab (kv8_store) and read back into one
// (kv8_load).  Both are copies of 3 bytes an element, bound by memory where a
// launch fills the GPU; a wave takes the keys or the values of 16 slots, so that
// short runs have waves enough (both in one wave, with a value's largest over 64
// lanes by floats: 188 us instead of 150 for the first of these, 9.2 instead of 3.8
// for the last).  MI355X, us stored / read back (a copy's 4.98 TB/s in brackets), 8 kv heads of 128
// channels: 32 x 4096 slots 150 / 151 (163), 16 x 2048 - / 43 (41), 8 x 1021 from
// slot 1003 14.9 / 15.6 (10.2), 1 x 512 3.8 / 3.5 (0.6; an empty launch takes 1.8).
#include "dma_dev.h"
#include "kv8_dev.h"
#include "qdec_kernels.h"

namespace qdec {

namespace {

constexpr int kGroup = 16;  // slots of one wave: a group of the V layout
constexpr int kWaves = 4;

template <int CTRL>
__device__ __forceinline__ uint32_t dpp_u(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
}
typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {  // of both halves
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2_t, a), __builtin_bit_cast(u16x2_t, b)));
}

// A wave's place: keys or values of 16-slot group g of a (sequence, kv head).
struct Place {
  int64_t cell;
  int g;
  bool keys;
};
__device__ __forceinline__ bool place_of(const Kv8CopyParams &p, Place &r) {
  const uint32_t x = blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), unit = x >> 1;
  if (unit >= (uint32_t)p.cells * (uint32_t)p.groups) return false;
  r.cell = unit / (uint32_t)p.groups;
  r.g = (int)(unit - (uint32_t)r.cell * (uint32_t)p.groups);
  r.keys = !(x & 1);
  return true;
}

// Magnitudes of bf16 numbers are ordered as their bits, and the bits from 0x7f80
// on are those that are not finite, so rows' largest are found on packed pairs.
template <int D>
__device__ __forceinline__ void store_keys(const Kv8CopyParams &p, int64_t cell, int s0, int s1) {
  constexpr int LPR = D / 8, RPW = 64 / LPR, N = kGroup / RPW;  // lanes to a row, 8 channels each; rows at once
  const int lane = threadIdx.x & 63, ch = lane % LPR * 8;
  const uint16_t *src = p.k_slab + (size_t)cell * p.slab_cap * D;
  int8_t *dst = p.k8 + (size_t)cell * p.cap * D;
  uint4 raw[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int slot = min(max(s0 + i * RPW + lane / LPR, p.pos0), s1 - 1);
    raw[i] = ld16(src + (size_t)slot * D + ch);
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int slot = s0 + i * RPW + lane / LPR;
    const u32x4_t v = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
    uint32_t m = max2(max2(v[0] & 0x7fff7fffu, v[1] & 0x7fff7fffu), max2(v[2] & 0x7fff7fffu, v[3] & 0x7fff7fffu));
    m = max(m >> 16, m & 0xffffu);
    m = max(m, dpp_u<0xB1>(m));
    m = max(m, dpp_u<0x4E>(m));
    m = max(m, dpp_u<0x141>(m));
    if constexpr (LPR == 16) m = max(m, dpp_u<0x140>(m));
    const float top = bf2f(m);
    const bool fin = m < 0x7f80u;
    const Kv8Div div(top, fin);
    float x[8];
    unpack8(raw[i], x);
    if (slot < p.pos0 || slot >= s1) continue;
    *reinterpret_cast<uint2 *>(dst + (size_t)slot * D + ch) =
        make_uint2(div.four(x[0], x[1], x[2], x[3]), div.four(x[4], x[5], x[6], x[7]));
    if (lane % LPR == 0) p.k_scale[(size_t)cell * p.cap + slot] = kv8_scale(top, fin);
  }
}

// Lane takes channels lane + 64 j of all 16 slots, as both layouts have them; lane
// c of each DPP row then holds what slot c is divided by.
template <int D>
__device__ __forceinline__ void store_values(const Kv8CopyParams &p, int64_t cell, int s0, int s1) {
  constexpr int N = D / 64;
  const int lane = threadIdx.x & 63, col = lane & 15;
  const uint16_t *src = p.v_slab + (size_t)cell * p.slab_cap * D;
  uint32_t w[N][8], m[8];  // slots 2 d, 2 d + 1
#pragma unroll
  for (int j = 0; j < N; ++j)
#pragma unroll
    for (int h = 0; h < 2; ++h) {  // (slab_cap is a multiple of 32)
      const uint4 v = ld16(src + ((size_t)((s0 >> 3) + h) * D + lane + 64 * j) * 8);
      w[j][4 * h] = v.x; w[j][4 * h + 1] = v.y; w[j][4 * h + 2] = v.z; w[j][4 * h + 3] = v.w;
    }
#pragma unroll
  for (int d = 0; d < 8; ++d) {
    m[d] = w[0][d] & 0x7fff7fffu;
    if constexpr (N == 2) m[d] = max2(m[d], w[1][d] & 0x7fff7fffu);
    m[d] = max2(m[d], dpp_u<0xB1>(m[d]));
    m[d] = max2(m[d], dpp_u<0x4E>(m[d]));
    m[d] = max2(m[d], dpp_u<0x141>(m[d]));
    m[d] = max2(m[d], dpp_u<0x140>(m[d]));
    const auto a = __builtin_amdgcn_permlane16_swap(m[d], m[d], false, false);
    m[d] = max2(a[0], a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(m[d], m[d], false, false);
    m[d] = max2(b[0], b[1]);
  }
  uint32_t mine = m[0];
#pragma unroll
  for (int d = 1; d < 8; ++d) mine = (col >> 1) == d ? m[d] : mine;
  mine = (col & 1) ? mine >> 16 : mine & 0xffffu;
  const float top = bf2f(mine);
  const bool fin = mine < 0x7f80u;
  const Kv8Div div(top, fin);
  if (lane < 16 && s0 + col >= p.pos0 && s0 + col < s1) p.v_scale[(size_t)cell * p.cap + s0 + col] = kv8_scale(top, fin);
  uint32_t q[N][4];
  auto four = [&](auto d) {  // slots 4 d ..
    constexpr int D4 = 4 * decltype(d)::value;
    Kv8Div k[4];
    k[0] = div.template at<D4>();
    k[1] = div.template at<D4 + 1>();
    k[2] = div.template at<D4 + 2>();
    k[3] = div.template at<D4 + 3>();
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const uint32_t u = w[j][D4 / 2], v = w[j][D4 / 2 + 1];
      q[j][D4 / 4] = low_bytes(k[0].one(lo16(u)), k[1].one(hi16(u)), k[2].one(lo16(v)), k[3].one(hi16(v)));
    }
  };
  four(Int<0>{});
  four(Int<1>{});
  four(Int<2>{});
  four(Int<3>{});
  int8_t *dst = p.v8 + (size_t)cell * p.cap * D + ((size_t)(s0 >> 4) * D + lane) * kGroup;
  if (s0 >= p.pos0 && s0 + kGroup <= s1) {
#pragma unroll
    for (int j = 0; j < N; ++j) *reinterpret_cast<uint4 *>(dst + 64 * kGroup * j) = make_uint4(q[j][0], q[j][1], q[j][2], q[j][3]);
  } else {
#pragma unroll
    for (int i = 0; i < kGroup; ++i)
      if (s0 + i >= p.pos0 && s0 + i < s1)
#pragma unroll
        for (int j = 0; j < N; ++j) dst[64 * kGroup * j + i] = (int8_t)(q[j][i >> 2] >> (8 * (i & 3)));
  }
}

template <int D>
__global__ void __launch_bounds__(64 * kWaves) kv8_store_kernel(const Kv8CopyParams p) {
  Place at;
  if (!place_of(p, at)) return;
  const int s0 = (p.pos0 / kGroup + at.g) * kGroup, s1 = p.pos0 + p.n;
  if (at.keys) store_keys<D>(p, at.cell, s0, s1);
  else store_values<D>(p, at.cell, s0, s1);
}

// Byte i of w, whose sign bits are turned, as an int8 times s: the byte is 128 more and
// the difference exact, so the product is rounded once.  (Taking 128 s off the product
// instead would leave fp32's range from s = 2^121 on, rows of the two largest bf16 numbers.)
__device__ __forceinline__ float byte_times(uint32_t w, int i, float s) {
  return ((float)((w >> (8 * i)) & 0xffu) - 128.f) * s;
}

template <int D>
__device__ __forceinline__ void load_keys(const Kv8CopyParams &p, int64_t cell, int r0, int64_t s0) {
  constexpr int LPR = D / 8, RPW = 64 / LPR, N = kGroup / RPW;
  const int lane = threadIdx.x & 63, ch = lane % LPR * 8;
  const int8_t *src = p.k8 + (size_t)cell * p.cap * D;
  const float *scale = p.k_scale + (size_t)cell * p.cap;
  uint16_t *dst = p.k_slab + (size_t)cell * p.slab_cap * D;
  uint2 w[N];
  float s[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int64_t slot = s0 + r0 + i * RPW + lane / LPR, at = min(max(slot, (int64_t)0), (int64_t)p.cap - 1);
    w[i] = *reinterpret_cast<const uint2 *>(src + (size_t)at * D + ch);
    s[i] = scale[at];
    if (slot != at) s[i] = __builtin_nanf("");  // outside the cache
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int r = r0 + i * RPW + lane / LPR;
    const uint32_t a = w[i].x ^ 0x80808080u, b = w[i].y ^ 0x80808080u;
    float x[8];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[e] = byte_times(a, e, s[i]);
      x[4 + e] = byte_times(b, e, s[i]);
    }
    if (r < p.n) *reinterpret_cast<uint4 *>(dst + (size_t)r * D + ch) = pack8(x);
  }
}

// The run begins at any slot of the 8-bit cache, so a lane's 16 values of a channel
// lie in two groups.
template <int D>
__device__ __forceinline__ void load_values(const Kv8CopyParams &p, int64_t cell, int r0, int64_t s0) {
  constexpr int N = D / 64;
  const int lane = threadIdx.x & 63, col = lane & 15;
  const int8_t *src = p.v8 + (size_t)cell * p.cap * D + lane * kGroup;
  uint16_t *dst = p.v_slab + (size_t)cell * p.slab_cap * D + (size_t)lane * 8;
  const int64_t s = s0 + r0, mine = s + col, at = min(max(mine, (int64_t)0), (int64_t)p.cap - 1);
  float scale = p.v_scale[(size_t)cell * p.cap + at];
  if (mine != at) scale = __builtin_nanf("");
  const int64_t last = p.cap / kGroup - 1, g0 = s >> 4;  // groups g0 and g0 + 1, where they are
  const int sh = (int)(s & 15);
  uint4 lo[N], hi[N];
#pragma unroll
  for (int j = 0; j < N; ++j) {
    lo[j] = *reinterpret_cast<const uint4 *>(src + ((size_t)min(max(g0, (int64_t)0), last) * D + 64 * j) * kGroup);
    hi[j] = lo[j];
    if (sh) hi[j] = *reinterpret_cast<const uint4 *>(src + ((size_t)min(max(g0 + 1, (int64_t)0), last) * D + 64 * j) * kGroup);
  }
#pragma unroll
  for (int j = 0; j < N; ++j) {
    uint32_t w[8] = {lo[j].x, lo[j].y, lo[j].z, lo[j].w, hi[j].x, hi[j].y, hi[j].z, hi[j].w};
    if (sh & 8)
#pragma unroll
      for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
    if (sh & 4)
#pragma unroll
      for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __builtin_amdgcn_alignbyte(w[i + 1], w[i], sh & 3) ^ 0x80808080u;
    auto eight = [&](auto half) {
      constexpr int H = decltype(half)::value;
      const float x[8] = {byte_times(w[2 * H], 0, dpp_f<0x150 + 8 * H>(scale)),     byte_times(w[2 * H], 1, dpp_f<0x151 + 8 * H>(scale)),
                          byte_times(w[2 * H], 2, dpp_f<0x152 + 8 * H>(scale)),     byte_times(w[2 * H], 3, dpp_f<0x153 + 8 * H>(scale)),
                          byte_times(w[2 * H + 1], 0, dpp_f<0x154 + 8 * H>(scale)), byte_times(w[2 * H + 1], 1, dpp_f<0x155 + 8 * H>(scale)),
                          byte_times(w[2 * H + 1], 2, dpp_f<0x156 + 8 * H>(scale)), byte_times(w[2 * H + 1], 3, dpp_f<0x157 + 8 * H>(scale))};
      const int r = r0 + 8 * H;
      uint16_t *out = dst + ((size_t)(r >> 3) * D + 64 * j) * 8;
      if (r + 8 <= p.n) {
        *reinterpret_cast<uint4 *>(out) = pack8(x);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (r + e < p.n) out[e] = (uint16_t)f2bf(x[e]);
      }
    };
    eight(Int<0>{});
    eight(Int<1>{});
  }
}

template <int D>
__global__ void __launch_bounds__(64 * kWaves) kv8_load_kernel(const Kv8CopyParams p) {
  Place at;
  if (!place_of(p, at)) return;
  const int64_t s0 = p.starts ? p.starts[(int)(at.cell / p.nkv)] : 0;
  if (at.keys) load_keys<D>(p, at.cell, at.g * kGroup, s0);
  else load_values<D>(p, at.cell, at.g * kGroup, s0);
}

template <class K>
hipError_t launch(const Kv8CopyParams &p, K k128, K k64, hipStream_t s) {
  const dim3 grid((unsigned)((2 * p.cells * p.groups + kWaves - 1) / kWaves)), block(64 * kWaves);
  hipLaunchKernelGGL(p.head_dim == 128 ? k128 : k64, grid, block, 0, s, p);
  return hipSuccess;
}

}  // namespace

hipError_t launch_kv8_store(const Kv8CopyParams &p, hipStream_t s) {
  return launch(p, kv8_store_kernel<128>, kv8_store_kernel<64>, s);
}

hipError_t launch_kv8_load(const Kv8CopyParams &p, hipStream_t s) {
  return launch(p, kv8_load_kernel<128>, kv8_load_kernel<64>, s);
}

}  // namespace qdec
