// Decode attention over the 8-bit KV cache, with the head RMSNorm, RoPE and the
// quantised write of the new rows folded in: t_rows query rows per sequence,
// row t at position lens[b] + t over slots 0 .. lens[b] + t.
//
// A workgroup of 8 waves takes up to 16 query rows and the 64-slot blocks j = c,
// c + splits, ... of one (sequence, kv head), its wave w every eighth of those.  Blocks are dealt by
// absolute slot numbers and a row is rescaled by its own scores alone, so a
// row's bits do not depend on t_rows.  Per block
// (v_mfma_f32_16x16x32_f16):
//   S^T = K . Q^T.  K's 8 bits are fp16 integers: a byte under the exponent byte
//     0x64 is 1024 + byte, so one byte permute makes two of them and one packed
//     subtraction takes 1152 off.  Q is held in two fp16 parts (22 bits) of the
//     row divided by a power of two; up to 8 query rows they are the two halves
//     of one MFMA's 16 columns.
//   p = 2^(S scale_k scale_q - m), fp32 statistics.
//   O^T += V^T . W^T with w = p scale_v in fp16: 2^-11 relative, an eighth of the
//     output's rounding.  fp16 reaches down to 2^-24 only, so a row's w are
//     held in units of 2^(u - 15), 2^u above the largest |w| so far.
// K's rows are dealt to MFMA rows so that a lane's 16 scores are the 16 slots of
// one V group, the operand of the second product; slot l's scales sit in lane
// l and reach the row by DPP.  K and V hold integers whatever lies behind the last slot, so
// only scores and scales are masked.
#include <algorithm>

#include "dma_dev.h"
#include "kv8_dev.h"
#include "qdec_kernels.h"

namespace qdec {

namespace {

constexpr int kW = 8;       // waves of a workgroup
constexpr int kPad = 8;     // fp16 behind an LDS query row (bank spread)

__device__ __forceinline__ f32x4_t mfma_f16(const f16x8_t &a, const f16x8_t &b, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// 16 int8 as two operands of 8 fp16.
__device__ __forceinline__ void to_f16(const uint4 &v, f16x8_t &a, f16x8_t &b) {
  const f16x2_t off = {(_Float16)1152.f, (_Float16)1152.f};
  auto two = [&](uint32_t w, uint32_t sel) {
    return __builtin_bit_cast(f16x2_t, __builtin_amdgcn_perm(0x64646464u, w, sel)) - off;
  };
  auto four = [&](uint32_t w, f16x8_t &o, int i) {
    w ^= 0x80808080u;
    const f16x2_t x = two(w, 0x04010400u), y = two(w, 0x04030402u);
    o[i] = x[0];
    o[i + 1] = x[1];
    o[i + 2] = y[0];
    o[i + 3] = y[1];
  };
  four(v.x, a, 0);
  four(v.y, a, 4);
  four(v.z, b, 0);
  four(v.w, b, 4);
}

// v of lane I of this lane's 16-lane row.
template <int I>
__device__ __forceinline__ float row_lane(float v) { return dpp_f<0x150 + I>(v); }

// Head RMSNorm and RoPE of channels 2 lane, 2 lane + 1 of a row, in fp32 (lanes
// from D / 2 on pass raw = 0).
template <int D>
__device__ __forceinline__ void norm_rope(uint32_t raw, uint32_t w, uint32_t cw, uint32_t sw, float eps, float &o0, float &o1) {
  const int lane = threadIdx.x & 63;
  const float x0 = lo16(raw), x1 = hi16(raw);
  const float rstd = 1.0f / sqrtf(wave_sum(x0 * x0 + x1 * x1) / (float)D + eps);
  const float y0 = x0 * rstd * lo16(w), y1 = x1 * rstd * hi16(w);
  const float p0 = shfl_xor(y0, D / 4), p1 = shfl_xor(y1, D / 4);
  const bool first = (lane & (D / 2 - 1)) < D / 4;
  o0 = y0 * lo16(cw) + (first ? -p0 : p0) * lo16(sw);
  o1 = y1 * hi16(cw) + (first ? -p1 : p1) * hi16(sw);
}

// A row's power-of-two factor: 2^-e with 2^e <= max|x| < 2^(e+1), and 2^e.
__device__ __forceinline__ void pow2_of(float top, float &down, float &up) {
  const int e = min(max((int)(__float_as_uint(top) >> 23) - 127, -100), 120);
  down = __uint_as_float((uint32_t)(127 - e) << 23);
  up = __uint_as_float((uint32_t)(127 + e) << 23);
}

template <int D>
struct Frag {  // one block
  uint4 k[4][D / 64];  // MFMA rows tile: row r = slot 16 (r >> 2) + 4 tile + (r & 3); 16 channels 64 h + 16 grp
  uint4 v[D / 16];     // channel 16 dt + col, slots 16 grp .. + 15
  float ks, vs;        // scales of slot `lane`
};

// LDS (bytes).
template <int D>
struct Lds {
  static constexpr int RS = D + kPad;
  static constexpr int q = 0;                            // [2][16][RS] fp16 query parts; then wave sums [kW][D / 16][64] f32x4
  static constexpr int qn = 2 * 16 * RS * 2;
  static constexpr int an = kW * (D / 16) * 64 * 16;
  static constexpr int qs = q + (qn > an ? qn : an);     // [16] query rows' factors
  static constexpr int k8 = qs + 16 * 4;                 // [kKv8MaxT][D]
  static constexpr int v8 = k8 + kKv8MaxT * D;           // [2][D][16]
  static constexpr int sk = v8 + 2 * D * 16;             // [kKv8MaxT]
  static constexpr int sv = sk + kKv8MaxT * 4;
  static constexpr int m = sv + kKv8MaxT * 4;            // [3][kW][16] wave statistics: maximum, sum, unit
  static constexpr int bytes = m + 3 * kW * 16 * 4;
};

// PK: at most 8 query rows in all, both parts in one tile.
template <int D, bool PK>
__global__ void __launch_bounds__(64 * kW) kv8_attn_kernel(const Kv8AttnParams p) {
  constexpr int NH = D / 64, DT = D / 16, LH = D / 2;
  constexpr int QPW = 16 / kW, KPW = kKv8MaxT / kW;
  using LY = Lds<D>;
  constexpr int RS = LY::RS;
  __shared__ __attribute__((aligned(16))) unsigned char smem[LY::bytes];
  _Float16 *s_q = reinterpret_cast<_Float16 *>(smem + LY::q);
  f32x4_t *s_acc = reinterpret_cast<f32x4_t *>(smem + LY::q);
  float *s_qs = reinterpret_cast<float *>(smem + LY::qs);
  unsigned char *s_k8 = smem + LY::k8, *s_v8 = smem + LY::v8;
  float *s_sk = reinterpret_cast<float *>(smem + LY::sk), *s_sv = reinterpret_cast<float *>(smem + LY::sv);
  float *s_m = reinterpret_cast<float *>(smem + LY::m);

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, grp = lane >> 4;
  const int c = blockIdx.x, kvh = blockIdx.y, C = p.splits, z = blockIdx.z;
  const int tile = (z >= p.batch) + (z >= 2 * p.batch) + (z >= 3 * p.batch), b = z - tile * p.batch;
  const int T = p.t_rows, nq = p.nq, nkv = p.nkv, G = nq / nkv, R = T * G;
  const int r0 = tile * 16, nr = min(R - r0, 16);  // this workgroup's query rows
  const int width = (nq + 2 * nkv) * D;
  const size_t cell = (size_t)b * nkv + kvh;
  int8_t *k8 = p.k8 + cell * p.cap * D, *v8 = p.v8 + cell * p.cap * D;
  float *kscale = p.k_scale + cell * p.cap, *vscale = p.v_scale + cell * p.cap;
  const float NEG_INF = -__builtin_huge_valf();
  const int blocks = p.cap / kKv8Block;

  auto load_block = [&](int j, Frag<D> &f) {
    const int s0 = j * kKv8Block;
    const int8_t *kb = k8 + (size_t)(s0 + 16 * (col >> 2) + (col & 3)) * D + 16 * grp;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int h = 0; h < NH; ++h) f.k[t][h] = ld_nt(kb + (4 * t) * D + 64 * h);
    const int8_t *vb = v8 + ((size_t)((s0 >> 4) + grp) * D + col) * 16;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) f.v[dt] = ld_nt(vb + dt * 256);
    f.ks = kscale[s0 + lane];
    f.vs = vscale[s0 + lane];
  };
  // This wave's i-th block; the first one's addresses do not depend on the length.
  auto nth = [&](int i) { return c + C * (wave + kW * i); };
  Frag<D> f0, f1;
  if (nth(0) < blocks) load_block(nth(0), f0);

  const int L = p.lens[b];
  if (L < 0 || L > p.cap - T) {  // no cache access; the rows become NaN
    if (c == 0)
      for (int i = threadIdx.x; i < nr * (D / 4); i += blockDim.x) {
        const int y = i / (D / 4), ch = (i - y * (D / 4)) * 4, r = r0 + y, row = b * T + r / G, k = (kvh * G + r % G) * D + ch;
        uint16_t *o = p.out + (p.ofrag ? frag_off(row, k, p.ofrag) : (size_t)row * nq * D + k);
        *reinterpret_cast<uint2 *>(o) = make_uint2(0x7fc07fc0u, 0x7fc07fc0u);
      }
    return;
  }
  const int last = L + T - 1, nb = last / kKv8Block + 1;
  if (c >= nb) return;
  if (nth(1) < nb) load_block(nth(1), f1);

  // ---- the query rows in two fp16 parts, the new keys and values in 8 bits, to LDS
  const int ch = 2 * min(lane, LH - 1);
  const bool lv = lane < LH;
  const uint16_t *rows = p.qkv + (size_t)b * T * width;
  auto pair = [&](const uint16_t *x) { return *reinterpret_cast<const uint32_t *>(x + ch); };
  const uint32_t qw = pair(p.q_norm_w), kw = pair(p.k_norm_w);
  for (int i = 0; i < QPW; ++i) {
    const int y = wave + kW * i, r = r0 + y;
    if (y >= nr) break;
    const int t = r / G, h = kvh * G + r - t * G;
    float x0, x1;
    norm_rope<D>(lv ? pair(rows + (size_t)t * width + (size_t)h * D) : 0u, qw, pair(p.cos_tab + (size_t)(L + t) * D),
                 pair(p.sin_tab + (size_t)(L + t) * D), p.eps, x0, x1);
    float down, up;
    pow2_of(wave_max(lv ? fmaxf(fabsf(x0), fabsf(x1)) : 0.f), down, up);
    x0 *= down;
    x1 *= down;
    const f16x2_t hi = {(_Float16)x0, (_Float16)x1};
    const f16x2_t lo = {(_Float16)(x0 - (float)hi[0]), (_Float16)(x1 - (float)hi[1])};
    if (lv) {
      *reinterpret_cast<f16x2_t *>(s_q + y * RS + ch) = hi;
      *reinterpret_cast<f16x2_t *>(s_q + (16 + y) * RS + ch) = lo;
    }
    if (lane == 0) s_qs[y] = up * p.scale_log2;
  }
  const int b_lo = L / kKv8Block, b_hi = last / kKv8Block;  // (new rows lie in two blocks at most)
  const bool mine = b_lo % C == c || b_hi % C == c;
  if (mine) {
    for (int i = 0; i < KPW; ++i) {
      const int t = wave + kW * i;
      if (t >= T) break;
      const uint16_t *x = rows + (size_t)t * width + (size_t)(nq + kvh) * D;
      const uint32_t vr = lv ? pair(x + (size_t)nkv * D) : 0u;
      float k0, k1;
      norm_rope<D>(lv ? pair(x) : 0u, kw, pair(p.cos_tab + (size_t)(L + t) * D), pair(p.sin_tab + (size_t)(L + t) * D), p.eps,
                   k0, k1);
      if (!lv) k0 = k1 = 0.f;
      const float v0 = lo16(vr), v1 = hi16(vr);
      const float kt = wave_max(fmaxf(fabsf(k0), fabsf(k1))), vt = wave_max(fmaxf(fabsf(v0), fabsf(v1)));
      const bool kf = __all(finite_f(k0) && finite_f(k1)), vf = __all(finite_f(v0) && finite_f(v1));
      const float kd = kv8_div(kt, kf), vd = kv8_div(vt, vf);
      const uint32_t q0 = kv8_round(k0, kd), q1 = kv8_round(k1, kd), w0 = kv8_round(v0, vd), w1 = kv8_round(v1, vd);
      const int slot = L + t, gi = (slot >> 4) - (L >> 4), e = slot & 15;
      const bool put = tile == 0 && (slot / kKv8Block) % C == c;
      if (lv) {
        *reinterpret_cast<uint16_t *>(s_k8 + t * D + ch) = (uint16_t)(q0 | (q1 << 8));
        s_v8[(gi * D + ch) * 16 + e] = (unsigned char)w0;
        s_v8[(gi * D + ch + 1) * 16 + e] = (unsigned char)w1;
        if (put) {
          *reinterpret_cast<uint16_t *>(k8 + (size_t)slot * D + ch) = (uint16_t)(q0 | (q1 << 8));
          int8_t *vo = v8 + ((size_t)(slot >> 4) * D + ch) * 16 + e;
          vo[0] = (int8_t)w0;
          vo[16] = (int8_t)w1;
        }
      }
      if (lane == 0) {
        const float sk = kv8_scale(kt, kf), sv = kv8_scale(vt, vf);
        s_sk[t] = sk;
        s_sv[t] = sv;
        if (put) {
          kscale[slot] = sk;
          vscale[slot] = sv;
        }
      }
    }
  }
  lds_barrier();

  // ---- this wave's blocks
  const int y = PK ? col & 7 : col;
  const bool row_in = y < nr;
  const float qs = row_in ? s_qs[y] : 0.f;
  const int lim = row_in ? L + (r0 + y) / G : -1;  // the last slot the row sees
  float m_run = NEG_INF, l_run = 0.f;
  int unit = -200;  // 2^unit > |w| so far
  f32x4_t acc[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) acc[dt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  // Query operands: 8 channels 64 h + 16 grp + 8 e of the column's row.
  f16x8_t qh[NH][2], ql[PK ? 1 : NH][2];
#pragma unroll
  for (int h = 0; h < NH; ++h)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      auto part = [&](int i) {
        const f16x8_t z = {};
        return row_in ? *reinterpret_cast<const f16x8_t *>(s_q + (16 * i + y) * RS + 64 * h + 16 * grp + 8 * e) : z;
      };
      qh[h][e] = part(PK ? col >> 3 : 0);
      if constexpr (!PK) ql[h][e] = part(1);
    }

  // The new rows of a block that holds some, from LDS.
  auto patch = [&](Frag<D> &f, int s0) {
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int i = s0 + 16 * (col >> 2) + 4 * t + (col & 3) - L;
      const bool is = (unsigned)i < (unsigned)T;
#pragma unroll
      for (int h = 0; h < NH; ++h) {
        const uint4 x = *reinterpret_cast<const uint4 *>(s_k8 + min(max(i, 0), kKv8MaxT - 1) * D + 64 * h + 16 * grp);
        if (is) f.k[t][h] = x;
      }
    }
    const int v0 = s0 + 16 * grp, gi = min(max((v0 >> 4) - (L >> 4), 0), 1);
    uint32_t take[4];
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      take[d] = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int s = v0 + 4 * d + e;
        if (s >= L && s <= last) take[d] |= 0xffu << (8 * e);
      }
    }
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      const uint4 x = *reinterpret_cast<const uint4 *>(s_v8 + (gi * D + dt * 16 + col) * 16);
      uint4 &v = f.v[dt];
      v.x = (v.x & ~take[0]) | (x.x & take[0]);
      v.y = (v.y & ~take[1]) | (x.y & take[1]);
      v.z = (v.z & ~take[2]) | (x.z & take[2]);
      v.w = (v.w & ~take[3]) | (x.w & take[3]);
    }
    const int i = s0 + lane - L;
    if ((unsigned)i < (unsigned)T) {
      f.ks = s_sk[i];
      f.vs = s_sv[i];
    }
  };

  auto process = [&](Frag<D> &f, int j) {
    const int s0 = j * kKv8Block;
    const bool edge = s0 + kKv8Block > L;  // slots that not every row sees
    if (edge) patch(f, s0);
    float s[16];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      f32x4_t hi = f32x4_t{0.f, 0.f, 0.f, 0.f}, lo = hi;
#pragma unroll
      for (int h = 0; h < NH; ++h) {
        f16x8_t a[2];
        to_f16(f.k[t][h], a[0], a[1]);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          hi = mfma_f16(a[e], qh[h][e], hi);
          if constexpr (!PK) lo = mfma_f16(a[e], ql[h][e], lo);
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (PK) s[4 * t + i] = hi[i] + dpp_f<0x128>(hi[i]);  // row_ror:8, the other part's column
        else s[4 * t + i] = hi[i] + lo[i];
      }
    }
    // lane (col, grp) holds slots s0 + 16 grp + i of its row
    auto each = [&](auto fn) {
      fn(Int<0>{}); fn(Int<1>{}); fn(Int<2>{}); fn(Int<3>{}); fn(Int<4>{}); fn(Int<5>{}); fn(Int<6>{}); fn(Int<7>{});
      fn(Int<8>{}); fn(Int<9>{}); fn(Int<10>{}); fn(Int<11>{}); fn(Int<12>{}); fn(Int<13>{}); fn(Int<14>{}); fn(Int<15>{});
    };
    const int seen = lim - s0 - 16 * grp;  // of them, those up to here
    float top = NEG_INF;
    each([&](auto n) {
      constexpr int i = decltype(n)::value;
      s[i] = s[i] * row_lane<i>(f.ks) * qs;
      if (edge && i > seen) s[i] = NEG_INF;
      top = fmaxf(top, s[i]);
    });
    const float m_new = fmaxf(m_run, max_xor16_32(top));
    const float m_sub = m_new == NEG_INF ? 0.f : m_new;
    const float alpha = __builtin_amdgcn_exp2f(m_run - m_sub);
    float psum = 0.f, big = 0.f;
    each([&](auto n) {
      constexpr int i = decltype(n)::value;
      const float e = __builtin_amdgcn_exp2f(s[i] - m_sub);
      psum += e;
      const float w = e * row_lane<i>(f.vs);
      s[i] = edge && i > seen ? 0.f : w;
      big = fmaxf(big, s[i]);
    });
    l_run = l_run * alpha + psum;
    // The unit: above this block's w and, moved to the new maximum, above the old.
    big = max_xor16_32(big);
    const int ub = (int)(__float_as_uint(big) >> 23) - 126;
    const int uo = unit - (int)fminf(m_new - m_run, 1000.f);
    const int un = min(max(max(ub, uo), -100), 125);
    const float ra = __builtin_ldexpf(alpha, max(unit - un, -300));
    m_run = m_new;
    unit = un;
    const float to = __uint_as_float((uint32_t)(127 + 15 - un) << 23);
    f16x8_t w[2];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      w[0][e] = (_Float16)(s[e] * to);
      w[1][e] = (_Float16)(s[8 + e] * to);
    }
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      f16x8_t a[2];
      to_f16(f.v[dt], a[0], a[1]);
      acc[dt] *= ra;
      acc[dt] = mfma_f16(a[0], w[0], acc[dt]);
      acc[dt] = mfma_f16(a[1], w[1], acc[dt]);
    }
  };
  for (int i = 0; nth(i) < nb; i += 2) {
    process(f0, nth(i));
    if (nth(i + 2) < nb) load_block(nth(i + 2), f0);
    if (nth(i + 1) < nb) {
      process(f1, nth(i + 1));
      if (nth(i + 3) < nb) load_block(nth(i + 3), f1);
    }
  }

  // ---- the waves' sums, in wave order; then the output or a partial: the
  // normalised row, its maximum and its sum.
  const int n_active = min(C, nb);
  float *part = p.partial + (cell * C + c) * (size_t)(R * (D + 2));
  const int r = r0 + y;
  const bool out_in = row_in && !(PK && col >= 8);
  float lw = l_run + shfl_xor(l_run, 16);
  lw += shfl_xor(lw, 32);
  lds_barrier();  // the queries have been read
  if (grp == 0) {
    s_m[wave * 16 + col] = m_run;
    s_m[(kW + wave) * 16 + col] = lw;
    s_m[(2 * kW + wave) * 16 + col] = __int_as_float(unit);
  }
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) s_acc[(wave * DT + dt) * 64 + lane] = acc[dt];
  lds_barrier();
  float M = NEG_INF, sum = 0.f, fac[kW];
  int U = -1000;
#pragma unroll
  for (int w = 0; w < kW; ++w) M = fmaxf(M, s_m[w * 16 + col]);
#pragma unroll
  for (int w = 0; w < kW; ++w) {
    const float mw = s_m[w * 16 + col];
    if (mw != NEG_INF) U = max(U, __float_as_int(s_m[(2 * kW + w) * 16 + col]) - (int)fminf(M - mw, 1000.f));
  }
  U = min(max(U, -100), 125);
#pragma unroll
  for (int w = 0; w < kW; ++w) {
    const float mw = s_m[w * 16 + col], l = s_m[(kW + w) * 16 + col];
    const float e = mw == NEG_INF ? l * 0.f : __builtin_amdgcn_exp2f(mw - M);  // (a NaN among its scores stays)
    sum += l * e;
    fac[w] = __builtin_ldexpf(e, max(__float_as_int(s_m[(2 * kW + w) * 16 + col]) - U, -300));
  }
  const float back = __builtin_ldexpf(1.f, U - 15);
  for (int dt = wave; dt < DT; dt += kW) {
    f32x4_t o = s_acc[dt * 64 + lane] * fac[0];
#pragma unroll
    for (int w = 1; w < kW; ++w) o += s_acc[(w * DT + dt) * 64 + lane] * fac[w];
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = o[i] / sum * back;
    if (!out_in) continue;
    const int k = dt * 16 + grp * 4;
    if (n_active == 1) {
      const int t = r / G, row = b * T + t, kk = (kvh * G + r - t * G) * D + k;
      uint16_t *dst = p.out + (p.ofrag ? frag_off(row, kk, p.ofrag) : (size_t)row * nq * D + kk);
      *reinterpret_cast<uint2 *>(dst) = make_uint2(pack2(o[0], o[1]), pack2(o[2], o[3]));
    } else {
      *reinterpret_cast<f32x4_t *>(part + (size_t)r * D + k) = sum == 0.f ? f32x4_t{0.f, 0.f, 0.f, 0.f} : o;
    }
  }
  if (n_active > 1 && wave == 0 && grp == 0 && out_in) {
    part[(size_t)R * D + r] = M;
    part[(size_t)R * D + R + r] = sum;
  }
}

// Merge of the splits' partials, in order: D / 4 threads per query row.
template <int D>
__global__ void __launch_bounds__(256) kv8_merge_kernel(const Kv8AttnParams p) {
  constexpr int TR = D / 4;
  const int G = p.nq / p.nkv, R = p.t_rows * G, kvh = blockIdx.y, b = blockIdx.z;
  const int r = blockIdx.x * (256 / TR) + threadIdx.x / TR;
  const int L = p.lens[b];
  if (r >= R || L < 0 || L > p.cap - p.t_rows) return;
  const int n = min(p.splits, (L + p.t_rows - 1) / kKv8Block + 1);
  if (n == 1) return;  // written by its workgroup
  const int ch = (int)(threadIdx.x % TR) * 4;
  const size_t stride = (size_t)R * (D + 2);
  const float *part = p.partial + ((size_t)b * p.nkv + kvh) * p.splits * stride;
  const float NEG_INF = -__builtin_huge_valf();
  float M = NEG_INF, l = 0.f;
  f32x4_t o = f32x4_t{0.f, 0.f, 0.f, 0.f};
  for (int i0 = 0; i0 < n; i0 += 8) {
    float mi[8], li[8];
    f32x4_t a[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float *pr = part + (size_t)min(i0 + i, n - 1) * stride;
      mi[i] = pr[(size_t)R * D + r];
      li[i] = pr[(size_t)R * D + R + r];
      a[i] = *reinterpret_cast<const f32x4_t *>(pr + (size_t)r * D + ch);
    }
    float Mn = M;
#pragma unroll
    for (int i = 0; i < 8; ++i) Mn = fmaxf(Mn, mi[i]);  // (the last partial repeats)
    const float w0 = M == NEG_INF ? l * 0.f : __builtin_amdgcn_exp2f(M - Mn);
    l *= w0;
    o *= w0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (i0 + i >= n) continue;
      const float w = li[i] * (mi[i] == NEG_INF ? 0.f : __builtin_amdgcn_exp2f(mi[i] - Mn));
      l += w;
      o += a[i] * w;
    }
    M = Mn;
  }
  const float inv = 1.f / l;
  const int t = r / G, row = b * p.t_rows + t, k = (kvh * G + r - t * G) * D + ch;
  uint16_t *dst = p.out + (p.ofrag ? frag_off(row, k, p.ofrag) : (size_t)row * p.nq * D + k);
  *reinterpret_cast<uint2 *>(dst) = make_uint2(pack2(o[0] * inv, o[1] * inv), pack2(o[2] * inv, o[3] * inv));
}

template <int D>
hipError_t launch_d(const Kv8AttnParams &p, hipStream_t s) {
  const int R = p.t_rows * (p.nq / p.nkv);
  const dim3 grid(p.splits, p.nkv, p.batch * ((R + 15) / 16)), block(64 * kW);
  if (R <= 8) hipLaunchKernelGGL((kv8_attn_kernel<D, true>), grid, block, 0, s, p);
  else hipLaunchKernelGGL((kv8_attn_kernel<D, false>), grid, block, 0, s, p);
  if (p.splits > 1) {
    const int per = 256 / (D / 4);
    hipLaunchKernelGGL((kv8_merge_kernel<D>), dim3((R + per - 1) / per, p.nkv, p.batch), dim3(256), 0, s, p);
  }
  return hipSuccess;
}

}  // namespace

int kv8_attn_splits(int batch, int nkv, int cap) {
  const int64_t cells = (int64_t)batch * nkv;
  const int64_t n = std::min<int64_t>(256 / cells, cap / (kW * kKv8Block));
  return (int)std::max<int64_t>(1, n);
}

hipError_t launch_kv8_attn(const Kv8AttnParams &p, hipStream_t s) {
  return p.head_dim == 128 ? launch_d<128>(p, s) : launch_d<64>(p, s);
}

}  // namespace qdec
