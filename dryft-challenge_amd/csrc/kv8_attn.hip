// Decode attention over the 8-bit KV cache, with the head RMSNorm, RoPE and the
// quantised write of the new rows folded in: t_rows query rows per sequence,
// row t at position lens[b] + t over slots 0 .. lens[b] + t.
//
// A workgroup takes up to 16 query rows of one (sequence, kv head) and, for split c,
// the runs c, c + splits, ... of 4 or 8 consecutive 64-slot blocks, one block of
// each to a wave.  Blocks are dealt by absolute slot numbers and a row is
// rescaled by its own scores alone, so a row's bits do not depend on t_rows.  Per
// block
//   S^T = K . Q^T (v_mfma_i32_16x16x64_i8), exact: K as it is held, q in 21 bits,
//     relative to its row's largest, as three digits of 7 bits.  The columns that few
//     query rows leave hold their other digits: up to 4 rows take one matrix instruction
//     where fp16 parts of q took two, and K no conversion, a quarter of a block's
//     vector instructions (32 x 4160 slots: 52.6 us with fp16 parts, 49.9 so).
//   p = 2^((S scale_k - m) scale_q), fp32 statistics.  The difference comes first: it is as
//     exact as the scores, where m scale_q, rounded by itself, is off by whole powers of 2 from
//     2^24 on and takes p and w out of range.
//   O^T += V^T . W^T (v_mfma_f32_16x16x32_f16) with w = p scale_v in fp16: 2^-11
//     relative, an eighth of the output's rounding.  V's 8 bits are fp16 integers: a byte under
//     the exponent byte 0x64 is 1024 + byte, so one byte permute makes two of them
//     and one packed subtraction takes 1152 off.  fp16 reaches down to 2^-24 only, so
//     a row's w are held in units of 2^(level - 15), 2^level the largest |w| so far, like p
//     relative to the maximum so far, so that level is a small number whatever the scores.
// K's rows are dealt to MFMA rows so that a lane's 16 scores are the 16 slots of
// one V group, the operand of the second product; slot l's scales sit in lane
// l and reach the row by DPP.  K and V hold integers whatever lies behind the last
// slot, so only scores and scales are masked.
//
// What bounds it, 32 query heads on 8 kv heads of 128 (MI355X, replayed graphs whose
// caches take turns): where a launch fills the GPU, the cache's bytes, which arithmetic
// lengthens by 1 to 2 us.  32 sequences of 4096 to 4220 slots: 281 MB in 49.4 us, 5.7
// TB/s (47.3 with no arithmetic; a read of as much takes 40): 6.8 from round to round
// by the cycle counter, the rest launch, first loads and merge.  131000 slots, 64 heads: 53.5 us, 7 of them the
// merge.  A small launch is a chain: length, then rows and tables, then their
// preparation, then the blocks that were loaded meanwhile: one sequence of 640 slots
// 6.8 us before its partials are merged (an empty launch takes 1.8) and 9.3 with the
// merge's launch, of 4100 slots in 9 splits 12.1.
#include <algorithm>

#include "dma_dev.h"
#include "kv8_dev.h"
#include "qdec_kernels.h"

// A row has the same bits in every form of the kernel, so products and sums are fused
// where it is written and nowhere else.
#pragma clang fp contract(off)

namespace qdec {

namespace {

__device__ __forceinline__ int div_by(const FastDiv &d, int n) { return (int)(((uint64_t)(uint32_t)n * d.mul) >> d.shift); }

typedef int i32x4_t __attribute__((ext_vector_type(4)));
__device__ __forceinline__ i32x4_t mfma_i8(const uint4 &a, const uint4 &b, i32x4_t c) {
  return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4_t, a), __builtin_bit_cast(i32x4_t, b), c, 0, 0, 0);
}
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

__device__ __forceinline__ float sum_xor16_32(float v) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// A head row on the 16 lanes of a DPP row, N = D / 16 consecutive channels to a
// lane, so that a wave prepares four rows at once; the rotation's partner
// channels are the lane's 8 further round.
template <int N>
struct Part {
  uint32_t v[N / 2];
  __device__ __forceinline__ void load(const uint16_t *p) {
    if constexpr (N == 8) {
      const uint4 x = ld16(p);
      v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
    } else {
      const uint2 x = *reinterpret_cast<const uint2 *>(p);
      v[0] = x.x; v[1] = x.y;
    }
  }
  __device__ __forceinline__ float operator[](int i) const { return (i & 1) ? hi16(v[i >> 1]) : lo16(v[i >> 1]); }
};

// Its RMSNorm (gain w) and RoPE (tables c, s), in fp32.
template <int N>
__device__ __forceinline__ void norm_rope(const Part<N> &raw, const Part<N> &w, const Part<N> &c, const Part<N> &s, float eps,
                                          float (&o)[N]) {
  float ss = 0.f, y[N];
#pragma unroll
  for (int i = 0; i < N; ++i) ss = __builtin_fmaf(raw[i], raw[i], ss);
  ss += dpp_f<0xB1>(ss);
  ss += dpp_f<0x4E>(ss);
  ss += dpp_f<0x141>(ss);
  ss += dpp_f<0x140>(ss);
  const float rstd = __builtin_amdgcn_rsqf(__builtin_fmaf(ss, 1.f / (16 * N), eps));
  Part<N> sn = s;  // the first half's partner counts negative
#pragma unroll
  for (int i = 0; i < N / 2; ++i) sn.v[i] ^= (threadIdx.x & 8) ? 0u : 0x80008000u;
#pragma unroll
  for (int i = 0; i < N; ++i) y[i] = raw[i] * (rstd * w[i]);
#pragma unroll
  for (int i = 0; i < N; ++i) o[i] = __builtin_fmaf(dpp_f<0x128>(y[i]), sn[i], y[i] * c[i]);
}

// The largest magnitude of such a row as its bits (from 0x7f800000 on: one of
// them is not finite).
template <int N>
__device__ __forceinline__ uint32_t top_bits(const float (&x)[N]) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) m = max(m, __float_as_uint(x[i]) & 0x7fffffffu);
  auto step = [&](auto ctrl) {
    m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, decltype(ctrl)::value, 0xf, 0xf, true));
  };
  step(Int<0xB1>{});
  step(Int<0x4E>{});
  step(Int<0x141>{});
  step(Int<0x140>{});
  return m;
}

// The factors 2^(20 - e) and 2^(e - 1) of a row with 2^(e-1) <= max|x| < 2^e <= 2^128 (a row
// below 2^-108 takes those of 2^-107: steps of 2^-127).
__device__ __forceinline__ void grid_of(uint32_t top, float &down, float &half_up) {
  const int e = min(max((int)(top >> 23), 19), 254) - 126;
  down = __uint_as_float((uint32_t)(127 + 20 - e) << 23);
  half_up = __uint_as_float((uint32_t)(126 + e) << 23);
}
// Four numbers of at most 2^20, rounded, as a 2^14 + b 2^7 + c, 0 <= b, c < 128, each
// digit an int8.  (1.5 * 2^23 added: the sum's low 22 bits are the whole number.)
__device__ __forceinline__ void digits4(const float *x, float down, uint32_t &a, uint32_t &b, uint32_t &c) {
  uint32_t q[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) q[i] = __float_as_uint(__builtin_fmaf(x[i], down, 12582912.f));
  a = low_bytes(q[0] >> 14, q[1] >> 14, q[2] >> 14, q[3] >> 14);
  b = low_bytes(q[0] >> 7, q[1] >> 7, q[2] >> 7, q[3] >> 7) & 0x7f7f7f7fu;
  c = low_bytes(q[0], q[1], q[2], q[3]) & 0x7f7f7f7fu;
}

// LDS (bytes).
template <int D, int AC, int BW>
struct Lds {
  static constexpr int RS = D + 16;                              // bytes per query row (bank spread)
  static constexpr int q = 0;                                    // [3][AC][RS] digits of the queries
  static constexpr int acc = q + 3 * AC * RS;                    // [BW][D / 16][4][AC] f32x4
  static constexpr int qs = acc + BW * (D / 16) * 4 * AC * 16;   // [16] query rows' factors
  static constexpr int k8 = qs + 16 * 4;                         // [kKv8MaxT][D]
  static constexpr int v8 = k8 + kKv8MaxT * D;                   // [2][D][16]
  static constexpr int sk = v8 + 2 * D * 16;                     // [kKv8MaxT]
  static constexpr int sv = sk + kKv8MaxT * 4;
  static constexpr int m = sv + kKv8MaxT * 4;                    // [3][16][BW] the waves' maximum, sum and level
  static constexpr int bytes = m + 3 * BW * 16 * 4;
};

// AC: 4, 8 or 16, the columns of 16 that query rows take, at most so many rows; the
// others hold other digits of them (one, two or three matrix instructions for 64
// channels).  BW: waves that take blocks, a run's; NW waves in all, 4 rows to prepare for
// each.  FOLD: several splits to a workgroup.
template <int D, int AC, int BW, bool FOLD>
__global__ void __launch_bounds__(64 * (AC == 16 ? 8 : BW)) kv8_attn_kernel(const Kv8AttnParams p) {
  constexpr int NH = D / 64, DT = D / 16, NW = AC == 16 ? 8 : BW, RUN = BW * kKv8Block;
  using LY = Lds<D, AC, BW>;
  constexpr int RS = LY::RS;
  __shared__ __attribute__((aligned(16))) unsigned char smem[LY::bytes];
  unsigned char *s_q = smem + LY::q;
  f32x4_t *s_acc = reinterpret_cast<f32x4_t *>(smem + LY::acc);
  float *s_qs = reinterpret_cast<float *>(smem + LY::qs);
  unsigned char *s_k8 = smem + LY::k8, *s_v8 = smem + LY::v8;
  float *s_sk = reinterpret_cast<float *>(smem + LY::sk), *s_sv = reinterpret_cast<float *>(smem + LY::sv);
  float *s_m = reinterpret_cast<float *>(smem + LY::m);

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, grp = lane >> 4;
  // The tiles of one (sequence, kv head, split) read the same blocks: their
  // workgroups are numbered 8 apart, 8 XCDs, so that they share an L2.
  const int C = p.splits, T = p.t_rows, nq = p.nq, nkv = p.nkv, G = p.by_g.d, R = T * G;
  const int P = FOLD ? (int)p.by_parts.d : C;  // c0, c0 + P, ... are this workgroup's splits
  int tile = 0, unit = blockIdx.x;             // unit = (b * nkv + kvh) * P + c0
  if constexpr (AC == 16) {
    const int tiles = (R + 15) / 16, units = p.batch * nkv * P, whole = units & ~7, x = blockIdx.x;
    if (tiles > 1) {
      const int w = x < whole * tiles ? x >> 3 : x - whole * tiles, q = div_by(p.by_tiles, w);
      tile = w - q * tiles;
      unit = x < whole * tiles ? q * 8 + (x & 7) : whole + q;
    }
  }
  const int cell = div_by(p.by_parts, unit), c0 = unit - cell * P, b = div_by(p.by_nkv, cell), kvh = cell - b * nkv;
  const int r0 = tile * 16, nr = min(R - r0, 16);  // this workgroup's query rows
  const int width = (nq + 2 * nkv) * D;
  int8_t *k8 = p.k8 + (size_t)cell * p.cap * D, *v8 = p.v8 + (size_t)cell * p.cap * D;
  float *kscale = p.k_scale + (size_t)cell * p.cap, *vscale = p.v_scale + (size_t)cell * p.cap;
  const float NEG_INF = -__builtin_huge_valf();

  // One block's keys, values and scales.  MFMA row r of K's tile t is slot 16 (r
  // >> 2) + 4 t + (r & 3), its channels 64 h + 16 grp .. + 15; V's are channel 16 dt +
  // col, slots 16 grp .. + 15; the scales those of slot `lane`.
  uint4 kf[4][NH], vf[DT];
  float ks, vs;
  auto load_k = [&](int j) {
    const int s0 = j * kKv8Block;
    const int8_t *kb = k8 + (size_t)(s0 + 16 * (col >> 2) + (col & 3)) * D + 16 * grp;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int h = 0; h < NH; ++h) kf[t][h] = ld_nt(kb + (4 * t) * D + 64 * h);
    ks = __builtin_nontemporal_load(kscale + s0 + lane);
  };
  auto load_v = [&](int j) {
    const int s0 = j * kKv8Block;
    const int8_t *vb = v8 + ((size_t)((s0 >> 4) + grp) * D + col) * 16;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) vf[dt] = ld_nt(vb + dt * 256);
    vs = __builtin_nontemporal_load(vscale + s0 + lane);
  };
  // This wave's first block, and one round's step.
  const bool takes = BW == NW || wave < BW;
  const int j0 = takes ? BW * c0 + wave : 0x7fffffff, step = BW * C;
  const uint16_t *rows = p.qkv + (size_t)b * T * width;
  const int L = p.lens[b];
  if (L < 0 || L > p.cap - T) {  // no cache access that counts; the rows become NaN
    if (c0 == 0 && !p.out_partials)
      for (int i = threadIdx.x; i < nr * (D / 4); i += blockDim.x) {
        const int y = i / (D / 4), ch = (i - y * (D / 4)) * 4, r = r0 + y, t = div_by(p.by_g, r), row = b * T + t,
                  k = (kvh * G + r - t * G) * D + ch;
        uint16_t *o = p.out + (p.ofrag ? frag_off(row, k, p.ofrag) : (size_t)row * nq * D + k);
        *reinterpret_cast<uint2 *>(o) = make_uint2(0x7fc07fc0u, 0x7fc07fc0u);
      }
    return;
  }
  const int last = L + T - 1, nb = last / kKv8Block + 1;
  if (BW * c0 >= nb) return;
  auto ours = [&](int slot) {  // its run is of one of this workgroup's splits
    const int run = slot / RUN, c = run - div_by(p.by_splits, run) * C;
    return FOLD ? c - div_by(p.by_parts, c) * P == c0 : c == c0;
  };
  const bool mine = ours(L) || ours(last);
  // Rows to prepare, four to a wave: this tile's queries from the last wave on, behind them
  // the new keys and values (for a workgroup that takes some of their blocks).  Every wave's
  // row loads leave before any wave's block loads: the rows' chain (length, tables,
  // preparation) is what the first block waits for, and behind the blocks of a full
  // launch each of its steps would take microseconds.
  constexpr int N = D / 16;
  const int quad = NW - 1 - wave, quads = (nr + 3) / 4;
  const bool query = quad < quads, job = query || (mine && quad < quads + (T + 3) / 4);
  const int i = 4 * (query ? quad : quad - quads) + grp, n = query ? nr : T, at = min(i, n - 1);
  const int t = query ? div_by(p.by_g, r0 + at) : at, head = query ? kvh * G + r0 + at - t * G : nq + kvh, ch = N * col;
  Part<N> raw, vraw, w, cw, sw;
  if (job) {
    const uint16_t *x = rows + (size_t)t * width + (size_t)head * D + ch;
    raw.load(x);
    w.load((query ? p.q_norm_w : p.k_norm_w) + ch);
    cw.load(p.cos_tab + (size_t)(L + t) * D + ch);
    sw.load(p.sin_tab + (size_t)(L + t) * D + ch);
    if (!query) vraw.load(x + (size_t)nkv * D);
  }
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  if (!job && j0 < nb) {
    load_k(j0);
    load_v(j0);
  }
  if (job) {
    float o[N];
    norm_rope<N>(raw, w, cw, sw, p.eps, o);
    const uint32_t top = top_bits<N>(o);
    if (query) {
      // 21 bits, relative to the row's largest, as three digits
      const bool fin = top < 0x7f800000u;
      float down, half_up;
      grid_of(top, down, half_up);
      if (i < n) {
#pragma unroll
        for (int e = 0; e < N; e += 4) {
          uint32_t d[3];
          digits4(o + e, down, d[0], d[1], d[2]);
#pragma unroll
          for (int k = 0; k < 3; ++k) *reinterpret_cast<uint32_t *>(s_q + (k * AC + i) * RS + ch + e) = d[k];
        }
        // (never 0, so that it leaves -inf, a slot not seen, as it is)
        if (col == 0) s_qs[i] = fin ? fmaxf(half_up * p.scale_log2 * 2.f, 0x1p-149f) : __builtin_nanf("");
      }
    } else {
      const bool fin = top < 0x7f800000u;
      const Kv8Div kd(__uint_as_float(top), fin);
      const float sk = kv8_scale(__uint_as_float(top), fin);
      uint32_t kq[N / 4], vq[N / 4];
#pragma unroll
      for (int e = 0; e < N; e += 4) kq[e / 4] = kd.four(o[e], o[e + 1], o[e + 2], o[e + 3]);
#pragma unroll
      for (int e = 0; e < N; ++e) o[e] = vraw[e];
      const uint32_t vtop = top_bits<N>(o);
      const bool vfin = vtop < 0x7f800000u;
      const Kv8Div vd(__uint_as_float(vtop), vfin);
      const float sv = kv8_scale(__uint_as_float(vtop), vfin);
#pragma unroll
      for (int e = 0; e < N; e += 4) vq[e / 4] = vd.four(o[e], o[e + 1], o[e + 2], o[e + 3]);
      const int slot = L + t, byte = slot & 15;
      if (i < n) {
        const bool put = tile == 0 && ours(slot);
        unsigned char *vl = s_v8 + (((slot >> 4) - (L >> 4)) * D + ch) * 16 + byte;
        int8_t *vg = v8 + ((size_t)(slot >> 4) * D + ch) * 16 + byte;
#pragma unroll
        for (int e = 0; e < N; e += 4) {
          *reinterpret_cast<uint32_t *>(s_k8 + t * D + ch + e) = kq[e / 4];
          if (put) *reinterpret_cast<uint32_t *>(k8 + (size_t)slot * D + ch + e) = kq[e / 4];
        }
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const uint32_t x = vq[e / 4] >> (8 * (e & 3));
          vl[16 * e] = (unsigned char)x;
          if (put) vg[16 * e] = (int8_t)x;
        }
        if (col == 0) {
          s_sk[t] = sk;
          s_sv[t] = sv;
          if (put) {
            kscale[slot] = sk;
            vscale[slot] = sv;
          }
        }
      }
    }
    if (j0 < nb) {
      load_k(j0);
      load_v(j0);
    }
  }
  lds_barrier();

  // ---- this wave's blocks
  const int y = col & (AC - 1);
  const bool row_in = y < nr;
  const float qs = row_in ? s_qs[y] : 0.f;
  const int lim = row_in ? L + div_by(p.by_g, r0 + y) : -1;  // the last slot the row sees
  // Query operands: 16 channels 64 h + 16 grp of the column's row, the digits so that
  // scores are (a 2^-6 + c 2^-20) + b 2^-13 in every form: four columns each of a,
  // b, c and nothing; eight of a and c, and b in a second operand; or three operands.
  constexpr int NO = AC == 4 ? 1 : AC == 8 ? 2 : 3;
  uint4 qf[NO][NH];
  constexpr float WA = 0x1p-6f, WB = 0x1p-13f, WC = 0x1p-20f;
  const float weight = AC == 16 ? WA : AC == 8 ? (col < 8 ? WA : WC) : col < 4 ? WA : col < 8 ? WB : WC;
#pragma unroll
  for (int o = 0; o < NO; ++o)
#pragma unroll
    for (int h = 0; h < NH; ++h) {
      const int k = AC == 4 ? col >> 2 : AC == 8 ? (o ? 1 : col >> 3 << 1) : o;
      qf[o][h] = row_in && k < 3 ? *reinterpret_cast<const uint4 *>(s_q + (k * AC + y) * RS + 64 * h + 16 * grp) : zero4();
    }
  auto each = [&](auto fn) {
    fn(Int<0>{}); fn(Int<1>{}); fn(Int<2>{}); fn(Int<3>{}); fn(Int<4>{}); fn(Int<5>{}); fn(Int<6>{}); fn(Int<7>{});
    fn(Int<8>{}); fn(Int<9>{}); fn(Int<10>{}); fn(Int<11>{}); fn(Int<12>{}); fn(Int<13>{}); fn(Int<14>{}); fn(Int<15>{});
  };

  const int n_active = min(C, (nb + BW - 1) / BW);
  for (int c = c0; c < n_active; c += P) {
    // Of the split's blocks so far: the largest score (before scale_q) and, in powers of 2, the largest
    // |w| beside it; acc is in units of 2^(level - 15).
    float m_run = NEG_INF, l_run = 0.f, level = NEG_INF;
    f32x4_t acc[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) acc[dt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    for (int j = takes ? BW * c + wave : nb; j < nb; j += step) {
      const int next = j + step < nb ? j + step : FOLD && c + P < n_active ? BW * (c + P) + wave : nb;
      const int s0 = j * kKv8Block;
      const bool edge = s0 + kKv8Block > L;  // slots that not every row sees, the new rows among them
      if (edge) {                            // which come from LDS
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const int i = s0 + 16 * (col >> 2) + 4 * t + (col & 3) - L;
          const bool is = (unsigned)i < (unsigned)T;
#pragma unroll
          for (int h = 0; h < NH; ++h) {
            const uint4 x = *reinterpret_cast<const uint4 *>(s_k8 + min(max(i, 0), kKv8MaxT - 1) * D + 64 * h + 16 * grp);
            if (is) kf[t][h] = x;
          }
        }
        const int v0 = s0 + 16 * grp, gi = min(max((v0 >> 4) - (L >> 4), 0), 1);
        // byte i of this lane's 16: slot v0 + i, a new row's from L to `last`
        auto from = [&](int s, int d) {  // dword d's bytes from slot s on
          const int n = min(max(s - v0 - 4 * d, 0), 4);
          return (uint32_t)(0xffffffffull << (8 * n));
        };
        uint32_t take[4];
#pragma unroll
        for (int d = 0; d < 4; ++d) take[d] = from(L, d) & ~from(last + 1, d);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          const uint4 x = *reinterpret_cast<const uint4 *>(s_v8 + (gi * D + dt * 16 + col) * 16);
          uint4 &v = vf[dt];
          v.x = (v.x & ~take[0]) | (x.x & take[0]);
          v.y = (v.y & ~take[1]) | (x.y & take[1]);
          v.z = (v.z & ~take[2]) | (x.z & take[2]);
          v.w = (v.w & ~take[3]) | (x.w & take[3]);
        }
        const int i = s0 + lane - L;
        if ((unsigned)i < (unsigned)T) {
          ks = s_sk[i];
          vs = s_sv[i];
        }
      }
      float s[16];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        i32x4_t d[NO];
#pragma unroll
        for (int o = 0; o < NO; ++o) {
          d[o] = i32x4_t{0, 0, 0, 0};
#pragma unroll
          for (int h = 0; h < NH; ++h) d[o] = mfma_i8(kf[t][h], qf[o][h], d[o]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float x = (float)d[0][i] * weight;
          if constexpr (AC == 16) {
            x = __builtin_fmaf((float)d[1][i], WB, __builtin_fmaf((float)d[2][i], WC, x));
          } else {
            x += dpp_f<0x128>(x);  // row_ror:8, a + c
            if constexpr (AC == 8) x = __builtin_fmaf((float)d[1][i], WB, x);
            else x += dpp_f<0x124>(x);  // row_ror:4
          }
          s[4 * t + i] = x;
        }
      }
      // lane (col, grp) holds slots s0 + 16 grp + i of its row
      each([&](auto n) {
        constexpr int i = decltype(n)::value;
        s[i] *= row_lane<i>(ks);
        pin(s[i]);
      });
      if (next < nb) load_k(next);
      // of them, those up to `seen` (pins: a branch around the selects, not sixteen in every block)
      int seen = lim - s0 - 16 * grp;
      if (edge) {
        pin(seen);
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = i > seen ? NEG_INF : s[i];
      }
      float top = s[0];
#pragma unroll
      for (int i = 1; i < 16; ++i) top = fmaxf(top, s[i]);
      const float m_old = m_run;
      m_run = fmaxf(m_run, max_xor16_32(top));
      const float base = m_run == NEG_INF ? 0.f : m_run;
      float psum = 0.f, big = 0.f;
      each([&](auto n) {
        constexpr int i = decltype(n)::value;
        const float e = __builtin_amdgcn_exp2f((s[i] - base) * qs);
        psum += e;
        s[i] = e * row_lane<i>(vs);
      });
      if (edge) {
        pin(seen);
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = i > seen ? 0.f : s[i];
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) big = fmaxf(big, s[i]);
      const float fall = (m_old - base) * qs;  // of what is there, in powers of 2
      l_run = __builtin_fmaf(l_run, __builtin_amdgcn_exp2f(fall), psum);
      const float level_old = level + fall;
      // (Not below -111, so that w's factor stays in range also where a slot with values of zero has
      // raised the maximum, not level: a normal w is 1 or more then, which fp16 rounds as ever.)
      level = fmaxf(fmaxf(level_old, __builtin_amdgcn_logf(max_xor16_32(big))), -111.f);
      const float up = __builtin_amdgcn_exp2f(15.f - level);
      f16x8_t w[2];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        w[0][e] = (_Float16)(s[e] * up);
        w[1][e] = (_Float16)(s[8 + e] * up);
      }
      if (__any(level_old < level)) {
        const float ra = level_old < level ? __builtin_amdgcn_exp2f(level_old - level) : 1.f;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) acc[dt] *= ra;
      }
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        f16x8_t a[2];
        to_f16(vf[dt], a[0], a[1]);
        acc[dt] = mfma_f16(a[0], w[0], acc[dt]);
        acc[dt] = mfma_f16(a[1], w[1], acc[dt]);
      }
      if (next < nb) load_v(next);
    }

    // ---- the waves' sums, in wave order; then the output or a partial: the
    // row's sum of values and of probabilities, both times 2^-20 (no value overflows
    // with so many slots), and its maximum.
    if (FOLD && c > c0) lds_barrier();  // the last split's are read
    if (takes && col < AC) {
      const float lw = sum_xor16_32(l_run);
      if (grp == 0) {
        s_m[col * BW + wave] = m_run;
        s_m[(16 + col) * BW + wave] = lw;
        s_m[(32 + col) * BW + wave] = level;
      }
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) s_acc[((wave * DT + dt) * 4 + grp) * AC + col] = acc[dt];
    }
    lds_barrier();
    if (row_in && col < AC) {
      float mw[BW], lw[BW], uw[BW], M = NEG_INF, U = NEG_INF, sum = 0.f;
#pragma unroll
      for (int w = 0; w < BW; w += 4) {
        *reinterpret_cast<f32x4_t *>(mw + w) = *reinterpret_cast<const f32x4_t *>(s_m + col * BW + w);
        *reinterpret_cast<f32x4_t *>(lw + w) = *reinterpret_cast<const f32x4_t *>(s_m + (16 + col) * BW + w);
        *reinterpret_cast<f32x4_t *>(uw + w) = *reinterpret_cast<const f32x4_t *>(s_m + (32 + col) * BW + w);
      }
#pragma unroll
      for (int w = 0; w < BW; ++w) M = fmaxf(M, mw[w]);
#pragma unroll
      for (int w = 0; w < BW; ++w) {
        const float fall = mw[w] == NEG_INF ? NEG_INF : (mw[w] - M) * qs;
        // (a NaN among a wave's scores stays, also where it saw nothing else)
        sum = __builtin_fmaf(lw[w], __builtin_amdgcn_exp2f(fall), sum);
        uw[w] += fall;
        U = fmaxf(U, uw[w]);
      }
#pragma unroll
      for (int w = 0; w < BW; ++w) uw[w] = uw[w] == NEG_INF ? 0.f : __builtin_amdgcn_exp2f(uw[w] - U);
      const int r = r0 + y;
      float *part = p.partial + ((size_t)cell * C + c) * kv8_partial_floats(R, D);
      const bool direct = n_active == 1 && !p.out_partials;
      // (2^(U - 15), a normal number for every row that is held, and 2^-20 by itself: together they
      // would be 0 for values below 2^-84)
      const float scale = U == NEG_INF ? 0.f : __builtin_amdgcn_exp2f(U - 15.f), wt = sum * 0x1p-20f;
      for (int dt = wave; dt < DT; dt += NW) {
        f32x4_t o = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < BW; ++w) {
          const f32x4_t a = s_acc[((w * DT + dt) * 4 + grp) * AC + col];
#pragma unroll
          for (int i = 0; i < 4; ++i) o[i] = __builtin_fmaf(a[i], uw[w], o[i]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = o[i] * 0x1p-20f * scale;
        const int k = dt * 16 + grp * 4;
        if (direct) {  // (as the merge has it of one partial)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[i] /= wt;
          const int t = div_by(p.by_g, r), row = b * T + t, kk = (kvh * G + r - t * G) * D + k;
          uint16_t *dst = p.out + (p.ofrag ? frag_off(row, kk, p.ofrag) : (size_t)row * nq * D + kk);
          *reinterpret_cast<uint2 *>(dst) = make_uint2(pack2(o[0], o[1]), pack2(o[2], o[3]));
        } else {
          *reinterpret_cast<f32x4_t *>(part + (size_t)r * D + k) = o;
        }
      }
      if (!direct && wave == 0 && grp == 0) {  // (a maximum of -inf: nothing seen)
        part[(size_t)R * D + r] = M != NEG_INF ? M * qs : sum != 0.f ? 0.f : M;
        part[(size_t)R * D + R + r] = wt;
      }
    }
    if constexpr (!FOLD) break;
  }
}

// Merge of the splits' partials, in order: D / 4 threads per query row.  The operations
// are those of attn_merge8 (gemm_dev.h), so a GEMM that merges has the same bits.
// CB partials are loaded at a time, 8 or (from 9 splits on) 16.  Workgroups of one wave
// reach more CUs than those of four (call and merge, us, 256 / 64 threads: 13 sequences of
// 1100 slots 13.8 / 13.5, one of 131000 in 32 splits 54.1 / 53.2).
template <int D, int CB>
__global__ void __launch_bounds__(64) kv8_merge_kernel(const Kv8AttnParams p) {
  constexpr int TR = D / 4;
  const int G = p.by_g.d, R = p.t_rows * G, kvh = blockIdx.y, b = blockIdx.z;
  const int r = blockIdx.x * (64 / TR) + threadIdx.x / TR;
  const int L = p.lens[b];
  if (r >= R || L < 0 || L > p.cap - p.t_rows) return;
  const int n = min(p.splits, ((L + p.t_rows - 1) >> p.run_log2) + 1);
  if (n == 1) return;  // written by its workgroup
  const int ch = (int)(threadIdx.x % TR) * 4;
  const size_t stride = kv8_partial_floats(R, D);
  const float *part = p.partial + ((size_t)b * p.nkv + kvh) * p.splits * stride;
  const float NEG_INF = -__builtin_huge_valf();
  float m[CB], l[CB];
  f32x4_t a[CB];
  auto load_group = [&](int i0) {
#pragma unroll
    for (int i = 0; i < CB; ++i) {
      const float *pr = part + (size_t)min(i0 + i, n - 1) * stride;
      m[i] = pr[(size_t)R * D + r];
      l[i] = pr[(size_t)R * D + R + r];
      a[i] = *reinterpret_cast<const f32x4_t *>(pr + (size_t)r * D + ch);
    }
  };
  load_group(0);
  float M = NEG_INF, sum = 0.f;
  f32x4_t o = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < CB; ++i) M = fmaxf(M, m[i]);  // (the last partial repeats)
  for (int i0 = CB; i0 < n; i0 += CB) {
    float x[CB];
#pragma unroll
    for (int i = 0; i < CB; ++i) x[i] = part[(size_t)min(i0 + i, n - 1) * stride + (size_t)R * D + r];
#pragma unroll
    for (int i = 0; i < CB; ++i) M = fmaxf(M, x[i]);
  }
  for (int i0 = 0; i0 < n; i0 += CB) {
    if (i0 > 0) load_group(i0);
#pragma unroll
    for (int i = 0; i < CB; ++i) {
      if (i0 + i >= n || m[i] == NEG_INF) continue;
      const float w = exp2f(m[i] - M);
      sum = __builtin_fmaf(l[i], w, sum);
#pragma unroll
      for (int d = 0; d < 4; ++d) o[d] = __builtin_fmaf(a[i][d], w, o[d]);
    }
  }
  const int t = div_by(p.by_g, r), row = b * p.t_rows + t, k = (kvh * G + r - t * G) * D + ch;
  uint16_t *dst = p.out + (p.ofrag ? frag_off(row, k, p.ofrag) : (size_t)row * p.nq * D + k);
  *reinterpret_cast<uint2 *>(dst) = make_uint2(pack2(o[0] / sum, o[1] / sum), pack2(o[2] / sum, o[3] / sum));
}

template <int D, int BW>
hipError_t launch_d(const Kv8AttnParams &p, hipStream_t s) {
  const int R = p.t_rows * (p.nq / p.nkv);
  const dim3 grid((unsigned)(p.batch * p.nkv * (int)p.by_parts.d * ((R + 15) / 16)));
  const dim3 block(64 * (R <= 8 ? BW : 8));
  if (R <= 4) hipLaunchKernelGGL((kv8_attn_kernel<D, 4, BW, false>), grid, block, 0, s, p);
  else if (R <= 8) hipLaunchKernelGGL((kv8_attn_kernel<D, 8, BW, false>), grid, block, 0, s, p);
  else if ((int)p.by_parts.d == p.splits) hipLaunchKernelGGL((kv8_attn_kernel<D, 16, BW, false>), grid, block, 0, s, p);
  else hipLaunchKernelGGL((kv8_attn_kernel<D, 16, BW, true>), grid, block, 0, s, p);
  if (p.splits > 1 && !p.out_partials) {
    const int per = 64 / (D / 4);
    const auto merge = p.splits > 8 ? kv8_merge_kernel<D, 16> : kv8_merge_kernel<D, 8>;
    hipLaunchKernelGGL(merge, dim3((R + per - 1) / per, p.nkv, p.batch), dim3(64), 0, s, p);
  }
  return hipSuccess;
}

}  // namespace

// Slots of a run: 8 blocks, or 4 where a workgroup for each of those finds a CU of its own.  A CU
// has about 64 KB in flight, half of what 8 waves ask for at once, so more CUs take
// less time until their partials cost more than that.  us with runs of 512 / 256, each in
// its splits and with the merge, 32 heads on 8: one sequence of 1500 slots 11.1 / 9.4, of
// 4000 12.1 / 12.0 and with 9 rows 13.1 / 14.9, of 6100 12.5 / 12.9; two of 1100 11.1 /
// 9.2, four 11.4 / 9.7.  Up to 512 slots a run of 8 blocks needs no merge.  The rules must not
// look at t_rows: a row keeps its bits.
static bool short_runs(int batch, int nkv, int cap) {
  return cap > 512 && cap <= 2048 && (int64_t)batch * nkv * ((cap + 255) / 256) <= 256;
}
// In one split: also where there are more workgroups than CUs, since registers hold two of 4
// waves, which start and end beside each other (us, 64 sequences of 300 slots 18.0 /
// 13.4, of 500 21.4 / 17.7, of 1100 33.6 / 30.5, of 2100 53.6 / 50.6, 40 of 500 18.9 / 15.5; but
// 32 of 1100 18.4 / 19.3), and for short caches of more than a few sequences (32 of 200 8.7 /
// 8.3; one of 60 6.2 / 6.6).
int kv8_attn_run(int batch, int nkv, int cap, int splits) {
  const int64_t cells = (int64_t)batch * nkv;
  if (splits > 1) return short_runs(batch, nkv, cap) ? 256 : 512;
  return cells > 256 || (cells > 64 && cap <= 512) ? 256 : 512;
}

// At most one workgroup of few rows to a CU (registers hold one of 8 waves: a second
// would run behind it).  us for runs of 512 in 1 / 2 / 4 splits: 8 sequences of 1100
// slots 13.8 / 12.8 / 12.1; 13 of 1100 15.2 / 14.1 / 21.3; 20 of 1100 16.2 / 23.4 / -; 16
// of 4200 41.6 / 30.9 / 35.6.  Up to 1024 slots a merge costs as much as it gives: one
// sequence of 640 slots in 1 split 9.7, in 3 of short runs 9.3 in a replayed graph, but 11.5
// and 12.9 launch by launch.  A caller that has the merge done elsewhere asks for 3.
int kv8_attn_splits(int batch, int nkv, int cap) {
  const int64_t cells = (int64_t)batch * nkv;
  if (cap <= 1024) return 1;
  if (short_runs(batch, nkv, cap)) return (cap + 255) / 256;
  return (int)std::max<int64_t>(1, std::min<int64_t>(256 / cells, (cap + 511ll) / 512));
}

// Workgroups that share the splits of a (sequence, kv head, row tile): with several
// tiles of rows, so many that all run at once.  us for 8 sequences of 2000 slots and
// 8 rows, 4 splits, a workgroup each / shared: 32 heads on 8 23.9 / 20.7, 64 on 8 41.0 /
// 31.7; 500 slots in 4 splits 20.9 / 12.3.
int kv8_attn_parts(int batch, int nkv, int splits, int tiles) {
  if (tiles == 1) return splits;
  const int64_t n = 256 / ((int64_t)batch * nkv * tiles);
  return (int)std::max<int64_t>(1, std::min<int64_t>(splits, n));
}

hipError_t launch_kv8_attn(const Kv8AttnParams &p, hipStream_t s) {
  if (p.run_log2 == 8) return p.head_dim == 128 ? launch_d<128, 4>(p, s) : launch_d<64, 4>(p, s);
  return p.head_dim == 128 ? launch_d<128, 8>(p, s) : launch_d<64, 8>(p, s);
}

}  // namespace qdec
