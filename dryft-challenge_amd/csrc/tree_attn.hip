// Attention of a tree of drafted tokens over a KV cache, with the head
// RMSNorm and RoPE of the nodes folded in: T nodes per sequence, each seeing
// all L cached slots, its ancestors and itself.
//
// With G = nq / nkv query heads per kv head, query row r = G*t + h of a kv head
// is node t's query head h.  A workgroup of four waves takes up to 64 rows of
// one (sequence, kv head) -- MTQ M tiles of 16 -- and a contiguous run of the
// 32-row key/value blocks, of which there are ceil(L / 32) in the cache and
// ceil(T / 32) of nodes behind them.  The run's blocks are dealt to the waves
// round robin; every wave holds all the workgroup's rows, so a key or value
// fragment goes straight from memory into the registers of the one wave that
// uses it, and no LDS traffic or barrier is in the loop.
//
//   1. Ancestor sets: lane t of a wave holds node t's set as 64 bits and a
//      pointer to its parent; pointer doubling unites the sets in at most six
//      rounds.  A set that does not reach the root is no node's.  The depth
//      is the size of the set less one.
//   2. Queries: D/8 lanes per row, 8 channels each; normalised, rotated rows
//      go to LDS and come back as B operands of v_mfma_f32_16x16x32_bf16.  The
//      workgroups that take node blocks prepare the new keys the same way.
//   3. Per block S^T = K . Q^T, online softmax in base 2 on fp32 scores, O^T
//      += V^T . P^T (P rounded to bf16, the operand type).  The running
//      maximum is only moved, and the sums rescaled, in blocks where some
//      row's maximum grows.
//   4. The waves merge in LDS; with more than one workgroup per row group the
//      partials go to memory and the last workgroup to arrive merges them in
//      order.
#include "qdec_common.h"
#include "qdec_kernels.h"

namespace qdec {

namespace {

constexpr int kTW = 4;  // waves per workgroup

template <int D>
struct TreeLds {
  static constexpr int RS = D + 8;  // bf16 per LDS row of queries or keys (bank spread)
  static constexpr int q = 0;       // queries [64][RS], then the waves' partials
  static constexpr int part_bytes = kTW * (D / 16) * 64 * 16;
  static constexpr int q_bytes = kTreeGroupRows * RS * 2 > part_bytes ? kTreeGroupRows * RS * 2 : part_bytes;
  static constexpr int k = q + q_bytes;                 // new keys [64][RS]
  static constexpr int v = k + kTreeMaxT * RS * 2;      // new values [8][D][8]
  static constexpr int m = v + kTreeMaxT * D * 2;       // wave row maxima [kTW][16]
  static constexpr int l = m + kTW * 16 * 4;            // wave row sums [kTW][16]
  static constexpr int bad = l + kTW * 16 * 4;          // nodes with a value that is not finite
  static constexpr int flag = bad + kTreeMaxT * 4;
  static constexpr int bytes = flag + 16;
};

__device__ __forceinline__ float max16_32(float v) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

__device__ __forceinline__ uint64_t shfl64(uint64_t v, int l) {
  const uint32_t lo = (uint32_t)__shfl((int)(uint32_t)v, l, 64);
  const uint32_t hi = (uint32_t)__shfl((int)(uint32_t)(v >> 32), l, 64);
  return ((uint64_t)hi << 32) | lo;
}

// Head RMSNorm and RoPE of one head row held by D/8 consecutive lanes, 8
// channels each (raw, w, cos and sin as bf16).  The sum of squares is the
// balanced tree over the channels that head_norm_rope builds and the products
// of bf16 squares are exact, so both give the same bits.
template <int D>
__device__ __forceinline__ uint4 head_row(const uint4 &raw, const uint4 &w, const uint4 &cw, const uint4 &sw, float eps) {
  constexpr int LPR = D / 8;
  float x[8], g[8], c[8], s[8], y[8];
  unpack8(raw, x);
  unpack8(w, g);
  unpack8(cw, c);
  unpack8(sw, s);
  float ss = ((x[0] * x[0] + x[1] * x[1]) + (x[2] * x[2] + x[3] * x[3])) +
             ((x[4] * x[4] + x[5] * x[5]) + (x[6] * x[6] + x[7] * x[7]));
  ss += dpp_f<0xB1>(ss);                           // lane ^ 1
  ss += dpp_f<0x4E>(ss);                           // lane ^ 2
  ss += dpp_f<0x141>(ss);                          // the other quad of 8
  if constexpr (LPR == 16) ss += dpp_f<0x140>(ss); // the other 8 of 16
  const float rstd = 1.0f / sqrtf(ss / (float)D + eps);
#pragma unroll
  for (int e = 0; e < 8; ++e) y[e] = rbf(g[e] * rbf(x[e] * rstd));
  const uint4 mine = pack8(y);
  uint4 other;  // channels i +- D/2: bf16 values, so four words
  other.x = (uint32_t)__shfl_xor((int)mine.x, LPR / 2, 64);
  other.y = (uint32_t)__shfl_xor((int)mine.y, LPR / 2, 64);
  other.z = (uint32_t)__shfl_xor((int)mine.z, LPR / 2, 64);
  other.w = (uint32_t)__shfl_xor((int)mine.w, LPR / 2, 64);
  float r[8];
  unpack8(other, r);
  const bool first = (threadIdx.x & (LPR - 1)) < LPR / 2;
#pragma unroll
  for (int e = 0; e < 8; ++e) y[e] = rbf(y[e] * c[e]) + rbf((first ? -r[e] : r[e]) * s[e]);
  return pack8(y);
}

__device__ __forceinline__ bool finite8(const uint4 &v) {
  auto two = [](uint32_t w) { return (w & 0x7f80u) != 0x7f80u && (w & 0x7f800000u) != 0x7f800000u; };
  return two(v.x) && two(v.y) && two(v.z) && two(v.w);
}

__device__ __forceinline__ uint4 ld16(const uint16_t *p) { return *reinterpret_cast<const uint4 *>(p); }

template <int D, int MTQ>
__global__ void __launch_bounds__(64 * kTW, MTQ <= 1 ? 2 : 1) tree_attn_kernel(const TreeAttnParams p) {
  using LY = TreeLds<D>;
  constexpr int RS = LY::RS;
  constexpr int DS = D / 32, DT = D / 16, DTW = DT / kTW;
  constexpr int LPR = D / 8, RPW = 64 / LPR;  // lanes per prepared row, rows per wave and pass
  __shared__ __align__(16) unsigned char smem[LY::bytes];
  uint16_t *s_q = reinterpret_cast<uint16_t *>(smem + LY::q);
  f32x4_t *s_acc = reinterpret_cast<f32x4_t *>(smem + LY::q);
  uint16_t *s_k = reinterpret_cast<uint16_t *>(smem + LY::k);
  uint16_t *s_v = reinterpret_cast<uint16_t *>(smem + LY::v);
  float *s_m = reinterpret_cast<float *>(smem + LY::m);
  float *s_l = reinterpret_cast<float *>(smem + LY::l);
  int *s_bad = reinterpret_cast<int *>(smem + LY::bad);
  uint32_t *s_flag = reinterpret_cast<uint32_t *>(smem + LY::flag);
  const float NEG_INF = -__builtin_huge_valf();

  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int col = lane & 15, grp = lane >> 4;

  // The row groups of one (sequence, kv head, split) read the same keys and
  // values: they get numbers that are equal modulo 8, the number of XCDs, and
  // close together, so that they share an L2.
  const int ng = p.groups, C = p.splits;
  const int units = p.batch * p.nkv * C, whole = units & ~7;
  int unit, g;
  if ((int)blockIdx.x < whole * ng) {
    const int q = blockIdx.x >> 3;
    g = q % ng;
    unit = (q / ng) * 8 + (blockIdx.x & 7);
  } else {
    const int y = blockIdx.x - whole * ng;
    g = y % ng;
    unit = whole + y / ng;
  }
  const int c = unit % C, cell = unit / C;  // cell = b * nkv + kvh
  const int kvh = cell % p.nkv, b = cell / p.nkv;

  const int T = p.t_rows, nq = p.nq, nkv = p.nkv, G = nq / nkv;
  const int R = T * G, r0 = g * 16 * MTQ;  // this workgroup's rows r0 .. r0 + rows - 1
  const int rows = min(16 * MTQ, R - r0);
  const int width = (nq + 2 * nkv) * D;
  const uint16_t *qkv = p.qkv + (size_t)b * T * width;
  auto out_at = [&](int m, int k) { return p.ofrag ? p.out + frag_off(m, k, p.ofrag) : p.out + (size_t)m * nq * D + k; };

  const int L = p.lens[b];
  if (L < 0 || L > p.cap - T) {
    if (c == 0)
      for (int i = threadIdx.x; i < rows * (D / 4); i += 64 * kTW) {
        const int r = r0 + i / (D / 4), k4 = i % (D / 4) * 4;
        *reinterpret_cast<uint2 *>(out_at(b * T + r / G, (kvh * G + r % G) * D + k4)) = make_uint2(0x7fc07fc0u, 0x7fc07fc0u);
      }
    return;
  }
  const int nb = (L + 31) >> 5, ntot = nb + ((T + 31) >> 5);
  const int n_active = max(1, min(C, (ntot + p.min_blocks - 1) / p.min_blocks));
  if (c >= n_active) return;
  const int j0 = (int)((int64_t)ntot * c / n_active), j1 = (int)((int64_t)ntot * (c + 1) / n_active);

  const size_t slab = (size_t)cell * p.cap * D;
  const uint16_t *kc = p.k_cache + slab, *vc = p.v_cache + slab;
  struct Frag {
    uint4 ka[DS], kb[DS], vf[DT];
  };
  // Key rows of tile a: 8*(m >> 2) + (m & 3), of tile b 4 further, so that a
  // lane's 8 scores are 8 consecutive rows, the B operand of the P.V product.
  const int ra = 8 * (col >> 2) + (col & 3);
  auto load_block = [&](int j, Frag &f) {
    const uint16_t *kp = kc + (size_t)(32 * j + ra) * D + 8 * grp;
    const uint16_t *vp = vc + ((size_t)(4 * j + grp) * D + col) * 8;
#pragma unroll
    for (int s = 0; s < DS; ++s) {
      f.ka[s] = ld_nt(kp + s * 32);
      f.kb[s] = ld_nt(kp + 4 * D + s * 32);
    }
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) f.vf[dt] = ld_nt(vp + dt * 128);
  };
  Frag f0, f1;
  if (j0 + wave < min(j1, nb)) load_block(j0 + wave, f0);

  // ---- 1. ancestor sets.
  uint64_t anc;
  {
    int up = lane < T ? p.parents[(size_t)b * T + lane] : -1;
    if (lane == 0) up = 0;
    if (up < 0 || up > lane || (up == lane && lane > 0)) up = lane;  // no node: a root of its own
    anc = 1ull << lane;
    for (int i = 0; i < 6; ++i) {
      const int up2 = __shfl(up, up, 64);
      anc |= shfl64(anc, up);
      if (!__any(up2 != up)) break;
      up = up2;
    }
    if (!(anc & 1) || lane >= T) anc = 0;
  }
  const int depth = (int)__popcll(anc) - 1;  // -1: no node (its rows are prepared at L and dropped)
  const int pos = depth > 0 ? L + depth : L;
  const uint64_t nodes = __ballot(anc != 0);

  // ---- 2. queries, and the new keys and values of this run's node blocks.
  const int sub = lane % LPR, ch = sub * 8;
  {
    const uint4 w = ld16(p.q_norm_w + ch);
    for (int i = wave * RPW + lane / LPR; i < 16 * MTQ; i += kTW * RPW) {
      const int r = r0 + min(i, rows - 1), t = r / G;
      const int pt = __shfl(pos, t, 64);
      const uint4 raw = ld16(qkv + (size_t)t * width + (size_t)(kvh * G + r % G) * D + ch);
      const uint4 cw = ld16(p.cos_tab + (size_t)pt * D + ch), sw = ld16(p.sin_tab + (size_t)pt * D + ch);
      *reinterpret_cast<uint4 *>(s_q + i * RS + ch) = head_row<D>(raw, w, cw, sw, p.eps);
    }
  }
  const int n0 = max(j0 - nb, 0) * 32, n1 = min((j1 - nb) * 32, kTreeMaxT);  // nodes of this run, n1 <= n0: none
  if (n1 > n0) {
    const uint4 w = ld16(p.k_norm_w + ch);
    for (int t = n0 + wave * RPW + lane / LPR; t < n1; t += kTW * RPW) {
      const bool node = (nodes >> t) & 1;
      const int tr = min(t, T - 1);
      const int pt = __shfl(pos, tr, 64);
      const uint16_t *row = qkv + (size_t)tr * width + (size_t)(nq + kvh) * D + ch;
      const uint4 cw = ld16(p.cos_tab + (size_t)pt * D + ch), sw = ld16(p.sin_tab + (size_t)pt * D + ch);
      const uint4 k = head_row<D>(ld16(row), w, cw, sw, p.eps);
      const uint4 v = ld16(row + (size_t)nkv * D);
      if (node && g == 0) {
        const size_t at = ((size_t)cell * T + t) * D + ch;
        *reinterpret_cast<uint4 *>(p.k_nodes + at) = k;
        *reinterpret_cast<uint4 *>(p.v_nodes + at) = v;
      }
      *reinterpret_cast<uint4 *>(s_k + t * RS + ch) = k;
      // A value that is not finite would reach every row through 0 * inf:
      // such a node's values are zero here and added below to the rows that
      // see it.
      const uint64_t part = __ballot(!finite8(v)) >> (lane & ~(LPR - 1));
      const bool bad = node && (part & ((1ull << LPR) - 1));
      if (sub == 0) s_bad[t] = bad;
      const uint32_t keep = node && !bad ? ~0u : 0u;
      const uint32_t vw[4] = {v.x & keep, v.y & keep, v.z & keep, v.w & keep};
      uint16_t *dst = s_v + ((size_t)(t >> 3) * D + ch) * 8 + (t & 7);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        dst[16 * e] = (uint16_t)(vw[e] & 0xffffu);
        dst[16 * e + 8] = (uint16_t)(vw[e] >> 16);
      }
    }
  }
  lds_barrier();
  uint64_t badset = 0;
  if (n1 > n0) badset = __ballot(lane >= n0 && lane < n1 && s_bad[lane]);

  uint4 qf[MTQ][DS];
  uint64_t sees[MTQ];
  f32x4_t acc[MTQ][DT];
  float m_run[MTQ], l_run[MTQ];
#pragma unroll
  for (int mt = 0; mt < MTQ; ++mt) {
#pragma unroll
    for (int s = 0; s < DS; ++s) qf[mt][s] = *reinterpret_cast<const uint4 *>(s_q + (mt * 16 + col) * RS + s * 32 + grp * 8);
    sees[mt] = shfl64(anc, min(r0 + mt * 16 + col, R - 1) / G);
    m_run[mt] = NEG_INF;
    l_run[mt] = 0.f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) acc[mt][dt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }

  // ---- 3. the blocks.
  const float scale = p.scale_log2;
  auto process = [&](Frag &f, int j) {
    f32x4_t sa[MTQ], sb[MTQ];
    if (j >= nb) {  // node rows 32*(j - nb) ..
      const int t0 = 32 * (j - nb);
#pragma unroll
      for (int s = 0; s < DS; ++s) {
        f.ka[s] = *reinterpret_cast<const uint4 *>(s_k + (t0 + ra) * RS + s * 32 + grp * 8);
        f.kb[s] = *reinterpret_cast<const uint4 *>(s_k + (t0 + ra + 4) * RS + s * 32 + grp * 8);
      }
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
        f.vf[dt] = *reinterpret_cast<const uint4 *>(s_v + ((size_t)((t0 >> 3) + grp) * D + dt * 16 + col) * 8);
    } else if (32 * j + 32 > L) {  // the last cached block: slots from L on hold anything
      const int v0 = 32 * j + 8 * grp;
      uint32_t keep[4];
#pragma unroll
      for (int d = 0; d < 4; ++d)
        keep[d] = (v0 + 2 * d < L ? 0x0000ffffu : 0u) | (v0 + 2 * d + 1 < L ? 0xffff0000u : 0u);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        f.vf[dt].x &= keep[0];
        f.vf[dt].y &= keep[1];
        f.vf[dt].z &= keep[2];
        f.vf[dt].w &= keep[3];
      }
    }
#pragma unroll
    for (int mt = 0; mt < MTQ; ++mt) {
      sa[mt] = sb[mt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < DS; ++s) {
        sa[mt] = mfma16x16x32(f.ka[s], qf[mt][s], sa[mt]);
        sb[mt] = mfma16x16x32(f.kb[s], qf[mt][s], sb[mt]);
      }
    }
    if (32 * j + 32 > L || j >= nb) {
#pragma unroll
      for (int mt = 0; mt < MTQ; ++mt) {
        const uint32_t bits = j >= nb ? (uint32_t)(sees[mt] >> (32 * (j - nb))) >> (8 * grp)
                                      : (uint32_t)((1ull << min(max(L - 32 * j - 8 * grp, 0), 8)) - 1);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (!((bits >> i) & 1)) sa[mt][i] = NEG_INF;
          if (!((bits >> (4 + i)) & 1)) sb[mt][i] = NEG_INF;
        }
      }
    }
#pragma unroll
    for (int mt = 0; mt < MTQ; ++mt) {
      const float bmax = fmaxf(fmaxf(fmaxf(sa[mt][0], sa[mt][1]), fmaxf(sa[mt][2], sa[mt][3])),
                               fmaxf(fmaxf(sb[mt][0], sb[mt][1]), fmaxf(sb[mt][2], sb[mt][3])));
      if (__any(bmax > m_run[mt])) {
        const float m_new = fmaxf(m_run[mt], max16_32(bmax));
        const float alpha = m_new == NEG_INF ? 1.f : __builtin_amdgcn_exp2f((m_run[mt] - m_new) * scale);
        l_run[mt] *= alpha;
        m_run[mt] = m_new;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) acc[mt][dt] *= alpha;
      }
      const float mc = m_run[mt] == NEG_INF ? 0.f : m_run[mt] * scale;
      float pj[8];
#pragma unroll
      for (int e = 0; e < 8; ++e)
        pj[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(e < 4 ? sa[mt][e] : sb[mt][e - 4], scale, -mc));
      l_run[mt] += ((pj[0] + pj[1]) + (pj[2] + pj[3])) + ((pj[4] + pj[5]) + (pj[6] + pj[7]));
      const uint4 pf = pack8(pj);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) acc[mt][dt] = mfma16x16x32(f.vf[dt], pf, acc[mt][dt]);
      if (j >= nb && (badset >> (32 * (j - nb))) & 0xffffffffu) {
        for (uint32_t left = (uint32_t)(badset >> (32 * (j - nb))); left; left &= left - 1) {
          const int i = __builtin_ctz(left), t = 32 * (j - nb) + i;
          float mine = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) mine = (i & 7) == e ? rbf(pj[e]) : mine;
          const float pr = __shfl(mine, col + 16 * (i >> 3), 64);
          if (!((sees[mt] >> t) & 1)) continue;
          const uint16_t *vr = qkv + (size_t)t * width + (size_t)(nq + nkv + kvh) * D;
#pragma unroll
          for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[mt][dt][e] += pr * bf2f(vr[dt * 16 + grp * 4 + e]);
        }
      }
    }
  };
  const int jc = min(j1, nb);  // blocks before jc come from the cache
  for (int j = j0 + wave; j < j1; j += 2 * kTW) {
    if (j + kTW < jc) load_block(j + kTW, f1);
    process(f0, j);
    if (j + 2 * kTW < jc) load_block(j + 2 * kTW, f0);
    if (j + kTW < j1) process(f1, j + kTW);
  }

  // ---- 4. merge.  A part whose rows saw nothing has maximum -inf and sum 0;
  // its weight is its sum times zero, so that a NaN among its scores stays.
  const bool direct = n_active == 1;
  constexpr int RG = 16 * MTQ;
  constexpr size_t kPart = (size_t)RG * (D + 2);  // floats of a partial: acc [RG][D], m [RG], l [RG]
  float *part0 = p.partial + (direct ? (size_t)0 : ((size_t)cell * ng + g) * C * kPart);
  float *part = part0 + (size_t)c * kPart;
  auto weight = [&](float m, float l, float M) {
    return m == NEG_INF ? l * 0.f : __builtin_amdgcn_exp2f((m - M) * scale);
  };
#pragma unroll
  for (int mt = 0; mt < MTQ; ++mt) {
    const int r = mt * 16 + col;
    float lw = l_run[mt] + shfl_xor(l_run[mt], 16);
    lw += shfl_xor(lw, 32);
    __syncthreads();  // the queries / the previous tile's partials are consumed
    if (grp == 0) {
      s_m[wave * 16 + col] = m_run[mt];
      s_l[wave * 16 + col] = lw;
    }
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) s_acc[(wave * DT + dt) * 64 + lane] = acc[mt][dt];
    __syncthreads();
    float M = NEG_INF;
#pragma unroll
    for (int w = 0; w < kTW; ++w) M = fmaxf(M, s_m[w * 16 + col]);
    float sc[kTW], lsum = 0.f;
#pragma unroll
    for (int w = 0; w < kTW; ++w) {
      const float l = s_l[w * 16 + col];
      sc[w] = weight(s_m[w * 16 + col], l, M);
      lsum += l * sc[w];
    }
#pragma unroll
    for (int i = 0; i < DTW; ++i) {
      const int dt = wave + kTW * i;
      f32x4_t tot = s_acc[dt * 64 + lane] * sc[0];
#pragma unroll
      for (int w = 1; w < kTW; ++w) tot += s_acc[(w * DT + dt) * 64 + lane] * sc[w];
      if (r >= rows) continue;
      if (direct) {
        const int t = (r0 + r) / G, hq = (r0 + r) % G;
        uint2 o = make_uint2(pack2(tot[0] / lsum, tot[1] / lsum), pack2(tot[2] / lsum, tot[3] / lsum));
        if (!((nodes >> t) & 1)) o = make_uint2(0u, 0u);
        *reinterpret_cast<uint2 *>(out_at(b * T + t, (kvh * G + hq) * D + dt * 16 + grp * 4)) = o;
      } else {
        store_coherent4(part + (size_t)r * D + dt * 16 + grp * 4, tot);
      }
    }
    if (!direct && wave == 0 && grp == 0 && r < rows) {
      store_coherent(part + (size_t)RG * D + r, M);
      store_coherent(part + (size_t)RG * D + RG + r, lsum);
    }
  }
  if (direct) return;
  if (!arrive_last(p.counters + (size_t)cell * ng + g, (uint32_t)n_active, s_flag)) return;
#pragma unroll
  for (int mt = 0; mt < MTQ; ++mt) {
    const int r = mt * 16 + col;
    if (r >= rows) continue;
    float M = NEG_INF;
    for (int i = 0; i < n_active; ++i) M = fmaxf(M, load_coherent(part0 + i * kPart + (size_t)RG * D + r));
    float lsum = 0.f;
    f32x4_t o[DTW];
#pragma unroll
    for (int i = 0; i < DTW; ++i) o[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    for (int i = 0; i < n_active; ++i) {
      const float *pr = part0 + i * kPart;
      const float l = load_coherent(pr + (size_t)RG * D + RG + r);
      const float w = weight(load_coherent(pr + (size_t)RG * D + r), l, M);
      lsum += l * w;
#pragma unroll
      for (int k = 0; k < DTW; ++k) o[k] += load_coherent4(pr + (size_t)r * D + (wave + kTW * k) * 16 + grp * 4) * w;
    }
    const int t = (r0 + r) / G, hq = (r0 + r) % G;
#pragma unroll
    for (int k = 0; k < DTW; ++k) {
      uint2 v = make_uint2(pack2(o[k][0] / lsum, o[k][1] / lsum), pack2(o[k][2] / lsum, o[k][3] / lsum));
      if (!((nodes >> t) & 1)) v = make_uint2(0u, 0u);
      *reinterpret_cast<uint2 *>(out_at(b * T + t, (kvh * G + hq) * D + (wave + kTW * k) * 16 + grp * 4)) = v;
    }
  }
}

template <int D>
hipError_t launch_d(const TreeAttnParams &p, hipStream_t s) {
  const dim3 grid((unsigned)(p.batch * p.nkv * p.groups * p.splits)), block(64 * kTW);
  switch (p.mtq) {
    case 1: hipLaunchKernelGGL((tree_attn_kernel<D, 1>), grid, block, 0, s, p); break;
    case 2: hipLaunchKernelGGL((tree_attn_kernel<D, 2>), grid, block, 0, s, p); break;
    case 3: hipLaunchKernelGGL((tree_attn_kernel<D, 3>), grid, block, 0, s, p); break;
    case 4: hipLaunchKernelGGL((tree_attn_kernel<D, 4>), grid, block, 0, s, p); break;
    default: return hipErrorInvalidValue;
  }
  return hipSuccess;
}

}  // namespace

// Row groups of equal size, and (splits = 0) about as many workgroups as the
// CUs hold at once, each with at least min_blocks blocks of a full cache.
void tree_attn_plan(TreeAttnParams *p, int splits) {
  const int tiles = (p->t_rows * (p->nq / p->nkv) + 15) / 16;
  p->groups = (16 * tiles + kTreeGroupRows - 1) / kTreeGroupRows;
  p->mtq = (tiles + p->groups - 1) / p->groups;
  p->min_blocks = 4;
  const int blocks = p->cap / 32;
  if (splits == 0) {
    const int64_t cells = (int64_t)p->batch * p->nkv * p->groups;
    splits = (int)std::max<int64_t>(1, std::min<int64_t>(256 * (p->mtq <= 1 ? 2 : 1) / cells, blocks / p->min_blocks));
  }
  p->splits = std::min(splits, 256);
}

hipError_t launch_tree_attn(const TreeAttnParams &p, hipStream_t s) {
  return p.head_dim == 128 ? launch_d<128>(p, s) : launch_d<64>(p, s);
}

}  // namespace qdec
