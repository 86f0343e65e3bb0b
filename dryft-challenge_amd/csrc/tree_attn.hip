// Attention of a tree of drafted tokens over a KV cache, with the head
// RMSNorm and RoPE of the nodes folded in: T nodes per sequence, each seeing
// all L cached slots, its ancestors and itself.
//
// With G = nq / nkv query heads per kv head, query row r = G*t + h of a kv head
// is node t's query head h.  A workgroup takes a group of rows of one
// (sequence, kv head) and a contiguous run of the 32-row key/value blocks, of
// which there are ceil(L / 32) in the cache and ceil(T / 32) of nodes behind
// them; runs are equal to within a block whatever L is.  Up to 32 rows go to
// tree_attn_kernel, whose waves split the run's blocks; more go to
// tree_wide_kernel, whose waves split the rows.
//
// Common to both:
//   * Ancestor sets: lane t of a wave holds node t's set as 64 bits and a
//     pointer to its parent; pointer doubling unites the sets in at most six
//     rounds.  A set that does not reach the root is no node's.  The depth is
//     the size of the set less one.
//   * Per block S^T = K . Q^T (v_mfma_f32_16x16x32_bf16), online softmax in
//     base 2 on fp32 scores, O^T += V^T . P^T (P rounded to bf16, the operand
//     type).  The running maximum is only moved, and the sums rescaled, in
//     blocks where some row's maximum grows.
//   * With more than one workgroup per row group the partials go to memory and
//     the last workgroup to arrive merges them in order.  A part whose rows saw
//     nothing has maximum -inf and sum 0.
#include "dma_dev.h"
#include "qdec_common.h"
#include "qdec_kernels.h"

namespace qdec {

namespace {

constexpr int kTW = 4;  // waves per workgroup

template <int D>
struct TreeLds {
  static constexpr int RS = D + 8;  // bf16 per LDS row of queries or keys (bank spread)
  static constexpr int q = 0;       // queries [32][RS], then the waves' partials
  static constexpr int part_bytes = kTW * (D / 16) * 64 * 16;
  static constexpr int q_bytes = 32 * RS * 2 > part_bytes ? 32 * RS * 2 : part_bytes;
  static constexpr int k = q + q_bytes;                 // new keys [64][RS]
  static constexpr int v = k + kTreeMaxT * RS * 2;      // new values [8][D][8]
  static constexpr int m = v + kTreeMaxT * D * 2;       // wave row maxima [kTW][16]
  static constexpr int l = m + kTW * 16 * 4;            // wave row sums [kTW][16]
  static constexpr int bad = l + kTW * 16 * 4;          // nodes with a value that is not finite
  static constexpr int flag = bad + kTreeMaxT * 4;
  static constexpr int bytes = flag + 16;
};

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

// A workgroup's place: split c of row group g of cell = b * nkv + kvh.  The row
// groups of one (cell, split) read the same keys and values: they get numbers
// that are equal modulo 8, the number of XCDs, and close together, so that
// they share an L2.
struct TreeUnit {
  int c, cell, g, kvh, b;
};
__device__ __forceinline__ TreeUnit tree_unit(const TreeAttnParams &p) {
  const int ng = p.groups, units = p.batch * p.nkv * p.splits, whole = units & ~7;
  TreeUnit r;
  int unit;
  if ((int)blockIdx.x < whole * ng) {
    const int q = blockIdx.x >> 3;
    r.g = q % ng;
    unit = (q / ng) * 8 + (blockIdx.x & 7);
  } else {
    const int y = blockIdx.x - whole * ng;
    r.g = y % ng;
    unit = whole + y / ng;
  }
  r.c = unit % p.splits;
  r.cell = unit / p.splits;
  r.kvh = r.cell % p.nkv;
  r.b = r.cell / p.nkv;
  return r;
}

// The blocks j0 .. j1 - 1 of split c of a sequence of L cached slots, the first
// nb of all from the cache; n_active splits hold any (c >= n_active: -1).
struct TreeRun {
  int nb, n_active, j0, j1;
};
__device__ __forceinline__ TreeRun tree_run(const TreeAttnParams &p, int L, int c) {
  TreeRun r;
  r.nb = (L + 31) >> 5;
  const int ntot = r.nb + ((p.t_rows + 31) >> 5);
  r.n_active = max(1, min(p.splits, (ntot + p.min_blocks - 1) / p.min_blocks));
  r.j0 = (int)((int64_t)ntot * c / r.n_active);
  r.j1 = (int)((int64_t)ntot * (c + 1) / r.n_active);
  if (c >= r.n_active) r.n_active = -1;
  return r;
}

// Lane t: the nodes from the root to node t as bits, 0 where row t holds none.
// up: parents[t] as loaded (anything on lanes from T on).
__device__ __forceinline__ uint64_t tree_ancestors(int up, int T, int lane) {
  if (lane == 0) up = 0;
  if (lane >= T || up < 0 || up > lane || (up == lane && lane > 0)) up = lane;  // no node: a root of its own
  uint64_t anc = 1ull << lane;
  for (int i = 0; i < 6; ++i) {
    const int up2 = __shfl(up, up, 64);
    anc |= shfl64(anc, up);
    if (!__any(up2 != up)) break;
    up = up2;
  }
  return (anc & 1) && lane < T ? anc : 0;
}

// Weight of a part in a merge: its sum times zero where it saw nothing, so that
// a NaN among its scores stays.
__device__ __forceinline__ float tree_weight(float m, float l, float M, float scale) {
  return m == -__builtin_huge_valf() ? l * 0.f : __builtin_amdgcn_exp2f((m - M) * scale);
}

// Values of a node that are not finite would reach every row through 0 * inf:
// they are zero in LDS and added here, to the rows that see their node.  bad,
// sees: bits of the 32 nodes of the block; pf: this lane's 8 probabilities; vr:
// the first node's raw value row.
template <int D>
__device__ __forceinline__ void add_not_finite(f32x4_t (&acc)[D / 16], const uint4 &pf, uint32_t bad, uint64_t sees,
                                               const uint16_t *vr, int width) {
  const int col = threadIdx.x & 15, grp = (threadIdx.x >> 4) & 3;
  const u32x4_t w = {pf.x, pf.y, pf.z, pf.w};
  for (; bad; bad &= bad - 1) {
    const int i = __builtin_ctz(bad);
    const uint32_t pair = w[(i >> 1) & 3];
    const float pr = __shfl((i & 1) ? hi16(pair) : lo16(pair), col + 16 * (i >> 3), 64);
    if (!((sees >> i) & 1)) continue;
    const uint16_t *v = vr + (size_t)i * width + grp * 4;
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t x = v[dt * 16 + e];
        if ((x & 0x7f80u) == 0x7f80u) acc[dt][e] += pr * bf2f(x);
      }
  }
}

template <int D, int MTQ>
__global__ void __launch_bounds__(64 * kTW, 2) tree_attn_kernel(const TreeAttnParams p) {
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

  const TreeUnit u_ = tree_unit(p);
  const int c = u_.c, cell = u_.cell, kvh = u_.kvh, b = u_.b, C = p.splits;  // one row group
  const int T = p.t_rows, nq = p.nq, nkv = p.nkv, G = nq / nkv;
  const int rows = T * G;  // query rows, at most 16 * MTQ
  const int width = (nq + 2 * nkv) * D;
  const uint16_t *qkv = p.qkv + (size_t)b * T * width;
  auto out_at = [&](int m, int k) { return p.ofrag ? p.out + frag_off(m, k, p.ofrag) : p.out + (size_t)m * nq * D + k; };

  // The raw query rows of this lane, before anything that waits.
  const int sub = lane % LPR, ch = sub * 8;
  constexpr int QP = (16 * MTQ + kTW * RPW - 1) / (kTW * RPW);
  uint4 qraw[QP];
  int qt[QP];
#pragma unroll
  for (int i = 0; i < QP; ++i) {
    const int r = min((i * kTW + wave) * RPW + lane / LPR, rows - 1);
    qt[i] = r / G;
    qraw[i] = ld16(qkv + (size_t)qt[i] * width + (size_t)(kvh * G + r % G) * D + ch);
  }
  const int up = lane < T ? p.parents[(size_t)b * T + lane] : -1;
  const int L = p.lens[b];
  if (L < 0 || L > p.cap - T) {
    if (c == 0)
      for (int i = threadIdx.x; i < rows * (D / 4); i += 64 * kTW) {
        const int r = i / (D / 4), k4 = i % (D / 4) * 4;
        *reinterpret_cast<uint2 *>(out_at(b * T + r / G, (kvh * G + r % G) * D + k4)) = make_uint2(0x7fc07fc0u, 0x7fc07fc0u);
      }
    return;
  }
  const TreeRun run = tree_run(p, L, c);
  if (run.n_active < 0) return;
  const int nb = run.nb, n_active = run.n_active, j0 = run.j0, j1 = run.j1;

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
  const uint64_t anc = tree_ancestors(up, T, lane);
  const int depth = (int)__popcll(anc) - 1;  // -1: no node (its rows are prepared at L and dropped)
  const int pos = depth > 0 ? L + depth : L;
  const uint64_t nodes = __ballot(anc != 0);

  // ---- 2. queries, and the new keys and values of this run's node blocks.
  {
    const uint4 w = ld16(p.q_norm_w + ch);
    uint4 cw[QP], sw[QP];
#pragma unroll
    for (int i = 0; i < QP; ++i) {
      const size_t at = (size_t)__shfl(pos, qt[i], 64) * D + ch;
      cw[i] = ld16(p.cos_tab + at);
      sw[i] = ld16(p.sin_tab + at);
    }
#pragma unroll
    for (int i = 0; i < QP; ++i) {
      const int r = (i * kTW + wave) * RPW + lane / LPR;
      const uint4 q = head_row<D>(qraw[i], w, cw[i], sw[i], p.eps);
      if (r < 16 * MTQ) *reinterpret_cast<uint4 *>(s_q + r * RS + ch) = q;
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
      if (node) {
        const size_t at = ((size_t)cell * T + t) * D + ch;
        *reinterpret_cast<uint4 *>(p.k_nodes + at) = k;
        *reinterpret_cast<uint4 *>(p.v_nodes + at) = v;
      }
      *reinterpret_cast<uint4 *>(s_k + t * RS + ch) = k;
      const uint64_t part = __ballot(!finite8(v)) >> (lane & ~(LPR - 1));
      if (sub == 0) s_bad[t] = node && (part & ((1ull << LPR) - 1));
      uint32_t vw[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {  // no node, or not finite (add_not_finite): zero
        if (!node || (vw[e] & 0x7f80u) == 0x7f80u) vw[e] &= 0xffff0000u;
        if (!node || (vw[e] & 0x7f800000u) == 0x7f800000u) vw[e] &= 0xffffu;
      }
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
    sees[mt] = shfl64(anc, min(mt * 16 + col, rows - 1) / G);
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
        const float m_new = fmaxf(m_run[mt], max_xor16_32(bmax));
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
      if (j >= nb) {
        const uint32_t bad = (uint32_t)(badset >> (32 * (j - nb)));
        if (bad)
          add_not_finite<D>(acc[mt], pf, bad, sees[mt] >> (32 * (j - nb)),
                            qkv + (size_t)(32 * (j - nb)) * width + (size_t)(nq + nkv + kvh) * D, width);
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

  // ---- 4. merge.
  const bool direct = n_active == 1;
  constexpr int RG = 16 * MTQ;
  constexpr size_t kPart = (size_t)RG * (D + 2);  // floats of a partial: acc [RG][D], m [RG], l [RG]
  float *part0 = p.partial + (direct ? (size_t)0 : (size_t)cell * C * kPart);
  float *part = part0 + (size_t)c * kPart;
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
      sc[w] = tree_weight(s_m[w * 16 + col], l, M, scale);
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
        const int t = r / G, hq = r % G;
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
  if (!arrive_last(p.counters + cell, (uint32_t)n_active, s_flag)) return;
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
      const float w = tree_weight(load_coherent(pr + (size_t)RG * D + r), l, M, scale);
      lsum += l * w;
#pragma unroll
      for (int k = 0; k < DTW; ++k) o[k] += load_coherent4(pr + (size_t)r * D + (wave + kTW * k) * 16 + grp * 4) * w;
    }
    const int t = r / G, hq = r % G;
#pragma unroll
    for (int k = 0; k < DTW; ++k) {
      uint2 v = make_uint2(pack2(o[k][0] / lsum, o[k][1] / lsum), pack2(o[k][2] / lsum, o[k][3] / lsum));
      if (!((nodes >> t) & 1)) v = make_uint2(0u, 0u);
      *reinterpret_cast<uint2 *>(out_at(b * T + t, (kvh * G + hq) * D + (wave + kTW * k) * 16 + grp * 4)) = v;
    }
  }
}

// ---------------------------------------------------------------- many rows
// From 33 query rows per kv head every wave has 16 * MT rows of its own and
// the NW waves share the blocks through a ring in LDS, filled by
// global_load_lds_dwordx4 with per-lane gather addresses so that every
// fragment lands in MFMA operand order (as the prefill attention stages its
// blocks):
//   K fragment 2s + h: lane (c, g) holds row 8*(c >> 2) + (c & 3) + 4h of the
//     block, channels 32s + 8g .. +8;
//   V fragment dt: lane (c, g) holds channel 16dt + c, rows 8g .. 8g + 7.
// The node blocks are prepared into the same order behind the ring.  A lane's
// 16 * MT query rows are prepared in registers, where they are used: lane
// (c, g) holds channels 32s + 8g .. +8 of row c for every s, so the rotation's
// partner channel is the lane's own and only the sum of squares crosses lanes.
// While block j's softmax runs on the vector units, the matrix cores form
// block j + 1's scores, one MFMA per exponential.
template <int D, int NT>
struct WideLds {
  static constexpr int KF = D / 16, VF = D / 16;  // fragments of a block
  static constexpr int BV = (KF + VF) * 64;       // uint4 per block
  static constexpr int RING = 4;
  static constexpr int vecs = (RING + NT) * BV;   // NT node blocks
};

// Head RMSNorm and RoPE of one row spread over the four lanes of a column, 8
// channels 32s + 8g .. of every k step s, with the bits of head_norm_rope:
// the same balanced sum over the channels (8 in the lane, 16 and 32 across
// lanes, 64 and 128 in the lane).
template <int D>
__device__ __forceinline__ void head_frags(uint4 (&f)[D / 32], const uint16_t *w, const uint16_t *cos_t,
                                           const uint16_t *sin_t, float eps) {
  constexpr int DS = D / 32;
  uint4 wv[DS], cv[DS], sv[DS];
#pragma unroll
  for (int s = 0; s < DS; ++s) {
    cv[s] = ld16(cos_t + 32 * s);
    sv[s] = ld16(sin_t + 32 * s);
    wv[s] = ld16(w + 32 * s);
  }
  float part[DS];
#pragma unroll
  for (int s = 0; s < DS; ++s) {
    float x[8];
    unpack8(f[s], x);
    float ss = ((x[0] * x[0] + x[1] * x[1]) + (x[2] * x[2] + x[3] * x[3])) +
               ((x[4] * x[4] + x[5] * x[5]) + (x[6] * x[6] + x[7] * x[7]));
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(ss), __float_as_uint(ss), false, false);
    ss = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(ss), __float_as_uint(ss), false, false);
    part[s] = __uint_as_float(b[0]) + __uint_as_float(b[1]);
  }
  float ss = part[0] + part[1];
  if constexpr (DS == 4) ss = ss + (part[2] + part[3]);
  const float rstd = 1.0f / sqrtf(ss / (float)D + eps);
#pragma unroll
  for (int s = 0; s < DS; ++s) {
    float x[8], g[8];
    unpack8(f[s], x);
    unpack8(wv[s], g);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = g[e] * rbf(x[e] * rstd);
    f[s] = pack8(x);
  }
#pragma unroll
  for (int s = 0; s < DS / 2; ++s) {
    float lo[8], hi[8], c[8], n[8], o[8];
    unpack8(f[s], lo);
    unpack8(f[s + DS / 2], hi);
    unpack8(cv[s], c);
    unpack8(sv[s], n);
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = rbf(lo[e] * c[e]) + rbf(-hi[e] * n[e]);
    f[s] = pack8(o);
    unpack8(cv[s + DS / 2], c);
    unpack8(sv[s + DS / 2], n);
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = rbf(hi[e] * c[e]) + rbf(lo[e] * n[e]);
    f[s + DS / 2] = pack8(o);
  }
}

template <int D, int NW, int MT, int NT>
__global__ void __launch_bounds__(64 * NW, D == 128 && NW == 4 && NT == 2 ? 1 : 2) tree_wide_kernel(const TreeAttnParams p) {
  using LY = WideLds<D, NT>;
  constexpr int DS = D / 32, DT = D / 16, KF = LY::KF, BV = LY::BV, RING = LY::RING;
  constexpr int FPW = (KF + LY::VF) / NW;  // fragments each wave loads per block
  constexpr int RG = 16 * MT * NW;         // rows of a group
  static_assert(KF % NW == 0 || (KF + LY::VF) % NW == 0, "whole fragments per wave");
  __shared__ uint4 ring[LY::vecs];         // [RING + NT][fragment][lane]
  uint4 *const tail = ring + RING * BV;
  // Flags of the nodes with a value that is not finite: in the last ring
  // slot, which takes its first block after they were read.
  uint32_t *s_bad = reinterpret_cast<uint32_t *>(ring + (RING - 1) * BV);
  const float NEG_INF = -__builtin_huge_valf();
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, grp = lane >> 4;

  const TreeUnit u_ = tree_unit(p);
  const int c = u_.c, cell = u_.cell, g = u_.g, kvh = u_.kvh, b = u_.b;
  const int ng = p.groups, C = p.splits;
  const int T = p.t_rows, nq = p.nq, nkv = p.nkv, G = nq / nkv;
  const int R = T * G, r0 = g * RG;
  const int rows = min(RG, R - r0);
  const int width = (nq + 2 * nkv) * D;
  const uint16_t *qkv = p.qkv + (size_t)b * T * width;
  auto out_at = [&](int m, int k) { return p.ofrag ? p.out + frag_off(m, k, p.ofrag) : p.out + (size_t)m * nq * D + k; };

  uint4 qf[MT][DS];
  int row[MT];
#pragma unroll
  for (int u = 0; u < MT; ++u) {
    row[u] = r0 + min((wave * MT + u) * 16 + col, rows - 1);
    const uint16_t *q = qkv + (size_t)(row[u] / G) * width + (size_t)(kvh * G + row[u] % G) * D + 8 * grp;
#pragma unroll
    for (int s = 0; s < DS; ++s) qf[u][s] = ld16(q + 32 * s);
  }
  const int up = lane < T ? p.parents[(size_t)b * T + lane] : -1;
  const int L = p.lens[b];
  if (L < 0 || L > p.cap - T) {
    if (c == 0)
      for (int i = threadIdx.x; i < rows * (D / 4); i += 64 * NW) {
        const int r = r0 + i / (D / 4), k4 = i % (D / 4) * 4;
        *reinterpret_cast<uint2 *>(out_at(b * T + r / G, (kvh * G + r % G) * D + k4)) = make_uint2(0x7fc07fc0u, 0x7fc07fc0u);
      }
    return;
  }
  const TreeRun run = tree_run(p, L, c);
  if (run.n_active < 0) return;
  const int nb = run.nb, n_active = run.n_active, j0 = run.j0, n = run.j1 - run.j0;
  const int nd = max(0, min(run.j1, nb) - j0);  // of the n blocks, those from the cache

  // Block jj of this run into its ring slot: this wave gathers fragments wave,
  // wave + NW, ...
  const size_t slab = (size_t)cell * p.cap * D;
  const uint32_t lds0 = lds_addr(ring);
  const uint16_t *kc = p.k_cache + slab, *vc = p.v_cache + slab;
  const uint32_t koff = (uint32_t)((8 * (col >> 2) + (col & 3)) * D + 8 * grp) * 2;
  const uint32_t voff = (uint32_t)(grp * D + col) * 16;
  auto dma_block = [&](int jj) {
    const size_t at = (size_t)(j0 + jj) * 32 * D;  // of either cache
    const uint32_t base = __builtin_amdgcn_readfirstlane(lds0 + (uint32_t)((jj & (RING - 1)) * BV * 16));
#pragma unroll
    for (int i = 0; i < FPW; ++i) {
      const int f = wave + NW * i;
      if (f < KF)
        dma16u(kc + at + 4 * D * (f & 1) + 32 * (f >> 1), koff, base + f * 1024);
      else
        dma16u(vc + at + (f - KF) * 128, voff, base + f * 1024);
    }
  };
#pragma unroll
  for (int jj = 0; jj < RING - 1; ++jj)
    if (jj < nd) dma_block(jj);

  // ---- ancestor sets and queries.
  const uint64_t anc = tree_ancestors(up, T, lane);
  const int depth = (int)__popcll(anc) - 1;  // -1: no node (its rows are prepared at L and dropped)
  const int pos = depth > 0 ? L + depth : L;
  const uint64_t nodes = __ballot(anc != 0);
  uint64_t sees[MT];
#pragma unroll
  for (int u = 0; u < MT; ++u) {
    sees[u] = shfl64(anc, row[u] / G);
    const size_t at = (size_t)__shfl(pos, row[u] / G, 64) * D + 8 * grp;
    head_frags<D>(qf[u], p.q_norm_w + 8 * grp, p.cos_tab + at, p.sin_tab + at, p.eps);
  }

  // ---- the node blocks of this run.
  uint64_t badset = 0;
  const int tb0 = max(j0 - nb, 0), tb1 = run.j1 - nb;  // node blocks, none when tb1 <= tb0
  if (tb1 > tb0) {
    if (threadIdx.x < 2) s_bad[threadIdx.x] = 0;
    lds_barrier();
    for (int i = 2 * tb0 + wave; i < 2 * tb1; i += NW) {  // key tile h of block i / 2
      const int h = i & 1, t = 32 * (i >> 1) + 8 * (col >> 2) + (col & 3) + 4 * h, tr = min(t, T - 1);
      const bool node = (nodes >> t) & 1;
      const uint16_t *kr = qkv + (size_t)tr * width + (size_t)(nq + kvh) * D + 8 * grp;
      uint4 k[DS], v[DS];
#pragma unroll
      for (int s = 0; s < DS; ++s) {
        k[s] = ld16(kr + 32 * s);
        v[s] = ld16(kr + (size_t)nkv * D + 32 * s);
      }
      const size_t at = (size_t)__shfl(pos, tr, 64) * D + 8 * grp;
      head_frags<D>(k, p.k_norm_w + 8 * grp, p.cos_tab + at, p.sin_tab + at, p.eps);
      bool fin = true;
#pragma unroll
      for (int s = 0; s < DS; ++s) {
        tail[(i >> 1) * BV + (2 * s + h) * 64 + lane] = k[s];
        fin = fin && finite8(v[s]);
      }
      if (node && !fin) atomicOr(s_bad + (t >> 5), 1u << (t & 31));
      if (node && g == 0) {
        const size_t o = ((size_t)cell * T + t) * D + 8 * grp;
#pragma unroll
        for (int s = 0; s < DS; ++s) {
          *reinterpret_cast<uint4 *>(p.k_nodes + o + 32 * s) = k[s];
          *reinterpret_cast<uint4 *>(p.v_nodes + o + 32 * s) = v[s];
        }
      }
    }
    for (int i = DT * tb0 + wave; i < DT * tb1; i += NW) {  // value fragment dt of block i / DT
      const int dt = i % DT, t0 = 32 * (i / DT) + 8 * grp;
      const uint16_t *vr = qkv + (size_t)(nq + nkv + kvh) * D + 16 * dt + col;
      uint32_t w[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = vr[(size_t)min(t0 + e, T - 1) * width];
#pragma unroll
      for (int e = 0; e < 8; ++e)  // no node, or not finite (added below to the rows that see it): zero
        if (!((nodes >> (t0 + e)) & 1) || (w[e] & 0x7f80u) == 0x7f80u) w[e] = 0;
      tail[(i / DT) * BV + (KF + dt) * 64 + lane] =
          make_uint4(w[0] | w[1] << 16, w[2] | w[3] << 16, w[4] | w[5] << 16, w[6] | w[7] << 16);
    }
    lds_barrier();
    badset = (uint64_t)s_bad[0] | (uint64_t)s_bad[1] << 32;
  }

  f32x4_t acc[MT][DT];
  float m_run[MT], l_run[MT];
#pragma unroll
  for (int u = 0; u < MT; ++u) {
    m_run[u] = NEG_INF;
    l_run[u] = 0.f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) acc[u][dt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
  auto src = [&](int jj) -> const uint4 * {
    return (jj < nd ? ring + (jj & (RING - 1)) * BV : tail + (j0 + jj - nb) * BV) + lane;
  };
  uint4 kf[KF];  // keys of the next block to score
  auto read_k = [&](int jj) {
    const uint4 *B = src(jj);
#pragma unroll
    for (int f = 0; f < KF; ++f) kf[f] = B[f * 64];
  };
  struct Scores {
    f32x4_t a[MT], b[MT];
  };
  auto score1 = [&](Scores &S, int s, int u, int h) {
    f32x4_t &d = h ? S.b[u] : S.a[u];
    d = mfma16x16x32(kf[2 * s + h], qf[u][s], s ? d : f32x4_t{0.f, 0.f, 0.f, 0.f});
  };
  // Block jj (if from the cache) is in LDS after every wave has waited for
  // its own loads of it, `newest` being the last block issued.
  auto await = [&](int jj, int newest) {
    const int younger = min(newest, nd - 1) - jj;
    if (younger >= 2)
      __builtin_amdgcn_s_waitcnt(vmcnt_enc(2 * FPW) & ~(15 << 8));
    else if (younger == 1)
      __builtin_amdgcn_s_waitcnt(vmcnt_enc(FPW) & ~(15 << 8));
    else
      __builtin_amdgcn_s_waitcnt(kVmcnt0 & ~(15 << 8));
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  __builtin_amdgcn_s_waitcnt(kVmcnt0);  // all that was loaded above, so the loop's counts are its own
  await(0, RING - 2);
  read_k(0);
  Scores s0, s1;
#pragma unroll
  for (int i = 0; i < 2 * DS * MT; ++i) score1(s0, i / (2 * MT), (i >> 1) % MT, i & 1);
  await(min(1, n - 1), RING - 2);
  if (RING - 1 < nd) dma_block(RING - 1);
  read_k(min(1, n - 1));

  const float scale = p.scale_log2;
  auto block = [&](int jj, Scores &S, Scores &N, auto lastc) {
    constexpr bool LAST = decltype(lastc)::value != 0;
    const int j = j0 + jj;
    if (32 * j + 32 > L) {  // the last cached block, or nodes
#pragma unroll
      for (int u = 0; u < MT; ++u) {
        const uint32_t bits = j >= nb ? (uint32_t)(sees[u] >> (32 * (j - nb))) >> (8 * grp)
                                      : (uint32_t)((1ull << min(max(L - 32 * j - 8 * grp, 0), 8)) - 1);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (!((bits >> i) & 1)) S.a[u][i] = NEG_INF;
          if (!((bits >> (4 + i)) & 1)) S.b[u][i] = NEG_INF;
        }
      }
    }
#pragma unroll
    for (int u = 0; u < MT; ++u) {
      const float bmax = fmaxf(fmaxf(fmaxf(S.a[u][0], S.a[u][1]), fmaxf(S.a[u][2], S.a[u][3])),
                               fmaxf(fmaxf(S.b[u][0], S.b[u][1]), fmaxf(S.b[u][2], S.b[u][3])));
      if (!__any(bmax > m_run[u])) continue;  // no row's maximum moves
      const float m_new = fmaxf(m_run[u], max_xor16_32(bmax));
      const float alpha = m_new == NEG_INF ? 1.f : __builtin_amdgcn_exp2f((m_run[u] - m_new) * scale);
      l_run[u] *= alpha;
      m_run[u] = m_new;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) acc[u][dt] *= alpha;
    }
    uint4 vf[DT];
    const uint4 *B = src(jj);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) vf[dt] = B[(KF + dt) * 64];
    uint4 pf[MT];
    float pj[MT][8], mc[MT], psum[MT];
#pragma unroll
    for (int u = 0; u < MT; ++u) {
      mc[u] = m_run[u] == NEG_INF ? 0.f : m_run[u] * scale;
      psum[u] = 0.f;
    }
#pragma unroll
    for (int u = 0; u < MT; ++u)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int i = u * 8 + e;  // MFMA i of the scores: k step, tile, row half
        float x = e < 4 ? S.a[u][e] : S.b[u][e - 4];
        pin(x);
        pj[u][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(x, scale, -mc[u]));
        if constexpr (!LAST) {
          if (i < 2 * DS * MT) {
            score1(N, i / (2 * MT), (i >> 1) % MT, i & 1);
            pin((i & 1) ? N.b[(i >> 1) % MT] : N.a[(i >> 1) % MT]);
          }
        }
        if (i > 0) psum[(i - 1) >> 3] += pj[(i - 1) >> 3][(i - 1) & 7];
        pin(pj[u][e]);
      }
    psum[MT - 1] += pj[MT - 1][7];
#pragma unroll
    for (int u = 0; u < MT; ++u) {
      l_run[u] += psum[u];
      pf[u] = pack8(pj[u]);
    }
    if constexpr (!LAST) {
      await(min(jj + 2, n - 1), jj + RING - 1);
      if (jj + RING < nd) dma_block(jj + RING);
    }
    if (j < nb && 32 * j + 32 > L) {  // slots from L on hold anything
      uint32_t keep[4];
      const int sb = 32 * j + 8 * grp;
#pragma unroll
      for (int d = 0; d < 4; ++d)
        keep[d] = (sb + 2 * d < L ? 0x0000ffffu : 0u) | (sb + 2 * d + 1 < L ? 0xffff0000u : 0u);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        vf[dt].x &= keep[0];
        vf[dt].y &= keep[1];
        vf[dt].z &= keep[2];
        vf[dt].w &= keep[3];
      }
    }
    if constexpr (!LAST) read_k(min(jj + 2, n - 1));
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int u = 0; u < MT; ++u) acc[u][dt] = mfma16x16x32(vf[dt], pf[u], acc[u][dt]);
    if (j >= nb) {
      const uint32_t bad = (uint32_t)(badset >> (32 * (j - nb)));
      if (bad) {
#pragma unroll
        for (int u = 0; u < MT; ++u)
          add_not_finite<D>(acc[u], pf[u], bad, sees[u] >> (32 * (j - nb)),
                            qkv + (size_t)(32 * (j - nb)) * width + (size_t)(nq + nkv + kvh) * D, width);
      }
    }
  };
  int jj = 0;
  if (!(n & 1)) {  // pairs, then the last block by itself
    block(0, s0, s1, Int<0>{});
    s0 = s1;
    jj = 1;
  }
  for (; jj + 1 < n; jj += 2) {
    block(jj, s0, s1, Int<0>{});
    block(jj + 1, s1, s0, Int<0>{});
  }
  block(jj, s0, s1, Int<1>{});

  // ---- output, or a partial per row and the merge by the last workgroup.
  const bool direct = n_active == 1;
  constexpr size_t kPart = (size_t)RG * (D + 2);
  float *part0 = p.partial + (direct ? (size_t)0 : ((size_t)cell * ng + g) * C * kPart);
  float lsum[MT];
#pragma unroll
  for (int u = 0; u < MT; ++u) {
    lsum[u] = l_run[u] + shfl_xor(l_run[u], 16);
    lsum[u] += shfl_xor(lsum[u], 32);
  }
  auto store_rows = [&](int u, const f32x4_t (&o)[DT], float l) {
    const int t = row[u] / G, hq = row[u] % G;
    const bool node = (nodes >> t) & 1;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      uint2 v = make_uint2(pack2(o[dt][0] / l, o[dt][1] / l), pack2(o[dt][2] / l, o[dt][3] / l));
      if (!node) v = make_uint2(0u, 0u);
      *reinterpret_cast<uint2 *>(out_at(b * T + t, (kvh * G + hq) * D + dt * 16 + grp * 4)) = v;
    }
  };
  if (direct) {
#pragma unroll
    for (int u = 0; u < MT; ++u)
      if ((wave * MT + u) * 16 + col < rows) store_rows(u, acc[u], lsum[u]);
    return;
  }
  float *part = part0 + (size_t)c * kPart;
#pragma unroll
  for (int u = 0; u < MT; ++u) {
    const int r = (wave * MT + u) * 16 + col;
    if (r >= rows) continue;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) store_coherent4(part + (size_t)r * D + dt * 16 + grp * 4, acc[u][dt]);
    if (grp == 0) {
      store_coherent(part + (size_t)RG * D + r, m_run[u]);
      store_coherent(part + (size_t)RG * D + RG + r, lsum[u]);
    }
  }
  if (!arrive_last(p.counters + (size_t)cell * ng + g, (uint32_t)n_active, reinterpret_cast<uint32_t *>(ring))) return;
#pragma unroll
  for (int u = 0; u < MT; ++u) {
    const int r = (wave * MT + u) * 16 + col;
    if (r >= rows) continue;
    float M = NEG_INF, l = 0.f;
    for (int i = 0; i < n_active; ++i) M = fmaxf(M, load_coherent(part0 + i * kPart + (size_t)RG * D + r));
    f32x4_t o[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[dt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    for (int i = 0; i < n_active; ++i) {
      const float *pr = part0 + i * kPart;
      const float li = load_coherent(pr + (size_t)RG * D + RG + r);
      const float w = tree_weight(load_coherent(pr + (size_t)RG * D + r), li, M, scale);
      l += li * w;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) o[dt] += load_coherent4(pr + (size_t)r * D + dt * 16 + grp * 4) * w;
    }
    store_rows(u, o, l);
  }
}

template <int D>
hipError_t launch_d(const TreeAttnParams &p, hipStream_t s) {
  const dim3 grid((unsigned)(p.batch * p.nkv * p.groups * p.splits));
  const bool two = p.t_rows > 32;  // node blocks
  switch (p.group_rows) {
    case 16: hipLaunchKernelGGL((tree_attn_kernel<D, 1>), grid, dim3(64 * kTW), 0, s, p); break;
    case 32: hipLaunchKernelGGL((tree_attn_kernel<D, 2>), grid, dim3(64 * kTW), 0, s, p); break;
    case 64:
      if (two) hipLaunchKernelGGL((tree_wide_kernel<D, 4, 1, 2>), grid, dim3(256), 0, s, p);
      else hipLaunchKernelGGL((tree_wide_kernel<D, 4, 1, 1>), grid, dim3(256), 0, s, p);
      break;
    case 128:
      if (two) hipLaunchKernelGGL((tree_wide_kernel<D, 4, 2, 2>), grid, dim3(256), 0, s, p);
      else hipLaunchKernelGGL((tree_wide_kernel<D, 4, 2, 1>), grid, dim3(256), 0, s, p);
      break;
    case 256:
      if (two) hipLaunchKernelGGL((tree_wide_kernel<D, 8, 2, 2>), grid, dim3(512), 0, s, p);
      else hipLaunchKernelGGL((tree_wide_kernel<D, 8, 2, 1>), grid, dim3(512), 0, s, p);
      break;
    default: return hipErrorInvalidValue;
  }
  return hipSuccess;
}

}  // namespace

// The row group (16 or 32: the narrow kernel, all rows; 64, 128 or 256: the
// wide one) and the splits.
void tree_attn_plan(TreeAttnParams *p, int splits) {
  const int rows = p->t_rows * (p->nq / p->nkv);
  const int64_t cells = (int64_t)p->batch * p->nkv;
  const int blocks = p->cap / 32;
  p->group_rows = rows <= 16 ? 16 : rows <= 32 ? 32 : rows <= 64 ? 64 : rows <= 128 ? 128 : 256;
  p->min_blocks = 4;
  p->groups = (rows + p->group_rows - 1) / p->group_rows;
  if (splits == 0) {
    const int64_t fill = p->group_rows == 256 ? 256 : 512;  // workgroups the CUs hold at once
    splits = (int)std::max<int64_t>(1, std::min<int64_t>(fill / (cells * p->groups), blocks / p->min_blocks));
  }
  p->splits = std::min(splits, 256);
}

hipError_t launch_tree_attn(const TreeAttnParams &p, hipStream_t s) {
  return p.head_dim == 128 ? launch_d<128>(p, s) : launch_d<64>(p, s);
}

}  // namespace qdec
