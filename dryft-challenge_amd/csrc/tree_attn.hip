// Attention of a tree of drafted tokens over a KV cache, with the head
// RMSNorm and RoPE of the nodes folded in: T nodes per sequence, each seeing
// all L cached slots, its ancestors and itself.
//
// With G = nq / nkv query heads per kv head, query row r = G*t + h of a kv head
// is node t's query head h.  A workgroup takes a group of rows of one
// (sequence, kv head) and a contiguous run of the 32-row key/value blocks, of
// which there are ceil(L / 32) in the cache and ceil(T / 32) of nodes behind
// them; runs are equal to within a block whatever L is, the node blocks
// counting for kTailWeight each (their rows are prepared first).  Two kernels:
// tree_narrow_kernel, 16 rows per workgroup, whose waves split the run's
// blocks, and tree_wide_kernel, 64 to 256 rows, whose waves split the rows.
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
//   * A lane's query rows are prepared in registers, in the place where the
//     MFMA's B operand wants them: lane (c, g) holds channels 32s + 8g .. +8 of
//     row c for every k step s, so the rotation's partner channel is the
//     lane's own and only the sum of squares crosses lanes.  The node blocks'
//     keys are prepared the same way as A operands.
//   * With more than one workgroup per row group the partials go to memory and
//     are merged in order: by the last workgroup to arrive (narrow), or by
//     tree_merge_kernel (wide, whose partials are too much for one CU).  A part
//     whose rows saw nothing has maximum -inf and sum 0.
#include "dma_dev.h"
#include "qdec_common.h"
#include "qdec_kernels.h"

namespace qdec {

namespace {

constexpr int kTW = 4;  // waves of a narrow workgroup
// Blocks that a node block counts for when a sequence's blocks are dealt.
constexpr int kTailWeight = 3;

__device__ __forceinline__ uint64_t shfl64(uint64_t v, int l) {
  const uint32_t lo = (uint32_t)__shfl((int)(uint32_t)v, l, 64);
  const uint32_t hi = (uint32_t)__shfl((int)(uint32_t)(v >> 32), l, 64);
  return ((uint64_t)hi << 32) | lo;
}

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
// nb of all from the cache; every one of the n_active splits holds some
// (c >= n_active: n_active = -1), the last one the node blocks.
struct TreeRun {
  int nb, n_active, j0, j1;
};
__host__ __device__ __forceinline__ int tree_active(int splits, int min_blocks, int nb, int ntb) {
  // at least tail / 2 + 1 blocks per split, so that the one before the last
  // has one left
  const int tail = kTailWeight * ntb, least = min_blocks > tail / 2 ? min_blocks : tail / 2 + 1;
  const int n = (nb + tail) / least;
  return n < 1 ? 1 : n < splits ? n : splits;
}
__device__ __forceinline__ TreeRun tree_run(const TreeAttnParams &p, int L, int c) {
  TreeRun r;
  r.nb = (L + 31) >> 5;
  const int ntb = (p.t_rows + 31) >> 5, total = r.nb + kTailWeight * ntb;
  r.n_active = tree_active(p.splits, p.min_blocks, r.nb, ntb);
  r.j0 = min((int)((int64_t)total * c / r.n_active), r.nb);
  r.j1 = c + 1 == r.n_active ? r.nb + ntb : min((int)((int64_t)total * (c + 1) / r.n_active), r.nb);
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

// Merge of the n partials of row r (acc [RG][D], m [RG], l [RG] each, RG * (D +
// 2) floats apart): this thread's f32x4 at channels ch[k].  8 partials' loads
// are in flight at a time.  Returns the row's sum.
template <int D, int NV, bool COH>
__device__ __forceinline__ float tree_merge(const float *part0, int n, int RG, int r, const int (&ch)[NV], float scale,
                                            f32x4_t (&o)[NV]) {
  const size_t stride = (size_t)RG * (D + 2);
  auto ld1 = [](const float *q) { return COH ? load_coherent(q) : *q; };
  auto ld4 = [](const float *q) { return COH ? load_coherent4(q) : *reinterpret_cast<const f32x4_t *>(q); };
  float M = -__builtin_huge_valf(), l = 0.f;
#pragma unroll
  for (int k = 0; k < NV; ++k) o[k] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  for (int i0 = 0; i0 < n; i0 += 8) {
    float mi[8], li[8];
    f32x4_t a[NV][8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float *pr = part0 + (size_t)min(i0 + i, n - 1) * stride;
      mi[i] = ld1(pr + (size_t)RG * D + r);
      li[i] = ld1(pr + (size_t)RG * D + RG + r);
#pragma unroll
      for (int k = 0; k < NV; ++k) a[k][i] = ld4(pr + (size_t)r * D + ch[k]);
    }
    float Mn = M;
#pragma unroll
    for (int i = 0; i < 8; ++i) Mn = fmaxf(Mn, i0 + i < n ? mi[i] : M);
    const float w0 = tree_weight(M, l, Mn, scale);
    l *= w0;
#pragma unroll
    for (int k = 0; k < NV; ++k) o[k] *= w0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (i0 + i >= n) continue;
      const float w = tree_weight(mi[i], li[i], Mn, scale);
      l += li[i] * w;
#pragma unroll
      for (int k = 0; k < NV; ++k) o[k] += a[k][i] * w;
    }
    M = Mn;
  }
  return l;
}

__device__ __forceinline__ uint16_t *tree_out(const TreeAttnParams &p, int m, int k) {
  return p.ofrag ? p.out + frag_off(m, k, p.ofrag) : p.out + (size_t)m * p.nq * p.head_dim + k;
}

// The rows r0 .. r0 + rows - 1 of a sequence whose length is out of range.
__device__ __forceinline__ void tree_nan_rows(const TreeAttnParams &p, int b, int kvh, int r0, int rows) {
  const int D = p.head_dim, G = p.nq / p.nkv;
  for (int i = threadIdx.x; i < rows * (D / 4); i += blockDim.x) {
    const int r = r0 + i / (D / 4), k4 = i % (D / 4) * 4;
    *reinterpret_cast<uint2 *>(tree_out(p, b * p.t_rows + r / G, (kvh * G + r % G) * D + k4)) =
        make_uint2(0x7fc07fc0u, 0x7fc07fc0u);
  }
}

// ----------------------------------------------------------------- few rows
// Four waves hold the same 16 rows and take the run's blocks in turn, two
// blocks in flight each: a key or value fragment goes straight from memory
// into the registers of the one wave that uses it, and there is no barrier
// before the merge.  The wave that takes a node block prepares its keys in
// place and turns its values in LDS of its own.
template <int D>
struct NarrowLds {
  static constexpr int v = 0;                                 // new values [8][D][8]
  static constexpr int acc = v + kTreeMaxT * D * 2;           // waves' partials [kTW][D / 16][64] f32x4
  static constexpr int m = acc + kTW * (D / 16) * 64 * 16;    // wave row maxima [kTW][16]
  static constexpr int l = m + kTW * 16 * 4;                  // wave row sums [kTW][16]
  static constexpr int flag = l + kTW * 16 * 4;
  static constexpr int bytes = flag + 16;
};

template <int D>
__global__ void __launch_bounds__(64 * kTW, 2) tree_narrow_kernel(const TreeAttnParams p) {
  using LY = NarrowLds<D>;
  constexpr int DS = D / 32, DT = D / 16, DTW = DT / kTW, RG = 16;
  __shared__ __align__(16) unsigned char smem[LY::bytes];
  uint16_t *s_v = reinterpret_cast<uint16_t *>(smem + LY::v);
  f32x4_t *s_acc = reinterpret_cast<f32x4_t *>(smem + LY::acc);
  float *s_m = reinterpret_cast<float *>(smem + LY::m);
  float *s_l = reinterpret_cast<float *>(smem + LY::l);
  uint32_t *s_flag = reinterpret_cast<uint32_t *>(smem + LY::flag);
  const float NEG_INF = -__builtin_huge_valf();
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, grp = lane >> 4;

  const TreeUnit u_ = tree_unit(p);
  const int c = u_.c, cell = u_.cell, g = u_.g, kvh = u_.kvh, b = u_.b;
  const int T = p.t_rows, nq = p.nq, nkv = p.nkv, G = nq / nkv;
  const int r0 = g * RG, rows = min(RG, T * G - r0);
  const int width = (nq + 2 * nkv) * D;
  const uint16_t *qkv = p.qkv + (size_t)b * T * width;

  // What does not depend on the length is loaded first.
  const int row = r0 + min(col, rows - 1), rt = row / G;  // lane's query row and node
  uint4 qf[DS];
  {
    const uint16_t *q = qkv + (size_t)rt * width + (size_t)(kvh * G + row % G) * D + 8 * grp;
#pragma unroll
    for (int s = 0; s < DS; ++s) qf[s] = ld16(q + 32 * s);
  }
  const int up = lane < T ? p.parents[(size_t)b * T + lane] : -1;
  const int L = p.lens[b];
  if (L < 0 || L > p.cap - T) {
    if (c == 0) tree_nan_rows(p, b, kvh, r0, rows);
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
  // The last split's node blocks go to its last waves, which take them first.
  const int jc = min(j1, nb), tb = j1 > nb ? wave - (kTW - (j1 - nb)) : -1;
  Frag f0, f1;
  if (tb >= 0) {  // raw node rows: keys in place, values by rows (vf[0 .. 2 DS - 1])
    const int ta = min(32 * tb + ra, T - 1), tc = min(32 * tb + ra + 4, T - 1);
    const uint16_t *ka = qkv + (size_t)ta * width + (size_t)(nq + kvh) * D + 8 * grp;
    const uint16_t *kb = qkv + (size_t)tc * width + (size_t)(nq + kvh) * D + 8 * grp;
#pragma unroll
    for (int s = 0; s < DS; ++s) {
      f1.ka[s] = ld16(ka + s * 32);
      f1.kb[s] = ld16(kb + s * 32);
      f1.vf[s] = ld16(ka + (size_t)nkv * D + s * 32);
      f1.vf[DS + s] = ld16(kb + (size_t)nkv * D + s * 32);
    }
  }
  if (j0 + wave < jc) load_block(j0 + wave, f0);

  const uint64_t anc = tree_ancestors(up, T, lane);
  const int depth = (int)__popcll(anc) - 1;  // -1: no node (its rows are prepared at L and dropped)
  const int pos = depth > 0 ? L + depth : L;
  const uint64_t nodes = __ballot(anc != 0);
  const uint64_t sees = shfl64(anc, rt);
  {
    const size_t at = (size_t)__shfl(pos, rt, 64) * D + 8 * grp;
    head_frags<D>(qf, p.q_norm_w + 8 * grp, p.cos_tab + at, p.sin_tab + at, p.eps);
  }

  f32x4_t acc[DT];
  float m_run = NEG_INF, l_run = 0.f;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) acc[dt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  const float scale = p.scale_log2;

  // A node block's raw rows into operands; returns the nodes with a value that
  // is not finite.
  auto prepare = [&](int t0, Frag &f) -> uint32_t {
    uint16_t *sv = s_v + (size_t)t0 * D;
    uint32_t bad = 0;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int t = t0 + ra + 4 * h;
      const bool node = (nodes >> t) & 1;
      const size_t at = (size_t)__shfl(pos, min(t, T - 1), 64) * D + 8 * grp;
      head_frags<D>(h ? f.kb : f.ka, p.k_norm_w + 8 * grp, p.cos_tab + at, p.sin_tab + at, p.eps);
      bool fin = true;
#pragma unroll
      for (int s = 0; s < DS; ++s) {
        const uint4 v = f.vf[DS * h + s];
        fin = fin && finite8(v);
        if (node && g == 0) {
          const size_t o = ((size_t)cell * T + t) * D + 32 * s + 8 * grp;
          *reinterpret_cast<uint4 *>(p.k_nodes + o) = h ? f.kb[s] : f.ka[s];
          *reinterpret_cast<uint4 *>(p.v_nodes + o) = v;
        }
        uint32_t w[4] = {v.x, v.y, v.z, v.w};
        uint16_t *dst = sv + ((size_t)((t - t0) >> 3) * D + 32 * s + 8 * grp) * 8 + (t & 7);
#pragma unroll
        for (int e = 0; e < 4; ++e) {  // no node, or not finite (add_not_finite): zero
          if (!node || (w[e] & 0x7f80u) == 0x7f80u) w[e] &= 0xffff0000u;
          if (!node || (w[e] & 0x7f800000u) == 0x7f800000u) w[e] &= 0xffffu;
          dst[16 * e] = (uint16_t)(w[e] & 0xffffu);
          dst[16 * e + 8] = (uint16_t)(w[e] >> 16);
        }
      }
      // lane t: is row t of the block one of this tile's, and not finite?
      const uint64_t nf = __ballot(node && !fin);
      const uint32_t m16 = (uint32_t)((nf | nf >> 16 | nf >> 32 | nf >> 48) & 0xffffu);
      bad |= (uint32_t)__ballot(lane < 32 && ((lane >> 2) & 1) == h && ((m16 >> (4 * (lane >> 3) + (lane & 3))) & 1));
    }
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
      f.vf[dt] = *reinterpret_cast<const uint4 *>(sv + ((size_t)grp * D + dt * 16 + col) * 8);
    return bad;
  };

  // Block j, from the cache or (NODES) of nodes.
  auto process = [&](Frag &f, int j, auto nodesc) {
    constexpr bool NODES = decltype(nodesc)::value != 0;
    uint32_t bad = 0;
    if constexpr (NODES) {
      bad = prepare(32 * (j - nb), f);
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
    f32x4_t sa = f32x4_t{0.f, 0.f, 0.f, 0.f}, sb = sa;
#pragma unroll
    for (int s = 0; s < DS; ++s) {
      sa = mfma16x16x32(f.ka[s], qf[s], sa);
      sb = mfma16x16x32(f.kb[s], qf[s], sb);
    }
    if (NODES || 32 * j + 32 > L) {
      const uint32_t bits = NODES ? (uint32_t)(sees >> (32 * (j - nb))) >> (8 * grp)
                                  : (uint32_t)((1ull << min(max(L - 32 * j - 8 * grp, 0), 8)) - 1);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (!((bits >> i) & 1)) sa[i] = NEG_INF;
        if (!((bits >> (4 + i)) & 1)) sb[i] = NEG_INF;
      }
    }
    const float bmax = fmaxf(fmaxf(fmaxf(sa[0], sa[1]), fmaxf(sa[2], sa[3])), fmaxf(fmaxf(sb[0], sb[1]), fmaxf(sb[2], sb[3])));
    if (__any(bmax > m_run)) {  // some row's maximum moves
      const float m_new = fmaxf(m_run, max_xor16_32(bmax));
      const float alpha = m_new == NEG_INF ? 1.f : __builtin_amdgcn_exp2f((m_run - m_new) * scale);
      l_run *= alpha;
      m_run = m_new;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) acc[dt] *= alpha;
    }
    const float mc = m_run == NEG_INF ? 0.f : m_run * scale;
    float pj[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) pj[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(e < 4 ? sa[e] : sb[e - 4], scale, -mc));
    l_run += ((pj[0] + pj[1]) + (pj[2] + pj[3])) + ((pj[4] + pj[5]) + (pj[6] + pj[7]));
    const uint4 pf = pack8(pj);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) acc[dt] = mfma16x16x32(f.vf[dt], pf, acc[dt]);
    if constexpr (NODES) {
      if (bad)
        add_not_finite<D>(acc, pf, bad, sees >> (32 * (j - nb)),
                          qkv + (size_t)(32 * (j - nb)) * width + (size_t)(nq + nkv + kvh) * D, width);
    }
  };
  if (tb >= 0) process(f1, nb + tb, Int<1>{});
  for (int j = j0 + wave; j < jc; j += 2 * kTW) {
    if (j + kTW < jc) load_block(j + kTW, f1);
    process(f0, j, Int<0>{});
    if (j + 2 * kTW < jc) load_block(j + 2 * kTW, f0);
    if (j + kTW < jc) process(f1, j + kTW, Int<0>{});
  }

  // ---- merge of the waves, in wave order.
  float lw = l_run + shfl_xor(l_run, 16);
  lw += shfl_xor(lw, 32);
  if (grp == 0) {
    s_m[wave * 16 + col] = m_run;
    s_l[wave * 16 + col] = lw;
  }
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) s_acc[(wave * DT + dt) * 64 + lane] = acc[dt];
  lds_barrier();
  float M = NEG_INF;
#pragma unroll
  for (int w = 0; w < kTW; ++w) M = fmaxf(M, s_m[w * 16 + col]);
  float sc[kTW], l = 0.f;
#pragma unroll
  for (int w = 0; w < kTW; ++w) {
    const float li = s_l[w * 16 + col];
    sc[w] = tree_weight(s_m[w * 16 + col], li, M, scale);
    l += li * sc[w];
  }
  f32x4_t o[DTW];
  int ch[DTW];
#pragma unroll
  for (int i = 0; i < DTW; ++i) {
    const int dt = wave + kTW * i;
    ch[i] = dt * 16 + grp * 4;
    o[i] = s_acc[dt * 64 + lane] * sc[0];
#pragma unroll
    for (int w = 1; w < kTW; ++w) o[i] += s_acc[(w * DT + dt) * 64 + lane] * sc[w];
  }
  if (n_active > 1) {
    constexpr size_t kPart = (size_t)RG * (D + 2);
    float *part0 = p.partial + ((size_t)cell * p.groups + g) * p.splits * kPart;
    float *part = part0 + (size_t)c * kPart;
    if (col < rows) {
#pragma unroll
      for (int i = 0; i < DTW; ++i) store_coherent4(part + (size_t)col * D + ch[i], o[i]);
      if (wave == 0 && grp == 0) {
        store_coherent(part + (size_t)RG * D + col, M);
        store_coherent(part + (size_t)RG * D + RG + col, l);
      }
    }
    if (!arrive_last(p.counters + (size_t)cell * p.groups + g, (uint32_t)n_active, s_flag)) return;
    l = tree_merge<D, DTW, true>(part0, n_active, RG, min(col, rows - 1), ch, scale, o);
  }
  if (col >= rows) return;
  const float inv = 1.f / l;
  const bool node = (nodes >> rt) & 1;
#pragma unroll
  for (int i = 0; i < DTW; ++i) {
    uint2 v = make_uint2(pack2(o[i][0] * inv, o[i][1] * inv), pack2(o[i][2] * inv, o[i][3] * inv));
    if (!node) v = make_uint2(0u, 0u);
    *reinterpret_cast<uint2 *>(tree_out(p, b * T + rt, (kvh * G + row % G) * D + ch[i])) = v;
  }
}

// ---------------------------------------------------------------- many rows
// Every wave has 16 * MT rows of its own and the NW waves share the blocks
// through a ring in LDS, filled by global_load_lds_dwordx4 with per-lane gather
// addresses so that every fragment lands in MFMA operand order (as the prefill
// attention stages its blocks):
//   K fragment 2s + h: lane (c, g) holds row 8*(c >> 2) + (c & 3) + 4h of the
//     block, channels 32s + 8g .. +8;
//   V fragment dt: lane (c, g) holds channel 16dt + c, rows 8g .. 8g + 7.
// The node blocks are prepared into the same order behind the ring.  While
// block j's softmax runs on the vector units, the matrix cores form block j +
// 1's scores, one MFMA per exponential.
template <int D, int NT>
struct WideLds {
  static constexpr int KF = D / 16, VF = D / 16;  // fragments of a block
  static constexpr int BV = (KF + VF) * 64;       // uint4 per block
  static constexpr int RING = 4;
  static constexpr int vecs = (RING + NT) * BV;   // NT node blocks
};

template <int D, int NW, int MT, int NT>
__global__ void __launch_bounds__(64 * NW, D == 128 && NW == 4 && NT == 2 ? 1 : 2) tree_wide_kernel(const TreeAttnParams p) {
  using LY = WideLds<D, NT>;
  constexpr int DS = D / 32, DT = D / 16, KF = LY::KF, BV = LY::BV, RING = LY::RING;
  constexpr int FPW = (KF + LY::VF) / NW;  // fragments each wave loads per block
  constexpr int RG = 16 * MT * NW;         // rows of a group
  static_assert(KF % NW == 0 || (KF + LY::VF) % NW == 0, "whole fragments per wave");
  __shared__ uint4 ring[LY::vecs];         // [RING + NT][fragment][lane]
  uint4 *const tail = ring + RING * BV;
  // Rows with a value that is not finite, a word per key tile: in the last
  // ring slot, which takes its first block after they were read.
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
    if (c == 0) tree_nan_rows(p, b, kvh, r0, rows);
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
    // Value fragment dt of node block i / DT: its loads go out before the keys
    // are worked on.
    constexpr int VW = DT * NT / NW > 0 ? DT * NT / NW : 1;  // per wave, at most
    uint32_t vr[VW][8];
    const uint16_t *v0 = qkv + (size_t)(nq + nkv + kvh) * D + col;
#pragma unroll
    for (int k = 0; k < VW; ++k) {
      const int i = DT * tb0 + wave + NW * k;
      if (i >= DT * tb1) break;
#pragma unroll
      for (int e = 0; e < 8; ++e) vr[k][e] = v0[(size_t)min(32 * (i / DT) + 8 * grp + e, T - 1) * width + 16 * (i % DT)];
    }
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
      const uint64_t nf = __ballot(node && !fin);
      if (lane == 0) s_bad[i] = (uint32_t)((nf | nf >> 16 | nf >> 32 | nf >> 48) & 0xffffu);
      if (node && g == 0) {
        const size_t o = ((size_t)cell * T + t) * D + 8 * grp;
#pragma unroll
        for (int s = 0; s < DS; ++s) {
          *reinterpret_cast<uint4 *>(p.k_nodes + o + 32 * s) = k[s];
          *reinterpret_cast<uint4 *>(p.v_nodes + o + 32 * s) = v[s];
        }
      }
    }
#pragma unroll
    for (int k = 0; k < VW; ++k) {
      const int i = DT * tb0 + wave + NW * k;
      if (i >= DT * tb1) break;
      const int t0 = 32 * (i / DT) + 8 * grp;
#pragma unroll
      for (int e = 0; e < 8; ++e)  // no node, or not finite (add_not_finite): zero
        if (!((nodes >> (t0 + e)) & 1) || (vr[k][e] & 0x7f80u) == 0x7f80u) vr[k][e] = 0;
      tail[(i / DT) * BV + (KF + i % DT) * 64 + lane] =
          make_uint4(vr[k][0] | vr[k][1] << 16, vr[k][2] | vr[k][3] << 16, vr[k][4] | vr[k][5] << 16, vr[k][6] | vr[k][7] << 16);
    }
    lds_barrier();
    // lane t: its row's place among the key tiles
    const int tile = 2 * (lane >> 5) + ((lane >> 2) & 1);
    badset = __ballot(tile >= 2 * tb0 && tile < 2 * tb1 && ((s_bad[tile] >> (4 * ((lane >> 3) & 3) + (lane & 3))) & 1));
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

  // ---- output, or a partial per row (m = -inf and l = 0 where a row holds no
  // node, which is how the merge knows it).
  float *part = p.partial + (n_active == 1 ? (size_t)0 : (((size_t)cell * ng + g) * C + c) * ((size_t)RG * (D + 2)));
#pragma unroll
  for (int u = 0; u < MT; ++u) {
    const int r = (wave * MT + u) * 16 + col, t = row[u] / G;
    const bool node = (nodes >> t) & 1;
    float l = l_run[u] + shfl_xor(l_run[u], 16);
    l += shfl_xor(l, 32);
    if (r >= rows) continue;
    if (n_active == 1) {
      const float inv = 1.f / l;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        uint2 v = make_uint2(pack2(acc[u][dt][0] * inv, acc[u][dt][1] * inv), pack2(acc[u][dt][2] * inv, acc[u][dt][3] * inv));
        if (!node) v = make_uint2(0u, 0u);
        *reinterpret_cast<uint2 *>(tree_out(p, b * T + t, (kvh * G + row[u] % G) * D + dt * 16 + grp * 4)) = v;
      }
    } else {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<f32x4_t *>(part + (size_t)r * D + dt * 16 + grp * 4) = acc[u][dt];
      if (grp == 0) {
        part[(size_t)RG * D + r] = node ? m_run[u] : NEG_INF;
        part[(size_t)RG * D + RG + r] = node ? l : 0.f;
      }
    }
  }
}

// Merge of the wide kernel's partials: D / 4 threads per row.
template <int D>
__global__ void __launch_bounds__(256) tree_merge_kernel(const TreeAttnParams p) {
  constexpr int TR = D / 4;
  const int T = p.t_rows, G = p.nq / p.nkv, R = T * G, RG = p.group_rows;
  const int per = (R + 256 / TR - 1) / (256 / TR);  // workgroups per cell
  const int cell = blockIdx.x / per, kvh = cell % p.nkv, b = cell / p.nkv;
  const int r = (blockIdx.x - cell * per) * (256 / TR) + threadIdx.x / TR;
  const int L = p.lens[b];
  if (L < 0 || L > p.cap - T || r >= R) return;
  const int n = tree_active(p.splits, p.min_blocks, (L + 31) >> 5, (T + 31) >> 5);
  if (n == 1) return;  // written by the one workgroup
  const int g = r / RG;
  const int ch[1] = {(int)(threadIdx.x % TR) * 4};
  f32x4_t o[1];
  const float l = tree_merge<D, 1, false>(p.partial + ((size_t)cell * p.groups + g) * p.splits * ((size_t)RG * (D + 2)), n, RG,
                                          r - g * RG, ch, p.scale_log2, o);
  const float inv = 1.f / l;
  uint2 v = make_uint2(pack2(o[0][0] * inv, o[0][1] * inv), pack2(o[0][2] * inv, o[0][3] * inv));
  if (l == 0.f) v = make_uint2(0u, 0u);  // no node
  *reinterpret_cast<uint2 *>(tree_out(p, b * T + r / G, (kvh * G + r % G) * D + ch[0])) = v;
}

template <int D>
hipError_t launch_d(const TreeAttnParams &p, hipStream_t s) {
  const dim3 grid((unsigned)(p.batch * p.nkv * p.groups * p.splits));
  const bool two = p.t_rows > 32;  // node blocks
  switch (p.group_rows) {
    case 16: hipLaunchKernelGGL((tree_narrow_kernel<D>), grid, dim3(64 * kTW), 0, s, p); return hipSuccess;
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
  if (p.splits > 1) {
    const int rows = p.t_rows * (p.nq / p.nkv), per = 256 / (D / 4);
    hipLaunchKernelGGL((tree_merge_kernel<D>), dim3(p.batch * p.nkv * ((rows + per - 1) / per)), dim3(256), 0, s, p);
  }
  return hipSuccess;
}

}  // namespace

// The row group (16: the narrow kernel; 64, 128 or 256: the wide one) and the
// splits.
void tree_attn_plan(TreeAttnParams *p, int splits) {
  const int rows = p->t_rows * (p->nq / p->nkv);
  const int64_t cells = (int64_t)p->batch * p->nkv;
  const int blocks = p->cap / 32;
  p->group_rows = rows <= 32 ? 16 : rows <= 64 ? 64 : rows <= 128 ? 128 : 256;
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
