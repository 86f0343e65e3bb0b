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
// tree_narrow_kernel, 16 or 32 rows per workgroup, all in every wave, whose
// waves split the run's blocks; and tree_wide_kernel, 128 or 256 rows, 32 per
// wave, whose waves share every block.
//
// Common to both:
//   * Ancestor sets: lane t of a wave holds node t's set as 64 bits and a
//     pointer to its parent; pointer doubling unites the sets in at most six
//     rounds.  A set that does not reach the root is no node's.  The depth is
//     the size of the set less one.
//   * Per block S^T = K . Q^T (v_mfma_f32_16x16x32_bf16), online softmax in
//     base 2 on fp32 scores, O^T += V^T . P^T.  The matrix instructions take
//     bf16: P goes in as two parts whose sum has 16 bits of it, and so do the
//     narrow kernel's queries (the wide one's, which is bound by its
//     arithmetic, are rounded once).  Each of these roundings would otherwise
//     add as much error to the result as its own rounding to bf16 (relative
//     to 64 bits 0.0040 with q, k as qdec_attn rounds them and P rounded, 0.0023
//     with P in two parts, 0.0017 with both: the output's rounding alone).
//     Node keys are rounded once, to what k_nodes holds: up to 0.0020 where the
//     nodes outweigh the cache.
//   * A lane's query rows are prepared in registers, in the place where the
//     MFMA's B operand wants them: lane (c, g) holds channels 32s + 8g .. +8 of
//     row c for every k step s, so the rotation's partner channel is the
//     lane's own and only the sum of squares crosses lanes.  The node blocks'
//     keys are prepared the same way as A operands.
//   * With more than one split every workgroup leaves a partial (sums, running
//     maximum and sum of a row) and tree_merge_kernel merges them in order.  (A
//     merge by the last workgroup to arrive took 5.4 us for 8 splits of 16
//     rows: its stores, the counter and its loads follow one another at memory
//     latency.  The second launch takes 3.5, and every CU shares its work.)
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

// 8 channels 32s + 8g .. of a row for every k step s: a head row spread over the
// four lanes of a column.
template <int D>
struct Head {
  uint4 v[D / 32];
  __device__ __forceinline__ void load(const uint16_t *p) {
#pragma unroll
    for (int s = 0; s < D / 32; ++s) v[s] = ld16(p + 32 * s);
  }
};

__device__ __forceinline__ uint4 vec(const u32x4_t &v) { return make_uint4(v[0], v[1], v[2], v[3]); }

// Eight numbers as two bf16 vectors whose sum has 16 bits of them.
__device__ __forceinline__ void split8(const float (&p)[8], uint4 &hi, uint4 &lo) {
  hi = pack8(p);
  float h[8], d[8];
  unpack8(hi, h);
#pragma unroll
  for (int e = 0; e < 8; ++e) d[e] = p[e] - h[e];
  lo = pack8(d);
}

// Head RMSNorm (gain w) and RoPE (cos c, sin n) of such a row, in fp32; rounded
// to bf16, the operand type, at the end, lo taking what f leaves (LO).
template <int D, bool LO>
__device__ __forceinline__ void head_rows(uint4 (&f)[D / 32], uint4 (&lo)[D / 32], const Head<D> &w, const Head<D> &cw,
                                          const Head<D> &sw, float eps) {
  constexpr int DS = D / 32;
  float ss = 0.f;
#pragma unroll
  for (int s = 0; s < DS; ++s) {
    float x[8];
    unpack8(f[s], x);
#pragma unroll
    for (int e = 0; e < 8; ++e) ss += x[e] * x[e];
  }
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(ss), __float_as_uint(ss), false, false);
  ss = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(ss), __float_as_uint(ss), false, false);
  ss = __uint_as_float(b[0]) + __uint_as_float(b[1]);
  const float rstd = 1.0f / sqrtf(ss / (float)D + eps);
  auto put = [&](int s, const float (&o)[8]) {
    if constexpr (LO)
      split8(o, f[s], lo[s]);
    else
      f[s] = pack8(o);
  };
#pragma unroll
  for (int s = 0; s < DS / 2; ++s) {
    float x[8], y[8], g[8], c[8], n[8], o[8];
    unpack8(f[s], x);
    unpack8(w.v[s], g);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] *= rstd * g[e];
    unpack8(f[s + DS / 2], y);
    unpack8(w.v[s + DS / 2], g);
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] *= rstd * g[e];
    unpack8(cw.v[s], c);
    unpack8(sw.v[s], n);
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = x[e] * c[e] - y[e] * n[e];
    put(s, o);
    unpack8(cw.v[s + DS / 2], c);
    unpack8(sw.v[s + DS / 2], n);
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = y[e] * c[e] + x[e] * n[e];
    put(s + DS / 2, o);
  }
}

__device__ __forceinline__ bool finite8(const uint4 &v) {
  auto two = [](uint32_t w) { return (w & 0x7f80u) != 0x7f80u && (w & 0x7f800000u) != 0x7f800000u; };
  return two(v.x) && two(v.y) && two(v.z) && two(v.w);
}

__device__ __forceinline__ int div_by(const FastDiv &d, int n) { return (int)(((uint64_t)(uint32_t)n * d.mul) >> d.shift); }

__device__ __forceinline__ bool tree_valid(const TreeAttnParams &p, int L) { return L >= 0 && L <= p.cap - p.t_rows; }
// Workgroups that share a sequence of L slots: `splits`, or fewer where they
// would get less than `least` blocks each (>= kTailWeight per node block, so that
// none before the last is empty); one where L is out of range.  The other
// sequences' lengths do not count, so that they do not move this one's sums.  us,
// this / the batch's splits dealt by the sequences' lengths: 8 x 8 nodes on 0 to
// 1600 slots, 32 query heads on 8, 17.4 / 17.4; 4 x 8 on 0 to 4000 18.5 / 19.0;
// 2 x 16 on 0 and 8000 22.6 / 21.3; 4 x 32 on 0 to 15000, 64 heads, 83 / 68.
__device__ __forceinline__ int tree_active(const TreeAttnParams &p, int L) {
  const int tail = kTailWeight * ((p.t_rows + 31) >> 5), least = max(p.min_blocks, tail);
  const int blocks = tree_valid(p, L) ? ((L + 31) >> 5) + tail : 1;
  return blocks < 2 * least ? 1 : min(p.splits, blocks / least);
}

// A workgroup's place: row group g of unit = (b * splits + c) * nkv + kvh, split c
// of sequence b.  The row groups of one unit read the same keys and values:
// they get numbers that are equal modulo 8, the number of XCDs, and close
// together, so that they share an L2.
struct TreeUnit {
  int unit, b, c, g, kvh;
};
__device__ __forceinline__ TreeUnit tree_unit(const TreeAttnParams &p) {
  const int ng = p.groups, x = blockIdx.x, whole = (p.batch * p.nkv * p.splits) & ~7;
  TreeUnit r;
  r.unit = x;
  r.g = 0;
  if (ng > 1) {
    const bool main = x < whole * ng;
    const int y = main ? x >> 3 : x - whole * ng, q = div_by(p.by_groups, y);
    r.g = y - q * ng;
    r.unit = main ? q * 8 + (x & 7) : whole + q;
  }
  const int w = div_by(p.by_nkv, r.unit);
  r.kvh = r.unit - w * p.nkv;
  r.b = div_by(p.by_splits, w);
  r.c = w - r.b * p.splits;
  return r;
}

// The blocks j0 .. j1 - 1 of split c of n, the first nb of all from the cache,
// the node blocks (the last split's) behind them.
struct TreeRun {
  int nb, j0, j1;
};
__device__ __forceinline__ TreeRun tree_run(const TreeAttnParams &p, int L, int c, int n) {
  TreeRun r;
  r.nb = (L + 31) >> 5;
  const int ntb = (p.t_rows + 31) >> 5, total = r.nb + kTailWeight * ntb;
  const int each = total / n, more = total - each * n;
  r.j0 = min(each * c + min(c, more), r.nb);
  r.j1 = c + 1 == n ? r.nb + ntb : min(each * (c + 1) + min(c + 1, more), r.nb);
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

// The running maximum only moves when a score exceeds it by kTreeMaxSlack / scale:
// probabilities then stay below 2^kTreeMaxSlack, which fp32 sums and bf16 operands
// carry as well as those below 1, and the sums are rescaled in a few of the
// first blocks only.
// Moves a row's running maximum m to a block's maximum `top` if that exceeds it by
// the slack (only then, so that no other row of the wave decides where this one
// rescales) and returns the factor of its sums.
__device__ __forceinline__ float raise_max(float &m, float top, float slack, float scale) {
  if (!(top > m + slack)) return 1.f;
  const float alpha = __builtin_amdgcn_exp2f((m - top) * scale);
  m = top;
  return alpha;
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

// The same of a row spread over D / 8 consecutive lanes, 8 channels each.
template <int D>
__device__ __forceinline__ uint4 head_row(const uint4 &raw, const uint4 &w, const uint4 &cw, const uint4 &sw, float eps) {
  constexpr int LPR = D / 8;
  float x[8], g[8], c[8], s[8], r[8];
  unpack8(raw, x);
  unpack8(w, g);
  unpack8(cw, c);
  unpack8(sw, s);
  float ss = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) ss += x[e] * x[e];
  ss += dpp_f<0xB1>(ss);                            // lane ^ 1
  ss += dpp_f<0x4E>(ss);                            // lane ^ 2
  ss += dpp_f<0x141>(ss);                           // the other quad of 8
  if constexpr (LPR == 16) ss += dpp_f<0x140>(ss);  // the other 8 of 16
  const float rstd = 1.0f / sqrtf(ss / (float)D + eps);
  const bool first = (threadIdx.x & (LPR - 1)) < LPR / 2;
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] *= rstd * g[e];
#pragma unroll
  for (int e = 0; e < 8; ++e) r[e] = shfl_xor(x[e], LPR / 2);  // channels i +- D / 2
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = x[e] * c[e] + (first ? -r[e] : r[e]) * s[e];
  return pack8(x);
}

// The node blocks, prepared by all NW waves of the workgroup into LDS in operand
// order (fragments as the wide kernel's ring holds them): wave and lane take
// rows (k * NW + wave) * RPW + lane / LPR, 8 channels of each.  load() issues the
// raw rows, before the lengths' and sets' dependent work, load_tables() the
// rotation tables' rows; store() does the rest.  One wave alone took 5 us for 32 rows.
template <int D, int NW, int NT>
struct TreeTail {
  static constexpr int KF = D / 16, BV = D / 8 * 64;  // fragments of K, uint4 per block
  static constexpr int LPR = D / 8, RPW = 64 / LPR, N = (32 * NT + NW * RPW - 1) / (NW * RPW);
  uint4 k[N], v[N], cw[N], sw[N], w;

  static __device__ __forceinline__ int row(int i) {
    return (i * NW + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * RPW + (threadIdx.x & 63) / LPR;
  }
  __device__ __forceinline__ void load(const TreeAttnParams &p, const uint16_t *qkv, int kvh, int ntb) {
    const int width = (p.nq + 2 * p.nkv) * D, ch = threadIdx.x % LPR * 8;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (i * NW * RPW >= 32 * ntb) break;
      const uint16_t *x = qkv + (size_t)min(row(i), p.t_rows - 1) * width + (size_t)(p.nq + kvh) * D + ch;
      k[i] = ld16(x);
      v[i] = ld16(x + (size_t)p.nkv * D);
    }
  }
  __device__ __forceinline__ void load_tables(const TreeAttnParams &p, int ntb, int pos) {
    const int ch = threadIdx.x % LPR * 8;
    w = ld16(p.k_norm_w + ch);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (i * NW * RPW >= 32 * ntb) break;
      const size_t at = (size_t)__shfl(pos, min(row(i), p.t_rows - 1), 64) * D + ch;
      cw[i] = ld16(p.cos_tab + at);
      sw[i] = ld16(p.sin_tab + at);
    }
  }
  // s_bad: 32 words per block.  The workgroup has to meet before it reads.
  __device__ __forceinline__ void store(const TreeAttnParams &p, uint4 *tail, int *s_bad, int cell, bool keep, int ntb,
                                        uint64_t nodes) {
    const int lane = threadIdx.x & 63, sub = lane % LPR, ch = sub * 8, T = p.t_rows;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (i * NW * RPW >= 32 * ntb) break;
      const int t = row(i), r = t & 31;
      const bool node = (nodes >> t) & 1;
      const uint4 kr = head_row<D>(k[i], w, cw[i], sw[i], p.eps);
      if (node && keep) {
        const size_t o = ((size_t)cell * T + t) * D + ch;
        *reinterpret_cast<uint4 *>(p.k_nodes + o) = kr;
        *reinterpret_cast<uint4 *>(p.v_nodes + o) = v[i];
      }
      const uint64_t nf = __ballot(!finite8(v[i])) >> (lane & ~(LPR - 1));
      if (t >= 32 * ntb) continue;  // (more rows per pass than a block has)
      if (sub == 0) s_bad[t] = node && (nf & ((1ull << LPR) - 1));
      uint4 *blk = tail + (t >> 5) * BV;
      // K fragment 2s + h, lane (c, g): row 8*(c >> 2) + (c & 3) + 4h, channels 32s + 8g ..
      blk[(2 * (sub >> 2) + ((r >> 2) & 1)) * 64 + 4 * (r >> 3) + (r & 3) + 16 * (sub & 3)] = kr;
      // V fragment dt, lane (c, g): channel 16dt + c, rows 8g ..
      uint16_t *dst = reinterpret_cast<uint16_t *>(blk + (KF + (ch >> 4)) * 64 + (ch & 15) + 16 * (r >> 3)) + (r & 7);
      uint32_t x[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {  // no node, or not finite (add_not_finite): zero
        if (!node || (x[e] & 0x7f80u) == 0x7f80u) x[e] &= 0xffff0000u;
        if (!node || (x[e] & 0x7f800000u) == 0x7f800000u) x[e] &= 0xffffu;
        dst[16 * e] = (uint16_t)(x[e] & 0xffffu);
        dst[16 * e + 8] = (uint16_t)(x[e] >> 16);
      }
    }
  }
};

__device__ __forceinline__ uint16_t *tree_out(const TreeAttnParams &p, int m, int k) {
  return p.ofrag ? p.out + frag_off(m, k, p.ofrag) : p.out + (size_t)m * p.nq * p.head_dim + k;
}
// Four channels of node t's query head hq: o / l, zeros where the row holds no
// node.
__device__ __forceinline__ void tree_store(const TreeAttnParams &p, int b, int t, int hq, int ch, const f32x4_t &o, float inv,
                                           bool node) {
  uint2 v = make_uint2(pack2(o[0] * inv, o[1] * inv), pack2(o[2] * inv, o[3] * inv));
  if (!node) v = make_uint2(0u, 0u);
  *reinterpret_cast<uint2 *>(tree_out(p, b * p.t_rows + t, hq * p.head_dim + ch)) = v;
}
// The partial of a unit's row group: acc [RG][D], m [RG], l [RG], with m = -inf
// and l = 0 where a row holds no node.
template <int D>
__device__ __forceinline__ float *tree_part(const TreeAttnParams &p, int unit, int g) {
  return p.partial + ((size_t)unit * p.groups + g) * ((size_t)p.group_rows * (D + 2));
}

// The sum of a partial: not 0 for a node, whatever it saw (scores of -inf only have
// the sum 0, weight 0 beside others and a NaN result by themselves).
__device__ __forceinline__ float part_sum(bool node, float m, float l) {
  if (!node) return 0.f;
  return m == -__builtin_huge_valf() && l == 0.f ? 1.f : l;
}

// The rows r0 .. r0 + rows - 1 of a sequence whose length is out of range.
__device__ __forceinline__ void tree_nan_rows(const TreeAttnParams &p, int b, int kvh, int r0, int rows) {
  const int D = p.head_dim, G = p.by_g.d;
  for (int i = threadIdx.x; i < rows * (D / 4); i += blockDim.x) {
    const int r = r0 + i / (D / 4), k4 = i % (D / 4) * 4, t = div_by(p.by_g, r);
    *reinterpret_cast<uint2 *>(tree_out(p, b * p.t_rows + t, (kvh * G + r - t * G) * D + k4)) =
        make_uint2(0x7fc07fc0u, 0x7fc07fc0u);
  }
}

// ----------------------------------------------------------------- few rows
// Four waves hold the same 16 * MT rows and take the run's blocks in turn, two
// blocks in flight each: a key or value fragment goes straight from memory into
// the registers of the one wave that uses it, and there is no barrier before
// the merge of the waves, but for the one after the node blocks' preparation in
// the last split.  With one M tile every wave
// prepares the queries for itself, in registers; with more, wave u prepares
// tile u and the operands stay in LDS (in registers they spilled: two blocks and
// 32 rows' sums are 192).
//
// What bounds it: the cache read when it is long (MI355X, 32 x 4 nodes on 2000 to
// 4224 slots, 16 query heads on 8: 74 us, 5.5 TB/s), else the chain of dependent
// loads before the first block (16 nodes on 640 slots: 8 us, 4 of them that; 64 nodes
// on 4100: 22, at 10 TB/s from L2).
template <int D, int MT, int NT>
struct NarrowLds {
  static constexpr int tail = 0;                            // node blocks in operand order
  static constexpr int bad = tail + NT * (D / 8) * 64 * 16;  // node rows with a value that is not finite
  static constexpr int acc = bad + kTreeMaxT * 4;        // waves' sums [MT][kTW][D / 16][64] f32x4
  static constexpr int m = acc + MT * kTW * (D / 16) * 64 * 16;  // wave row maxima [MT][kTW][16]
  static constexpr int l = m + MT * kTW * 16 * 4;        // wave row sums
  static constexpr int q = l + MT * kTW * 16 * 4;        // query operands [MT][2][D / 32][64] (MT > 1)
  static constexpr int bytes = q + (MT > 1 ? MT * (D / 32) * 2048 : 0);
};

// 512 threads for the registers, as the wide kernel's (with accumulation registers
// the two M tiles were 2% slower).
template <int D, int MT, int NT, bool SHARED>
__global__ void __launch_bounds__(512, 2) tree_narrow_kernel(const TreeAttnParams p) {
  using LY = NarrowLds<D, MT, NT>;
  constexpr int DS = D / 32, DT = D / 16, DTW = DT / kTW, RG = 16 * MT;
  __shared__ __align__(16) unsigned char smem[LY::bytes];
  f32x4_t *s_acc = reinterpret_cast<f32x4_t *>(smem + LY::acc);
  float *s_m = reinterpret_cast<float *>(smem + LY::m);
  float *s_l = reinterpret_cast<float *>(smem + LY::l);
  const float NEG_INF = -__builtin_huge_valf();
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, grp = lane >> 4;

  const TreeUnit u_ = tree_unit(p);
  const int kvh = u_.kvh, g = u_.g, b = u_.b, c = u_.c, L = p.lens[b], n_active = tree_active(p, L);
  if (c >= n_active) return;
  const int cell = b * p.nkv + kvh;
  const int T = p.t_rows, nq = p.nq, nkv = p.nkv, G = p.by_g.d;
  const int r0 = g * RG, rows = min(RG, T * G - r0);
  const int width = (nq + 2 * nkv) * D;
  const uint16_t *qkv = p.qkv + (size_t)b * T * width;

  // What does not depend on the length is loaded first: the tile of query rows
  // that this wave prepares.
  uint4 *s_q = reinterpret_cast<uint4 *>(smem + LY::q);
  uint4 qf[DS], ql[DS];  // the queries in two parts
  const int mine = MT == 1 ? 0 : min(wave, MT - 1);
  int rt[MT];  // the lane's query rows' nodes
#pragma unroll
  for (int u = 0; u < MT; ++u) rt[u] = div_by(p.by_g, r0 + min(u * 16 + col, rows - 1));
  const int qr = r0 + min(mine * 16 + col, rows - 1), qt = div_by(p.by_g, qr);
  {
    const uint16_t *q = qkv + (size_t)qt * width + (size_t)(kvh * G + qr - qt * G) * D + 8 * grp;
#pragma unroll
    for (int s = 0; s < DS; ++s) qf[s] = ld16(q + 32 * s);
  }
  const int up = lane < T ? p.parents[(size_t)b * T + lane] : -1;
  if (!tree_valid(p, L)) {
    if (c == 0) tree_nan_rows(p, b, kvh, r0, rows);
    return;
  }
  const TreeRun run = tree_run(p, L, c, n_active);
  const int nb = run.nb, j0 = run.j0, j1 = run.j1;

  const size_t slab = (size_t)cell * p.cap * D;
  const uint16_t *kc = p.k_cache + slab, *vc = p.v_cache + slab;
  struct Frag {
    uint4 ka[DS], kb[DS], vf[DT];
  };
  // Key rows of tile a: 8*(m >> 2) + (m & 3), of tile b 4 further, so that a
  // lane's 8 scores are 8 consecutive rows, the B operand of the P.V product.
  const int ra = 8 * (col >> 2) + (col & 3);
  // A key load takes half a cache line per row and the next one the other half: it
  // stays in the caches meanwhile.  A value load takes whole lines, which only other
  // row groups (SHARED) read again.  us with non-temporal loads of neither / values only /
  // both, on one cache again and again: 32 x 4 nodes on 2000 to 4224 slots, one row
  // group, 81 / 68 / 76; 2 x 16 on 8300, two, 25 / 28 / 30.
  auto load_block = [&](int j, Frag &f) {
    const uint16_t *kp = kc + (size_t)(32 * j + ra) * D + 8 * grp;
    const uint16_t *vp = vc + ((size_t)(4 * j + grp) * D + col) * 8;
#pragma unroll
    for (int s = 0; s < DS; ++s) {
      f.ka[s] = ld16(kp + s * 32);
      f.kb[s] = ld16(kp + 4 * D + s * 32);
    }
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) f.vf[dt] = SHARED ? ld16(vp + dt * 128) : ld_nt(vp + dt * 128);
  };
  const int jc = min(j1, nb), ntb = max(j1 - nb, 0);  // the last split has the node blocks
  uint4 *tail = reinterpret_cast<uint4 *>(smem + LY::tail);
  int *s_bad = reinterpret_cast<int *>(smem + LY::bad);
  TreeTail<D, kTW, NT> nt;
  if (ntb > 0) nt.load(p, qkv, kvh, ntb);
  Frag f0, f1;

  const uint64_t anc = tree_ancestors(up, T, lane);
  const int depth = (int)__popcll(anc) - 1;  // -1: no node (its rows are prepared at L and dropped)
  const int pos = depth > 0 ? L + depth : L;
  const uint64_t nodes = __ballot(anc != 0);
  uint64_t sees[MT];
  // The tables of the rows' positions, then the first block: what follows works
  // while the block is on its way.
  Head<D> qw, cw, sw;
  {
    const size_t at = (size_t)__shfl(pos, qt, 64) * D + 8 * grp;
    qw.load(p.q_norm_w + 8 * grp);
    cw.load(p.cos_tab + at);
    sw.load(p.sin_tab + at);
  }
  if (ntb > 0) nt.load_tables(p, ntb, pos);
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
  if (j0 + wave < jc) load_block(j0 + wave, f0);
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
#pragma unroll
  for (int u = 0; u < MT; ++u) sees[u] = shfl64(anc, rt[u]);
  head_rows<D, true>(qf, ql, qw, cw, sw, p.eps);
  if constexpr (MT > 1) {
    if (wave < MT) {
#pragma unroll
      for (int s = 0; s < DS; ++s) {
        s_q[(2 * wave * DS + s) * 64 + lane] = qf[s];
        s_q[((2 * wave + 1) * DS + s) * 64 + lane] = ql[s];
      }
    }
  }
  uint64_t badset = 0;
  if (ntb > 0) {
    nt.store(p, tail, s_bad, cell, g == 0, ntb, nodes);
    lds_barrier();
    badset = __ballot(lane < 32 * ntb && s_bad[lane]);
  } else if (MT > 1) {
    lds_barrier();
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
  const float scale = p.scale_log2;
  const float slack = kTreeMaxSlack / scale;

  // Block j, from the cache or (NODES) of nodes.
  auto process = [&](Frag &f, int j, auto nodesc) {
    constexpr bool NODES = decltype(nodesc)::value != 0;
    if constexpr (NODES) {
      const uint4 *B = tail + (j - nb) * ((D / 8) * 64) + lane;
#pragma unroll
      for (int s = 0; s < DS; ++s) {
        f.ka[s] = B[(2 * s) * 64];
        f.kb[s] = B[(2 * s + 1) * 64];
      }
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) f.vf[dt] = B[(D / 16 + dt) * 64];
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
    f32x4_t sa[MT], sb[MT];
#pragma unroll
    for (int u = 0; u < MT; ++u) {
      sa[u] = sb[u] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < DS; ++s) {
        if (MT > 1 && s % 2 == 0) __atomic_signal_fence(__ATOMIC_SEQ_CST);  // a few operands at a time (registers)
        const uint4 q = MT > 1 ? s_q[(2 * u * DS + s) * 64 + lane] : qf[s];
        const uint4 r = MT > 1 ? s_q[((2 * u + 1) * DS + s) * 64 + lane] : ql[s];
        sa[u] = mfma16x16x32(f.ka[s], r, sa[u]);
        sb[u] = mfma16x16x32(f.kb[s], r, sb[u]);
        sa[u] = mfma16x16x32(f.ka[s], q, sa[u]);
        sb[u] = mfma16x16x32(f.kb[s], q, sb[u]);
      }
    }
    if (NODES || 32 * j + 32 > L) {
#pragma unroll
      for (int u = 0; u < MT; ++u) {
        const uint32_t bits = NODES ? (uint32_t)(sees[u] >> (32 * (j - nb))) >> (8 * grp)
                                    : (uint32_t)((1ull << min(max(L - 32 * j - 8 * grp, 0), 8)) - 1);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (!((bits >> i) & 1)) sa[u][i] = NEG_INF;
          if (!((bits >> (4 + i)) & 1)) sb[u][i] = NEG_INF;
        }
      }
    }
#pragma unroll
    for (int u = 0; u < MT; ++u) {
      const float bmax = fmaxf(fmaxf(fmaxf(sa[u][0], sa[u][1]), fmaxf(sa[u][2], sa[u][3])),
                               fmaxf(fmaxf(sb[u][0], sb[u][1]), fmaxf(sb[u][2], sb[u][3])));
      if (__any(bmax > m_run[u] + slack)) {
        const float alpha = raise_max(m_run[u], max_xor16_32(bmax), slack, scale);
        l_run[u] *= alpha;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) acc[u][dt] *= alpha;
      }
      const float mc = m_run[u] == NEG_INF ? 0.f : m_run[u] * scale;
      float pj[8];
#pragma unroll
      for (int e = 0; e < 8; ++e)
        pj[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(e < 4 ? sa[u][e] : sb[u][e - 4], scale, -mc));
      l_run[u] += ((pj[0] + pj[1]) + (pj[2] + pj[3])) + ((pj[4] + pj[5]) + (pj[6] + pj[7]));
      uint4 pf, pl;
      split8(pj, pf, pl);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) acc[u][dt] = mfma16x16x32(f.vf[dt], pl, acc[u][dt]);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) acc[u][dt] = mfma16x16x32(f.vf[dt], pf, acc[u][dt]);
      if constexpr (NODES) {
        const uint32_t bad = (uint32_t)(badset >> (32 * (j - nb)));
        if (bad)
          add_not_finite<D>(acc[u], pf, bad, sees[u] >> (32 * (j - nb)),
                            qkv + (size_t)(32 * (j - nb)) * width + (size_t)(nq + nkv + kvh) * D, width);
      }
    }
  };
  if (wave >= kTW - ntb) process(f1, nb + wave - (kTW - ntb), Int<1>{});  // the last waves
  for (int j = j0 + wave; j < jc; j += 2 * kTW) {
    if (j + kTW < jc) load_block(j + kTW, f1);
    process(f0, j, Int<0>{});
    if (j + 2 * kTW < jc) load_block(j + 2 * kTW, f0);
    if (j + kTW < jc) process(f1, j + kTW, Int<0>{});
  }

  // ---- merge of the waves, in wave order; output or partial.
#pragma unroll
  for (int u = 0; u < MT; ++u) {
    float lw = l_run[u] + shfl_xor(l_run[u], 16);
    lw += shfl_xor(lw, 32);
    if (grp == 0) {
      s_m[(u * kTW + wave) * 16 + col] = m_run[u];
      s_l[(u * kTW + wave) * 16 + col] = lw;
    }
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) s_acc[((u * kTW + wave) * DT + dt) * 64 + lane] = acc[u][dt];
  }
  lds_barrier();
  float *part = n_active > 1 ? tree_part<D>(p, u_.unit, g) : nullptr;
#pragma unroll
  for (int u = 0; u < MT; ++u) {
    float M = NEG_INF;
#pragma unroll
    for (int w = 0; w < kTW; ++w) M = fmaxf(M, s_m[(u * kTW + w) * 16 + col]);
    float sc[kTW], l = 0.f;
#pragma unroll
    for (int w = 0; w < kTW; ++w) {
      const float li = s_l[(u * kTW + w) * 16 + col];
      sc[w] = tree_weight(s_m[(u * kTW + w) * 16 + col], li, M, scale);
      l += li * sc[w];
    }
    const float inv = 1.f / l;
    const int r = u * 16 + col;
    const bool node = (nodes >> rt[u]) & 1;
#pragma unroll
    for (int i = 0; i < DTW; ++i) {
      const int dt = wave + kTW * i, ch = dt * 16 + grp * 4;
      f32x4_t o = s_acc[((u * kTW) * DT + dt) * 64 + lane] * sc[0];
#pragma unroll
      for (int w = 1; w < kTW; ++w) o += s_acc[((u * kTW + w) * DT + dt) * 64 + lane] * sc[w];
      if (r >= rows) continue;
      if (n_active == 1)
        tree_store(p, b, rt[u], kvh * G + r0 + r - rt[u] * G, ch, o, inv, node);
      else
        *reinterpret_cast<f32x4_t *>(part + (size_t)r * D + ch) = o;
    }
    if (n_active > 1 && wave == 0 && grp == 0 && r < rows) {
      part[(size_t)RG * D + r] = node ? M : NEG_INF;
      part[(size_t)RG * D + RG + r] = part_sum(node, M, l);
    }
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
// block j's exponentials run on the vector units, the matrix cores form block j +
// 1's scores, one MFMA per exponential; the probabilities' low parts are formed
// between the products of the high ones, the next scores' maxima between those of
// the low ones.  The values are read as the keys' registers come free and the
// other way round.  Cached blocks before the last run without its checks, and the
// workgroup meets every second block when the ring has 8 slots.
//
// MI355X, 2 x 64 nodes, 64 query heads on 8, 30000 slots: 178 us at full clock, 0.74
// PFLOP/s (1.1 with both parts of the probabilities), and 8 for the merge.  A block of 256 rows takes about 2700
// cycles of a CU, of which the matrix cores have 1560 and the LDS reads 530; the
// rest is the two waves of a SIMD waiting for each other's vector instructions.
// (The call took 209 us with the checks in every block and the softmax's steps one
// after the other, 184 now.  64 rows per wave would halve the LDS reads, but then the sums live in
// the accumulation registers, and the scores with them: every score tile moved
// between the two files.)
template <int D, int NW, int NT>
struct WideLds {
  static constexpr int KF = D / 16, VF = D / 16;  // fragments of a block
  static constexpr int BV = (KF + VF) * 64;       // uint4 per block
  static constexpr int RING = NW == 8 ? 8 : 4;    // 4 waves: 8 slots take 2 us longer to fill
  static constexpr int vecs = (RING + NT) * BV;   // NT node blocks
};

template <int D, int NW, int NT>
// 512 threads also where it runs with 256: the registers of two waves per SIMD.
// More would be accumulation registers (64 nodes on 30000 slots, 16 query heads on
// 8: 47.5 us, 54 with them).
__global__ void __launch_bounds__(512, 2) tree_wide_kernel(const TreeAttnParams p) {
  using LY = WideLds<D, NW, NT>;
  constexpr int MT = 2;
  constexpr int DS = D / 32, DT = D / 16, KF = LY::KF, BV = LY::BV, RING = LY::RING;
  constexpr int FPW = (KF + LY::VF) / NW;  // fragments each wave loads per block
  constexpr int RG = 16 * MT * NW;         // rows of a group
  constexpr bool PAIRS = RING >= 8;        // one barrier per two blocks: the ring holds blocks jj .. jj + 3 meanwhile
  static_assert((KF + LY::VF) % NW == 0 && (RING - 2) * FPW < 64, "whole fragments per wave, counted in vmcnt");
  __shared__ uint4 ring[LY::vecs];         // [RING + NT][fragment][lane]
  uint4 *const tail = ring + RING * BV;
  // Node rows with a value that is not finite: in the last ring slot, which
  // takes its first block after they were read.
  int *s_bad = reinterpret_cast<int *>(ring + (RING - 1) * BV);
  const float NEG_INF = -__builtin_huge_valf();
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, grp = lane >> 4;

  const TreeUnit u_ = tree_unit(p);
  const int kvh = u_.kvh, g = u_.g, b = u_.b, c = u_.c, L = p.lens[b], n_active = tree_active(p, L);
  if (c >= n_active) return;
  const int cell = b * p.nkv + kvh;
  const int T = p.t_rows, nq = p.nq, nkv = p.nkv, G = p.by_g.d;
  const int R = T * G, r0 = g * RG;
  const int rows = min(RG, R - r0);
  const int width = (nq + 2 * nkv) * D;
  const uint16_t *qkv = p.qkv + (size_t)b * T * width;
  uint4 qf[MT][DS];
  int row[MT], rt[MT];
#pragma unroll
  for (int u = 0; u < MT; ++u) {
    row[u] = r0 + min((wave * MT + u) * 16 + col, rows - 1);
    rt[u] = div_by(p.by_g, row[u]);
    const uint16_t *q = qkv + (size_t)rt[u] * width + (size_t)(kvh * G + row[u] - rt[u] * G) * D + 8 * grp;
#pragma unroll
    for (int s = 0; s < DS; ++s) qf[u][s] = ld16(q + 32 * s);
  }
  const int up = lane < T ? p.parents[(size_t)b * T + lane] : -1;
  if (!tree_valid(p, L)) {
    if (c == 0) tree_nan_rows(p, b, kvh, r0, rows);
    return;
  }
  const TreeRun run = tree_run(p, L, c, n_active);
  const int nb = run.nb, j0 = run.j0, n = run.j1 - run.j0;
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
      if (NW * (i + 1) <= KF || (NW * i < KF && f < KF))
        dma16u(kc + at + 4 * D * (f & 1) + 32 * (f >> 1), koff, base + f * 1024);
      else
        dma16u(vc + at + (f - KF) * 128, voff, base + f * 1024);
    }
  };
#pragma unroll
  for (int jj = 0; jj < RING - 1; ++jj)
    if (jj < nd) dma_block(jj);

  const int ntb = max(run.j1 - nb, 0);  // the last split has the node blocks
  TreeTail<D, NW, NT> nt;
  if (ntb > 0) nt.load(p, qkv, kvh, ntb);

  // ---- ancestor sets and queries.
  const uint64_t anc = tree_ancestors(up, T, lane);
  const int depth = (int)__popcll(anc) - 1;  // -1: no node (its rows are prepared at L and dropped)
  const int pos = depth > 0 ? L + depth : L;
  const uint64_t nodes = __ballot(anc != 0);
  uint64_t sees[MT];
#pragma unroll
  for (int u = 0; u < MT; ++u) {
    sees[u] = shfl64(anc, rt[u]);
    const size_t at = (size_t)__shfl(pos, rt[u], 64) * D + 8 * grp;
    Head<D> qw, cw, sw;
    qw.load(p.q_norm_w + 8 * grp);
    cw.load(p.cos_tab + at);
    sw.load(p.sin_tab + at);
    head_rows<D, false>(qf[u], qf[u], qw, cw, sw, p.eps);
    __atomic_signal_fence(__ATOMIC_SEQ_CST);  // one tile's tables at a time (registers)
  }

  // ---- the node blocks.
  uint64_t badset = 0;
  if (ntb > 0) {
    nt.load_tables(p, ntb, pos);
    nt.store(p, tail, s_bad, cell, g == 0, ntb, nodes);
    lds_barrier();
    badset = __ballot(lane < 32 * ntb && s_bad[lane]);
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
    float mx[MT];  // a lane's largest
    __device__ __forceinline__ float at(int u, int e) const { return e < 4 ? a[u][e] : b[u][e - 4]; }
    __device__ __forceinline__ void max_to(int u, int e) {  // entries up to odd e
      mx[u] = fmaxf(e == 1 ? at(u, 0) : fmaxf(mx[u], at(u, e - 1)), at(u, e));
    }
  };
  auto score1 = [&](Scores &S, int s, int u, int h) {
    f32x4_t &d = h ? S.b[u] : S.a[u];
    d = mfma16x16x32(kf[2 * s + h], qf[u][s], s ? d : f32x4_t{0.f, 0.f, 0.f, 0.f});
  };
  // Block jj (if from the cache) is in LDS after every wave has waited for
  // its own loads of it, `newest` being the last block issued.
  auto await = [&](int jj, int newest) {
    switch (min(newest, nd - 1) - jj) {  // younger blocks may stay in flight
      case 6: if constexpr (RING >= 8) { __builtin_amdgcn_s_waitcnt(vmcnt_enc(6 * FPW) & ~(15 << 8)); break; } [[fallthrough]];
      case 5: if constexpr (RING >= 8) { __builtin_amdgcn_s_waitcnt(vmcnt_enc(5 * FPW) & ~(15 << 8)); break; } [[fallthrough]];
      case 4: if constexpr (RING >= 8) { __builtin_amdgcn_s_waitcnt(vmcnt_enc(4 * FPW) & ~(15 << 8)); break; } [[fallthrough]];
      case 3: if constexpr (RING >= 8) { __builtin_amdgcn_s_waitcnt(vmcnt_enc(3 * FPW) & ~(15 << 8)); break; } [[fallthrough]];
      case 2: __builtin_amdgcn_s_waitcnt(vmcnt_enc(2 * FPW) & ~(15 << 8)); break;
      case 1: __builtin_amdgcn_s_waitcnt(vmcnt_enc(FPW) & ~(15 << 8)); break;
      default: __builtin_amdgcn_s_waitcnt(kVmcnt0 & ~(15 << 8));
    }
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  __builtin_amdgcn_s_waitcnt(kVmcnt0);  // all that was loaded above, so the loop's counts are its own
  await(0, RING - 2);
  read_k(0);
  Scores s0, s1;
#pragma unroll
  for (int i = 0; i < 2 * DS * MT; ++i) score1(s0, i / (2 * MT), (i >> 1) % MT, i & 1);
#pragma unroll
  for (int i = 1; i < 8 * MT; i += 2) s0.max_to(i >> 3, i & 7);
  await(min(1, n - 1), RING - 2);
  if (RING - 1 < nd) dma_block(RING - 1);
  int issued = RING - 1;  // the newest block asked for, if there is one
  read_k(min(1, n - 1));

  const float scale = p.scale_log2, slack = kTreeMaxSlack / scale;
  // AHEAD: 2 or 3, the workgroup meets and blocks up to jj + AHEAD are in LDS
  // after that; 0, the last meeting covers this block; -1, the last block.
  // INNER: blocks up to jj + RING are whole ones from the cache and the last
  // meeting brought its loads up to date.
  auto block = [&](int jj, Scores &S, Scores &N, auto ahead, auto inner) {
    constexpr int AHEAD = decltype(ahead)::value;
    constexpr bool LAST = AHEAD < 0, INNER = decltype(inner)::value != 0;
    auto at = [&](int k) { return INNER ? ring + (k & (RING - 1)) * BV + lane : src(k); };
    const int j = j0 + jj;
    if (!INNER && 32 * j + 32 > L) {  // the last cached block, or nodes
#pragma unroll
      for (int u = 0; u < MT; ++u) {
        const uint32_t bits = j >= nb ? (uint32_t)(sees[u] >> (32 * (j - nb))) >> (8 * grp)
                                      : (uint32_t)((1ull << min(max(L - 32 * j - 8 * grp, 0), 8)) - 1);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (!((bits >> i) & 1)) S.a[u][i] = NEG_INF;
          if (!((bits >> (4 + i)) & 1)) S.b[u][i] = NEG_INF;
        }
#pragma unroll
        for (int e = 1; e < 8; e += 2) S.max_to(u, e);
      }
    }
    if (__builtin_expect(__any(S.mx[0] > m_run[0] + slack || S.mx[1] > m_run[1] + slack), 0)) {
#pragma unroll
      for (int u = 0; u < MT; ++u) {
        const float alpha = raise_max(m_run[u], max_xor16_32(S.mx[u]), slack, scale);
        l_run[u] *= alpha;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) acc[u][dt] *= alpha;
      }
    }
    uint4 vf[DT];
    const uint4 *B = at(jj) + KF * 64;
    auto read_v = [&](int dt) {
      __atomic_signal_fence(__ATOMIC_SEQ_CST);
      vf[dt] = B[dt * 64];
      vf[dt + 1] = B[(dt + 1) * 64];
      __atomic_signal_fence(__ATOMIC_SEQ_CST);
    };
    read_v(0);
    u32x4_t ph[MT], pl[MT];  // the probabilities' two parts
    float pj[MT][8], mc[MT], psum[MT];
    auto high = [&](int u, int e) { ph[u][e >> 1] = pack2(pj[u][e - 1], pj[u][e]); };  // e odd
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
        float x = S.at(u, e);
        pin(x);
        pj[u][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(x, scale, -mc[u]));
        if constexpr (!LAST) {
          if (i < 2 * DS * MT) {
            score1(N, i / (2 * MT), (i >> 1) % MT, i & 1);
            pin((i & 1) ? N.b[(i >> 1) % MT] : N.a[(i >> 1) % MT]);
          }
        }
        if (i % 4 == 3 && i / 2 + 1 < DT) read_v(i / 2 + 1);  // as the keys' registers come free
        if (i > 0) psum[(i - 1) >> 3] += pj[(i - 1) >> 3][(i - 1) & 7];
        if (i > 0 && !(i & 1)) high((i - 1) >> 3, (i - 1) & 7);
        pin(pj[u][e]);
      }
    psum[MT - 1] += pj[MT - 1][7];
    high(MT - 1, 7);
#pragma unroll
    for (int u = 0; u < MT; ++u) l_run[u] += psum[u];
    if constexpr (INNER && AHEAD > 0) {
      constexpr int STEP = AHEAD - 1;  // blocks between meetings
      __builtin_amdgcn_s_waitcnt(vmcnt_enc((RING - AHEAD - STEP) * FPW) & ~(15 << 8));
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
#pragma unroll
      for (int i = STEP - 1; i >= 0; --i) dma_block(jj + RING - i);
      issued = jj + RING;
    } else if constexpr (AHEAD > 0) {
      await(min(jj + AHEAD, n - 1), issued);
      for (; issued < jj + RING; ++issued)  // slots up to jj's were read by all
        if (issued + 1 < nd) dma_block(issued + 1);
    }
    if (!INNER && j < nb && 32 * j + 32 > L) {  // slots from L on hold anything
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
    const uint4 *K2 = at(INNER ? jj + 2 : min(jj + 2, n - 1));
    constexpr int VPM = 8 / DT;  // probabilities per MFMA
#pragma unroll
    for (int i = 0; i < DT * MT; ++i) {
      const int dt = i / MT, u = i % MT;
      acc[u][dt] = mfma16x16x32(vf[dt], vec(ph[u]), acc[u][dt]);
#pragma unroll
      for (int x = i * VPM; x < (i + 1) * VPM; ++x) {
        const int w = x >> 3, e = x & 7;
        pj[w][e] -= (e & 1) ? hi16(ph[w][e >> 1]) : lo16(ph[w][e >> 1]);
        if (e & 1) pl[w][e >> 1] = pack2(pj[w][e - 1], pj[w][e]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int i = 0; i < DT * MT; ++i) {
      const int dt = i / MT, u = i % MT;
      acc[u][dt] = mfma16x16x32(vf[dt], vec(pl[u]), acc[u][dt]);
      if constexpr (!LAST) {
#pragma unroll
        for (int x = i * VPM; x < (i + 1) * VPM; ++x)
          if (x & 1) N.max_to(x >> 3, x & 7);
        if (u == MT - 1) {  // as the values' registers come free
          __atomic_signal_fence(__ATOMIC_SEQ_CST);
          kf[dt] = K2[dt * 64];
          __atomic_signal_fence(__ATOMIC_SEQ_CST);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    if (!INNER && j >= nb) {
      const uint32_t bad = (uint32_t)(badset >> (32 * (j - nb)));
      if (bad) {
#pragma unroll
        for (int u = 0; u < MT; ++u)
          add_not_finite<D>(acc[u], vec(ph[u]), bad, sees[u] >> (32 * (j - nb)),
                            qkv + (size_t)(32 * (j - nb)) * width + (size_t)(nq + nkv + kvh) * D, width);
      }
    }
  };
  int jj = 0;
  if (!(n & 1)) {  // pairs, then the last block by itself
    block(0, s0, s1, Int<2>{}, Int<0>{});
    s0 = s1;
    jj = 1;
  }
  constexpr Int<PAIRS ? 3 : 2> first;
  constexpr Int<PAIRS ? 0 : 2> second;
  while (jj + 1 < n) {
    block(jj, s0, s1, first, Int<0>{});
    block(jj + 1, s1, s0, second, Int<0>{});
    jj += 2;
    for (; jj + 1 + RING < nd; jj += 2) {
      block(jj, s0, s1, first, Int<1>{});
      block(jj + 1, s1, s0, second, Int<1>{});
    }
  }
  block(jj, s0, s1, Int<-1>{}, Int<0>{});

  // ---- output or partial.
  float *part = n_active > 1 ? tree_part<D>(p, u_.unit, g) : nullptr;
#pragma unroll
  for (int u = 0; u < MT; ++u) {
    const int r = (wave * MT + u) * 16 + col;
    const bool node = (nodes >> rt[u]) & 1;
    float l = l_run[u] + shfl_xor(l_run[u], 16);
    l += shfl_xor(l, 32);
    if (r >= rows) continue;
    if (n_active == 1) {
      const float inv = 1.f / l;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) tree_store(p, b, rt[u], kvh * G + row[u] - rt[u] * G, dt * 16 + grp * 4, acc[u][dt], inv, node);
    } else {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<f32x4_t *>(part + (size_t)r * D + dt * 16 + grp * 4) = acc[u][dt];
      if (grp == 0) {
        part[(size_t)RG * D + r] = node ? m_run[u] : NEG_INF;
        part[(size_t)RG * D + RG + r] = part_sum(node, m_run[u], l);
      }
    }
  }
}

// Merge of the splits' partials, in order: D / 4 threads per query row, the loads
// of 8 partials in flight at a time.
template <int D>
__global__ void __launch_bounds__(256) tree_merge_kernel(const TreeAttnParams p) {
  constexpr int TR = D / 4;
  const int G = p.by_g.d, R = p.t_rows * G, RG = p.group_rows;
  const int per = (R + 256 / TR - 1) / (256 / TR);  // workgroups per (sequence, kv head)
  const int cell = blockIdx.x / per, b = div_by(p.by_nkv, cell), kvh = cell - b * p.nkv;
  const int r = (blockIdx.x - cell * per) * (256 / TR) + threadIdx.x / TR;
  const int n = tree_active(p, p.lens[b]);
  // one split: written by its workgroup, as the rows of a length out of range
  if (n == 1 || r >= R) return;
  const int g = r / RG, rg = r - g * RG, ch = (int)(threadIdx.x % TR) * 4;
  const float *part = tree_part<D>(p, b * p.splits * p.nkv + kvh, g);
  const size_t stride = (size_t)p.nkv * p.groups * RG * (D + 2);  // to the next workgroup's
  const float scale = p.scale_log2;
  float M = -__builtin_huge_valf(), l = 0.f;
  bool node = false;
  f32x4_t o = f32x4_t{0.f, 0.f, 0.f, 0.f};
  for (int i0 = 0; i0 < n; i0 += 8) {
    float mi[8], li[8];
    f32x4_t a[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float *pr = part + (size_t)min(i0 + i, n - 1) * stride;
      mi[i] = pr[(size_t)RG * D + rg];
      li[i] = pr[(size_t)RG * D + RG + rg];
      a[i] = *reinterpret_cast<const f32x4_t *>(pr + (size_t)rg * D + ch);
    }
    float Mn = M;
#pragma unroll
    for (int i = 0; i < 8; ++i) Mn = fmaxf(Mn, mi[i]);  // (the last partial repeats)
    const float w0 = tree_weight(M, l, Mn, scale);
    l *= w0;
    o *= w0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (i0 + i >= n) continue;
      const float w = tree_weight(mi[i], li[i], Mn, scale);
      l += li[i] * w;
      o += a[i] * w;
      node |= li[i] != 0.f;
    }
    M = Mn;
  }
  const int t = div_by(p.by_g, r);
  tree_store(p, b, t, kvh * G + r - t * G, ch, o, 1.f / l, node);
}

template <int D>
hipError_t launch_d(const TreeAttnParams &p, hipStream_t s) {
  const dim3 grid((unsigned)(p.batch * p.nkv * p.groups * p.splits));
  const bool two = p.t_rows > 32;  // node blocks
  switch (p.group_rows) {
    case 16:  // more than 32 nodes are more than one group
      if (two) hipLaunchKernelGGL((tree_narrow_kernel<D, 1, 2, true>), grid, dim3(64 * kTW), 0, s, p);
      else if (p.groups > 1) hipLaunchKernelGGL((tree_narrow_kernel<D, 1, 1, true>), grid, dim3(64 * kTW), 0, s, p);
      else hipLaunchKernelGGL((tree_narrow_kernel<D, 1, 1, false>), grid, dim3(64 * kTW), 0, s, p);
      break;
    case 32:  // more than 32 nodes are more than one group
      if (two) hipLaunchKernelGGL((tree_narrow_kernel<D, 2, 2, true>), grid, dim3(64 * kTW), 0, s, p);
      else if (p.groups > 1) hipLaunchKernelGGL((tree_narrow_kernel<D, 2, 1, true>), grid, dim3(64 * kTW), 0, s, p);
      else hipLaunchKernelGGL((tree_narrow_kernel<D, 2, 1, false>), grid, dim3(64 * kTW), 0, s, p);
      break;
    case 128:
      if (two) hipLaunchKernelGGL((tree_wide_kernel<D, 4, 2>), grid, dim3(256), 0, s, p);
      else hipLaunchKernelGGL((tree_wide_kernel<D, 4, 1>), grid, dim3(256), 0, s, p);
      break;
    case 256:
      if (two) hipLaunchKernelGGL((tree_wide_kernel<D, 8, 2>), grid, dim3(512), 0, s, p);
      else hipLaunchKernelGGL((tree_wide_kernel<D, 8, 1>), grid, dim3(512), 0, s, p);
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

// The row group and the splits.  Below, us on MI355X with 32 query heads on 8.
//
// The narrow kernel reads the cache once per row group, from an L2 that its
// groups share; the wide one once per 128 or 256 rows, but its pipeline takes
// longer to fill.  The narrow one is ahead until its reads come to about 200 MB,
// and with up to 64 rows always: narrow / wide, 2 x 32 nodes on 4200 slots (138 MB)
// 24.8 / 25.6, on 8300 (272 MB) 34.9 / 31.7, 32 on 30000 (492 MB) 52 / 44; 64 nodes on
// 8300 (272 MB) 36.3 / 37.5, on 30000 (980 MB) 88 / 63; 4 x 16 nodes on 30000 114 / 119.
//
// 16 rows per workgroup give more workgroups, 32 half the reads.  16 where 32
// would leave CUs idle and the reads are under 130 MB: 16 / 32 rows, 16 nodes on
// 4100 slots (67 MB) 15.1 / 17.0, 32 on 2000 (65 MB) 15.2 / 16.1, on 4200 (138 MB)
// 20.1 / 19.2, 2 x 16 on 4200 (138 MB) 20.5 / 19.4.
//
// One workgroup per CU, none of fewer than four blocks of a full cache: more
// splits read no faster and merge more (16 nodes on 4100 slots, 4 / 8 / 16 / 32
// splits: 19 / 15.5 / 18.5 / 27; 2 x 32 nodes on 30000 slots, 8 / 16 / 32: 92 / 63 / 67).
void tree_attn_plan(TreeAttnParams *p, int splits) {
  const int rows = p->t_rows * (p->nq / p->nkv), tiles = (rows + 15) / 16;
  const int64_t cells = (int64_t)p->batch * p->nkv;
  const int blocks = p->cap / 32;
  const int64_t cache = cells * p->cap * p->head_dim * 4;  // bytes of both caches
  if (rows > 64 && cache * ((rows + 31) / 32) > 200000000)
    p->group_rows = rows <= 128 ? 128 : 256;
  else
    p->group_rows = rows <= 16 || (cells * tiles < 128 && cache * tiles < 130000000) ? 16 : 32;
  p->min_blocks = 4;
  p->groups = (rows + p->group_rows - 1) / p->group_rows;
  if (splits == 0) {
    const int64_t units = cells * p->groups;
    int64_t n = std::min<int64_t>(256 / units, blocks / p->min_blocks);
    splits = (int)std::max<int64_t>(1, n);
  }
  p->splits = std::min(splits, 256);
  p->by_groups = fast_div(p->groups);
  p->by_nkv = fast_div(p->nkv);
  p->by_splits = fast_div(p->splits);
  p->by_g = fast_div(p->nq / p->nkv);
}

hipError_t launch_tree_attn(const TreeAttnParams &p, hipStream_t s) {
  return p.head_dim == 128 ? launch_d<128>(p, s) : launch_d<64>(p, s);
}

}  // namespace qdec
