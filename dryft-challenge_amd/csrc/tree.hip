// Small kernels of tree speculation: the drafter that merges the
// continuations of earlier occurrences into one tree, the acceptance walk,
// and the copy of the accepted path's keys and values into the cache.  The
// tree attention is tree_attn.hip.
#include "qdec_common.h"
#include "qdec_kernels.h"

namespace qdec {

namespace {

__device__ __forceinline__ int64_t lane_i64(int64_t v, int l) {
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(uint64_t)v, l);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)((uint64_t)v >> 32), l);
  return (int64_t)(((uint64_t)hi << 32) | lo);
}

// One workgroup per sequence.
//   1. The history is scanned from its end in windows of kDraftU * 1024
//      positions, the next window's loads in flight while one is searched in
//      LDS.  Position e ends an earlier occurrence of the pattern of n tokens
//      when hist[e - i] = hist[L - i], i < n.  A wave's hits are a ballot; one
//      wave per pattern then appends them to its list in order, most recent
//      first, while the others store the next window.  Both lists full ends
//      the scan.
//   2. The candidates' tokens go to LDS.
//   3. The first wave builds the tree with one lane per node: a token's child
//      is found by one ballot.
// What bounds it: a history of 20K tokens is 160 KB through one CU.  MI355X: 16
// histories of 8000 to 32000 tokens 15.7 us (36 with every position's pattern read
// from memory), one of 600 tokens 3.8.
constexpr int kDraftThreads = 1024;
constexpr int kDraftU = 8;
constexpr int kDraftWindow = kDraftU * kDraftThreads;
constexpr int kDraftGram = 64;  // tokens of a pattern, at most
__global__ void __launch_bounds__(kDraftThreads) tree_draft_kernel(const qdec_tree_draft_args p) {
  constexpr int NW = kDraftThreads / 64, WORDS = kDraftU * NW;
  static_assert(WORDS == 128 && 2 * kTreeMaxMatches * (kTreeMaxT - 1) <= kDraftWindow, "two words per lane; the drafts fit");
  __shared__ int64_t s_tok[kDraftWindow + kDraftGram];  // the window, newest first; then the drafts
  __shared__ int64_t s_pat[kDraftGram];                 // the last tokens, newest first
  __shared__ uint64_t s_hit[2][WORDS];
  __shared__ int s_end[2][kTreeMaxMatches];
  __shared__ int s_found[2];
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int T = p.t_rows, K = p.depth, M = p.matches;
  const int64_t *h = p.hist + (size_t)b * p.cap;
  int L = p.lens[b];
  if (L < 0) L = 0;
  if (L >= p.cap) L = p.cap - 1;
  const int ngram[2] = {p.primary, p.backoff};
  int64_t r[kDraftU], over = 0;
  auto load = [&](int top) {
#pragma unroll
    for (int u = 0; u < kDraftU; ++u) {
      const int e = top - u * kDraftThreads - tid;
      r[u] = e >= 0 ? h[e] : 0;
    }
    const int e = top - kDraftWindow - tid;
    if (tid < kDraftGram) over = e >= 0 ? h[e] : 0;
  };
  if (tid < 2) s_found[tid] = 0;
  if (tid < kDraftGram) s_pat[tid] = L >= tid ? h[L - tid] : 0;
  if (T > 1) load(L - 1);
  for (int top = T > 1 ? L - 1 : -1; top >= 0; top -= kDraftWindow) {
#pragma unroll
    for (int u = 0; u < kDraftU; ++u) s_tok[u * kDraftThreads + tid] = r[u];
    if (tid < kDraftGram) s_tok[kDraftWindow + tid] = over;
    __syncthreads();  // the window; the hits of the one before are listed
    if (s_found[0] == M && s_found[1] == M) break;
    if (top >= kDraftWindow) load(top - kDraftWindow);
    const int64_t newest = s_pat[0];
    uint64_t last[kDraftU];  // the newest token itself: most waves go no further
#pragma unroll
    for (int u = 0; u < kDraftU; ++u) {
      const int q = u * kDraftThreads + tid;
      last[u] = __ballot(q <= top && s_tok[q] == newest);
    }
#pragma unroll
    for (int u = 0; u < kDraftU; ++u) {
      const int q = u * kDraftThreads + tid, e = top - q;
      uint64_t hit[2] = {0, 0};
      if (last[u]) {
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          bool ok = ((last[u] >> lane) & 1) && e >= ngram[w] - 1;
          for (int i = 1; i < ngram[w] && ok; ++i) ok = s_tok[q + i] == s_pat[i];
          hit[w] = __ballot(ok);
        }
      }
      if (lane < 2) s_hit[lane][u * NW + wave] = lane ? hit[1] : hit[0];
    }
    __syncthreads();
    if (wave < 2) {  // word k: window positions (k / NW) * 1024 + (k % NW) * 64 + bit
      uint64_t bits[2] = {s_hit[wave][2 * lane], s_hit[wave][2 * lane + 1]};
      const int count = __popcll(bits[0]) + __popcll(bits[1]), upto = wave_scan(count);
      const int had = s_found[wave];
      int at = had + upto - count;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int word = 2 * lane + k, q = word / NW * kDraftThreads + word % NW * 64;
        for (; bits[k] && at < M; bits[k] &= bits[k] - 1) s_end[wave][at++] = top - q - __builtin_ctzll(bits[k]);
      }
      if (lane == 63) s_found[wave] = min(M, had + upto);
    }
  }
  __syncthreads();
  const int found = s_found[0], total = found + s_found[1];
  for (int i = tid; i < total * K; i += kDraftThreads) {
    const int m = i / K, at = i - m * K;
    const int e = m < found ? s_end[0][m] : s_end[1][m - found];
    s_tok[i] = e + 1 + at <= L ? h[e + 1 + at] : 0;
  }
  __syncthreads();
  if (wave) return;
  const int64_t newest = s_pat[0];
  int64_t id = newest;  // lane t: node t's token and parent
  int par = -1;
  int count = 1;
  for (int m = 0; m < total && count < T; ++m) {
    const int e = m < found ? s_end[0][m] : s_end[1][m - found];
    const int n = min(K, L - e);
    const int64_t mine = s_tok[m * K + min(lane, K - 1)];
    int cur = 0;
    for (int i = 0; i < n; ++i) {
      const int64_t x = lane_i64(mine, i);
      const uint64_t child = __ballot(par == cur && id == x);
      if (child) {
        cur = __ffsll((unsigned long long)child) - 1;
        continue;
      }
      if (count == T) break;
      if (lane == count) {
        id = x;
        par = cur;
      }
      cur = count++;
    }
  }
  if (lane < T) {
    p.ids[(size_t)b * T + lane] = lane < count ? id : 0;
    p.parents[(size_t)b * T + lane] = par;
  }
}

// One wave per sequence, one lane per node: a step down the tree is one
// ballot over the lanes.  The launch bounds it (MI355X: one sequence 1.6 us, 32 2.6).
__global__ void __launch_bounds__(64) tree_accept_kernel(const qdec_tree_accept_args p) {
  const int b = blockIdx.x, lane = threadIdx.x;
  const int T = p.t_rows;
  const size_t row = (size_t)b * T + min(lane, T - 1);
  const int L = p.lens[b];
  const int64_t id = p.ids[row], pick = p.out_tok[row];
  const int par = lane < T ? p.parents[row] : -1;
  int a = -1, mine = -1;  // steps taken; lane i: the i-th node of the walk
  int64_t out = -1;
  if (L < p.stop_len) {
    int cur = 0;
    for (;;) {
      const int64_t want = lane_i64(pick, cur);
      if (lane == ++a) {
        mine = cur;
        out = want;
      }
      const uint64_t child = __ballot(par == cur && lane > cur && id == want);
      if (!child) break;
      cur = __ffsll((unsigned long long)child) - 1;
    }
    const int at = L + 1 + lane;
    if (lane <= a && at >= 0 && at < p.cap) p.hist[(size_t)b * p.cap + at] = out;
  }
  if (lane < T) {
    p.path[row] = mine;
    if (p.emit) p.emit[row] = out;
  }
  if (lane == 0) {
    p.naccept[b] = max(a, 0);
    p.lens_out[b] = L + a + 1;
  }
}

// One workgroup per (kv head, sequence, layer): the node rows of the path are
// 16-byte vectors; keys go to their slot's row as they are, the 8 channels of
// a value vector to their places of the channel-major cache.  A path has few rows,
// so the launch and one load after another bound it: MI355X, 36 layers of 8 kv
// heads, one sequence 3.1 us, eight 6.2.
template <int D>
__global__ void __launch_bounds__(256) tree_commit_kernel(const qdec_tree_commit_args p) {
  const int kvh = blockIdx.x, b = blockIdx.y;
  const int T = p.t_rows;
  const int a = p.naccept[b], L = p.lens[b];
  const int *path = p.path + (size_t)b * T;
  if (a < 0 || a >= T || L <= a || L > p.cap || path[0] != 0) return;
  const int n = a + 1;
  const int lane = threadIdx.x & 63;
  const int node = lane < n ? path[lane] : 0;  // every wave holds the path
  if (__any(node < 0 || node >= T)) return;
  const size_t slab = ((size_t)blockIdx.z * p.batch + b) * p.nkv + kvh;
  const uint16_t *kn = reinterpret_cast<const uint16_t *>(p.k_nodes) + slab * T * D;
  const uint16_t *vn = reinterpret_cast<const uint16_t *>(p.v_nodes) + slab * T * D;
  uint16_t *kc = reinterpret_cast<uint16_t *>(p.k_cache) + slab * p.cap * D;
  uint16_t *vc = reinterpret_cast<uint16_t *>(p.v_cache) + slab * p.cap * D;
  constexpr int VR = D / 8;  // vectors of a row
  for (int i0 = threadIdx.x & ~63; i0 < n * VR; i0 += 256) {
    const int i = i0 + lane;
    const int r = min(i / VR, n - 1), c = (i % VR) * 8;
    const int src = __shfl(node, r, 64);
    if (i >= n * VR) continue;
    const int slot = L - n + r;
    const uint4 k = *reinterpret_cast<const uint4 *>(kn + (size_t)src * D + c);
    const uint4 v = *reinterpret_cast<const uint4 *>(vn + (size_t)src * D + c);
    *reinterpret_cast<uint4 *>(kc + (size_t)slot * D + c) = k;
    uint16_t *dst = vc + ((size_t)(slot >> 3) * D + c) * 8 + (slot & 7);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      dst[16 * e] = (uint16_t)(w[e] & 0xffffu);
      dst[16 * e + 8] = (uint16_t)(w[e] >> 16);
    }
  }
}

}  // namespace

hipError_t launch_tree_draft(const qdec_tree_draft_args &a, hipStream_t s) {
  hipLaunchKernelGGL(tree_draft_kernel, dim3(a.batch), dim3(kDraftThreads), 0, s, a);
  return hipSuccess;
}

hipError_t launch_tree_accept(const qdec_tree_accept_args &a, hipStream_t s) {
  hipLaunchKernelGGL(tree_accept_kernel, dim3(a.batch), dim3(64), 0, s, a);
  return hipSuccess;
}

hipError_t launch_tree_commit(const qdec_tree_commit_args &a, hipStream_t s) {
  const dim3 grid(a.nkv, a.batch, a.n_layers);
  if (a.head_dim == 128)
    hipLaunchKernelGGL(tree_commit_kernel<128>, grid, dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL(tree_commit_kernel<64>, grid, dim3(256), 0, s, a);
  return hipSuccess;
}

}  // namespace qdec
