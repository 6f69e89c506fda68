// What the kernels over a tree of drafted tokens share: the parameters, the ancestors of the nodes, the masks of a row and
// the join of partial results.
//
// Node j of sequence b stands at position t_j = lens[b] + depth_j (depth 0: child of the last cached token).  It sees the
// cached token s if lo_j <= s < lens[b] and the drafted node i if i is j or an ancestor of j and t_i >= lo_j; a landmark
// position ((position + 1) % 64 == 0) is seen by nobody when mask_lmk is set.  lo_j = t_j - W + 1, rounded down to its chunk
// when `expand` is set; W = 0: everything.
// Rows of one key head are (node, member of the head group) pairs, row = node * G + member.  The keys come in tiles of 64:
// tile 0 is the drafted nodes, tile i > 0 the page of chunk c0 + i - 1, c0 the chunk of the leftmost visible token.
#pragma once
#include "common.cuh"

namespace hils {

typedef unsigned long long u64t;

constexpr int kTreeMaxNodes = 64;
constexpr float kLog2E = 1.4426950408889634f, kLn2F = 0.6931471805599453f;

struct TreeParams {
  const void* q; const void* k_new; const void* v_new; const void* k_pages; const void* v_pages;
  const int32_t* pages; const int32_t* lens; const int32_t* parents;
  void* o; float* lse;
  void* lse_act;                       // or null: lse again, rounded to the activation type
  float* part_o; float* part_ml;       // splits > 1: (split, b, node, head) rows of D unnormalised sums, and (log2 max, sum)
  int B, n, h_q, h_kv, W, mask_lmk, expand, page_stride, num_pages, splits, row_blocks;
  float scale;
};

// Ancestors of the tree's nodes.  anc[j]: bits of j and its ancestors, 0 when j is absent: its parent is no earlier node
// and not -1, or an ancestor is absent.  Pointer doubling: six rounds cover 64 nodes, and a bad parent cannot make it loop.
// Called by `threads` threads (at least 64, thread 0 among them) that meet at barrier `bar`; parent: that of node tid, which
// the caller loads early; par and anc: [2][64] in shared memory; the result is in anc[0].
__device__ __forceinline__ int tree_parent(const int32_t* parents, int n, int tid) { return tid < min(n, kTreeMaxNodes) ? parents[tid] : -2; }

__device__ __forceinline__ void tree_ancestors(int parent, int (*par)[kTreeMaxNodes], u64t (*anc)[kTreeMaxNodes], int tid, int bar, int threads) {
  auto meet = [&] { asm volatile("bar.sync %0, %1;" ::"r"(bar), "r"(threads) : "memory"); };
  if (tid < kTreeMaxNodes) {
    par[0][tid] = (parent >= -1 && parent < tid) ? parent : -2;      // -2: absent
    anc[0][tid] = 1ull << tid;
  }
  meet();
#pragma unroll
  for (int r = 0; r < 6; ++r) {
    const int a = r & 1;
    if (tid < kTreeMaxNodes) {
      const int pj = par[a][tid];
      par[a ^ 1][tid] = pj >= 0 ? par[a][pj] : pj;
      anc[a ^ 1][tid] = pj >= 0 ? (anc[a][tid] | anc[a][pj]) : anc[a][tid];
    }
    meet();
  }
  if (tid < kTreeMaxNodes && par[0][tid] != -1) anc[0][tid] = 0ull;
  meet();
}

__device__ __forceinline__ int tree_low(const TreeParams& p, int t) {      // leftmost position visible from position t
  if (p.W == 0) return 0;
  int lo = t - p.W + 1;
  if (p.expand) lo = floor_div(lo, 64) * 64;
  return max(lo, 0);
}

// bits of the drafted nodes that node j sees
__device__ __forceinline__ u64t tree_draft_mask(const TreeParams& p, const u64t* anc, int j, int len, int lo) {
  u64t m = anc[j], out = 0ull;
  for (u64t rest = m; rest; rest &= rest - 1) {
    const int i = __ffsll((long long)rest) - 1;
    const int t = len + __popcll(anc[i]) - 1;
    if (t >= lo && !(p.mask_lmk && (t & 63) == 63)) out |= 1ull << i;
  }
  return out;
}

// bits of a page tile's keys (tokens 64c .. 64c + 63) that a row with left edge lo sees
__device__ __forceinline__ u64t tree_page_mask(const TreeParams& p, int c, int len, int lo) {
  const int held = len - c * 64, skip = lo - c * 64;
  u64t m = held >= 64 ? ~0ull : (held <= 0 ? 0ull : (1ull << held) - 1);
  if (p.mask_lmk) m &= ~(1ull << 63);
  if (skip >= 64) return 0ull;
  if (skip > 0) m &= ~0ull << skip;
  return m;
}

// Tokens of sequence b; a length past the table's width is cut to it and `over` set.
__device__ __forceinline__ int tree_length(const TreeParams& p, int b, bool& over) {
  const int64_t cap = min((int64_t)p.page_stride * 64, (int64_t)0x7fffffff - 256);
  const int len = max(p.lens[b], 0);
  over = len > cap;
  return over ? (int)cap : len;
}

// page of chunk c of sequence b, or -1 (reported by the caller)
__device__ __forceinline__ int tree_page(const TreeParams& p, int b, int c) {
  const int pg = p.pages[(int64_t)b * p.page_stride + c];
  return (unsigned)pg < (unsigned)p.num_pages ? pg : -1;
}

}  // namespace hils
