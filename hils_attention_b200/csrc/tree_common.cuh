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
  unsigned call;                       // number of the call, of the kernel with waits (tree_attn_tc.cu)
};

// Ancestors of the tree's nodes.  anc[j]: bits of j and its ancestors, 0 when j is absent: its parent is no earlier node
// and not -1, or an ancestor is absent.  anc[64]: bits of the nodes at landmark positions, if those are masked.  Pointer
// doubling, log2 n rounds: a bad parent cannot make it loop.  One warp does it, two nodes to a lane (four times as fast as
// rounds that meet at a barrier).  Called by `threads` threads (thread 0 to 31 among them) that meet at barrier `bar` once at
// the end; parents: those of nodes tid and tid + 32, which the caller loads early; par [64], anc [65] in shared memory.
__device__ __forceinline__ int2 tree_parents(const int32_t* parents, int n, int tid) {
  return make_int2(tid < min(n, 32) ? parents[tid] : -2, tid < min(n, kTreeMaxNodes) - 32 ? parents[tid + 32] : -2);
}

__device__ __forceinline__ void tree_ancestors(int2 parents, int n, int len, int mask_lmk, int* par, u64t* anc, int tid, int bar, int threads) {
  if (tid < 32) {
    int p0 = (parents.x >= -1 && parents.x < tid) ? parents.x : -2, p1 = (parents.y >= -1 && parents.y < tid + 32) ? parents.y : -2;   // -2: absent
    u64t a0 = 1ull << tid, a1 = 1ull << (tid + 32);
    for (int far = 1; far < min(n, kTreeMaxNodes); far *= 2) {
      par[tid] = p0;
      par[tid + 32] = p1;
      anc[tid] = a0;
      anc[tid + 32] = a1;
      __syncwarp();
      if (p0 >= 0) { a0 |= anc[p0]; p0 = par[p0]; }
      if (p1 >= 0) { a1 |= anc[p1]; p1 = par[p1]; }
      __syncwarp();
    }
    anc[tid] = p0 == -1 ? a0 : 0ull;
    anc[tid + 32] = p1 == -1 ? a1 : 0ull;
    const uint32_t l0 = __ballot_sync(0xffffffffu, mask_lmk && ((len + __popcll(a0) - 1) & 63) == 63);
    const uint32_t l1 = __ballot_sync(0xffffffffu, mask_lmk && ((len + __popcll(a1) - 1) & 63) == 63);
    if (tid == 0) anc[kTreeMaxNodes] = (u64t)l1 << 32 | l0;
  }
  asm volatile("bar.sync %0, %1;" ::"r"(bar), "r"(threads) : "memory");
}

__device__ __forceinline__ int tree_low(const TreeParams& p, int t) {      // leftmost position visible from position t
  if (p.W == 0) return 0;
  int lo = t - p.W + 1;
  if (p.expand) lo = floor_div(lo, 64) * 64;
  return max(lo, 0);
}

// bits of the drafted nodes that node j sees
__device__ __forceinline__ u64t tree_draft_mask(const u64t* anc, int j, int len, int lo) {
  u64t m = anc[j] & ~anc[kTreeMaxNodes];
  if (lo > len)                                           // a window shorter than the path
    for (u64t rest = m; rest; rest &= rest - 1) {
      const int i = __ffsll((long long)rest) - 1;
      if (len + __popcll(anc[i]) - 1 < lo) m &= ~(1ull << i);
    }
  return m;
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
