// Attention of a tree of drafted tokens over the paged store (tree_common.cuh states what a row sees).
//
// fp32 kernel on the CUDA cores (a TF32 product would not keep fp32's accuracy), the join of the shares, the positions, and the
// plan of a call; bf16 runs tree_attn_tc.cu.  One CTA per (sequence, key head, 32 rows, share of the tiles).  K and V of a tile of
// 64 keys go from registers, where they arrive while the tile before is computed, to shared memory; a thread forms 2 x 4 scores
// and 2 x D/16 outputs; running maximum and sum per row.  What bounds it: latency at the sizes it is for.  9 nodes x 2 query heads
// a key head, 2 sequences of 2003 tokens, D 64: 15.2 us and 8.2 for the join with cold caches (23 us a call in a loop).  Where the
// arithmetic binds (64 nodes x 4 a key head, 8 of them, 6000 tokens, D 128: 344 us) 18 TFLOP/s, held by shared-memory reads.
#include <algorithm>

#include "tree_common.cuh"

namespace hils {

// Set when a page table holds an id outside the pool (8200001; the tile is skipped), a sequence reaches past the table's width
// (8200002; it is cut) or past the bound of a decode step (8200003).
static __device__ int g_tree_status = 0;

constexpr int kTreeThreads = 256, kTreeRows = 32;

template <int D>
constexpr size_t tree_smem_floats() { return (size_t)kTreeRows * D + 64 * (D + 4) + 64 * D + kTreeRows * 65 + kTreeRows; }

template <typename T, int D>
__global__ void __launch_bounds__(kTreeThreads) tree_attn_kernel(TreeParams p) {
  constexpr int CPT = D / 16;                             // output columns of a thread: float4 at 4 tx, and 64 + 4 tx
  __shared__ int par_s[kTreeMaxNodes];
  __shared__ u64t anc[kTreeMaxNodes + 1], vis_s[kTreeRows];
  __shared__ int lo_s[kTreeRows];
  __shared__ u64t dmask_s[kTreeRows];
  extern __shared__ __align__(16) float tsm[];
  float* q_s = tsm;                                       // [32][D]
  float* k_s = q_s + kTreeRows * D;                       // [64][D + 4]
  float* v_s = k_s + 64 * (D + 4);                        // [64][D]
  float* s_s = v_s + 64 * D;                              // [32][65]
  float* corr_s = s_s + kTreeRows * 65;                   // [32]
  const int tid = threadIdx.x, G = p.h_q / p.h_kv, R = p.n * G;
  const int rb = blockIdx.x % p.row_blocks, split = blockIdx.x / p.row_blocks, h = blockIdx.y, b = blockIdx.z;
  bool over;
  const int len = tree_length(p, b, over);
  if (over && tid == 0) atomicExch(&g_tree_status, 8200002);
  const int2 parents = tree_parents(p.parents + (int64_t)b * p.n, p.n, tid);
  const int64_t new0 = (int64_t)b * p.n;
  constexpr int kQ = kTreeRows * (D / 4) / kTreeThreads, kKv = 64 * (D / 4) / kTreeThreads;
  float4 qf[kQ], kf[kKv], vf[kKv];
#pragma unroll
  for (int i = 0; i < kQ; ++i) {
    const int x = tid + i * kTreeThreads, r = x / (D / 4), d = (x - r * (D / 4)) * 4, row = rb * kTreeRows + r;
    qf[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (row < R) qf[i] = load4(static_cast<const T*>(p.q) + ((new0 + row / G) * p.h_q + h * G + row % G) * D + d);
  }
  const int c0 = tree_low(p, len) >> 6, c1 = (len + 63) >> 6;
  const int nt = 1 + max(0, c1 - c0), per = (nt + p.splits - 1) / p.splits;
  const int t0 = split * per, t1 = min(nt, t0 + per);
  // K and V of a tile travel in registers while the tile before is computed, its page id one tile earlier
  auto page_of = [&](int t) { return t > 0 && t < t1 ? p.pages[(int64_t)b * p.page_stride + c0 + t - 1] : 0; };
  int pg = page_of(t0);
  u64t held = 0ull;                                       // keys of the tile that anybody may see
  bool in_pool = true;
  auto fetch = [&](int t) {
    in_pool = (unsigned)pg < (unsigned)p.num_pages;
    if (!in_pool && tid == 0) atomicExch(&g_tree_status, 8200001);
    held = !in_pool ? 0ull : (t == 0 ? (p.n >= 64 ? ~0ull : (1ull << p.n) - 1) : tree_page_mask(p, c0 + t - 1, len, 0));
    const T* kb = t == 0 ? static_cast<const T*>(p.k_new) + (new0 * p.h_kv + h) * D : static_cast<const T*>(p.k_pages) + ((int64_t)pg * p.h_kv + h) * 64 * D;
    const T* vb = t == 0 ? static_cast<const T*>(p.v_new) + (new0 * p.h_kv + h) * D : static_cast<const T*>(p.v_pages) + ((int64_t)pg * p.h_kv + h) * 64 * D;
    const int64_t rs = t == 0 ? (int64_t)p.h_kv * D : D;
#pragma unroll
    for (int i = 0; i < kKv; ++i) {
      const int x = tid + i * kTreeThreads, r = x / (D / 4), d = (x - r * (D / 4)) * 4;
      kf[i] = vf[i] = make_float4(0.f, 0.f, 0.f, 0.f);    // keys nobody may see hold anything, NaN too
      if (held >> r & 1ull) {
        kf[i] = load4(kb + r * rs + d);
        vf[i] = load4(vb + r * rs + d);
      }
    }
    pg = page_of(t + 1);
  };
  if (t0 < t1) fetch(t0);
  tree_ancestors(parents, p.n, len, p.mask_lmk, par_s, anc, tid, 0, kTreeThreads);
  if (tid < kTreeRows) {
    const int row = rb * kTreeRows + tid, j = row / G;
    const bool there = row < R && anc[j] != 0ull;
    const int lo = there ? tree_low(p, len + __popcll(anc[j]) - 1) : 0x7fffffff;
    lo_s[tid] = lo;
    dmask_s[tid] = there ? tree_draft_mask(anc, j, len, lo) : 0ull;
  }
#pragma unroll
  for (int i = 0; i < kQ; ++i) *reinterpret_cast<float4*>(q_s + (tid + i * kTreeThreads) * 4) = qf[i];
  const int ty = tid >> 4, tx = tid & 15, sr = tid >> 3, sl = tid & 7;
  float acc[2][CPT], m_run = -CUDART_INF_F, l_run = 0.f;   // m_run, l_run: of row sr, the same in its eight threads
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int e = 0; e < CPT; ++e) acc[i][e] = 0.f;
  for (int t = t0; t < t1; ++t) {
    const int c = c0 + t - 1;
    __syncthreads();
    if (tid < kTreeRows) vis_s[tid] = t == 0 ? dmask_s[tid] : (in_pool ? tree_page_mask(p, c, len, lo_s[tid]) : 0ull);
#pragma unroll
    for (int i = 0; i < kKv; ++i) {
      const int x = tid + i * kTreeThreads, r = x / (D / 4), d = (x - r * (D / 4)) * 4;
      *reinterpret_cast<float4*>(k_s + r * (D + 4) + d) = kf[i];
      *reinterpret_cast<float4*>(v_s + r * D + d) = vf[i];
    }
    const u64t tile_held = held;
    __syncthreads();
    if (t + 1 < t1) fetch(t + 1);
    // scores of rows 2 ty, 2 ty + 1 against keys tx, tx + 16, tx + 32, tx + 48
    float s[2][4] = {};
    for (int d = 0; d < D; d += 4) {
      const float4 qa = *reinterpret_cast<const float4*>(q_s + (2 * ty) * D + d), qb = *reinterpret_cast<const float4*>(q_s + (2 * ty + 1) * D + d);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 kv = *reinterpret_cast<const float4*>(k_s + (tx + 16 * i) * (D + 4) + d);
        s[0][i] = fmaf(qa.x, kv.x, fmaf(qa.y, kv.y, fmaf(qa.z, kv.z, fmaf(qa.w, kv.w, s[0][i]))));
        s[1][i] = fmaf(qb.x, kv.x, fmaf(qb.y, kv.y, fmaf(qb.z, kv.z, fmaf(qb.w, kv.w, s[1][i]))));
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      s_s[(2 * ty) * 65 + tx + 16 * i] = s[0][i];
      s_s[(2 * ty + 1) * 65 + tx + 16 * i] = s[1][i];
    }
    __syncthreads();
    {
      const u64t vis = vis_s[sr];
      float y[8], top = -CUDART_INF_F;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int key = sl + 8 * i;
        y[i] = (vis >> key & 1ull) ? s_s[sr * 65 + key] * p.scale : -CUDART_INF_F;
        top = fmaxf(top, y[i]);
      }
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      const float mn = fmaxf(m_run, top), ref = mn > -CUDART_INF_F ? mn : 0.f;     // a row whose scores are NaN stays NaN
      const float corr = m_run > -CUDART_INF_F ? expf(m_run - ref) : 0.f;
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int key = sl + 8 * i;
        const float e = (vis >> key & 1ull) ? expf(y[i] - ref) : 0.f;
        s_s[sr * 65 + key] = e;
        sum += e;
      }
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      l_run = l_run * corr + sum;
      m_run = mn;
      if (sl == 0) corr_s[sr] = corr;
    }
    __syncthreads();
    const float ca = corr_s[2 * ty], cb = corr_s[2 * ty + 1];
#pragma unroll
    for (int e = 0; e < CPT; ++e) { acc[0][e] *= ca; acc[1][e] *= cb; }
    const u64t va = vis_s[2 * ty], vbits = vis_s[2 * ty + 1];
    const bool mixed = va != tile_held || vbits != tile_held;       // a key that one row sees and another does not may hold NaN
    for (int key = 0; key < 64; ++key) {
      const float pa = s_s[(2 * ty) * 65 + key], pb = s_s[(2 * ty + 1) * 65 + key];
      float v[CPT];
#pragma unroll
      for (int e = 0; e < CPT; e += 4) *reinterpret_cast<float4*>(v + e) = *reinterpret_cast<const float4*>(v_s + key * D + e * 16 + tx * 4);
      if (!mixed) {
#pragma unroll
        for (int e = 0; e < CPT; ++e) { acc[0][e] = fmaf(pa, v[e], acc[0][e]); acc[1][e] = fmaf(pb, v[e], acc[1][e]); }
      } else {
        if (va >> key & 1ull)
#pragma unroll
          for (int e = 0; e < CPT; ++e) acc[0][e] = fmaf(pa, v[e], acc[0][e]);
        if (vbits >> key & 1ull)
#pragma unroll
          for (int e = 0; e < CPT; ++e) acc[1][e] = fmaf(pb, v[e], acc[1][e]);
      }
    }
  }
  __syncthreads();
  float* ml_s = s_s;                                      // [32][2]: max and sum of a row
  if (sl == 0) { ml_s[2 * sr] = m_run; ml_s[2 * sr + 1] = l_run; }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = 2 * ty + i, row = rb * kTreeRows + r;
    if (row >= R) continue;
    const float m = ml_s[2 * r], l = ml_s[2 * r + 1];
    const int64_t out = (new0 + row / G) * p.h_q + h * G + row % G;
    if (p.splits == 1) {
      const float inv = l > 0.f ? 1.f / l : (l == l ? 0.f : l);
#pragma unroll
      for (int e = 0; e < CPT; e += 4)
        store4(static_cast<T*>(p.o) + out * D + e * 16 + tx * 4,
               make_float4(acc[i][e] * inv, acc[i][e + 1] * inv, acc[i][e + 2] * inv, acc[i][e + 3] * inv));
      if (tx == 0) {
        const float lse = l > 0.f ? m + logf(l) : (l == l ? -CUDART_INF_F : l);
        p.lse[out] = lse;
        if (p.lse_act) static_cast<T*>(p.lse_act)[out] = from_f<T>(lse);
      }
    } else {
      const int64_t at = (int64_t)split * p.B * p.n * p.h_q + out;
#pragma unroll
      for (int e = 0; e < CPT; e += 4)
        store4(p.part_o + at * D + e * 16 + tx * 4, make_float4(acc[i][e], acc[i][e + 1], acc[i][e + 2], acc[i][e + 3]));
      if (tx == 0) { p.part_ml[2 * at] = m * kLog2E; p.part_ml[2 * at + 1] = l; }
    }
  }
}

// Joins the splits: o = sum 2^(m_i - M) O_i / sum 2^(m_i - M) l_i.  One warp per row.  A lane holds the weights of two shares
// (there are at most 64), then D / 4 lanes read a share's row, eight shares on their way at once: one after another, 33 shares
// took 9.3 us.
constexpr int kTreeMaxSplits = 64;

template <typename T, int D>
__global__ void __launch_bounds__(256) tree_join_kernel(TreeParams p) {
  constexpr int LPR = D / 4, SPP = 32 / LPR, UN = 8;      // lanes per share, shares per step
  const int lane = threadIdx.x & 31, sub = lane / LPR, d = (lane % LPR) * 4;
  const int64_t rows = (int64_t)p.B * p.n * p.h_q, row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (row >= rows) return;
  float2 ml[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int s = lane + 32 * i;
    ml[i] = s < p.splits ? *reinterpret_cast<const float2*>(p.part_ml + 2 * (s * rows + row)) : make_float2(-CUDART_INF_F, 0.f);
  }
  const float top = warp_max(fmaxf(ml[0].x, ml[1].x)), ref = top > -CUDART_INF_F ? top : 0.f;
  float w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) w[i] = ml[i].y == 0.f ? 0.f : exp2f(ml[i].x - ref);      // 0: nothing visible in this share
  const float l = warp_sum(fmaf(w[0], ml[0].y, w[1] * ml[1].y));
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s0 = 0; s0 < p.splits; s0 += UN * SPP) {
    float4 x[UN];
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      const int s = s0 + u * SPP + sub;
      x[u] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (s < p.splits) x[u] = *reinterpret_cast<const float4*>(p.part_o + (s * rows + row) * D + d);
    }
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      const int s = s0 + u * SPP + sub;
      const float wl = __shfl_sync(0xffffffffu, w[0], s & 31), wh = __shfl_sync(0xffffffffu, w[1], s & 31), ws = s < 32 ? wl : wh;
      if (ws == 0.f) continue;
      acc.x = fmaf(ws, x[u].x, acc.x);
      acc.y = fmaf(ws, x[u].y, acc.y);
      acc.z = fmaf(ws, x[u].z, acc.z);
      acc.w = fmaf(ws, x[u].w, acc.w);
    }
  }
  if constexpr (SPP == 2) {
    acc.x += __shfl_xor_sync(0xffffffffu, acc.x, 16);
    acc.y += __shfl_xor_sync(0xffffffffu, acc.y, 16);
    acc.z += __shfl_xor_sync(0xffffffffu, acc.z, 16);
    acc.w += __shfl_xor_sync(0xffffffffu, acc.w, 16);
  }
  const float inv = l > 0.f ? 1.f / l : (l == l ? 0.f : l);
  if (sub == 0) store4(static_cast<T*>(p.o) + row * D + d, make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv));
  if (lane == 0) {
    const float lse = l > 0.f ? (ref + log2f(l)) * kLn2F : (l == l ? -CUDART_INF_F : l);
    p.lse[row] = lse;
    if (p.lse_act) static_cast<T*>(p.lse_act)[row] = from_f<T>(lse);
  }
}

// Positions of the nodes, -1 for those that are absent.  A length past max_len is reported.
__global__ void __launch_bounds__(kTreeMaxNodes) tree_positions_kernel(const int32_t* parents, const int32_t* lens, int32_t* pos, int n, int max_len) {
  __shared__ int par_s[kTreeMaxNodes];
  __shared__ u64t anc[kTreeMaxNodes + 1];
  const int b = blockIdx.x, j = threadIdx.x;
  tree_ancestors(tree_parents(parents + (int64_t)b * n, n, j), n, 0, 0, par_s, anc, j, 0, kTreeMaxNodes);
  if (j == 0 && lens[b] > max_len) atomicExch(&g_tree_status, 8200003);
  if (j < n) pos[(int64_t)b * n + j] = anc[j] ? max(lens[b], 0) + __popcll(anc[j]) - 1 : -1;
}

// Tiles of a sequence of at most max_len tokens
static int tree_tiles(int max_len, int W) {
  const int all = (max_len + 63) / 64;
  return 1 + (W == 0 ? all : std::min<int64_t>(all, ((int64_t)W + 62) / 64 + 1));
}

// Shares of the tiles: the number that makes the busiest SM finish first, where a CTA costs what its tiles cost and about eight
// more to start and to write its partial result (measured with 1, 2, 4, 8, 12: 32 rows over 16000 tokens 118 us up to 4, 110 to
// 112 from 8 on; 384 rows 107 and 101; 256 rows over 32000 tokens the same).
static int tree_splits(int64_t ctas, int tiles, int slots) {
  int best = 1;
  int64_t cost = INT64_MAX;
  for (int s = 1; s <= std::min(tiles, kTreeMaxSplits); ++s) {
    const int64_t waves = (ctas * s + slots - 1) / slots, c = waves * ((tiles + s - 1) / s + 8) + (s > 1 ? 4 : 0);
    if (c < cost) { cost = c; best = s; }
  }
  return best;
}

// Rows of one key head that a CTA takes: fp32 the CUDA-core kernel's tile, bf16 the 128 of a tensor-core instruction.
static int tree_cta_rows(int dtype) { return dtype == HILS_BF16 ? 128 : kTreeRows; }

static TreeParams tree_plan(int B, int n, int h_q, int h_kv, int max_len, int W, int dtype) {
  TreeParams p = {};
  p.B = B; p.n = n; p.h_q = h_q; p.h_kv = h_kv; p.W = W;
  const int64_t R = (int64_t)n * (h_q / h_kv);
  const int rows = tree_cta_rows(dtype);
  p.row_blocks = (int)((R + rows - 1) / rows);
  p.splits = tree_splits((int64_t)B * h_kv * p.row_blocks, tree_tiles(max_len, W), 148 * 2);
  return p;
}

static size_t tree_workspace(const TreeParams& p, int D) {
  return p.splits > 1 ? (size_t)p.splits * p.B * p.n * p.h_q * (D + 2) * sizeof(float) : 0;
}

int take_status_tree() {
  int v = 0, zero = 0;
  if (cudaDeviceSynchronize() != cudaSuccess) return -1;
  if (cudaMemcpyFromSymbol(&v, g_tree_status, sizeof(int)) != cudaSuccess) return -1;
  if (v != 0) cudaMemcpyToSymbol(g_tree_status, &zero, sizeof(int));
  return v;
}

int tree_tc_launch(const TreeParams& p, int D, cudaStream_t st);   // tree_attn_tc.cu

template <typename T, int D>
static int launch_tree(const TreeParams& p, cudaStream_t st) {
  if constexpr (sizeof(T) == 2) {
    if (int rc = tree_tc_launch(p, D, st)) return rc;
  } else {
    const size_t smem = tree_smem_floats<D>() * sizeof(float);
    cudaFuncSetAttribute(tree_attn_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    tree_attn_kernel<T, D><<<dim3((unsigned)(p.row_blocks * p.splits), (unsigned)p.h_kv, (unsigned)p.B), kTreeThreads, smem, st>>>(p);
    HILS_LAUNCH_CHECK("tree_attn_paged");
  }
  if (p.splits > 1) {
    const int64_t rows = (int64_t)p.B * p.n * p.h_q;
    tree_join_kernel<T, D><<<(unsigned)((rows + 7) / 8), 256, 0, st>>>(p);
    HILS_LAUNCH_CHECK("tree_attn_paged (join)");
  }
  return HILS_OK;
}

size_t tree_attn_workspace(int B, int n, int h_q, int h_kv, int D, int max_len, int W, int dtype) {
  return tree_workspace(tree_plan(B, n, h_q, h_kv, max_len, W, dtype), D);
}

void tree_positions_launch(const int32_t* parents, const int32_t* lens, int32_t* positions, int B, int n, int max_len, cudaStream_t st) {
  tree_positions_kernel<<<(unsigned)B, kTreeMaxNodes, 0, st>>>(parents, lens, positions, n, max_len);
}

// Checked arguments; lse_act as in TreeParams.
int tree_attn_launch(const void* q, const void* k_new, const void* v_new, const void* k_pages, const void* v_pages, const int32_t* page_table,
                     int page_stride, int num_pages, const int32_t* lens, int max_len, const int32_t* parents, void* o, float* lse,
                     void* lse_act, int B, int n, int h_q, int h_kv, int D, int W, int mask_lmk, int expand, float scale, int dtype,
                     void* workspace, size_t workspace_bytes, cudaStream_t st) {
  TreeParams p = tree_plan(B, n, h_q, h_kv, max_len, W, dtype);
  const size_t need = tree_workspace(p, D);
  if (need > 0 && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15))) {
    set_error("tree_attn_paged: a 16-byte aligned workspace of %zu bytes needed, %zu given", need, workspace_bytes);
    return HILS_ERR_WORKSPACE;
  }
  p.q = q; p.k_new = k_new; p.v_new = v_new; p.k_pages = k_pages; p.v_pages = v_pages; p.pages = page_table; p.lens = lens;
  p.parents = parents; p.o = o; p.lse = lse; p.lse_act = lse_act; p.page_stride = page_stride; p.num_pages = num_pages;
  p.mask_lmk = mask_lmk; p.expand = expand; p.scale = scale;
  p.part_o = static_cast<float*>(workspace);
  p.part_ml = p.part_o + (size_t)p.splits * B * n * h_q * D;
  if (dtype == HILS_BF16) return D == 128 ? launch_tree<bf16, 128>(p, st) : launch_tree<bf16, 64>(p, st);
  return D == 128 ? launch_tree<float, 128>(p, st) : launch_tree<float, 64>(p, st);
}

}  // namespace hils

using namespace hils;

static int check_tree(int B, int n, int h_q, int h_kv, int D, int max_len, int window_size, int chunk_size, int dtype) {
  HILS_REQUIRE(dtype == HILS_BF16 || dtype == HILS_F32, "tree_attn_paged: dtype must be bf16 or fp32");
  HILS_REQUIRE(B >= 0 && B <= 65535, "tree_attn_paged: %d sequences (at most 65535)", B);
  HILS_REQUIRE(n >= 0 && n <= kTreeMaxNodes, "tree_attn_paged: %d nodes (at most %d)", n, kTreeMaxNodes);
  HILS_REQUIRE(h_q > 0 && h_kv > 0 && h_q % h_kv == 0, "tree_attn_paged: h_q must be a multiple of h_kv");
  HILS_REQUIRE(h_kv <= 65535 && h_q / h_kv <= 1024, "tree_attn_paged: too many heads");
  HILS_REQUIRE(D == 64 || D == 128, "tree_attn_paged: head dimension %d (64 or 128)", D);
  HILS_REQUIRE(chunk_size == 64, "tree_attn_paged: the page is the chunk and must hold 64 tokens (got %d)", chunk_size);
  HILS_REQUIRE(max_len >= 0 && max_len <= 0x7fffffff - 256, "tree_attn_paged: bad length %d", max_len);
  HILS_REQUIRE(window_size >= 0, "tree_attn_paged: negative window");
  return HILS_OK;
}

extern "C" size_t hils_tree_attn_paged_workspace_bytes(int B, int n, int h_q, int h_kv, int D, int max_len, int window_size, int dtype) {
  if (check_tree(B, n, h_q, h_kv, D, max_len, window_size, 64, dtype) || B == 0 || n == 0) return 0;
  return tree_attn_workspace(B, n, h_q, h_kv, D, max_len, window_size, dtype);
}

extern "C" int hils_tree_attn_paged(const void* q, const void* k_new, const void* v_new, const void* k_pages, const void* v_pages,
                                    const int32_t* page_table, int page_stride, int num_pages, const int32_t* lens, int max_len,
                                    const int32_t* parents, void* o, float* lse, int B, int n, int h_q, int h_kv, int D, int window_size,
                                    int chunk_size, int mask_lmk, int expand_to_chunk, float sm_scale, int dtype, void* workspace,
                                    size_t workspace_bytes, void* stream) {
  if (int rc = check_tree(B, n, h_q, h_kv, D, max_len, window_size, chunk_size, dtype)) return rc;
  HILS_REQUIRE(sm_scale > 0.f && sm_scale <= 3.4e38f, "tree_attn_paged: sm_scale must be positive");
  HILS_REQUIRE(page_stride > 0 && num_pages > 0, "tree_attn_paged: bad size");
  HILS_REQUIRE((int64_t)num_pages * h_kv * 64 <= 0x7fffffff, "tree_attn_paged: a pool of %d pages of %d heads is too large", num_pages, h_kv);
  HILS_REQUIRE((max_len + 63) / 64 <= page_stride, "tree_attn_paged: %d tokens do not fit a page table of %d pages", max_len, page_stride);
  if (B == 0 || n == 0) return HILS_OK;
  HILS_REQUIRE(q && k_new && v_new && k_pages && v_pages && page_table && lens && parents && o && lse, "tree_attn_paged: null pointer");
  HILS_REQUIRE(((((uintptr_t)q) | ((uintptr_t)k_new) | ((uintptr_t)v_new) | ((uintptr_t)k_pages) | ((uintptr_t)v_pages) | ((uintptr_t)o)) & 15) == 0,
               "tree_attn_paged: tensors must be 16-byte aligned");
  return hils::tree_attn_launch(q, k_new, v_new, k_pages, v_pages, page_table, page_stride, num_pages, lens, max_len, parents, o, lse, nullptr, B,
                                n, h_q, h_kv, D, window_size, mask_lmk, expand_to_chunk, sm_scale, dtype, workspace, workspace_bytes,
                                (cudaStream_t)stream);
}

extern "C" int hils_draft_positions(const int32_t* parents, const int32_t* lens, int32_t* positions, int B, int n, void* stream) {
  HILS_REQUIRE(B >= 0 && n >= 0 && n <= kTreeMaxNodes, "draft_positions: %d sequences of %d nodes (at most %d)", B, n, kTreeMaxNodes);
  if (B == 0 || n == 0) return HILS_OK;
  HILS_REQUIRE(parents && lens && positions, "draft_positions: null pointer");
  hils::tree_positions_launch(parents, lens, positions, B, n, 0x7fffffff, (cudaStream_t)stream);
  HILS_LAUNCH_CHECK("draft_positions");
  return HILS_OK;
}
