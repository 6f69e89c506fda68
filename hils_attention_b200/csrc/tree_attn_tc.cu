// Attention of a tree of drafted tokens over the paged store on the tensor cores (tcgen05 + TMEM + TMA), bf16.
//
// One CTA owns 128 (node, head) rows of one key head and a share of the 64-key tiles (tree_common.cuh: tile 0 is the
// drafted nodes, the others are pages).  A page of one head is a contiguous 64 x D block, so a tile is one TMA box per 64
// columns and the page table costs one 4-byte read per tile.  S = Q K^T goes to tensor memory (two buffers, so the next
// product runs under this tile's softmax), a thread owns a row of S, P = exp2(S - m), bf16, goes back over the columns its S
// had and is the A operand of O += P V from there: P costs no shared memory, and the rows never wait for a product.
//
// One sweep.  The reference point m of a row moves only when its maximum grows by more than 2^8 (then the row of O is read,
// scaled and written back); until then P is at most 256 and the sums, in fp32, are as exact as with the true maximum.  P is
// rounded to bf16 (half a step, 2^-8 relative, of the order of the output's own rounding); the row sum is not.
//
// Places nobody sees may hold NaN: their scores are selected away before the maximum, and their V rows are zeroed in shared
// memory before the product (0 * NaN would spoil the row).  A key that one row sees and another does not (a drafted branch,
// the edge of the window) cannot be zeroed; where its V holds a non-finite value it is zeroed all the same and added row by
// row at the end, from global memory.
//
// What bounds it (1965 MHz).  Many rows: 64 nodes x 4 query heads a key head, 4 sequences of 32000 tokens: 159 us, floor 83 (136
// GFLOP; 524 MB); 194 in a loop under the power cap.  An S product of 128 x 64 x 16 issues every 62 clocks instead of 32, since it
// reads 6 KB of operands from shared memory (Q would have to be in tensor memory, which is full), P V at the rate of the
// arithmetic: 763 clocks a tile, two CTAs an SM, 1526 of the 1950 clocks that two tiles take; the exponentials 1024 of them.
// 256 rows in one CTA, which brings a tile once, took 179 (171 with one group at that time); P through shared memory 224.
// Few rows: 16 nodes, 32 sequences x 32 heads, window 512: 83 us, floor 46 (302 MB).  While tiles run, 2 CTAs an SM ask for all
// the HBM gives; of a CTA's 31000 clocks 5900 pass before its first tile and 4700 after its last, and 1024 CTAs are 3.46 waves.
// Not faster for these: keys as the rows of the product (four CTAs an SM: 92 us against 80 in the same loop), rows dealt to other
// warps (D 64: 140 against 131).  Long caches with few rows run at 0.87 of the copy bandwidth (8 x 16000 tokens, 8 key heads: 92 us
// in a loop).
#include <algorithm>
#include <atomic>

#include "tc_rows.cuh"
#include "tree_common.cuh"
#include "umma.cuh"

namespace hils {

// A page outside the pool (8200001), a length past the table (8200002)
static __device__ int g_tree_tc_status = 0;
// A wait that ran out (8300001 ..), for the host alone.  g_tree_tc_given_up is the call (TreeParams::call) it happened in: CTAs of
// that call that start later return zeros at once, other calls have nothing to do with it.
static __device__ int g_tree_tc_expired = 0;
static __device__ unsigned g_tree_tc_given_up = 0u;

__device__ __forceinline__ void give_up(const TreeParams& p, int code) {
  atomicExch(&g_tree_tc_expired, code);
  atomicExch(&g_tree_tc_given_up, p.call);
}

// A replay of a captured call has the number of the capture: what an earlier replay left is cleared before it.
__global__ void tree_tc_begin_kernel(unsigned call) {
  if (g_tree_tc_given_up == call) g_tree_tc_given_up = 0u;
}

using namespace umma;

constexpr float kTtSlack = 8.f;              // log2 units a row's maximum may grow before O is rescaled

// Two CTAs share an SM.  KS, VS: places for the K and the V of a tile.
template <int D> struct TtShape {
  static constexpr int DB = D / 64, QBYTES = DB * 16384, TBYTES = DB * 8192;
  static constexpr int KS = D == 128 ? 2 : 4, VS = D == 128 ? 3 : 4;
  static constexpr int THREADS = 192;                      // row warps, a warp that issues the products, one that brings the tiles
  static constexpr int VAT = QBYTES + KS * TBYTES, BARS = VAT + VS * TBYTES;
  // The ancestors are worked out where the third V tile will be: it is sent for when they are known.
  static constexpr int SCRATCH = VAT + 2 * TBYTES, SMEM = BARS + 512;
};

__device__ __forceinline__ bool not_finite8(uint4 x) {     // eight bf16: an exponent of all ones
  bool bad = false;
#pragma unroll
  for (const uint32_t w : {x.x, x.y, x.z, x.w}) bad = bad || (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u;
  return bad;
}

// row `r` of a [64 x D] tile of DB column blocks, piece c of 16 bytes
__device__ __forceinline__ uint8_t* tile_at(uint8_t* tile, int r, int c) { return tile + (c >> 3) * 8192 + sw128_off(r, c & 7); }

// A second (2^18 polls of 3.95 us), shorter than the common limit: these waits are for copies and products of one tile, microseconds.
__device__ __forceinline__ bool wait_for(uint64_t* b, uint32_t parity) { return mbar_wait<1 << 18>(b, parity); }

// What the products left out for one row: the keys whose V rows were zeroed although this row sees them.  Rare (a value that
// is not finite in a drafted branch or at the edge of the window), so plainly: the score again, from global memory.
template <int D>
__device__ __forceinline__ void add_bad_keys(const TreeParams& p, const u64t* bad, int b, int h, int64_t out, const bf16* kn, const bf16* vn,
                                          int64_t nrs, int c0, int len, int lo, u64t dmask, float sl2, float ref, int cb, float (&ov)[32]) {
  const bf16* q = static_cast<const bf16*>(p.q) + out * D;
#pragma unroll 1
  for (int k = 0; k < 3; ++k) {
    const int c = c0 + k - 1;
#pragma unroll 1
    for (u64t rest = bad[k] & (k == 0 ? dmask : tree_page_mask(p, c, len, lo)); rest; rest &= rest - 1) {
      const int i = __ffsll((long long)rest) - 1;
      const int64_t at = k == 0 ? i * nrs : (((int64_t)tree_page(p, b, c) * p.h_kv + h) * 64 + i) * D;
      const bf16* kr = (k == 0 ? kn : static_cast<const bf16*>(p.k_pages)) + at;
      const bf16* vr = (k == 0 ? vn : static_cast<const bf16*>(p.v_pages)) + at;
      float s = 0.f;
#pragma unroll 1
      for (int d = 0; d < D; ++d) s = fmaf(to_f(q[d]), to_f(kr[d]), s);
      const float w = to_f(__float2bfloat16_rn(ex2(fmaf(s, sl2, -ref))));
#pragma unroll
      for (int j = 0; j < 32; ++j) ov[j] = fmaf(w, to_f(vr[cb * 32 + j]), ov[j]);
    }
  }
}

// two fp32 sums or products at a time
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  unsigned long long d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(reinterpret_cast<u64t&>(a)), "l"(reinterpret_cast<u64t&>(b)), "l"(reinterpret_cast<u64t&>(c)));
  return reinterpret_cast<float2&>(d);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  unsigned long long d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(reinterpret_cast<u64t&>(a)), "l"(reinterpret_cast<u64t&>(b)));
  return reinterpret_cast<float2&>(d);
}

// D[tmem] (+)= A[tmem] * B[smem]; A: 128 rows, two bf16 to a column
__device__ __forceinline__ void mma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t db, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}"
      ::"r"(tmem_d), "r"(tmem_a), "l"(db), "r"(idesc), "r"(accumulate)
      : "memory");
}

template <int D>
__global__ void __launch_bounds__(TtShape<D>::THREADS, 2) tree_attn_tc_kernel(const __grid_constant__ TreeParams p, const __grid_constant__ CUtensorMap tmK,
                                                                     const __grid_constant__ CUtensorMap tmV) {
  using Sh = TtShape<D>;
  constexpr int KS = Sh::KS, VS = Sh::VS, DB = Sh::DB, TB = Sh::TBYTES, kRows = 128, kThreads = Sh::THREADS;
  constexpr int kMmaWarp = 4, kLoadWarp = 5, kTmem = 256;
  extern __shared__ uint8_t tt_smem[];
  uint8_t* Qs = tt_smem;
  uint8_t* Ks = Qs + Sh::QBYTES;
  uint8_t* Vs = tt_smem + Sh::VAT;
  uint64_t* bars = reinterpret_cast<uint64_t*>(tt_smem + Sh::BARS);
  uint64_t* k_full = bars;                 // [KS]
  uint64_t* k_free = k_full + KS;          // [KS]
  uint64_t* v_full = k_free + KS;          // [VS]
  uint64_t* v_ready = v_full + VS;         // [VS] and cleared of what nobody sees
  uint64_t* v_free = v_ready + VS;         // [VS]
  uint64_t* s_full = v_free + VS;          // [2]
  uint64_t* p_full = s_full + 2;           // [2]: a warp may be a tile ahead of another, not two
  uint64_t* pv_done = p_full + 2;          // [1]
  uint64_t* done = pv_done + 1;            // [1] used once: the last product
  uint64_t* setup = done + 1;              // [1] the row warps have read the ancestors
  u64t* bad_s = reinterpret_cast<u64t*>(setup + 1);   // [3] keys with non-finite values: drafts, tiles c0, c0 + 1
  volatile int* tile_ok = reinterpret_cast<volatile int*>(bad_s + 3);   // [8]
  uint32_t& tmem_base_s = *reinterpret_cast<uint32_t*>(const_cast<int*>(tile_ok) + 8);
  volatile int& abort_s = const_cast<volatile int*>(tile_ok)[9];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if ((reinterpret_cast<uintptr_t>(tt_smem) & 1023) != 0) {   // the tiles need the 1 KB alignment of their swizzle
    if (tid == 0) give_up(p, 8300009);
    return;
  }
  const int G = p.h_q / p.h_kv, R = p.n * G;
  const int rb = blockIdx.x % p.row_blocks, split = blockIdx.x / p.row_blocks, h = blockIdx.y, b = blockIdx.z;
  bool over;
  const int len = tree_length(p, b, over);
  const int2 parents = tree_parents(p.parents + (int64_t)b * p.n, p.n, tid);
  // all loads that need no length are sent for first: the rows (a warp its 32, whole rows at a time), the drafted keys and values
  const int64_t new0 = (int64_t)b * p.n;
  const int row = rb * kRows + tid;
  const bool valid = tid < kRows && row < R, draft = split == 0;
  const int64_t out = valid ? (new0 + row / G) * p.h_q + h * G + row % G : 0;
  const bf16* kn = static_cast<const bf16*>(p.k_new) + (new0 * p.h_kv + h) * D;
  const bf16* vn = static_cast<const bf16*>(p.v_new) + (new0 * p.h_kv + h) * D;
  const int64_t nrs = (int64_t)p.h_kv * D;
  constexpr int kMeet = kThreads - 32, kDraft = (64 * (D / 8) + kMeet - 1) / kMeet;
  uint4 qv[D / 8], kx[kDraft], vx[kDraft];
  if (tid < kRows) {
    const uint32_t real = __ballot_sync(0xffffffffu, valid);
#pragma unroll
    for (int i = 0; i < D / 8; ++i) {
      const int x = i * 32 + lane, rr = x / (D / 8), c = x % (D / 8);
      const int64_t from = __shfl_sync(0xffffffffu, out, rr);
      qv[i] = make_uint4(0u, 0u, 0u, 0u);
      if (real >> rr & 1u) qv[i] = *reinterpret_cast<const uint4*>(static_cast<const bf16*>(p.q) + from * D + c * 8);
    }
  }
  if (draft && warp != kLoadWarp) {
#pragma unroll
    for (int i = 0; i < kDraft; ++i) {
      const int x = i * kMeet + tid, r = x / (D / 8), c = x % (D / 8);
      kx[i] = vx[i] = make_uint4(0u, 0u, 0u, 0u);
      if (r < p.n) {
        kx[i] = *reinterpret_cast<const uint4*>(kn + r * nrs + c * 8);
        vx[i] = *reinterpret_cast<const uint4*>(vn + r * nrs + c * 8);
      }
    }
  }
  if (tid == 32 * kLoadWarp) {
    for (int s = 0; s < KS; ++s) { mbar_init(&k_full[s], 1); mbar_init(&k_free[s], 1); }
    for (int s = 0; s < VS; ++s) { mbar_init(&v_full[s], 1); mbar_init(&v_ready[s], 1); mbar_init(&v_free[s], 1); }
    for (int s = 0; s < 2; ++s) { mbar_init(&s_full[s], 1); mbar_init(&p_full[s], 128); }
    mbar_init(pv_done, 1);
    mbar_init(done, 1);
    mbar_init(setup, 4);
    mbar_init_fence();
    abort_s = *const_cast<volatile unsigned*>(&g_tree_tc_given_up) == p.call;
    bad_s[0] = bad_s[1] = bad_s[2] = 0ull;
    if (over) atomicExch(&g_tree_tc_status, 8200002);
  }
  if (warp == kMmaWarp) tmem_alloc(&tmem_base_s, kTmem);
  const int lo_min = tree_low(p, len), c0 = lo_min >> 6, c1 = (len + 63) >> 6;
  const int nt = 1 + max(0, c1 - c0), per = (nt + p.splits - 1) / p.splits;
  const int t0 = split * per, first = c0 + max(t0, 1) - 1;   // first: chunk of this CTA's first page tile
  int ids = -1;
  if (warp == kLoadWarp && first + lane < c1) ids = p.pages[(int64_t)b * p.page_stride + first + lane];
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base_s, tS = tmem, tO = tmem + 128;            // S: two buffers of 64 columns, O: D columns
  const int nit = abort_s ? 0 : max(0, min(nt, t0 + per) - t0);
  __syncthreads();                                         // nobody has set abort_s on the way

  // ---- ancestors, rows, drafted keys; the producer is already on its way ------------
  int lo = 0x7fffffff;
  u64t dmask = 0ull;
  if (warp != kLoadWarp) {
    u64t* anc = reinterpret_cast<u64t*>(tt_smem + Sh::SCRATCH);
    if (draft) {
#pragma unroll
      for (int i = 0; i < kDraft; ++i) {
        const int x = i * kMeet + tid, r = x / (D / 8), c = x % (D / 8);
        if (not_finite8(vx[i])) {                          // zero in the product, added row by row at the end
          atomicOr(&bad_s[0], 1ull << r);
          vx[i] = make_uint4(0u, 0u, 0u, 0u);
        }
        if (r < 64) {
          *reinterpret_cast<uint4*>(tile_at(Ks, r, c)) = kx[i];
          *reinterpret_cast<uint4*>(tile_at(Vs, r, c)) = vx[i];
        }
      }
    }
    if (tid < kRows) {
#pragma unroll
      for (int i = 0; i < D / 8; ++i) {
        const int x = i * 32 + lane, rr = x / (D / 8), c = x % (D / 8);
        *reinterpret_cast<uint4*>(Qs + (c >> 3) * 16384 + sw128_off(warp * 32 + rr, c & 7)) = qv[i];
      }
    }
    fence_async_smem();
    tree_ancestors(parents, p.n, len, p.mask_lmk, reinterpret_cast<int*>(anc + kTreeMaxNodes + 2), anc, tid, 2, kMeet);
    // behind that barrier the rows and the drafted tile are there
    if (draft && bad_s[0] != 0ull) {                       // rare: the other pieces of those rows
      for (int x = tid; x < 64 * (D / 8); x += kMeet)
        if (bad_s[0] >> (x / (D / 8)) & 1ull) *reinterpret_cast<uint4*>(tile_at(Vs, x / (D / 8), x % (D / 8))) = make_uint4(0u, 0u, 0u, 0u);
      fence_async_smem();
      named_bar_sync(2, kMeet);
    }
    if (draft && tid == 0) {
      mbar_arrive(&k_full[0]);
      mbar_arrive(&v_full[0]);
      mbar_arrive(&v_ready[0]);
    }
    if (warp < kMmaWarp) {                                 // the masks while the first product runs; then the ancestors' place is free
      if (valid && anc[row / G] != 0ull) {
        lo = tree_low(p, len + __popcll(anc[row / G]) - 1);
        dmask = tree_draft_mask(anc, row / G, len, lo);
      }
      fence_async_smem();                                  // the next to write there is a TMA copy
      __syncwarp();
      if (lane == 0) mbar_arrive(setup);
    }
  }

  const float sl2 = p.scale * kLog2E;
  if (warp == kLoadWarp) {
    // ---- producer: K of a tile one step before its V, the order in which their places become free; and when a V tile has
    // landed, the rows that nobody sees become zeros, and so do those that some rows see and others do not (the deepest
    // node's left edge is at most that of position len + n - 1) and that are not finite.
    const int lo_max = tree_low(p, len + p.n - 1);
    auto clear_v = [&](int it, bool in_pool) {
      const int s = it % VS, t = t0 + it, c = c0 + t - 1;
      if (t == 0) return true;                             // drafts: cleared and announced by the other warps
      const u64t unseen = ~(in_pool ? tree_page_mask(p, c, len, lo_min) : 0ull);
      const bool mixed = lo_max > c * 64 && c - c0 < 2, got = __all_sync(0xffffffffu, wait_for(&v_full[s], (it / VS) & 1));
      uint8_t* tile = Vs + s * TB;
      u64t gone = unseen;
      if (mixed) {
        u64t bad = 0ull;
        for (int x = lane; x < 64 * (D / 8); x += 32)
          if (!(unseen >> (x / (D / 8)) & 1ull) && not_finite8(*reinterpret_cast<const uint4*>(tile_at(tile, x / (D / 8), x % (D / 8)))))
            bad |= 1ull << (x / (D / 8));
        bad = (u64t)__reduce_or_sync(0xffffffffu, (uint32_t)bad) | (u64t)__reduce_or_sync(0xffffffffu, (uint32_t)(bad >> 32)) << 32;
        if (lane == 0) bad_s[1 + c - c0] = bad;
        gone |= bad;
      }
      if (gone == 1ull << 63) {                            // a full page: its landmark
        if (lane < D / 8) *reinterpret_cast<uint4*>(tile_at(tile, 63, lane)) = make_uint4(0u, 0u, 0u, 0u);
      } else if (gone != 0ull) {
        for (int x = lane; x < 64 * (D / 8); x += 32)
          if (gone >> (x / (D / 8)) & 1ull) *reinterpret_cast<uint4*>(tile_at(tile, x / (D / 8), x % (D / 8))) = make_uint4(0u, 0u, 0u, 0u);
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&v_ready[s]);
      return got;
    };
    int pg = 0, prev = 0, k_issued = 0, v_issued = 0;
    bool ok = true;
    auto bring = [&](uint64_t* full, uint8_t* tile, const CUtensorMap* map, bool draft, int page) {
      if (draft) return;                                   // written and announced by the other warps
      if ((unsigned)page >= (unsigned)p.num_pages) {
        mbar_arrive(full);
        return;
      }
      mbar_expect_tx(full, TB);
#pragma unroll
      for (int db = 0; db < DB; ++db) tma_load_2d(tile + db * 8192, map, full, db * 64, (page * p.h_kv + h) * 64);
    };
    // V of a tile is cleared when all of the ring behind it is on its way, so that waiting for it holds no load back
    constexpr int kLag = VS - 1;
    uint32_t pool_bits = 0u;                               // bit i: tile step - i is in the pool
    for (int step = 0; step < nit + kLag; ++step) {
      const int c = c0 + t0 + step - 1;
      prev = pg;                                           // page of tile step - 1, whose V is due
      if (step < nit) {
        if (t0 + step > 0) {
          if (c > first && ((c - first) & 31) == 0) ids = c + lane < c1 ? p.pages[(int64_t)b * p.page_stride + c + lane] : -1;
          pg = __shfl_sync(0xffffffffu, ids, (c - first) & 31);
        } else {
          pg = 0;
        }
      }
      pool_bits = pool_bits << 1 | ((unsigned)pg < (unsigned)p.num_pages ? 1u : 0u);
      if (lane == 0) {
        if (step < nit) {
          const int s = step % KS;
          if (step >= KS) ok = wait_for(&k_free[s], (step / KS - 1) & 1);
          if (ok) {
            const bool in_pool = (unsigned)pg < (unsigned)p.num_pages;
            tile_ok[step & 7] = in_pool;                   // reaches the row threads through k_full and s_full; they are past step - 8
            if (!in_pool) atomicExch(&g_tree_tc_status, 8200001);
            bring(&k_full[s], Ks + s * TB, &tmK, t0 + step == 0, pg);
            ++k_issued;
          }
        }
        if (ok && step > 0 && step <= nit) {
          const int it = step - 1, s = it % VS;
          if (it >= VS) ok = wait_for(&v_free[s], (it / VS - 1) & 1);
          else if (it == 2) ok = wait_for(setup, 0);       // the third place was the ancestors'
          if (ok) {
            bring(&v_full[s], Vs + s * TB, &tmV, t0 + it == 0, prev);
            ++v_issued;
          }
        }
      }
      ok = __shfl_sync(0xffffffffu, (int)ok, 0);
      if (ok && step >= kLag) ok = clear_v(step - kLag, pool_bits >> kLag & 1u);
      if (!__all_sync(0xffffffffu, ok && !abort_s)) break;
    }
    if (lane == 0) {
      if (!ok) { abort_s = 1; give_up(p, 8300001); }
      for (int it = max(0, k_issued - KS); it < k_issued; ++it) wait_for(&k_full[it % KS], (it / KS) & 1);   // no copy outlives the CTA
      for (int it = max(0, v_issued - VS); it < v_issued; ++it) wait_for(&v_full[it % VS], (it / VS) & 1);
    }
  } else if (warp == kMmaWarp) {
    // ---- products.  The whole warp runs the loop and one elected lane issues: descriptors then live in uniform registers,
    // where the instruction takes them from. ------------------------------------------------------------------------------
    if (nit > 0) {
      constexpr uint32_t idesc_qk = idesc_bf16(128, 64, 0);
      constexpr uint32_t idesc_pv = idesc_bf16(128, D, 1);
      const uint64_t q_d = desc_sw128(smem_u32(Qs), 16, 1024), k_d = desc_sw128(smem_u32(Ks), 16, 1024), v_d = desc_sw128(smem_u32(Vs), 8192, 1024);
      auto issue_qk = [&](int buf, int place) {
        if (elect_one()) {
          const uint64_t kb = k_d + place * (TB >> 4);
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk)
            mma_ss(tS + buf * 64, q_d + (((kk >> 2) * 16384 + (kk & 3) * 32) >> 4), kb + (((kk >> 2) * 8192 + (kk & 3) * 32) >> 4), idesc_qk, kk > 0);
          mma_commit(&s_full[buf]);
          mma_commit(&k_free[place]);
        }
        __syncwarp();
      };
      bool ok = __all_sync(0xffffffffu, wait_for(&k_full[0], 0));
      if (ok) {
        tc_fence_after();
        issue_qk(0, 0);
      }
      // places and phases are counted along: a division by VS costs as much as a barrier
      int ks = 0, vs = 0;
      uint32_t kp = 0, vp = 0;
      for (int it = 0; ok && it < nit; ++it) {
        const int buf = it & 1;
        if (it + 1 < nit) {                                // into the columns of S and P of it - 1
          if (++ks == KS) { ks = 0; kp ^= 1; }
          ok = wait_for(&k_full[ks], kp);
          if (it > 0) ok = wait_for(pv_done, buf ^ 1) && ok;
          if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
          tc_fence_after();
          issue_qk(buf ^ 1, ks);
        }
        ok = wait_for(&v_ready[vs], vp);
        ok = wait_for(&p_full[buf], (it >> 1) & 1) && ok;
        if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
        tc_fence_after();
        if (elect_one()) {
          const uint64_t b0 = v_d + vs * (TB >> 4);
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) mma_ts(tO, tS + buf * 64 + kk * 8, b0 + ((kk * 2048) >> 4), idesc_pv, it > 0 || kk > 0);
          mma_commit(pv_done);
          mma_commit(&v_free[vs]);
        }
        __syncwarp();
        if (++vs == VS) { vs = 0; vp ^= 1; }
      }
      if (!ok && lane == 0) { abort_s = 1; give_up(p, 8300002); }
      __threadfence_block();
      __syncwarp();
      if (elect_one()) mma_commit(done);               // no product outlives the CTA's tensor memory
      wait_for(done, 0);
    }
  } else {
    // ---- rows -----------------------------------------------------------------------------------------------------------
    const uint32_t lane_base = (uint32_t)(warp * 32) << 16, tSg = tS + lane_base, tOg = tO + lane_base;
    const bool rows_here = rb * kRows + warp * 32 < R;
    float m = -CUDART_INF_F, l = 0.f;                      // reference point (log2 units) and sum
    bool ok = true;
    for (int it = 0; it < nit; ++it) {
      const int s = it & 1, t = t0 + it, c = c0 + t - 1;
      ok = __all_sync(0xffffffffu, wait_for(&s_full[s], (it >> 1) & 1) && !abort_s);
      if (!ok) break;
      tc_fence_after();
      float sv[64];
      if (rows_here) {
        tmem_ld32(tSg + s * 64, sv);
        tmem_ld32(tSg + s * 64 + 32, sv + 32);
      }
      // (k_full of this tile cannot be asked here: with the product done the next tile of the place may have arrived too)
      const bool in_pool = tile_ok[it & 7] != 0;
      // rows past the last one hold zeros and go nowhere: they "see" everything, which keeps their warp on the short path
      const u64t vis = !valid ? ~0ull : (t == 0 ? dmask : (in_pool ? tree_page_mask(p, c, len, lo) : 0ull));
      bool moved = false;
      if (rows_here) {
        tmem_ld_wait64(sv);
        // a warp whose rows all see everything, or everything but the landmark, skips the selection
        if (__all_sync(0xffffffffu, (vis | 1ull << 63) == ~0ull)) {
          if (!(vis >> 63)) sv[63] = -CUDART_INF_F;
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            sv[j] = ((uint32_t)vis & (1u << j)) ? sv[j] : -CUDART_INF_F;
            sv[j + 32] = ((uint32_t)(vis >> 32) & (1u << j)) ? sv[j + 32] : -CUDART_INF_F;
          }
        }
        float m4[4] = {sv[0], sv[1], sv[2], sv[3]};
#pragma unroll
        for (int j = 4; j < 64; ++j) m4[j & 3] = fmaxf(m4[j & 3], sv[j]);
        const float top = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * sl2;
        float grow = 1.f;
        if (top > m + kTtSlack) {                          // also the first visible key: m is -inf
          moved = m > -CUDART_INF_F;
          grow = moved ? ex2(m - top) : 0.f;
          m = top;
          l *= grow;
        }
        if (it > 0 && __any_sync(0xffffffffu, moved)) {    // rare after the first tiles: O stands still once the last product is done
          // (never a phase off: S of this tile came after the product of it - 2, the product of `it` waits for this thread)
          ok = wait_for(pv_done, (it - 1) & 1) && ok;
          tc_fence_after();
          const float f = moved ? grow : 1.f;
#pragma unroll 1
          for (int cb = 0; cb < D / 32; ++cb) {
            float ov[32];
            tmem_ld32(tOg + cb * 32, ov);
            tmem_ld_wait32(ov);
#pragma unroll
            for (int j = 0; j < 32; ++j) ov[j] *= f;
            tmem_st32(tOg + cb * 32, ov);
          }
        }
        const float ref = m > -CUDART_INF_F ? m : 0.f;
        const float2 sl2x2 = make_float2(sl2, sl2), refx2 = make_float2(-ref, -ref);
        float2 s4[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        float pk[32];                                      // pairs of bf16
#pragma unroll
        for (int j = 0; j < 64; j += 2) {
          float2 w = fma2(make_float2(sv[j], sv[j + 1]), sl2x2, refx2);
          w = make_float2(ex2(w.x), ex2(w.y));             // -inf gives 0
          s4[j >> 1 & 1] = add2(s4[j >> 1 & 1], w);
          const __nv_bfloat162 hh = __floats2bfloat162_rn(w.x, w.y);
          pk[j >> 1] = __uint_as_float(*reinterpret_cast<const uint32_t*>(&hh));
        }
        tmem_st32(tSg + s * 64, pk);                       // over the first half of the columns S had
        const float2 sum = add2(s4[0], s4[1]);
        l += sum.x + sum.y;
        tmem_st_wait();
      }
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_before();
      mbar_arrive(&p_full[s]);
    }
    // The last product, by a barrier of its own with a single phase.  pv_done cannot be asked here: the products of the last
    // two tiles need nothing more from this thread, so its barrier may be one or two phases ahead of the thread, and a parity
    // does not tell two phases from none.
    if (ok && nit > 0) ok = __all_sync(0xffffffffu, wait_for(done, 0) && !abort_s);
    if (!ok && lane == 0) {
      abort_s = 1;
      give_up(p, 8300003);
    }
    if (ok) tc_fence_after();
    const bool have = ok && nit > 0 && rows_here;
    if (!have) { m = -CUDART_INF_F; l = 0.f; }             // given up halfway: as a row that sees nothing, in both outputs
    const float inv = p.splits > 1 ? 1.f : (l > 0.f ? 1.f / l : (l == l ? 0.f : l));
    const int64_t at = (int64_t)split * p.B * p.n * p.h_q + out;
#pragma unroll 1
    for (int cb = 0; cb < D / 32; ++cb) {
      float ov[32];
      if (have) {
        tmem_ld32(tOg + cb * 32, ov);
        tmem_ld_wait32(ov);
      }
      if (l == 0.f) {                                      // a row that sees nothing: its weights are 0, but 0 * V is NaN for an infinite V
#pragma unroll
        for (int j = 0; j < 32; ++j) ov[j] = 0.f;
      }
      if (have && valid && (bad_s[0] | bad_s[1] | bad_s[2]))
        add_bad_keys<D>(p, bad_s, b, h, out, kn, vn, nrs, c0, len, lo, dmask, sl2, m > -CUDART_INF_F ? m : 0.f, cb, ov);
      // through shared memory (Q's place: its last product is done), so that 128 bytes of a row leave together
      if (rows_here) {
        float4* stage = reinterpret_cast<float4*>(Qs + warp * 4096);
#pragma unroll
        for (int j = 0; j < 8; ++j)
          stage[lane * 8 + (j ^ (lane & 7))] = make_float4(ov[4 * j] * inv, ov[4 * j + 1] * inv, ov[4 * j + 2] * inv, ov[4 * j + 3] * inv);
        __syncwarp();
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int rr = 4 * j + (lane >> 3), e = lane & 7;
          const int64_t to = __shfl_sync(0xffffffffu, out, rr);
          const float4 v = stage[rr * 8 + (e ^ (rr & 7))];
          if (row - lane + rr < R) {
            if (p.splits > 1) store4(p.part_o + ((int64_t)split * p.B * p.n * p.h_q + to) * D + cb * 32 + e * 4, v);
            else store4(static_cast<bf16*>(p.o) + to * D + cb * 32 + e * 4, v);
          }
        }
        __syncwarp();
      }
    }
    if (valid) {
      if (p.splits > 1) {
        *reinterpret_cast<float2*>(p.part_ml + 2 * at) = make_float2(m, l);
      } else {
        const float lse = l > 0.f ? (m + log2f(l)) * kLn2F : (l == l ? -CUDART_INF_F : l);
        p.lse[out] = lse;
        if (p.lse_act) static_cast<bf16*>(p.lse_act)[out] = __float2bfloat16_rn(lse);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) tmem_dealloc(tmem, kTmem);
}

int take_status_tree_tc() {
  int v = 0, x = 0, zero = 0;
  if (cudaDeviceSynchronize() != cudaSuccess) return -1;
  if (cudaMemcpyFromSymbol(&v, g_tree_tc_status, sizeof(int)) != cudaSuccess) return -1;
  if (cudaMemcpyFromSymbol(&x, g_tree_tc_expired, sizeof(int)) != cudaSuccess) return -1;
  if (v != 0) cudaMemcpyToSymbol(g_tree_tc_status, &zero, sizeof(int));
  if (x != 0) cudaMemcpyToSymbol(g_tree_tc_expired, &zero, sizeof(int));
  return x != 0 ? x : v;
}

static std::atomic<unsigned> g_tree_tc_calls{0u};

template <int D>
static int launch_tree_tc(TreeParams p, cudaStream_t st) {
  while ((p.call = ++g_tree_tc_calls) == 0u) {}            // 0: nobody
  cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
  if (cudaStreamIsCapturing(st, &capture) != cudaSuccess) cudaGetLastError();   // the launch below reports what is wrong with the stream
  if (capture == cudaStreamCaptureStatusActive) tree_tc_begin_kernel<<<1, 1, 0, st>>>(p.call);
  CUtensorMap tmK, tmV;
  const uint64_t rows = (uint64_t)p.num_pages * p.h_kv * 64;
  if (int rc = make_tmap_bf16_rows(&tmK, p.k_pages, rows, D, D, 64)) return rc;
  if (int rc = make_tmap_bf16_rows(&tmV, p.v_pages, rows, D, D, 64)) return rc;
  using Sh = TtShape<D>;
  cudaFuncSetAttribute(tree_attn_tc_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, Sh::SMEM);
  tree_attn_tc_kernel<D><<<dim3((unsigned)(p.row_blocks * p.splits), (unsigned)p.h_kv, (unsigned)p.B), Sh::THREADS, Sh::SMEM, st>>>(p, tmK, tmV);
  HILS_LAUNCH_CHECK("tree_attn_paged (tensor-core path)");
  return HILS_OK;
}

int tree_tc_launch(const TreeParams& p, int D, cudaStream_t st) { return D == 128 ? launch_tree_tc<128>(p, st) : launch_tree_tc<64>(p, st); }

}  // namespace hils
