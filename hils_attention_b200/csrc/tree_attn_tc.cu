// Attention of a tree of drafted tokens over the paged store on the tensor cores (tcgen05 + TMEM + TMA), bf16.
//
// One CTA owns 128 (node, head) rows of one key head and a share of the 64-key tiles (tree_common.cuh: tile 0 is the drafted
// nodes, the others are pages).  A page of one head is a contiguous 64 x D block, so a tile is one TMA box per 64 columns and
// the page table costs one 4-byte read per tile.  S = Q K^T goes to TMEM (two buffers, so the next product runs under this
// tile's softmax), a thread owns a row of S, P = exp2(S - m) goes to shared memory as bf16, O += P V stays in TMEM.
//
// One sweep.  The reference point m of a row moves only when its maximum grows by more than 2^8 (then the row of O is read,
// scaled and written back); until then P is at most 256 and the sums, in fp32, are as exact as with the true maximum.
//
// Places nobody sees may hold NaN: their scores are selected away before the maximum, and their V rows are zeroed in shared
// memory before the product (0 * NaN would spoil the row).  A key that one row sees and another does not (a drafted branch,
// the edge of the window) cannot be zeroed; where its V holds a non-finite value it is zeroed all the same and added row by
// row at the end, from global memory.
#include <algorithm>

#include "tc_rows.cuh"
#include "tree_common.cuh"
#include "umma.cuh"

namespace hils {

// A page outside the pool (8200001), a length past the table (8200002)
static __device__ int g_tree_tc_status = 0;
// A wait that ran out (8300001 ..); CTAs that start later see it and write nothing but zeros
static __device__ int g_tree_tc_expired = 0;

using namespace umma;

constexpr float kTtSlack = 8.f;              // log2 units a row's maximum may grow before O is rescaled

// TG groups of 128 rows share the tiles of a CTA.  One group: two CTAs per SM, each with places for two tiles of D = 128.
// Two groups (more than 128 rows per key head): one CTA per SM, every tile is brought once for 256 rows, four places.
template <int D, int TG> struct TtShape {
  static constexpr int DB = D / 64, QBYTES = DB * 16384, TBYTES = DB * 8192;
  static constexpr int NS = TG == 1 ? (D == 128 ? 2 : 4) : (D == 128 ? 4 : 6);
  static constexpr int THREADS = 128 * TG + 64;            // row warps, one warp that issues the products, one that brings the tiles
  static constexpr int PAT = TG * QBYTES + 2 * NS * TBYTES, BARS = PAT + TG * 16384, SMEM = BARS + 512;
};

__device__ __forceinline__ bool not_finite8(uint4 x) {     // eight bf16: an exponent of all ones
  bool bad = false;
#pragma unroll
  for (const uint32_t w : {x.x, x.y, x.z, x.w}) bad = bad || (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u;
  return bad;
}

// row `r` of a [64 x D] tile of DB column blocks, piece c of 16 bytes
__device__ __forceinline__ uint8_t* tile_at(uint8_t* tile, int r, int c) { return tile + (c >> 3) * 8192 + sw128_off(r, c & 7); }

// Shorter than the common limit: these waits are for copies and products of one tile, microseconds.
__device__ __forceinline__ bool wait_for(uint64_t* b, uint32_t parity) { return mbar_wait<1 << 20>(b, parity); }

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

template <int D, int TG>
__global__ void __launch_bounds__(TtShape<D, TG>::THREADS, TG == 1 ? 2 : 1) tree_attn_tc_kernel(const __grid_constant__ TreeParams p, const __grid_constant__ CUtensorMap tmK,
                                                                     const __grid_constant__ CUtensorMap tmV) {
  using Sh = TtShape<D, TG>;
  constexpr int NS = Sh::NS, DB = Sh::DB, TB = Sh::TBYTES, QB = Sh::QBYTES, kRows = 128 * TG, kThreads = Sh::THREADS;
  constexpr int kMmaWarp = 4 * TG, kLoadWarp = 4 * TG + 1, kTmem = TG == 1 ? 256 : 512;
  extern __shared__ uint8_t tt_smem[];
  uint8_t* Qs = tt_smem;
  uint8_t* Ks = Qs + TG * QB;
  uint8_t* Vs = Ks + NS * TB;
  uint8_t* Ps = tt_smem + Sh::PAT;
  uint64_t* bars = reinterpret_cast<uint64_t*>(tt_smem + Sh::BARS);
  uint64_t* k_full = bars;                 // [NS]
  uint64_t* k_free = bars + NS;            // [NS]
  uint64_t* v_full = bars + 2 * NS;        // [NS]
  uint64_t* v_free = bars + 3 * NS;        // [NS]
  uint64_t* s_full = bars + 4 * NS;        // [TG][2]
  uint64_t* p_full = s_full + 2 * TG;      // [TG]
  uint64_t* pv_done = p_full + TG;         // [TG]
  uint64_t* done = pv_done + TG;           // [1]
  u64t* bad_s = reinterpret_cast<u64t*>(done + 1);   // [3] keys with non-finite values: drafts, tiles c0, c0 + 1
  volatile int* tile_ok = reinterpret_cast<volatile int*>(bad_s + 3);   // [8]
  uint32_t& tmem_base_s = *reinterpret_cast<uint32_t*>(const_cast<int*>(tile_ok) + 8);
  volatile int& abort_s = const_cast<volatile int*>(tile_ok)[9];
  int& lo_max_s = const_cast<int*>(tile_ok)[10];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if ((reinterpret_cast<uintptr_t>(tt_smem) & 1023) != 0) {   // the tiles need the 1 KB alignment of their swizzle
    if (tid == 0) atomicExch(&g_tree_tc_expired, 8300009);
    return;
  }
  const int G = p.h_q / p.h_kv, R = p.n * G;
  const int rb = blockIdx.x % p.row_blocks, split = blockIdx.x / p.row_blocks, h = blockIdx.y, b = blockIdx.z;
  bool over;
  const int len = tree_length(p, b, over);
  const int parent = tree_parent(p.parents + (int64_t)b * p.n, p.n, tid);
  if (tid == 32 * kLoadWarp) {
    for (int s = 0; s < NS; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_free[s], 1);
      mbar_init(&v_full[s], 1);
      mbar_init(&v_free[s], 1);
    }
    for (int g = 0; g < TG; ++g) {
      mbar_init(&s_full[2 * g], 1);
      mbar_init(&s_full[2 * g + 1], 1);
      mbar_init(&p_full[g], 128);
      mbar_init(&pv_done[g], 1);
    }
    mbar_init(done, 1);
    mbar_init_fence();
    abort_s = *const_cast<volatile int*>(&g_tree_tc_expired) != 0;
    lo_max_s = 0;
    bad_s[0] = bad_s[1] = bad_s[2] = 0ull;
    if (over) atomicExch(&g_tree_tc_status, 8200002);
  }
  if (warp == kMmaWarp) tmem_alloc(&tmem_base_s, kTmem);
  const int lo_min = tree_low(p, len), c0 = lo_min >> 6, c1 = (len + 63) >> 6;
  const int nt = 1 + max(0, c1 - c0), per = (nt + p.splits - 1) / p.splits;
  const int t0 = split * per;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base_s, tS = tmem, tO = tmem + 128 * TG;       // S: 2 buffers of 64 columns a group, O: D columns a group
  const int nit = abort_s ? 0 : max(0, min(nt, t0 + per) - t0);
  __syncthreads();                                         // nobody has set abort_s on the way

  // ---- ancestors, rows, drafted keys (the scratch lies where P will be); the producer is already on its way ------------
  const int64_t new0 = (int64_t)b * p.n;
  const int row = rb * kRows + tid;
  const bool valid = tid < kRows && row < R;
  const int64_t out = valid ? (new0 + row / G) * p.h_q + h * G + row % G : 0;
  const bf16* kn = static_cast<const bf16*>(p.k_new) + (new0 * p.h_kv + h) * D;
  const bf16* vn = static_cast<const bf16*>(p.v_new) + (new0 * p.h_kv + h) * D;
  const int64_t nrs = (int64_t)p.h_kv * D;
  int lo = 0x7fffffff, lo_max = 0;
  u64t dmask = 0ull;
  if (warp != kLoadWarp) {
    constexpr int kMeet = kThreads - 32;
    int (*par)[kTreeMaxNodes] = reinterpret_cast<int (*)[kTreeMaxNodes]>(Ps);
    u64t (*anc)[kTreeMaxNodes] = reinterpret_cast<u64t (*)[kTreeMaxNodes]>(Ps + 1024);
    if (t0 == 0 && nit > 0) {
      for (int x = tid; x < 64 * (D / 8); x += kMeet) {
        const int r = x / (D / 8), c = x % (D / 8);
        uint4 kx = make_uint4(0u, 0u, 0u, 0u), vx = kx;
        if (r < p.n) {
          kx = *reinterpret_cast<const uint4*>(kn + r * nrs + c * 8);
          vx = *reinterpret_cast<const uint4*>(vn + r * nrs + c * 8);
          if (not_finite8(vx)) {                           // zero in the product, added row by row at the end
            atomicOr(&bad_s[0], 1ull << r);
            vx = make_uint4(0u, 0u, 0u, 0u);
          }
        }
        *reinterpret_cast<uint4*>(tile_at(Ks, r, c)) = kx;
        *reinterpret_cast<uint4*>(tile_at(Vs, r, c)) = vx;
      }
    }
    if (tid < kRows) load_row_to_tile<D>(Qs + (tid >> 7) * QB, tid & 127, static_cast<const bf16*>(p.q) + out * D, valid);
    tree_ancestors(parent, par, anc, tid, 2, kMeet);
    if (valid && anc[0][row / G] != 0ull) {
      lo = tree_low(p, len + __popcll(anc[0][row / G]) - 1);
      dmask = tree_draft_mask(p, anc[0], row / G, len, lo);
    }
    if (tid < p.n && anc[0][tid] != 0ull) atomicMax(&lo_max_s, tree_low(p, len + __popcll(anc[0][tid]) - 1));
    named_bar_sync(2, kMeet);
    if (t0 == 0 && nit > 0 && bad_s[0] != 0ull)            // the other pieces of those rows
      for (int x = tid; x < 64 * (D / 8); x += kMeet)
        if (bad_s[0] >> (x / (D / 8)) & 1ull) *reinterpret_cast<uint4*>(tile_at(Vs, x / (D / 8), x % (D / 8))) = make_uint4(0u, 0u, 0u, 0u);
    fence_async_smem();
    named_bar_sync(2, kMeet);
    lo_max = lo_max_s;
    if (t0 == 0 && nit > 0 && tid == 0) {                  // the drafted tile is there
      mbar_arrive(&k_full[0]);
      mbar_arrive(&v_full[0]);
    }
  }

  const float sl2 = p.scale * kLog2E;
  if (warp == kLoadWarp) {
    // ---- producer: K of a tile one step before its V, the order in which their places become free ---------------------
    const int first = c0 + max(t0, 1) - 1;                 // chunk of this CTA's first page tile
    int ids = 0, pg = 0, k_issued = 0, v_issued = 0;
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
    for (int step = 0; step <= nit; ++step) {
      const int prev = pg, c = c0 + t0 + step - 1;         // prev: page of tile step - 1, whose V is due
      if (step < nit) {
        if (t0 + step > 0) {
          if (((c - first) & 31) == 0) ids = c + lane < c1 ? p.pages[(int64_t)b * p.page_stride + c + lane] : -1;
          pg = __shfl_sync(0xffffffffu, ids, (c - first) & 31);
        } else {
          pg = 0;
        }
      }
      if (lane == 0) {
        if (step < nit) {
          const int s = step % NS;
          if (step >= NS) ok = wait_for(&k_free[s], (step / NS - 1) & 1);
          if (ok) {
            const bool in_pool = (unsigned)pg < (unsigned)p.num_pages;
            tile_ok[step & 7] = in_pool;                   // reaches the row threads through k_full and s_full; they are past step - 8
            if (!in_pool) atomicExch(&g_tree_tc_status, 8200001);
            bring(&k_full[s], Ks + s * TB, &tmK, t0 + step == 0, pg);
            ++k_issued;
          }
        }
        if (ok && step > 0) {
          const int it = step - 1, s = it % NS;
          if (it >= NS) ok = wait_for(&v_free[s], (it / NS - 1) & 1);
          if (ok) {
            bring(&v_full[s], Vs + s * TB, &tmV, t0 + it == 0, prev);
            ++v_issued;
          }
        }
      }
      ok = __shfl_sync(0xffffffffu, (int)ok, 0);
      if (!ok || abort_s) break;
    }
    if (lane == 0) {
      if (!ok) { abort_s = 1; atomicExch(&g_tree_tc_expired, 8300001); }
      for (int it = max(0, k_issued - NS); it < k_issued; ++it) wait_for(&k_full[it % NS], (it / NS) & 1);   // no copy outlives the CTA
      for (int it = max(0, v_issued - NS); it < v_issued; ++it) wait_for(&v_full[it % NS], (it / NS) & 1);
    }
  } else if (warp == kMmaWarp) {
    // ---- products -----------------------------------------------------------------------------------------------------
    // The whole warp runs the loop and one elected lane issues: descriptors then live in uniform registers, where the
    // instruction takes them from (issued from a lane's own branch, each of them is moved there first).
    if (nit > 0) {
      constexpr uint32_t idesc_qk = idesc_bf16(128, 64, 0);
      constexpr uint32_t idesc_pv = idesc_bf16(128, D, 1);
      const uint64_t q_d = desc_sw128(smem_u32(Qs), 16, 1024), k_d = desc_sw128(smem_u32(Ks), 16, 1024),
                     p_d = desc_sw128(smem_u32(Ps), 16, 1024), v_d = desc_sw128(smem_u32(Vs), 8192, 1024);
      auto issue_qk = [&](int it) {
        if (elect_one()) {
          const uint64_t kb = k_d + (it % NS) * (TB >> 4);
#pragma unroll
          for (int g = 0; g < TG; ++g) {
            const uint64_t qa = q_d + g * (QB >> 4);
            const uint32_t ts = tS + g * 128 + (it & 1) * 64;
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk)
              mma_ss(ts, qa + (((kk >> 2) * 16384 + (kk & 3) * 32) >> 4), kb + (((kk >> 2) * 8192 + (kk & 3) * 32) >> 4), idesc_qk, kk > 0);
            mma_commit(&s_full[2 * g + (it & 1)]);
          }
          mma_commit(&k_free[it % NS]);
        }
        __syncwarp();
      };
      bool ok = wait_for(&k_full[0], 0);
      ok = __all_sync(0xffffffffu, ok);
      if (ok) {
        tc_fence_after();
        issue_qk(0);
      }
      for (int it = 0; ok && it < nit; ++it) {
        if (__any_sync(0xffffffffu, abort_s)) break;
        if (it + 1 < nit) {                                // its S buffers were consumed before the arrivals on p_full of it - 1
          ok = __all_sync(0xffffffffu, wait_for(&k_full[(it + 1) % NS], ((it + 1) / NS) & 1));
          if (!ok) break;
          tc_fence_after();
          issue_qk(it + 1);
        }
        ok = __all_sync(0xffffffffu, wait_for(&v_full[it % NS], (it / NS) & 1));
        if (!ok) break;
        const uint64_t b0 = v_d + (it % NS) * (TB >> 4);
#pragma unroll
        for (int g = 0; g < TG; ++g) {
          ok = ok && __all_sync(0xffffffffu, wait_for(&p_full[g], it & 1));
          if (ok) {
            tc_fence_after();
            if (elect_one()) {
              const uint64_t pa = p_d + g * (16384 >> 4);
#pragma unroll
              for (int kk = 0; kk < 4; ++kk)
                mma_ss(tO + g * D, pa + ((kk * 32) >> 4), b0 + ((kk * 2048) >> 4), idesc_pv, it > 0 || kk > 0);
              mma_commit(&pv_done[g]);
              if (g == TG - 1) mma_commit(&v_free[it % NS]);
            }
            __syncwarp();
          }
        }
        if (!ok) break;
      }
      if (!ok && lane == 0) { abort_s = 1; atomicExch(&g_tree_tc_expired, 8300002); }
      if (elect_one()) mma_commit(done);                   // no product outlives the CTA's tensor memory
      wait_for(done, 0);
    }
  } else {
    // ---- rows -----------------------------------------------------------------------------------------------------------
    const int grp = tid >> 7, r = tid & 127;
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16, tSg = tS + grp * 128 + lane_base, tOg = tO + grp * D + lane_base;
    uint8_t* Pg = Ps + grp * 16384;
    const bool rows_here = rb * kRows + warp * 32 < R;
    float m = -CUDART_INF_F, l = 0.f;                      // reference point (log2 units) and sum
    bool ok = true;
    for (int it = 0; it < nit; ++it) {
      const int s = it & 1, t = t0 + it, c = c0 + t - 1, vs = it % NS;
      ok = wait_for(&s_full[2 * grp + s], (it >> 1) & 1);
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
      float grow = 1.f;
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
        if (top > m + kTtSlack) {                          // also the first visible key: m is -inf
          moved = m > -CUDART_INF_F;
          grow = moved ? ex2(m - top) : 0.f;
          m = top;
          l *= grow;
        }
        const float ref = m > -CUDART_INF_F ? m : 0.f;
        float s4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < 64; ++j) {
          sv[j] = ex2(fmaf(sv[j], sl2, -ref));             // -inf gives 0
          s4[j & 3] += sv[j];
        }
        l += (s4[0] + s4[1]) + (s4[2] + s4[3]);
      }
      if (it > 0) ok = wait_for(&pv_done[grp], (it - 1) & 1) && ok;     // P is free, O stands still
      ok = __all_sync(0xffffffffu, ok) && !abort_s;
      if (!ok) break;
      if (rows_here) {
        if (it > 0 && __any_sync(0xffffffffu, moved)) {
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
          tmem_st_wait();
        }
        store_row_bf16_sw128(Pg, r, sv);
      }
      // V rows of this page that nobody sees become zeros (one warp, a row at a time), and so do those that some rows see
      // and others do not and that are not finite
      if (t > 0 && warp < 2) {
        const u64t held = in_pool ? tree_page_mask(p, c, len, lo_min) : 0ull;
        uint8_t* tile = Vs + vs * TB;
        if (warp == 0 && held != ~0ull) {
          ok = wait_for(&v_full[vs], (it / NS) & 1);
          for (u64t rest = ~held; rest; rest &= rest - 1)
            if (lane < D / 8) *reinterpret_cast<uint4*>(tile_at(tile, __ffsll((long long)rest) - 1, lane)) = make_uint4(0u, 0u, 0u, 0u);
        }
        if (lo_max > c * 64 && c - c0 < 2 && (held >> tid & 1ull)) {
          ok = wait_for(&v_full[vs], (it / NS) & 1) && ok;
          bool clear = false;
#pragma unroll
          for (int e = 0; e < D / 8; ++e) clear = clear || not_finite8(*reinterpret_cast<const uint4*>(tile_at(tile, tid, e)));
          if (clear) {
            atomicOr(&bad_s[1 + c - c0], 1ull << tid);
#pragma unroll
            for (int e = 0; e < D / 8; ++e) *reinterpret_cast<uint4*>(tile_at(tile, tid, e)) = make_uint4(0u, 0u, 0u, 0u);
          }
        }
      }
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      fence_async_smem();
      tc_fence_before();
      mbar_arrive(&p_full[grp]);
    }
    if (ok && nit > 0) ok = __all_sync(0xffffffffu, wait_for(&pv_done[grp], (nit - 1) & 1)) && !abort_s;
    if (!ok && lane == 0) {
      abort_s = 1;
      atomicExch(&g_tree_tc_expired, 8300003);
    }
    if (ok) tc_fence_after();
    named_bar_sync(1, kRows);                              // bad_s of all row threads
    const bool have = ok && nit > 0 && rows_here;
    const float inv = p.splits > 1 ? 1.f : (l > 0.f ? 1.f / l : (l == l ? 0.f : l));
    const int64_t at = (int64_t)split * p.B * p.n * p.h_q + out;
#pragma unroll 1
    for (int cb = 0; cb < D / 32; ++cb) {
      float ov[32];
      if (have) {
        tmem_ld32(tOg + cb * 32, ov);
        tmem_ld_wait32(ov);
      } else {
#pragma unroll
        for (int j = 0; j < 32; ++j) ov[j] = 0.f;
      }
      if (have && valid && (bad_s[0] | bad_s[1] | bad_s[2]))
        add_bad_keys<D>(p, bad_s, b, h, out, kn, vn, nrs, c0, len, lo, dmask, sl2, m > -CUDART_INF_F ? m : 0.f, cb, ov);
#pragma unroll
      for (int j = 0; j < 32; ++j) ov[j] *= inv;
      if (valid) {
        if (p.splits > 1) {
          float* po = p.part_o + at * D + cb * 32;
#pragma unroll
          for (int j = 0; j < 32; j += 4) store4(po + j, make_float4(ov[j], ov[j + 1], ov[j + 2], ov[j + 3]));
        } else {
          store32_bf16(static_cast<bf16*>(p.o) + out * D + cb * 32, ov);
        }
      }
    }
    if (valid) {
      if (p.splits > 1) {
        *reinterpret_cast<float2*>(p.part_ml + 2 * at) = make_float2(m, have ? l : 0.f);
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

template <int D, int TG>
static int launch_tree_tc(const TreeParams& p, cudaStream_t st) {
  CUtensorMap tmK, tmV;
  const uint64_t rows = (uint64_t)p.num_pages * p.h_kv * 64;
  if (int rc = make_tmap_bf16_rows(&tmK, p.k_pages, rows, D, D, 64)) return rc;
  if (int rc = make_tmap_bf16_rows(&tmV, p.v_pages, rows, D, D, 64)) return rc;
  using Sh = TtShape<D, TG>;
  cudaFuncSetAttribute(tree_attn_tc_kernel<D, TG>, cudaFuncAttributeMaxDynamicSharedMemorySize, Sh::SMEM);
  tree_attn_tc_kernel<D, TG><<<dim3((unsigned)(p.row_blocks * p.splits), (unsigned)p.h_kv, (unsigned)p.B), Sh::THREADS, Sh::SMEM, st>>>(p, tmK, tmV);
  HILS_LAUNCH_CHECK("tree_attn_paged (tensor-core path)");
  return HILS_OK;
}

// rows_per_cta: 128 or 256
int tree_tc_launch(const TreeParams& p, int D, int rows_per_cta, cudaStream_t st) {
  if (rows_per_cta == 256) return D == 128 ? launch_tree_tc<128, 2>(p, st) : launch_tree_tc<64, 2>(p, st);
  return D == 128 ? launch_tree_tc<128, 1>(p, st) : launch_tree_tc<64, 1>(p, st);
}

}  // namespace hils
