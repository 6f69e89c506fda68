// Attention of a tree of drafted tokens over the paged store for few rows per key head (at most 32), bf16: warp-level tensor
// instructions, tiles by TMA.
//
// With 16 rows a 128-row tile of the tensor memory is 7/8 padding and the work is streaming K and V.  A CTA (one key head of one
// sequence, a share of its tiles) is four warps over a ring of shared-memory places; the first warp also sends for the tiles, a
// place ahead (a fifth warp for that would leave 168 registers a thread instead of 255, and 32 rows would spill); two CTAs per
// SM keep about 130 KB on their way.  Warp w takes keys 16w .. 16w+15 of every tile for all rows, with a running
// maximum, sum and output of its own (registers), so the warps never wait for one another; they are joined once, at the end.
// Masks as in tree_common.cuh.  V of keys nobody sees is masked out of the operand registers (0 * NaN would spoil the row);
// a key that some rows see and others do not is masked out as well when it is not finite and added row by row.
#include <algorithm>

#include "tree_common.cuh"
#include "umma.cuh"

namespace hils {

// A page outside the pool (8200001), a length past the table (8200002)
static __device__ int g_tree_mma_status = 0;
// A wait that ran out (8400001 ..); CTAs that start later see it and write nothing but zeros
static __device__ int g_tree_mma_expired = 0;

using namespace umma;

constexpr int kTmWarps = 4, kTmThreads = 32 * kTmWarps;
constexpr float kTmSlack = 8.f;              // log2 units a row's maximum may grow before its sums are rescaled

// MT: 16-row fragments
template <int D, int MT> struct TmShape {
  static constexpr int DB = D / 64, TB = DB * 8192, NS = D == 128 ? 3 : 6, QB = MT * 16 * D * 2;
  static constexpr int RING = 2 * NS * TB, Q = RING, BARS = Q + QB, SCRATCH = BARS + 256, SMEM = SCRATCH + 1536;
  static_assert(kTmWarps * MT * 16 * (D + 4) * 4 <= RING, "the warps' outputs are joined where the tiles were");
};

__device__ __forceinline__ bool tm_wait(uint64_t* b, uint32_t parity) { return mbar_wait<1 << 20>(b, parity); }

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// byte offset of (row, 16-byte piece c) in a tile of column blocks of `rows` rows x 128 bytes with the 128-byte swizzle
__device__ __forceinline__ uint32_t tm_off(int rows, int r, int c) { return (c >> 3) * rows * 128 + sw128_off(r, c & 7); }

__device__ __forceinline__ bool bad8(uint4 x) {            // eight bf16: an exponent of all ones
  bool bad = false;
#pragma unroll
  for (const uint32_t w : {x.x, x.y, x.z, x.w}) bad = bad || (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u;
  return bad;
}

template <int D, int MT>
__global__ void __launch_bounds__(kTmThreads, 2) tree_attn_mma_kernel(const __grid_constant__ TreeParams p, const __grid_constant__ CUtensorMap tmK,
                                                                      const __grid_constant__ CUtensorMap tmV) {
  using Sh = TmShape<D, MT>;
  constexpr int NS = Sh::NS, DB = Sh::DB, TB = Sh::TB, CP = D / 8, NT = D / 8;      // CP: 16-byte pieces of a row; NT: output fragments
  extern __shared__ uint8_t tm_smem[];
  uint8_t* Ks = tm_smem;
  uint8_t* Vs = Ks + NS * TB;
  uint8_t* Qs = tm_smem + Sh::Q;
  uint64_t* full = reinterpret_cast<uint64_t*>(tm_smem + Sh::BARS);   // [NS]
  uint64_t* freed = full + NS;                                        // [NS]
  volatile int* tile_ok = reinterpret_cast<volatile int*>(freed + NS);   // [NS]
  volatile int& abort_s = const_cast<volatile int*>(tile_ok)[NS];
  int& lo_max_s = const_cast<int*>(tile_ok)[NS + 1];
  int (*par)[kTreeMaxNodes] = reinterpret_cast<int (*)[kTreeMaxNodes]>(tm_smem + Sh::SCRATCH);
  u64t (*anc)[kTreeMaxNodes] = reinterpret_cast<u64t (*)[kTreeMaxNodes]>(tm_smem + Sh::SCRATCH + 512);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if ((reinterpret_cast<uintptr_t>(tm_smem) & 1023) != 0) {           // the tiles need the 1 KB alignment of their swizzle
    if (tid == 0) atomicExch(&g_tree_mma_expired, 8400009);
    return;
  }
  const int G = p.h_q / p.h_kv, R = p.n * G, split = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  if (tid == 0) {
    for (int s = 0; s < NS; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&freed[s], kTmWarps);
    }
    mbar_init_fence();
    abort_s = *const_cast<volatile int*>(&g_tree_mma_expired) != 0;
    lo_max_s = 0;
  }
  bool over;
  const int len = tree_length(p, b, over);
  if (over && tid == 0) atomicExch(&g_tree_mma_status, 8200002);
  const int lo_min = tree_low(p, len), c0 = lo_min >> 6, c1 = (len + 63) >> 6;
  const int nt = 1 + max(0, c1 - c0), per = (nt + p.splits - 1) / p.splits;
  const int t0 = split * per;
  int nit = max(0, min(nt, t0 + per) - t0);
  const int64_t new0 = (int64_t)b * p.n;
  const bf16* kn = static_cast<const bf16*>(p.k_new) + (new0 * p.h_kv + h) * D;
  const bf16* vn = static_cast<const bf16*>(p.v_new) + (new0 * p.h_kv + h) * D;
  const int64_t nrs = (int64_t)p.h_kv * D;

  // ---- queries, drafted keys, ancestors ------------------------------------------------------------------------------
  for (int x = tid; x < MT * 16 * CP; x += kTmThreads) {
    const int r = x / CP, c = x % CP;
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    if (r < R) v = *reinterpret_cast<const uint4*>(static_cast<const bf16*>(p.q) + ((new0 + r / G) * p.h_q + h * G + r % G) * D + c * 8);
    *reinterpret_cast<uint4*>(Qs + tm_off(MT * 16, r, c)) = v;
  }
  if (t0 == 0 && nit > 0)
    for (int x = tid; x < 64 * CP; x += kTmThreads) {
      const int r = x / CP, c = x % CP;
      uint4 kx = make_uint4(0u, 0u, 0u, 0u), vx = kx;
      if (r < p.n) {
        kx = *reinterpret_cast<const uint4*>(kn + r * nrs + c * 8);
        vx = *reinterpret_cast<const uint4*>(vn + r * nrs + c * 8);
      }
      *reinterpret_cast<uint4*>(Ks + tm_off(64, r, c)) = kx;
      *reinterpret_cast<uint4*>(Vs + tm_off(64, r, c)) = vx;
    }
  tree_ancestors(tree_parent(p.parents + new0, p.n, tid), par, anc, tid, 0, kTmThreads);
  if (tid < p.n && anc[0][tid] != 0ull) atomicMax(&lo_max_s, tree_low(p, len + __popcll(anc[0][tid]) - 1));
  fence_async_smem();
  __syncthreads();
  const int lo_max = lo_max_s;
  if (abort_s) nit = 0;
  __syncthreads();                                         // nobody has set it on the way

  // ---- the four computing warps ------------------------------------------------------------------------------------------
  const int qr = lane >> 2, qj = lane & 3;                 // fragment row and column pair of this thread
  const float sl2 = p.scale * kLog2E;
  // this thread's rows: mt * 16 + qr and + 8
  u64t dmask[MT][2];
  int lo[MT][2];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int row = mt * 16 + qr + 8 * i, j = row / G;
      dmask[mt][i] = 0ull;
      lo[mt][i] = 0x7fffffff;
      if (row < R && anc[0][j] != 0ull) {
        lo[mt][i] = tree_low(p, len + __popcll(anc[0][j]) - 1);
        dmask[mt][i] = tree_draft_mask(p, anc[0], j, len, lo[mt][i]);
      }
    }
  float o[MT][NT][4], m[MT][2], l[MT][2];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
    for (int i = 0; i < 2; ++i) { m[mt][i] = -CUDART_INF_F; l[mt][i] = 0.f; }
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[mt][t][e] = 0.f;
  }
  const uint32_t q32 = smem_u32(Qs), k32 = smem_u32(Ks), v32 = smem_u32(Vs);
  const int lrow = lane & 15, lcol = lane >> 4;            // ldmatrix: the row this lane points at, and which 16-byte piece
  const int krow = warp * 16 + (lane & 7) + ((lane >> 4) & 1) * 8, kcol = (lane >> 3) & 1;
  const int vrow = warp * 16 + (lane & 15), vcol = lane >> 4;
  // the first warp sends for tile `it` once the tile before it in its place is done with
  const int first = c0 + max(t0, 1) - 1;
  int ids = 0, issued = 0;
  auto bring = [&](int it) {
    const int s = it % NS, c = c0 + t0 + it - 1;
    const bool draft = t0 + it == 0;
    int pg = 0;
    bool got = true;
    if (!draft) {
      if (((c - first) & 31) == 0) ids = c + lane < c1 ? p.pages[(int64_t)b * p.page_stride + c + lane] : -1;
      pg = __shfl_sync(0xffffffffu, ids, (c - first) & 31);
    }
    if (it >= NS) got = tm_wait(&freed[s], (it / NS - 1) & 1);
    if (!__all_sync(0xffffffffu, got)) return false;
    if (lane == 0) {
      const bool in_pool = (unsigned)pg < (unsigned)p.num_pages;
      tile_ok[s] = in_pool;
      if (!in_pool) atomicExch(&g_tree_mma_status, 8200001);
      if (draft || !in_pool) {
        mbar_arrive(&full[s]);
      } else {
        mbar_expect_tx(&full[s], 2 * TB);
#pragma unroll
        for (int db = 0; db < DB; ++db) {
          tma_load_2d(Ks + s * TB + db * 8192, &tmK, &full[s], db * 64, (pg * p.h_kv + h) * 64);
          tma_load_2d(Vs + s * TB + db * 8192, &tmV, &full[s], db * 64, (pg * p.h_kv + h) * 64);
        }
      }
    }
    ++issued;
    return true;
  };
  bool ok = true;
  if (warp == 0)
    for (int it = 0; it < min(NS - 1, nit); ++it) bring(it);
  for (int it = 0; it < nit; ++it) {
    const int s = it % NS, t = t0 + it, c = c0 + t - 1;
    if (warp == 0 && it + NS - 1 < nit) ok = bring(it + NS - 1);
    if (!ok) break;
    ok = tm_wait(&full[s], (it / NS) & 1);
    ok = __all_sync(0xffffffffu, ok && !abort_s);
    if (!ok) break;
    const bool in_pool = tile_ok[s] != 0;
    // this warp's sixteen keys: which anybody sees, which each row sees
    uint32_t held = (uint32_t)((t == 0 ? (p.n >= 64 ? ~0ull : (1ull << p.n) - 1) : (in_pool ? tree_page_mask(p, c, len, lo_min) : 0ull)) >> (16 * warp)) & 0xffffu;
    if (held != 0u) {
      const uint32_t kt = k32 + s * TB, vt = v32 + s * TB;
      float sc[MT][2][4];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[mt][x][e] = 0.f;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        uint32_t kb[4];
        ldsm4(kt + tm_off(64, krow, kk * 2 + kcol), kb);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          uint32_t qa[4];
          ldsm4(q32 + tm_off(MT * 16, mt * 16 + lrow, kk * 2 + lcol), qa);
          mma16816(sc[mt][0], qa, kb[0], kb[1]);
          mma16816(sc[mt][1], qa, kb[2], kb[3]);
        }
      }
      uint32_t pa[MT][4];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        float grow[2];
        bool moved = false;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t vis = (uint32_t)((t == 0 ? dmask[mt][i] : tree_page_mask(p, c, len, lo[mt][i])) >> (16 * warp)) & held;
          float y[4];                                      // keys 2 qj, 2 qj + 1, 2 qj + 8, 2 qj + 9
          float top = -CUDART_INF_F;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            y[e] = (vis >> (2 * qj + (e & 1) + 8 * (e >> 1)) & 1u) ? sc[mt][e >> 1][2 * i + (e & 1)] : -CUDART_INF_F;
            top = fmaxf(top, y[e]);
          }
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2)) * sl2;
          grow[i] = 1.f;
          if (top > m[mt][i] + kTmSlack) {                 // also the first visible key: m is -inf, the sums are zero
            grow[i] = ex2(m[mt][i] - top);
            m[mt][i] = top;
            l[mt][i] *= grow[i];
            moved = true;
          }
          const float ref = m[mt][i] > -CUDART_INF_F ? m[mt][i] : 0.f;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float w = ex2(fmaf(y[e], sl2, -ref));    // -inf gives 0
            sc[mt][e >> 1][2 * i + (e & 1)] = w;
            l[mt][i] += w;
          }
        }
        if (__any_sync(0xffffffffu, moved))
#pragma unroll
          for (int x = 0; x < NT; ++x) {
            o[mt][x][0] *= grow[0]; o[mt][x][1] *= grow[0];
            o[mt][x][2] *= grow[1]; o[mt][x][3] *= grow[1];
          }
        pa[mt][0] = pack2(sc[mt][0][0], sc[mt][0][1]);
        pa[mt][1] = pack2(sc[mt][0][2], sc[mt][0][3]);
        pa[mt][2] = pack2(sc[mt][1][0], sc[mt][1][1]);
        pa[mt][3] = pack2(sc[mt][1][2], sc[mt][1][3]);
      }
      if (t == 0 || lo_max > c * 64) {                     // some rows see keys that others do not
        uint32_t bad = 0u;
        for (int x = lane; x < 16 * CP; x += 32)
          if (bad8(*reinterpret_cast<const uint4*>(Vs + s * TB + tm_off(64, warp * 16 + x / CP, x % CP)))) bad |= 1u << (x / CP);
        bad = __reduce_or_sync(0xffffffffu, bad) & held;
        held &= ~bad;
        for (; bad; bad &= bad - 1) {                      // rare: the row's weight times the key's values, where the row sees the key
          const int key = __ffs(bad) - 1, src = (lane & ~3) | ((key & 7) >> 1);
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const float w0 = (key & 8) ? sc[mt][1][2 * i] : sc[mt][0][2 * i], w1 = (key & 8) ? sc[mt][1][2 * i + 1] : sc[mt][0][2 * i + 1];
              const float w = __shfl_sync(0xffffffffu, (key & 1) ? w1 : w0, src);
              const u64t vis = t == 0 ? dmask[mt][i] : tree_page_mask(p, c, len, lo[mt][i]);
              if (vis >> (16 * warp + key) & 1ull)
#pragma unroll
                for (int x = 0; x < NT; ++x) {
                  const float2 v = load2(reinterpret_cast<const bf16*>(Vs + s * TB + tm_off(64, warp * 16 + key, x)) + 2 * qj);
                  o[mt][x][2 * i] = fmaf(w, v.x, o[mt][x][2 * i]);
                  o[mt][x][2 * i + 1] = fmaf(w, v.y, o[mt][x][2 * i + 1]);
                }
            }
        }
      }
      const uint32_t f0 = held >> (2 * qj), f1 = held >> (2 * qj + 8);
      const uint32_t mask0 = ((f0 & 1u) ? 0xffffu : 0u) | ((f0 & 2u) ? 0xffff0000u : 0u), mask1 = ((f1 & 1u) ? 0xffffu : 0u) | ((f1 & 2u) ? 0xffff0000u : 0u);
#pragma unroll
      for (int x = 0; x < NT; x += 2) {
        uint32_t vb[4];
        ldsm4t(vt + tm_off(64, vrow, x + vcol), vb);
        vb[0] &= mask0; vb[1] &= mask1; vb[2] &= mask0; vb[3] &= mask1;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          mma16816(o[mt][x], pa[mt], vb[0], vb[1]);
          mma16816(o[mt][x + 1], pa[mt], vb[2], vb[3]);
        }
      }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&freed[s]);
  }
  if (!ok && lane == 0) {
    abort_s = 1;
    atomicExch(&g_tree_mma_expired, 8400001);
  }
  if (warp == 0 && !ok)
    for (int it = max(0, issued - NS); it < issued; ++it) tm_wait(&full[it % NS], (it / NS) & 1);   // no copy outlives the CTA
  // the sums of a row: over the four lanes that share it
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      l[mt][i] += __shfl_xor_sync(0xffffffffu, l[mt][i], 1);
      l[mt][i] += __shfl_xor_sync(0xffffffffu, l[mt][i], 2);
    }
  __syncthreads();                                         // the ring is free: every tile was waited for
  // ---- join the warps ------------------------------------------------------------------------------------------------------
  constexpr int OS = D + 4;
  float* osm = reinterpret_cast<float*>(tm_smem);          // [warps][MT * 16][OS]
  float* ml = reinterpret_cast<float*>(tm_smem + Sh::SCRATCH);   // [warps][MT * 16][2]: 1 KB at most
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int row = mt * 16 + qr + 8 * i;
#pragma unroll
      for (int x = 0; x < NT; ++x)
        *reinterpret_cast<float2*>(osm + (warp * MT * 16 + row) * OS + x * 8 + 2 * qj) = make_float2(o[mt][x][2 * i], o[mt][x][2 * i + 1]);
      if (qj == 0) *reinterpret_cast<float2*>(ml + (warp * MT * 16 + row) * 2) = make_float2(m[mt][i], l[mt][i]);
    }
  __syncthreads();
  for (int x = tid; x < R * (D / 4); x += 32 * kTmWarps) {
    const int row = x / (D / 4), d = (x % (D / 4)) * 4;
    float2 w[kTmWarps];
    float top = -CUDART_INF_F;
#pragma unroll
    for (int k = 0; k < kTmWarps; ++k) {
      w[k] = *reinterpret_cast<const float2*>(ml + (k * MT * 16 + row) * 2);
      top = fmaxf(top, w[k].x);
    }
    const float ref = top > -CUDART_INF_F ? top : 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < kTmWarps; ++k) {
      if (w[k].y == 0.f) continue;                         // nothing visible among this warp's keys
      const float f = w[k].x > -CUDART_INF_F ? ex2(w[k].x - ref) : 1.f;     // -inf with a sum: NaN scores, kept
      const float4 y = *reinterpret_cast<const float4*>(osm + (k * MT * 16 + row) * OS + d);
      sum = fmaf(f, w[k].y, sum);
      acc.x = fmaf(f, y.x, acc.x); acc.y = fmaf(f, y.y, acc.y); acc.z = fmaf(f, y.z, acc.z); acc.w = fmaf(f, y.w, acc.w);
    }
    const int64_t out = (new0 + row / G) * p.h_q + h * G + row % G;
    if (p.splits > 1) {
      const int64_t at = (int64_t)split * p.B * p.n * p.h_q + out;
      store4(p.part_o + at * D + d, acc);
      if (d == 0) *reinterpret_cast<float2*>(p.part_ml + 2 * at) = make_float2(top, ok ? sum : 0.f);
    } else {
      const float inv = sum > 0.f ? 1.f / sum : (sum == sum ? 0.f : sum);
      store4(static_cast<bf16*>(p.o) + out * D + d, make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv));
      if (d == 0) {
        const float lse = sum > 0.f ? (ref + log2f(sum)) * kLn2F : (sum == sum ? -CUDART_INF_F : sum);
        p.lse[out] = lse;
        if (p.lse_act) static_cast<bf16*>(p.lse_act)[out] = __float2bfloat16_rn(lse);
      }
    }
  }
}

int take_status_tree_mma() {
  int v = 0, x = 0, zero = 0;
  if (cudaDeviceSynchronize() != cudaSuccess) return -1;
  if (cudaMemcpyFromSymbol(&v, g_tree_mma_status, sizeof(int)) != cudaSuccess) return -1;
  if (cudaMemcpyFromSymbol(&x, g_tree_mma_expired, sizeof(int)) != cudaSuccess) return -1;
  if (v != 0) cudaMemcpyToSymbol(g_tree_mma_status, &zero, sizeof(int));
  if (x != 0) cudaMemcpyToSymbol(g_tree_mma_expired, &zero, sizeof(int));
  return x != 0 ? x : v;
}

template <int D, int MT>
static int launch_tree_mma(const TreeParams& p, cudaStream_t st) {
  CUtensorMap tmK, tmV;
  const uint64_t rows = (uint64_t)p.num_pages * p.h_kv * 64;
  if (int rc = make_tmap_bf16_rows(&tmK, p.k_pages, rows, D, D, 64)) return rc;
  if (int rc = make_tmap_bf16_rows(&tmV, p.v_pages, rows, D, D, 64)) return rc;
  constexpr int smem = TmShape<D, MT>::SMEM;
  cudaFuncSetAttribute(tree_attn_mma_kernel<D, MT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  tree_attn_mma_kernel<D, MT><<<dim3((unsigned)p.splits, (unsigned)p.h_kv, (unsigned)p.B), kTmThreads, smem, st>>>(p, tmK, tmV);
  HILS_LAUNCH_CHECK("tree_attn_paged (few rows)");
  return HILS_OK;
}

// rows of one key head: 16 or 32 at most
int tree_mma_launch(const TreeParams& p, int D, int rows, cudaStream_t st) {
  if (rows <= 16) return D == 128 ? launch_tree_mma<128, 1>(p, st) : launch_tree_mma<64, 1>(p, st);
  return D == 128 ? launch_tree_mma<128, 2>(p, st) : launch_tree_mma<64, 2>(p, st);
}

}  // namespace hils
