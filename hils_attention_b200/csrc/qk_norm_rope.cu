// Norm of queries and keys per head and the rotation of their positions, one pass over both tensors, forward and backward.
//
//   y = w * x * rsqrt(mean(x^2) + eps)            (w = NULL: y = x)
//   pair (a, b) of y at angle t = position * inv_freq[i], s = scaling:   a' = s (a cos t - b sin t), b' = s (b cos t + a sin t)
//
// The pairs are (i, i + rot/2) or, interleaved, (2i, 2i + 1) for i < rot/2; elements from rot on are not rotated.  All
// arithmetic is fp32, one rounding at the end.  Backward: dy = R(-t) dout, dx = rstd (w dy - x rstd^2 mean(w dy x)),
// dw = sum over rows of dy x rstd.
//
// Angles.  A position of a million times an angle per position in fp32 is off by a tenth of a radian.  The angle is kept in
// turns as a 64-bit fixed-point fraction instead: frac(inv_freq / 2 pi) * 2^64, formed once per CTA in fp64; its product
// with the position modulo 2^64 IS the fraction of a turn (the whole turns fall off the top), good to position * 2^-53
// turns, for the price of one integer multiplication.  So no cos/sin table is read, whatever the positions.
//
// Layout.  2V elements of a row (V pairs) are one unit, a lane owns one unit and a group of lanes (the next power of two of
// the units) one row, so the row's sums are a few shuffles and a group reads and writes whole rows with 16-byte accesses.
// A group forms the cos/sin of its token once and walks `hpg` heads with it, kHeads rows in flight.
#include <algorithm>

#include "common.cuh"

namespace hils {

constexpr int kQkThreads = 256;
constexpr int kQkMaxD = 256;
constexpr double kInvTwoPi = 0.15915494309189533577;

struct QkSide {
  const void* x; const void* w; void* out; const void* g; float* dw;   // dw: partial sums, one row of D per CTA
  int64_t xb, xl, xh, gb, gl, gh;
  int H, hpg, hsplit, cta0, ctas;
};

struct QkParams {
  QkSide side[2];
  const void* pos; const double* inv_freq;
  int64_t pos_b, pos_l;
  int B, L, D, rot, lpr, n_sides, pos64, w_f32;
  float eps, scaling;
};

template <typename T, int V>
__device__ __forceinline__ void load_v(const T* p, float (&f)[V]) {
  if constexpr (V == 1) {
    f[0] = to_f(*p);
  } else if constexpr (sizeof(T) == 2 && V == 8) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  } else {
    static_assert(V == 4, "a unit half is 1, 4 or (bf16) 8 elements");
    const float4 v = load4(p);
    f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
  }
}

template <typename T, int V>
__device__ __forceinline__ void store_v(T* p, const float (&f)[V]) {
  if constexpr (V == 1) {
    *p = from_f<T>(f[0]);
  } else if constexpr (sizeof(T) == 2 && V == 8) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
    store4(p, make_float4(f[0], f[1], f[2], f[3]));
  }
}

// where the two halves of unit u start
template <int V, bool INTER>
__device__ __forceinline__ void unit_at(const QkParams& p, int u, int& o1, int& o2) {
  const int ru = p.rot / (2 * V);
  if (INTER || u >= ru) {
    o1 = u * 2 * V;
    o2 = o1 + V;
  } else {
    o1 = u * V;
    o2 = (p.rot >> 1) + u * V;
  }
}

// rotate the V pairs of a unit held as its two halves (in memory order)
template <int V, bool INTER, bool BACK>
__device__ __forceinline__ void rotate(float (&e1)[V], float (&e2)[V], const float (&cs)[V], const float (&sn)[V]) {
#pragma unroll
  for (int j = 0; j < V; ++j) {
    float* a;
    float* b;
    if constexpr (INTER && V > 1) {
      float* e = (2 * j < V) ? e1 : e2;
      a = e + (2 * j) % V;
      b = e + (2 * j + 1) % V;
    } else {
      a = e1 + j;
      b = e2 + j;
    }
    const float x = *a, y = *b, s = BACK ? -sn[j] : sn[j];
    *a = x * cs[j] - y * s;
    *b = y * cs[j] + x * s;
  }
}

__device__ __forceinline__ float weight_at(const QkParams& p, const void* w, int d) {
  return p.w_f32 ? static_cast<const float*>(w)[d] : to_f(static_cast<const bf16*>(w)[d]);
}

template <typename T, int V, int UPL, bool INTER, bool BWD>
__global__ void __launch_bounds__(kQkThreads) qk_norm_rope_kernel(const __grid_constant__ QkParams p) {
  constexpr int kHeads = UPL > 1 ? 1 : (BWD ? 2 : 4);          // rows in flight per lane
  __shared__ unsigned long long turn_s[kQkMaxD / 2];
  __shared__ float dw_s[BWD ? kQkThreads / 32 : 1][BWD ? kQkMaxD : 1];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int si = (p.n_sides > 1 && (int)blockIdx.x >= p.side[1].cta0) ? 1 : 0;
  const QkSide& sd = p.side[si];
  for (int i = tid; i < (p.rot >> 1); i += kQkThreads) {
    const double t = p.inv_freq[i] * kInvTwoPi;
    turn_s[i] = (unsigned long long)((t - floor(t)) * 18446744073709551616.0);
  }
  __syncthreads();
  const int lpr = p.lpr, sub = lane & (lpr - 1), gpw = 32 / lpr;   // groups per warp
  const int units = p.D / (2 * V), ru = p.rot / (2 * V);
  int o1[UPL], o2[UPL];
  bool has[UPL];
  float w1[UPL][V], w2[UPL][V], dw1[UPL][V], dw2[UPL][V];
#pragma unroll
  for (int i = 0; i < UPL; ++i) {
    const int u = sub + i * 32;
    has[i] = u < units;
    unit_at<V, INTER>(p, has[i] ? u : 0, o1[i], o2[i]);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      w1[i][j] = sd.w ? weight_at(p, sd.w, o1[i] + j) : 1.f;
      w2[i][j] = sd.w ? weight_at(p, sd.w, o2[i] + j) : 1.f;
      dw1[i][j] = dw2[i][j] = 0.f;
    }
  }
  const int64_t items = (int64_t)p.B * p.L * sd.hsplit;
  const int64_t step = (int64_t)sd.ctas * (kQkThreads / 32) * gpw;
  const float inv_d = 1.f / (float)p.D;
  for (int64_t it0 = ((int64_t)(blockIdx.x - sd.cta0) * (kQkThreads / 32) + warp) * gpw; it0 < items; it0 += step) {
    const int64_t it = it0 + lane / lpr;
    const bool live = it < items;
    const int64_t tok = (live ? it : 0) / sd.hsplit;
    const int h0 = (int)((live ? it : 0) - tok * sd.hsplit) * sd.hpg, h1 = live ? min(sd.H, h0 + sd.hpg) : h0;
    const int64_t b = tok / p.L, l = tok - b * p.L;
    const int64_t po = b * p.pos_b + l * p.pos_l;
    const long long pos = p.pos64 ? static_cast<const long long*>(p.pos)[po] : (long long)static_cast<const int*>(p.pos)[po];
    float cs[UPL][V], sn[UPL][V];
#pragma unroll
    for (int i = 0; i < UPL; ++i) {
      const int u = sub + i * 32;
      const bool turns = u < ru;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        cs[i][j] = 1.f;
        sn[i][j] = 0.f;
        if (turns) {
          const long long frac = (long long)(turn_s[u * V + j] * (unsigned long long)pos);
          sincospif((float)frac * 1.0842021724855044e-19f, &sn[i][j], &cs[i][j]);    // 2^-63: twice the fraction of a turn
          cs[i][j] *= p.scaling;
          sn[i][j] *= p.scaling;
        }
      }
    }
    const T* x0 = static_cast<const T*>(sd.x) + b * sd.xb + l * sd.xl;
    const T* g0 = BWD ? static_cast<const T*>(sd.g) + b * sd.gb + l * sd.gl : nullptr;
    T* y0 = static_cast<T*>(sd.out) + tok * sd.H * (int64_t)p.D;
    for (int hh = 0; hh < sd.hpg; hh += kHeads) {               // the same trip count in the whole warp
      float a[kHeads][UPL][V], c[kHeads][UPL][V], ga[BWD ? kHeads : 1][UPL][V], gc[BWD ? kHeads : 1][UPL][V];
      float ss[kHeads], dot[kHeads];
#pragma unroll
      for (int k = 0; k < kHeads; ++k) {
        const int h = h0 + hh + k;
        const bool on = h < h1;
#pragma unroll
        for (int i = 0; i < UPL; ++i) {
#pragma unroll
          for (int j = 0; j < V; ++j) {
            a[k][i][j] = c[k][i][j] = 0.f;
            if (BWD) ga[k][i][j] = gc[k][i][j] = 0.f;
          }
          if (on && has[i]) {
            if (!BWD || sd.w) {
              load_v<T, V>(x0 + h * sd.xh + o1[i], a[k][i]);
              load_v<T, V>(x0 + h * sd.xh + o2[i], c[k][i]);
            }
            if constexpr (BWD) {
              load_v<T, V>(g0 + h * sd.gh + o1[i], ga[k][i]);
              load_v<T, V>(g0 + h * sd.gh + o2[i], gc[k][i]);
            }
          }
        }
      }
#pragma unroll
      for (int k = 0; k < kHeads; ++k) {
        ss[k] = dot[k] = 0.f;
#pragma unroll
        for (int i = 0; i < UPL; ++i) {
          if constexpr (BWD) rotate<V, INTER, true>(ga[k][i], gc[k][i], cs[i], sn[i]);
#pragma unroll
          for (int j = 0; j < V; ++j) {
            ss[k] = fmaf(a[k][i][j], a[k][i][j], fmaf(c[k][i][j], c[k][i][j], ss[k]));
            if constexpr (BWD) dot[k] = fmaf(ga[k][i][j] * w1[i][j], a[k][i][j], fmaf(gc[k][i][j] * w2[i][j], c[k][i][j], dot[k]));
          }
        }
      }
      if (sd.w) {
        for (int o = lpr >> 1; o > 0; o >>= 1)
#pragma unroll
          for (int k = 0; k < kHeads; ++k) {
            ss[k] += __shfl_xor_sync(0xffffffffu, ss[k], o);
            if (BWD) dot[k] += __shfl_xor_sync(0xffffffffu, dot[k], o);
          }
      }
#pragma unroll
      for (int k = 0; k < kHeads; ++k) {
        const int h = h0 + hh + k;
        const bool on = h < h1;
        const float rstd = sd.w ? rsqrtf(fmaf(ss[k], inv_d, p.eps)) : 1.f;
        const float m = BWD ? dot[k] * inv_d * rstd * rstd : 0.f;
#pragma unroll
        for (int i = 0; i < UPL; ++i) {
          float y1[V], y2[V];
#pragma unroll
          for (int j = 0; j < V; ++j) {
            if constexpr (BWD) {
              y1[j] = ga[k][i][j];
              y2[j] = gc[k][i][j];
              if (sd.w) {
                if (on) {                                       // rows past the end hold zeros, and rstd of a zero row is large
                  dw1[i][j] = fmaf(ga[k][i][j], a[k][i][j] * rstd, dw1[i][j]);
                  dw2[i][j] = fmaf(gc[k][i][j], c[k][i][j] * rstd, dw2[i][j]);
                }
                y1[j] = rstd * (ga[k][i][j] * w1[i][j] - a[k][i][j] * m);
                y2[j] = rstd * (gc[k][i][j] * w2[i][j] - c[k][i][j] * m);
              }
            } else {
              y1[j] = a[k][i][j] * rstd * w1[i][j];
              y2[j] = c[k][i][j] * rstd * w2[i][j];
            }
          }
          if constexpr (!BWD) rotate<V, INTER, false>(y1, y2, cs[i], sn[i]);
          if (on && has[i]) {
            store_v<T, V>(y0 + h * (int64_t)p.D + o1[i], y1);
            store_v<T, V>(y0 + h * (int64_t)p.D + o2[i], y2);
          }
        }
      }
    }
  }
  if constexpr (BWD) {
    if (sd.w) {
      // the CTA's share of dw, summed in a fixed order: over the groups of a warp, then over the warps
#pragma unroll
      for (int i = 0; i < UPL; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          for (int o = lpr; o < 32; o <<= 1) {
            dw1[i][j] += __shfl_xor_sync(0xffffffffu, dw1[i][j], o);
            dw2[i][j] += __shfl_xor_sync(0xffffffffu, dw2[i][j], o);
          }
          if (lane < lpr && has[i]) {
            dw_s[warp][o1[i] + j] = dw1[i][j];
            dw_s[warp][o2[i] + j] = dw2[i][j];
          }
        }
      __syncthreads();
      for (int d = tid; d < p.D; d += kQkThreads) {
        float s = 0.f;
        for (int w = 0; w < kQkThreads / 32; ++w) s += dw_s[w][d];
        sd.dw[(int64_t)(blockIdx.x - sd.cta0) * p.D + d] = s;
      }
    }
  }
}

// dw = the sum of the CTAs' shares, in a fixed order: warp w takes the rows w, w + 8, ..., then the warps are added up
struct QkSumParams {
  const float* part[2]; void* dw[2];
  int rows[2];
  int D, out_f32;
};

__global__ void __launch_bounds__(256) qk_weight_grad_kernel(QkSumParams p) {
  __shared__ float s[8][33];
  const int si = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, d = blockIdx.x * 32 + lane;
  float acc = 0.f;
  if (d < p.D)
    for (int r = warp; r < p.rows[si]; r += 8) acc += p.part[si][(int64_t)r * p.D + d];
  s[warp][lane] = acc;
  __syncthreads();
  if (warp == 0 && d < p.D) {
    for (int w = 1; w < 8; ++w) acc += s[w][lane];
    if (p.out_f32) static_cast<float*>(p.dw[si])[d] = acc;
    else static_cast<bf16*>(p.dw[si])[d] = __float2bfloat16_rn(acc);
  }
}

// CTAs of one side: enough to fill the device, never more than there are rows for
constexpr int kQkMaxCtas = 148 * 8;

template <typename T, int V, int UPL, bool INTER, bool BWD>
static void launch_qk(const QkParams& p, int ctas, cudaStream_t st) {
  qk_norm_rope_kernel<T, V, UPL, INTER, BWD><<<ctas, kQkThreads, 0, st>>>(p);
}

template <typename T, bool INTER, bool BWD>
static void launch_qk_v(const QkParams& p, int v, int ctas, cudaStream_t st) {
  if constexpr (sizeof(T) == 2) {
    if (v == 8) return launch_qk<T, 8, 1, INTER, BWD>(p, ctas, st);
  }
  if (v == 4) return launch_qk<T, 4, 1, INTER, BWD>(p, ctas, st);
  launch_qk<T, 1, 4, INTER, BWD>(p, ctas, st);
}

// Work split of one call: heads per group, CTAs per side.  Kept in one place so that the workspace query and the launch agree.
struct QkPlan { int v, lpr, hpg[2], hsplit[2], ctas[2]; };

static QkPlan qk_plan(const int* heads, int n, int64_t tokens, int D, int rot, int v) {
  QkPlan pl = {};
  pl.v = v;
  const int units = D / (2 * v);
  pl.lpr = 1;
  while (pl.lpr < units && pl.lpr < 32) pl.lpr <<= 1;
  int total = 0;
  for (int i = 0; i < n; ++i) total += heads[i];
  for (int i = 0; i < n; ++i) {
    const int H = std::max(1, heads[i]);
    // a group walks several heads with one set of cos/sin; fewer when that would leave the device empty
    int hpg = std::min(H, 16);
    while (hpg > 1 && tokens * ((total + hpg - 1) / hpg) * pl.lpr < (int64_t)148 * 1024) hpg = (hpg + 1) / 2;
    pl.hpg[i] = hpg;
    pl.hsplit[i] = (H + hpg - 1) / hpg;
    const int64_t groups = tokens * pl.hsplit[i], per_cta = kQkThreads / pl.lpr;
    pl.ctas[i] = (int)std::max<int64_t>(1, std::min<int64_t>((groups + per_cta - 1) / per_cta,
                                                             std::max(1, (int)((int64_t)kQkMaxCtas * heads[i] / std::max(1, total)))));
  }
  return pl;
}

}  // namespace hils

using namespace hils;

// widest access that the sizes, strides and addresses allow: halves of a unit must not straddle a rotation boundary
static int qk_width(const hils_rope_tensor* t, int n, int D, int rot, int es, bool bwd) {
  for (int v = 16 / es; v >= 4; v >>= 1) {
    if (D % (2 * v) || rot % (2 * v)) continue;
    bool ok = true;
    for (int i = 0; i < n; ++i) {
      const int64_t a = (int64_t)v * es;
      ok = ok && (uintptr_t)t[i].x % a == 0 && (uintptr_t)t[i].out % a == 0 && (t[i].x_stride_b * es) % a == 0 && (t[i].x_stride_l * es) % a == 0 &&
           (t[i].x_stride_h * es) % a == 0;
      if (bwd)
        ok = ok && (uintptr_t)t[i].d_out % a == 0 && (t[i].g_stride_b * es) % a == 0 && (t[i].g_stride_l * es) % a == 0 && (t[i].g_stride_h * es) % a == 0;
    }
    if (ok) return v;
  }
  return 1;
}

static int qk_run(const hils_rope_tensor* t, int n, const void* positions, int pos64, int64_t pos_b, int64_t pos_l, const double* inv_freq,
                  int rot, int B, int L, int D, int interleaved, float scaling, float eps, int dtype, int weight_dtype, void* workspace,
                  size_t workspace_bytes, cudaStream_t st, bool bwd) {
  const char* what = bwd ? "qk_norm_rope_bwd" : "qk_norm_rope_fwd";
  HILS_REQUIRE(dtype == HILS_BF16 || dtype == HILS_F32, "%s: unknown dtype %d", what, dtype);
  HILS_REQUIRE(weight_dtype == HILS_BF16 || weight_dtype == HILS_F32, "%s: unknown weight dtype %d", what, weight_dtype);
  HILS_REQUIRE(t && n >= 1 && n <= 2, "%s: one or two tensors, got %d", what, n);
  HILS_REQUIRE(B >= 0 && L >= 0 && D > 0 && D <= kQkMaxD && D % 2 == 0, "%s: D (%d) must be even and at most %d", what, D, kQkMaxD);
  HILS_REQUIRE(rot >= 0 && rot <= D && rot % 2 == 0, "%s: the rotated part (%d) must be even and at most D (%d)", what, rot, D);
  for (int i = 0; i < n; ++i) HILS_REQUIRE(t[i].heads >= 0, "%s: negative number of heads", what);
  const int64_t tokens = (int64_t)B * L;
  const int es = dtype == HILS_BF16 ? 2 : 4;
  int heads[2] = {0, 0};
  for (int i = 0; i < n; ++i) heads[i] = t[i].heads;
  const bool empty = tokens == 0 || (heads[0] == 0 && heads[1] == 0);
  if (!empty) {
    HILS_REQUIRE(positions && (inv_freq || rot == 0), "%s: null pointer", what);
    for (int i = 0; i < n; ++i)
      HILS_REQUIRE(heads[i] == 0 || ((t[i].x || (bwd && !t[i].weight)) && t[i].out && (!bwd || t[i].d_out)), "%s: null pointer", what);
  }
  for (int i = 0; i < n; ++i) HILS_REQUIRE(!bwd || !t[i].weight || t[i].d_weight, "%s: null pointer", what);
  const QkPlan pl = qk_plan(heads, n, std::max<int64_t>(1, tokens), D, rot, empty ? 1 : qk_width(t, n, D, rot, es, bwd));
  QkParams p = {};
  QkSumParams sum = {};
  int ctas = 0, sums = 0;
  size_t need = 0;
  for (int i = 0; i < n; ++i) {
    QkSide& s = p.side[i];
    s.x = t[i].x; s.w = t[i].weight; s.out = t[i].out; s.g = t[i].d_out;
    s.xb = t[i].x_stride_b; s.xl = t[i].x_stride_l; s.xh = t[i].x_stride_h;
    s.gb = t[i].g_stride_b; s.gl = t[i].g_stride_l; s.gh = t[i].g_stride_h;
    s.H = heads[i]; s.hpg = pl.hpg[i]; s.hsplit = pl.hsplit[i]; s.cta0 = ctas; s.ctas = pl.ctas[i];
    ctas += pl.ctas[i];
    if (bwd && t[i].weight) {
      s.dw = reinterpret_cast<float*>(static_cast<unsigned char*>(workspace) + need);
      sum.part[sums] = s.dw; sum.dw[sums] = t[i].d_weight; sum.rows[sums] = empty ? 0 : pl.ctas[i];
      ++sums;
      need += (size_t)pl.ctas[i] * D * sizeof(float);
    }
  }
  if (need > 0 && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15))) {
    set_error("%s: a 16-byte aligned workspace of %zu bytes needed, %zu given", what, need, workspace_bytes);
    return HILS_ERR_WORKSPACE;
  }
  p.pos = positions; p.inv_freq = inv_freq; p.pos_b = pos_b; p.pos_l = pos_l;
  p.B = B; p.L = L; p.D = D; p.rot = rot; p.lpr = pl.lpr; p.n_sides = n; p.pos64 = pos64; p.w_f32 = weight_dtype == HILS_F32;
  p.eps = eps; p.scaling = scaling;
  if (!empty) {
#define HILS_QK(T)                                                                          \
  (interleaved ? (bwd ? launch_qk_v<T, true, true>(p, pl.v, ctas, st) : launch_qk_v<T, true, false>(p, pl.v, ctas, st)) \
               : (bwd ? launch_qk_v<T, false, true>(p, pl.v, ctas, st) : launch_qk_v<T, false, false>(p, pl.v, ctas, st)))
    if (dtype == HILS_BF16) HILS_QK(bf16); else HILS_QK(float);
#undef HILS_QK
    HILS_LAUNCH_CHECK(what);
  }
  if (sums > 0) {
    sum.D = D; sum.out_f32 = weight_dtype == HILS_F32;
    qk_weight_grad_kernel<<<dim3((unsigned)((D + 31) / 32), (unsigned)sums), 256, 0, st>>>(sum);
    HILS_LAUNCH_CHECK(what);
  }
  return HILS_OK;
}

extern "C" int hils_qk_norm_rope_fwd(const hils_rope_tensor* tensors, int n_tensors, const void* positions, int positions_64,
                                     int64_t pos_stride_b, int64_t pos_stride_l, const double* inv_freq, int rot, int B, int L, int D,
                                     int interleaved, float scaling, float eps, int dtype, int weight_dtype, void* stream) {
  return qk_run(tensors, n_tensors, positions, positions_64, pos_stride_b, pos_stride_l, inv_freq, rot, B, L, D, interleaved, scaling, eps,
                dtype, weight_dtype, nullptr, 0, (cudaStream_t)stream, false);
}

extern "C" size_t hils_qk_norm_rope_bwd_workspace_bytes(int D) {
  return D > 0 && D <= kQkMaxD ? (size_t)(kQkMaxCtas + 2) * D * sizeof(float) : 0;
}

extern "C" int hils_qk_norm_rope_bwd(const hils_rope_tensor* tensors, int n_tensors, const void* positions, int positions_64,
                                     int64_t pos_stride_b, int64_t pos_stride_l, const double* inv_freq, int rot, int B, int L, int D,
                                     int interleaved, float scaling, float eps, int dtype, int weight_dtype, void* workspace,
                                     size_t workspace_bytes, void* stream) {
  return qk_run(tensors, n_tensors, positions, positions_64, pos_stride_b, pos_stride_l, inv_freq, rot, B, L, D, interleaved, scaling, eps,
                dtype, weight_dtype, workspace, workspace_bytes, (cudaStream_t)stream, true);
}
