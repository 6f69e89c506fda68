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
// A group forms the cos/sin of its token once and walks `hpg` heads with it, the rows of the next four steps on their way.
//
// What bounds it: the HBM.  Forward 2, backward 3 tensors' worth of bytes; 65536 tokens, 32 + 32 heads of 128, bf16: 348 us
// = 6.16 TB/s and 580 us = 5.55 TB/s (0.94 and 0.85 of the copy bandwidth; the issue slots are 60 to 70 % busy).  With the
// loads in registers, four rows at a time, it was 908 and 1682 us.  fp32, 16 + 16 heads: 388 us = 5.54 TB/s and 594 us = 5.42 TB/s.
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
    static_assert(V == 4 || V == 8, "a unit half is 1, 4 or 8 elements");
#pragma unroll
    for (int i = 0; i < V; i += 4) {
      const float4 v = load4(p + i);
      f[i] = v.x; f[i + 1] = v.y; f[i + 2] = v.z; f[i + 3] = v.w;
    }
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

// Rows per lane on their way from global memory (asynchronous copies into slots that only their own thread reads, so they
// need no barrier).  The kernel holds 80 (forward) or 128 (backward) registers of working values per thread; loads kept in
// registers as well leave too few warps to cover the memory's latency.  Four steps ahead with two CTAs per SM measured best:
// backward at 64K tokens 580 us, six ahead 697, three CTAs (which spill) 1854; the weights sit in shared memory, not in
// registers, for the same reason (808 us with them in registers).
template <typename T, int V>
constexpr bool kQkAsync = V * sizeof(T) >= 8;
constexpr int kQkStages = 4;

template <int BYTES>
__device__ __forceinline__ void copy_async(void* dst, const void* src) {
  const uint32_t d = (uint32_t)__cvta_generic_to_shared(dst);
  if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(d), "l"(src) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(d), "l"(src) : "memory");
}

template <typename T, int V, int UPL, bool BWD>
constexpr size_t qk_smem() {
  const size_t ring = kQkAsync<T, V> ? (size_t)kQkStages * (BWD ? 4 : 2) * kQkThreads * V * sizeof(T) : 0;
  const size_t dw = BWD ? (size_t)(kQkThreads / 32) * kQkMaxD * sizeof(float) : 0;
  return (kQkMaxD / 2) * sizeof(unsigned long long) + kQkMaxD * sizeof(float) + (ring > dw ? ring : dw);
}

template <typename T, int V, int UPL, bool INTER, bool BWD>
__global__ void __launch_bounds__(kQkThreads, 2) qk_norm_rope_kernel(const __grid_constant__ QkParams p) {
  constexpr bool kAsync = kQkAsync<T, V>;
  constexpr int kParts = BWD ? 4 : 2, kBytes = V * sizeof(T);
  extern __shared__ __align__(16) unsigned char qk_smem_raw[];
  unsigned long long* turn_s = reinterpret_cast<unsigned long long*>(qk_smem_raw);
  float* w_s = reinterpret_cast<float*>(turn_s + kQkMaxD / 2);
  unsigned char* ring = reinterpret_cast<unsigned char*>(w_s + kQkMaxD);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int si = (p.n_sides > 1 && (int)blockIdx.x >= p.side[1].cta0) ? 1 : 0;
  const QkSide& sd = p.side[si];
  for (int i = tid; i < (p.rot >> 1); i += kQkThreads) {
    const double t = p.inv_freq[i] * kInvTwoPi;
    turn_s[i] = (unsigned long long)((t - floor(t)) * 18446744073709551616.0);
  }
  for (int d = tid; d < p.D; d += kQkThreads) w_s[d] = sd.w ? weight_at(p, sd.w, d) : 1.f;
  __syncthreads();
  const int lpr = p.lpr, sub = lane & (lpr - 1), gpw = 32 / lpr;   // groups per warp
  const int units = p.D / (2 * V), ru = p.rot / (2 * V);
  int o1[UPL], o2[UPL];
  bool has[UPL];
  float dw1[UPL][V], dw2[UPL][V];
#pragma unroll
  for (int i = 0; i < UPL; ++i) {
    const int u = sub + i * 32;
    has[i] = u < units;
    unit_at<V, INTER>(p, has[i] ? u : 0, o1[i], o2[i]);
#pragma unroll
    for (int j = 0; j < V; ++j) dw1[i][j] = dw2[i][j] = 0.f;
  }
  const int64_t items = (int64_t)p.B * p.L * sd.hsplit;
  const int64_t step = (int64_t)sd.ctas * (kQkThreads / 32) * gpw;
  const int64_t first = ((int64_t)(blockIdx.x - sd.cta0) * (kQkThreads / 32) + warp) * gpw;
  const float inv_d = 1.f / (float)p.D;

  // A walk over this group's rows: item after item (a token and up to hpg of its heads), the same number of steps in the
  // whole warp.  `left` heads of the current item are real.
  struct Walk { int64_t it0; int hh, left; const T* x; const T* g; };
  auto decode = [&](int64_t it0, int64_t& tok, int64_t& b, int64_t& l, int& h0) {
    int64_t it = it0 + lane / lpr;
    if (it >= items) it = 0;
    if (items <= 0x7fffffff) {                                    // 32-bit divisions are several times cheaper
      const uint32_t t = (uint32_t)it / (uint32_t)sd.hsplit, bb = t / (uint32_t)p.L;
      tok = t; b = bb; l = t - bb * (uint32_t)p.L;
      h0 = (int)((uint32_t)it - t * (uint32_t)sd.hsplit) * sd.hpg;
    } else {
      tok = it / sd.hsplit; b = tok / p.L; l = tok - b * p.L;
      h0 = (int)(it - tok * sd.hsplit) * sd.hpg;
    }
    return it0 + lane / lpr < items ? min(sd.H - h0, sd.hpg) : 0;
  };
  auto enter = [&](Walk& w) {
    int64_t tok, b, l;
    int h0;
    w.left = decode(w.it0, tok, b, l, h0);
    w.hh = sd.hpg;
    w.x = static_cast<const T*>(sd.x) + b * sd.xb + l * sd.xl + h0 * sd.xh;
    if (BWD) w.g = static_cast<const T*>(sd.g) + b * sd.gb + l * sd.gl + h0 * sd.gh;
  };
  auto advance = [&](Walk& w) {
    --w.left;
    w.x += sd.xh;
    if (BWD) w.g += sd.gh;
    if (--w.hh == 0) {
      w.it0 += step;
      if (w.it0 < items) enter(w);
    }
  };
  auto slot = [&](int stage, int part) { return ring + ((size_t)(stage * kParts + part) * kQkThreads + tid) * kBytes; };
  auto issue = [&](Walk& w, int stage) {
    if (w.it0 < items) {
      if (w.left > 0 && has[0]) {
        if (!BWD || sd.w) {
          copy_async<kBytes>(slot(stage, 0), w.x + o1[0]);
          copy_async<kBytes>(slot(stage, 1), w.x + o2[0]);
        }
        if constexpr (BWD) {
          copy_async<kBytes>(slot(stage, kParts - 2), w.g + o1[0]);
          copy_async<kBytes>(slot(stage, kParts - 1), w.g + o2[0]);
        }
      }
      advance(w);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };

  Walk ahead = {first, 0, 0, nullptr, nullptr};                   // loads; without asynchronous copies the row in hand
  if (first < items) enter(ahead);
  if constexpr (kAsync)
    for (int s = 0; s < kQkStages; ++s) issue(ahead, s);
  int64_t it0 = first;                                            // the item in hand
  int stage = 0, hh = 0, left = 0;
  T* y = nullptr;
  float cs[UPL][V], sn[UPL][V];
  while (it0 < items) {
    if (hh == 0) {
      int64_t tok, b, l;
      int h0;
      left = decode(it0, tok, b, l, h0);
      y = static_cast<T*>(sd.out) + (tok * sd.H + h0) * (int64_t)p.D;
      const int64_t po = b * p.pos_b + l * p.pos_l;
      const long long pos = p.pos64 ? static_cast<const long long*>(p.pos)[po] : (long long)static_cast<const int*>(p.pos)[po];
#pragma unroll
      for (int i = 0; i < UPL; ++i) {
        const int u = sub + i * 32;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          cs[i][j] = 1.f;
          sn[i][j] = 0.f;
          if (u < ru) {
            const long long frac = (long long)(turn_s[u * V + j] * (unsigned long long)pos);
            sincospif((float)frac * 1.0842021724855044e-19f, &sn[i][j], &cs[i][j]);    // 2^-63: twice the fraction of a turn
            cs[i][j] *= p.scaling;
            sn[i][j] *= p.scaling;
          }
        }
      }
    }
    const bool on = hh < left;
    float a[UPL][V], c[UPL][V], ga[BWD ? UPL : 1][V], gc[BWD ? UPL : 1][V];
    if constexpr (kAsync) asm volatile("cp.async.wait_group %0;" ::"n"(kQkStages - 1) : "memory");
#pragma unroll
    for (int i = 0; i < UPL; ++i) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        a[i][j] = c[i][j] = 0.f;
        if (BWD) ga[i][j] = gc[i][j] = 0.f;
      }
      if (on && has[i]) {
        if (!BWD || sd.w) {
          const T* x = ahead.x;
          load_v<T, V>(kAsync ? reinterpret_cast<const T*>(slot(stage, 0)) : x + o1[i], a[i]);
          load_v<T, V>(kAsync ? reinterpret_cast<const T*>(slot(stage, 1)) : x + o2[i], c[i]);
        }
        if constexpr (BWD) {
          const T* g = ahead.g;
          load_v<T, V>(kAsync ? reinterpret_cast<const T*>(slot(stage, kParts - 2)) : g + o1[i], ga[i]);
          load_v<T, V>(kAsync ? reinterpret_cast<const T*>(slot(stage, kParts - 1)) : g + o2[i], gc[i]);
        }
      }
    }
    float ss = 0.f, dot = 0.f, gw1[BWD ? UPL : 1][V], gw2[BWD ? UPL : 1][V];
#pragma unroll
    for (int i = 0; i < UPL; ++i) {
      float w1[V], w2[V];
      if constexpr (BWD) {
        rotate<V, INTER, true>(ga[i], gc[i], cs[i], sn[i]);
        load_v<float, V>(w_s + o1[i], w1);
        load_v<float, V>(w_s + o2[i], w2);
      }
#pragma unroll
      for (int j = 0; j < V; ++j) {
        ss = fmaf(a[i][j], a[i][j], fmaf(c[i][j], c[i][j], ss));
        if constexpr (BWD) {
          gw1[i][j] = ga[i][j] * w1[j];
          gw2[i][j] = gc[i][j] * w2[j];
          dot = fmaf(gw1[i][j], a[i][j], fmaf(gw2[i][j], c[i][j], dot));
        }
      }
    }
    if (sd.w) {
      for (int o = lpr >> 1; o > 0; o >>= 1) {
        ss += __shfl_xor_sync(0xffffffffu, ss, o);
        if (BWD) dot += __shfl_xor_sync(0xffffffffu, dot, o);
      }
    }
    if constexpr (kAsync) {
      issue(ahead, stage);                                        // the slot's values are in registers now
      if (++stage == kQkStages) stage = 0;
    }
    const float rstd = sd.w ? rsqrtf(fmaf(ss, inv_d, p.eps)) : 1.f;
    const float m = BWD ? dot * inv_d * rstd * rstd : 0.f;
#pragma unroll
    for (int i = 0; i < UPL; ++i) {
      float y1[V], y2[V], w1[V], w2[V];
      if constexpr (!BWD) {
        load_v<float, V>(w_s + o1[i], w1);
        load_v<float, V>(w_s + o2[i], w2);
      }
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if constexpr (BWD) {
          y1[j] = ga[i][j];
          y2[j] = gc[i][j];
          if (sd.w) {
            if (on) {                                             // rows past the end hold zeros, and rstd of a zero row is large
              dw1[i][j] = fmaf(ga[i][j], a[i][j] * rstd, dw1[i][j]);
              dw2[i][j] = fmaf(gc[i][j], c[i][j] * rstd, dw2[i][j]);
            }
            y1[j] = rstd * (gw1[i][j] - a[i][j] * m);
            y2[j] = rstd * (gw2[i][j] - c[i][j] * m);
          }
        } else {
          y1[j] = a[i][j] * rstd * w1[j];
          y2[j] = c[i][j] * rstd * w2[j];
        }
      }
      if constexpr (!BWD) rotate<V, INTER, false>(y1, y2, cs[i], sn[i]);
      if (on && has[i]) {
        store_v<T, V>(y + o1[i], y1);
        store_v<T, V>(y + o2[i], y2);
      }
    }
    if constexpr (!kAsync) advance(ahead);
    y += p.D;
    if (++hh == sd.hpg) {
      hh = 0;
      it0 += step;
    }
  }
  if constexpr (kAsync) asm volatile("cp.async.wait_group 0;" ::: "memory");
  if constexpr (BWD) {
    if (sd.w) {
      // the CTA's share of dw, summed in a fixed order: over the groups of a warp, then over the warps
      float* dw_s = reinterpret_cast<float*>(ring);               // the copies are done: their slots are free
      __syncthreads();
#pragma unroll
      for (int i = 0; i < UPL; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          for (int o = lpr; o < 32; o <<= 1) {
            dw1[i][j] += __shfl_xor_sync(0xffffffffu, dw1[i][j], o);
            dw2[i][j] += __shfl_xor_sync(0xffffffffu, dw2[i][j], o);
          }
          if (lane < lpr && has[i]) {
            dw_s[warp * kQkMaxD + o1[i] + j] = dw1[i][j];
            dw_s[warp * kQkMaxD + o2[i] + j] = dw2[i][j];
          }
        }
      __syncthreads();
      for (int d = tid; d < p.D; d += kQkThreads) {
        float s = 0.f;
        for (int w = 0; w < kQkThreads / 32; ++w) s += dw_s[w * kQkMaxD + d];
        sd.dw[(int64_t)(blockIdx.x - sd.cta0) * p.D + d] = s;
      }
    }
  }
}

// dw = the sum of the CTAs' shares, in a fixed order: warp w takes the rows w, w + 32, ..., then the warps are added up
// (32 warps: all loads of a thread are on their way at once)
struct QkSumParams {
  const float* part[2]; void* dw[2];
  int rows[2];
  int D, out_f32;
};

__global__ void __launch_bounds__(1024) qk_weight_grad_kernel(QkSumParams p) {
  __shared__ float s[32][33];
  const int si = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, d = blockIdx.x * 32 + lane;
  float acc = 0.f;
  if (d < p.D)
#pragma unroll 5
    for (int r = warp; r < p.rows[si]; r += 32) acc += p.part[si][(int64_t)r * p.D + d];
  s[warp][lane] = acc;
  __syncthreads();
  acc = warp_sum(s[lane][warp]);
  const int at = blockIdx.x * 32 + warp;
  if (lane == 0 && at < p.D) {
    if (p.out_f32) static_cast<float*>(p.dw[si])[at] = acc;
    else static_cast<bf16*>(p.dw[si])[at] = __float2bfloat16_rn(acc);
  }
}

// CTAs of a call: one wave at two per SM (more of them cost 2 to 19 % at 64K tokens), never more than there are rows for
constexpr int kQkMaxCtas = 148 * 2;

template <typename T, int V, int UPL, bool INTER, bool BWD>
static void launch_qk(const QkParams& p, int ctas, cudaStream_t st) {
  constexpr size_t smem = qk_smem<T, V, UPL, BWD>();
  if (smem > 48 * 1024)
    cudaFuncSetAttribute(qk_norm_rope_kernel<T, V, UPL, INTER, BWD>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  qk_norm_rope_kernel<T, V, UPL, INTER, BWD><<<ctas, kQkThreads, smem, st>>>(p);
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
    qk_weight_grad_kernel<<<dim3((unsigned)((D + 31) / 32), (unsigned)sums), 1024, 0, st>>>(sum);
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
