// Group norm with an activation over channels-last tensors (tbg.h "GROUP NORM"): x [N][S][C], statistics over the S x C/G values of a
// (sample, group), forward and backward, with the input kept whole or as an 8-bit checkpoint of x - mean.
//
//   xh = (x - mean) rstd,  z = gamma xh + beta,  y = act(z)
//   dz = dy act'(z),  dbeta = sum dz,  dgamma = sum dz xh,  dx = rstd (gamma dz - mean(gamma dz) - xh mean(gamma dz xh))
//
// HBM-bound.  A block works on a tile of CT channels (every lane has V fixed neighbouring ones) and a range of rows, so all accesses are
// whole 16-byte pieces of rows whatever the group width: groups need not line up with tiles.  Direction forward / backward: a sums launch
// leaves partial sums per (sample, row range, tile, group), the second launch joins those of its groups in a fixed order (no atomics) and
// writes the result.
//
// The statistics are 64-bit sums of x and x^2: one pass, and mean(x^2) - mean^2 loses nothing that matters for fp32 values of
// |mean| = 10^5 standard deviations, nor for 16-bit ones, which do not resolve more than 2^11 of them.  The mean is used as fp32 + its remainder.
#include "act8.h"

#include <type_traits>

struct GnP {
  const void *x, *dy;
  const float *gamma, *beta;
  void *y;                             // forward: output; backward: dx
  unsigned char *q, *e;                // checkpoint of x - mean (written forward, read backward), or null
  unsigned char *yq, *ye;              // forward: checkpoint of y, or null
  double *stats;                       // [N][G][2] mean, rstd
  double *part;                        // forward: [N][nchunk][nslot][2] sum x, sum x^2; backward: sum gamma dz, sum gamma dz xh
  float *pch;                          // backward: [N][nchunk][C][2] sum dz, sum dz xh of a channel
  float *dgamma, *dbeta;
  long long xn, xs, dn, ds;            // sample / row pitches of x and dy in elements (y, dx: contiguous)
  int N, S, C, G, Cg, affn, nb;        // affn: affine parameters' sample pitch (0 or C); nb: 8-bit blocks a row
  int CT, ntile, lanes;                // channels a tile (a power of two), tiles, lanes a row
  int nchunk, crows, nslot;            // row ranges of the sums launch
  int split, arows;                    // the second launch's part of a row range: `split` pieces of arows rows
  int pblocks;                         // backward: first blocks of the second launch that sum dgamma / dbeta
  float eps;
};

#ifndef GN_BLOCKS
#define GN_BLOCKS 2048
#endif
constexpr int GN_T = 256, GN_TS = 1024, GN_TB = 512, GN_CT = 128;  // threads a block: second launches, forward sums, backward sums; most channels a tile

template <int ACT>
__device__ __forceinline__ float gn_act(float z) {
  if constexpr (ACT == TBG_ACT_LRELU) return 1.41421356237309515f * (z > 0.f ? z : 0.2f * z);
  if constexpr (ACT == TBG_ACT_SILU) return z * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.44269504088896341f * z));
  return z;
}
// dy act'(z).  positive: LeakyReLU's side of the kink, decided in 64 bits so that it does not hang on the last bit of a 32-bit product
template <int ACT>
__device__ __forceinline__ float gn_dact(float dy, float z, bool positive) {
  if constexpr (ACT == TBG_ACT_LRELU) return dy * (positive ? 1.41421356237309515f : 0.282842712474619f);
  if constexpr (ACT == TBG_ACT_SILU) {  // z comes times -log2(e): s = 1 / (1 + e^-z), act' = s + z s (1 - s)
    const float s = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(z)), u = z * s;
    return dy * fmaf(fmaf(-u, s, u), -0.693147180559945309f, s);
  }
  return dy;
}

// group of channel c, and of the channels after it one by one
struct GnGroup {
  int g, left;
  __device__ __forceinline__ GnGroup(int c, int Cg) : g(c / Cg), left(Cg - (c - c / Cg * Cg)) {}
  __device__ __forceinline__ void next(int Cg) {
    if (--left == 0) { ++g; left = Cg; }
  }
};

// what a block of the sums launch works on: row range k of a tile of a sample.  Row ranges vary fastest in both launches and their count is
// a multiple of 8 where there are that many: a row range then stays on one of the 8 XCDs, whose L2 still holds it for the second launch
struct GnTile {
  int n, tile, k, c0, ct;
};
__device__ __forceinline__ GnTile gn_tile(const GnP &p, int b) {
  GnTile t;
  t.k = b % p.nchunk; b /= p.nchunk;
  t.tile = b % p.ntile;
  t.n = b / p.ntile;
  t.c0 = t.tile * p.CT;
  t.ct = min(p.CT, p.C - t.c0);
  return t;
}

// sums of one group's partial pairs over its tiles and the row ranges, by `sub` neighbouring lanes (a power of two), all of which get it
__device__ __forceinline__ void gn_join(const GnP &p, int n, int g, int lane, int sub, double &a, double &b) {
  const int t0 = g * p.Cg / p.CT, t1 = ((g + 1) * p.Cg - 1) / p.CT, nt = t1 - t0 + 1;
  a = b = 0.0;
  const double *base = p.part + (long long)n * p.nchunk * p.nslot * 2;
  for (int i = lane; i < nt * p.nchunk; i += sub) {
    const int k = i / nt, t = t0 + i - k * nt;
    const double2 s = *reinterpret_cast<const double2 *>(base + ((long long)k * p.nslot + t + g) * 2);
    a += s.x;
    b += s.y;
  }
  for (int off = sub >> 1; off > 0; off >>= 1) {
    a += __shfl_xor(a, off, 64);
    b += __shfl_xor(b, off, 64);
  }
}

// ---- forward, first launch: sums of x and x^2.  V / A neighbouring channels share a group (A accumulators a lane)
template <class E, int V, int A>
__global__ __launch_bounds__(GN_TS) void gn_sums_kernel(GnP p) {
  constexpr int U = 4, NW = GN_TS / 64;
  __shared__ double red[NW * (GN_CT / V) * A * 2];
  const GnTile t = gn_tile(p, blockIdx.x);
  const int lane = threadIdx.x & (p.lanes - 1), rl = threadIdx.x / p.lanes, RL = GN_TS / p.lanes;
  const int r1 = min(p.S, (t.k + 1) * p.crows);
  double s1[A], s2[A];
#pragma unroll
  for (int i = 0; i < A; ++i) s1[i] = s2[i] = 0.0;
  if (lane * V < t.ct) {
    const typename E::type *x = reinterpret_cast<const typename E::type *>(p.x) + t.n * p.xn + t.c0 + lane * V;
    // 16-bit types: 8 values and 8 squares are added in fp32 before they are in fp64 (values of 8 or 11 bits within 13 or 10 binades: the
    // first sum is exact, the second off by 2^-24 at most, random over the sums of a group)
    constexpr bool PRE = E::BYTES == 2;
    constexpr int B = PRE ? (A < U ? A : U) : 1;  // rows added up before
    const auto add = [&](const Pack<E, V> *v, auto rows) {
#pragma unroll
      for (int a = 0; a < A; ++a) {
        if constexpr (PRE) {
          float t1 = 0.f, t2 = 0.f;
#pragma unroll
          for (int u = 0; u < rows.value; ++u)
#pragma unroll
            for (int i = a * V / A; i < (a + 1) * V / A; ++i) {
              const float d = E::get(v[u].v[i]);
              t1 += d;
              t2 = fmaf(d, d, t2);
            }
          s1[a] += (double)t1;
          s2[a] += (double)t2;
        } else {
#pragma unroll
          for (int u = 0; u < rows.value; ++u)
#pragma unroll
            for (int i = a * V / A; i < (a + 1) * V / A; ++i) {
              const double d = E::get(v[u].v[i]);
              s1[a] += d;
              s2[a] = fma(d, d, s2[a]);
            }
        }
      }
    };
    int r = t.k * p.crows + rl;
    const typename E::type *xr = x + r * p.xs;
    const long long step = RL * p.xs;
    for (; r + (U - 1) * RL < r1; r += U * RL) {
      Pack<E, V> v[U];
#pragma unroll
      for (int u = 0; u < U; ++u, xr += step) v[u] = ld_pack<E, V>(xr);
#pragma unroll
      for (int u = 0; u < U; u += B) add(v + u, std::integral_constant<int, B>());
    }
    for (; r < r1; r += RL, xr += step) {
      const Pack<E, V> v = ld_pack<E, V>(xr);
      add(&v, std::integral_constant<int, 1>());
    }
  }
  // rows of a wave by lane exchanges, the waves through LDS
  for (int off = p.lanes; off < 64; off <<= 1)
#pragma unroll
    for (int i = 0; i < A; ++i) {
      s1[i] += __shfl_xor(s1[i], off, 64);
      s2[i] += __shfl_xor(s2[i], off, 64);
    }
  const int wave = threadIdx.x >> 6, cols = p.lanes * A;  // partial sums a wave: cols of (64 / lanes rows joined)
  if ((threadIdx.x & 63) < p.lanes)
#pragma unroll
    for (int i = 0; i < A; ++i) {
      red[(wave * cols + lane * A + i) * 2] = s1[i];
      red[(wave * cols + lane * A + i) * 2 + 1] = s2[i];
    }
  __syncthreads();
  if (threadIdx.x < 2 * cols) {
    double a = red[threadIdx.x];
#pragma unroll
    for (int w = 1; w < NW; ++w) a += red[w * 2 * cols + threadIdx.x];
    red[threadIdx.x] = a;
  }
  __syncthreads();
  const int g0 = t.c0 / p.Cg, g1 = (t.c0 + t.ct - 1) / p.Cg, step = V / A;
  for (int g = g0 + threadIdx.x; g <= g1; g += GN_TS) {
    const int a0 = max(g * p.Cg - t.c0, 0) / step, a1 = min((g + 1) * p.Cg - t.c0, t.ct) / step;
    double2 o = {0.0, 0.0};
    for (int c = a0; c < a1; ++c) {
      o.x += red[c * 2];
      o.y += red[c * 2 + 1];
    }
    *reinterpret_cast<double2 *>(p.part + (((long long)t.n * p.nchunk + t.k) * p.nslot + t.tile + g) * 2) = o;
  }
}

// ---- forward, second launch.  Q: checkpoints are written
template <class E, int V, int ACT, bool Q>
__global__ __launch_bounds__(GN_T) void gn_apply_kernel(GnP p) {
  constexpr int U = 4;
  __shared__ double st[2 * GN_CT];  // mean, rstd of the tile's groups
  const int piece = blockIdx.x / p.nchunk % p.split;
  const GnTile t = gn_tile(p, blockIdx.x / p.nchunk / p.split * p.nchunk + blockIdx.x % p.nchunk);
  const int g0 = t.c0 / p.Cg, ng = (t.c0 + t.ct - 1) / p.Cg - g0 + 1;
  int sub = 64;
  while (sub > 1 && ng * sub > GN_T) sub >>= 1;
  for (int i = threadIdx.x; i < ng * sub; i += GN_T) {
    const int g = g0 + i / sub;
    double a, q;
    gn_join(p, t.n, g, i % sub, sub, a, q);
    const double m = (double)p.S * p.Cg, mean = a / m, var = q / m - mean * mean;
    const double rstd = 1.0 / sqrt((var < 0.0 ? 0.0 : var) + (double)p.eps);  // (a NaN stays one)
    if (i % sub == 0) {
      st[(g - g0) * 2] = mean;
      st[(g - g0) * 2 + 1] = rstd;
      if (p.stats && t.k == 0 && piece == 0 && g * p.Cg >= t.c0) {  // the tile in which the group begins
        p.stats[((long long)t.n * p.G + g) * 2] = mean;
        p.stats[((long long)t.n * p.G + g) * 2 + 1] = rstd;
      }
    }
  }
  __syncthreads();
  const int lane = threadIdx.x & (p.lanes - 1), rl = threadIdx.x / p.lanes, RL = GN_T / p.lanes;
  const int c = t.c0 + lane * V;
  if (c >= p.nb * A8_BLOCK) return;    // whole 8-bit blocks leave together
  const bool in = lane * V < t.ct;     // the others of the last block write the checkpoints' padding
  float mu[V], sc[V], sh[V];
  double sc64[V], be64[V];  // LeakyReLU's kink in 64 bits, as the backward pass has it
  GnGroup at(c, p.Cg);
#pragma unroll
  for (int i = 0; i < V; ++i, at.next(p.Cg)) {
    mu[i] = sc[i] = sh[i] = 0.f;
    sc64[i] = be64[i] = 0.0;
    if (in) {
      const int g = at.g - g0;
      const double mean = st[g * 2], rstd = st[g * 2 + 1];
      const float ga = p.gamma[(long long)t.n * p.affn + c + i], be = p.beta[(long long)t.n * p.affn + c + i];
      mu[i] = (float)mean;
      sc[i] = ga * (float)rstd;
      sh[i] = (float)((double)be - (mean - (double)mu[i]) * rstd * (double)ga);
      sc64[i] = rstd * (double)ga;
      be64[i] = be;
    }
  }
  const int r1 = min(p.S, min((t.k + 1) * p.crows, t.k * p.crows + (piece + 1) * p.arows));
  int r = t.k * p.crows + piece * p.arows + rl;
  const typename E::type *x = reinterpret_cast<const typename E::type *>(p.x) + t.n * p.xn + r * p.xs + c;
  typename E::type *y = reinterpret_cast<typename E::type *>(p.y) + ((long long)t.n * p.S + r) * p.C + c;
  const long long xstep = RL * p.xs, ystep = (long long)RL * p.C;
  const long long row0 = (long long)t.n * p.S;
  const auto keep = [&](const float (&v)[V], unsigned char *q, unsigned char *e, long long row, bool kink) {
    const unsigned code = a8_code(a8_block_max<V>(v));
    float k[V];
    a8_round<V>(v, code, k);
    if (ACT == TBG_ACT_LRELU && kink) {  // one step back where rounding has crossed the kink: the backward pass takes the value's own slope
      const float scale = a8_scale(code);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float kept = (k[i] - A8_MAGIC) * scale;
        if ((fma((double)v[i], sc64[i], be64[i]) > 0.0) != (fma((double)kept, sc64[i], be64[i]) > 0.0))
          k[i] = fminf(fmaxf(k[i] + (v[i] > kept ? 1.f : -1.f), A8_MAGIC - 127.f), A8_MAGIC + 127.f);
      }
    }
    a8_store<V>(q + row * p.nb * A8_BLOCK + c, code, k);
    if ((c & (A8_BLOCK - 1)) == 0) e[row * p.nb + c / A8_BLOCK] = (unsigned char)code;
  };
  const auto write = [&](int row, const Pack<E, V> &v) {
    float d[V], o[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      d[i] = E::get(v.v[i]) - mu[i];
      o[i] = gn_act<ACT>(fmaf(d[i], sc[i], sh[i]));
    }
    const Pack<E, V> w = put_pack<E, V>(o);
    if (!Q || in) st_pack<E, V>(y, w);
    y += ystep;
    if constexpr (Q) {
#pragma unroll
      for (int i = 0; i < V; ++i) o[i] = in ? E::get(w.v[i]) : 0.f;  // (beyond the channels x and mu are 0 already)
      if (p.q) keep(d, p.q, p.e, row0 + row, true);
      if (p.yq) keep(o, p.yq, p.ye, row0 + row, false);
    }
  };
  if (!Q && !in) return;
  const Pack<E, V> zero = {};
  for (; r + (U - 1) * RL < r1; r += U * RL) {
    Pack<E, V> v[U];
#pragma unroll
    for (int u = 0; u < U; ++u, x += xstep) v[u] = in ? ld_pack<E, V>(x) : zero;
#pragma unroll
    for (int u = 0; u < U; ++u) write(r + u * RL, v[u]);
  }
  for (; r < r1; r += RL, x += xstep) write(r, in ? ld_pack<E, V>(x) : zero);
}

// ---- backward.  With d = x - mean (or its checkpoint), xh = d rstd: a lane keeps z = sc d + be of its V channels
template <int V>
struct GnCh {
  float mu[V], lo[V], sc[V], za[V], zb[V];  // za, zb: the same times -log2(e), for the exponential
  double sc64[V], be64[V];
};
template <int V, bool Q8>
__device__ __forceinline__ void gn_channels(const GnP &p, int n, int c, GnCh<V> &h) {
  GnGroup at(c, p.Cg);
#pragma unroll
  for (int i = 0; i < V; ++i, at.next(p.Cg)) {
    const double2 s = *reinterpret_cast<const double2 *>(p.stats + ((long long)n * p.G + at.g) * 2);
    const float ga = p.gamma[(long long)n * p.affn + c + i];
    h.mu[i] = Q8 ? 0.f : (float)s.x;
    h.lo[i] = Q8 ? 0.f : (float)(s.x - (double)(float)s.x);
    h.sc64[i] = s.y * (double)ga;
    h.sc[i] = (float)h.sc64[i];
    h.be64[i] = p.beta[(long long)n * p.affn + c + i];
    h.za[i] = (float)(-1.44269504088896341 * h.sc64[i]);
    h.zb[i] = (float)(-1.44269504088896341 * h.be64[i]);
  }
}
// a row's operands as they lie in memory
template <class E, int V, bool Q8>
struct GnRow {
  Pack<E, V> g, x;
  u32x2 q;
  unsigned e;
};
// where a lane stands, and a step of `rows` rows
template <class E, int V, bool Q8>
struct GnAt {
  const typename E::type *x, *g;
  const unsigned char *q, *e;
  __device__ __forceinline__ GnAt(const GnP &p, int n, int r, int c) {
    const long long row = (long long)n * p.S + r;
    x = reinterpret_cast<const typename E::type *>(p.x) + n * p.xn + r * p.xs + c;
    g = reinterpret_cast<const typename E::type *>(p.dy) + n * p.dn + r * p.ds + c;
    q = p.q + row * p.nb * A8_BLOCK + c;
    e = p.e + row * p.nb + c / A8_BLOCK;
  }
  __device__ __forceinline__ GnRow<E, V, Q8> next(const GnP &p, int rows) {
    GnRow<E, V, Q8> w;
    if constexpr (Q8) {
      w.e = *e;
      if constexpr (V == 8) w.q = *reinterpret_cast<const u32x2 *>(q);
      else w.q[0] = *q;
      q += (long long)rows * p.nb * A8_BLOCK;
      e += (long long)rows * p.nb;
    } else {
      w.x = ld_pack<E, V>(x);
      x += rows * p.xs;
    }
    w.g = ld_pack<E, V>(g);
    g += rows * p.ds;
    return w;
  }
};
// d and dz of a row
template <class E, int V, int ACT, bool Q8>
__device__ __forceinline__ void gn_row(const GnRow<E, V, Q8> &w, const GnCh<V> &h, float (&d)[V], float (&dz)[V]) {
  const float scale = Q8 ? a8_scale(w.e) : 1.f;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    if constexpr (Q8) d[i] = (float)(int)(signed char)(w.q[i >> 2] >> (8 * (i & 3)) & 0xff) * scale;
    else d[i] = (E::get(w.x.v[i]) - h.mu[i]) - h.lo[i];
    const float z = ACT == TBG_ACT_SILU ? fmaf(d[i], h.za[i], h.zb[i]) : 0.f;
    const bool pos = ACT == TBG_ACT_LRELU ? fma((double)d[i], h.sc64[i], h.be64[i]) > 0.0 : false;
    dz[i] = gn_dact<ACT>(E::get(w.g.v[i]), z, pos);
  }
}

// ---- backward, first launch: sums of dz and dz xh of every channel, and of gamma dz and gamma dz xh of every group
template <class E, int V, int ACT, bool Q8>
__global__ __launch_bounds__(GN_TB, V == 8 ? 4 : 8) void gn_bwd_sums_kernel(GnP p) {
  constexpr int U = 2, NW = GN_TB / 64;
  __shared__ float red[NW * GN_CT * 2];
  const GnTile t = gn_tile(p, blockIdx.x);
  const int lane = threadIdx.x & (p.lanes - 1), rl = threadIdx.x / p.lanes, RL = GN_TB / p.lanes;
  const int r1 = min(p.S, (t.k + 1) * p.crows), c = t.c0 + lane * V;
  float s1[V], s2[V];
#pragma unroll
  for (int i = 0; i < V; ++i) s1[i] = s2[i] = 0.f;
  if (lane * V < t.ct) {
    GnCh<V> h;
    gn_channels<V, Q8>(p, t.n, c, h);
    const auto add = [&](const GnRow<E, V, Q8> &w) {
      float d[V], dz[V];
      gn_row<E, V, ACT, Q8>(w, h, d, dz);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        s1[i] += dz[i];
        s2[i] = fmaf(dz[i], d[i], s2[i]);
      }
    };
    int r = t.k * p.crows + rl;
    GnAt<E, V, Q8> at(p, t.n, r, c);
    for (; r + (U - 1) * RL < r1; r += U * RL) {
      GnRow<E, V, Q8> w[U];
#pragma unroll
      for (int u = 0; u < U; ++u) w[u] = at.next(p, RL);
#pragma unroll
      for (int u = 0; u < U; ++u) add(w[u]);
    }
    for (; r < r1; r += RL) add(at.next(p, RL));
  }
  for (int off = p.lanes; off < 64; off <<= 1)
#pragma unroll
    for (int i = 0; i < V; ++i) {
      s1[i] += __shfl_xor(s1[i], off, 64);
      s2[i] += __shfl_xor(s2[i], off, 64);
    }
  const int wave = threadIdx.x >> 6;
  if ((threadIdx.x & 63) < p.lanes)
#pragma unroll
    for (int i = 0; i < V; ++i) {
      red[(wave * p.CT + lane * V + i) * 2] = s1[i];
      red[(wave * p.CT + lane * V + i) * 2 + 1] = s2[i];
    }
  __syncthreads();
  if (threadIdx.x < 2 * t.ct) {
    float a = red[threadIdx.x];
#pragma unroll
    for (int w = 1; w < NW; ++w) a += red[w * 2 * p.CT + threadIdx.x];
    if (threadIdx.x & 1) a *= (float)p.stats[((long long)t.n * p.G + (t.c0 + (threadIdx.x >> 1)) / p.Cg) * 2 + 1];  // d -> xh
    red[threadIdx.x] = a;
    p.pch[(((long long)t.n * p.nchunk + t.k) * p.C + t.c0) * 2 + threadIdx.x] = a;
  }
  __syncthreads();
  const int g0 = t.c0 / p.Cg, g1 = (t.c0 + t.ct - 1) / p.Cg;
  for (int g = g0 + threadIdx.x; g <= g1; g += GN_TB) {
    const int a0 = max(g * p.Cg - t.c0, 0), a1 = min((g + 1) * p.Cg - t.c0, t.ct);
    double2 o = {0.0, 0.0};
    for (int j = a0; j < a1; ++j) {
      const double ga = p.gamma[(long long)t.n * p.affn + t.c0 + j];
      o.x = fma(ga, (double)red[j * 2], o.x);
      o.y = fma(ga, (double)red[j * 2 + 1], o.y);
    }
    *reinterpret_cast<double2 *>(p.part + (((long long)t.n * p.nchunk + t.k) * p.nslot + t.tile + g) * 2) = o;
  }
}

// ---- backward, second launch: dx, and in its first blocks dgamma / dbeta
template <class E, int V, int ACT, bool Q8>
__global__ __launch_bounds__(GN_T, V == 8 ? 4 : 8) void gn_bwd_dx_kernel(GnP p) {
  constexpr int U = 2;
  __shared__ double st[2 * GN_CT];  // of the tile's groups: rstd mean(gamma dz), rstd^2 mean(gamma dz xh)
  int b = blockIdx.x;
  if (b < p.pblocks) {  // 8 lanes a channel: the row ranges (and samples, where the parameters are shared) in a fixed order
    const long long idx = (long long)b * (GN_T / 8) + threadIdx.x / 8;
    const int sub = threadIdx.x & 7;
    const long long count = p.affn ? (long long)p.N * p.C : p.C;
    if (idx < count) {
      const int n = p.affn ? (int)(idx / p.C) : 0, c = (int)(idx % p.C);
      const long long len = (long long)(p.affn ? 1 : p.N) * p.nchunk;
      double a = 0.0, q = 0.0;
      for (long long i = sub; i < len; i += 8) {
        const float2 s = *reinterpret_cast<const float2 *>(p.pch + (((long long)n * p.nchunk + i) * p.C + c) * 2);
        a += s.x;
        q += s.y;
      }
#pragma unroll
      for (int off = 4; off > 0; off >>= 1) {
        a += __shfl_xor(a, off, 64);
        q += __shfl_xor(q, off, 64);
      }
      if (sub == 0) {
        p.dbeta[idx] = (float)a;
        p.dgamma[idx] = (float)q;
      }
    }
    return;
  }
  b -= p.pblocks;
  const int piece = b / p.nchunk % p.split;
  const GnTile t = gn_tile(p, b / p.nchunk / p.split * p.nchunk + b % p.nchunk);
  const int g0 = t.c0 / p.Cg, ng = (t.c0 + t.ct - 1) / p.Cg - g0 + 1;
  int sub = 64;
  while (sub > 1 && ng * sub > GN_T) sub >>= 1;
  for (int i = threadIdx.x; i < ng * sub; i += GN_T) {
    double a, q;
    gn_join(p, t.n, g0 + i / sub, i % sub, sub, a, q);
    const double m = (double)p.S * p.Cg;
    if (i % sub == 0) {
      const double rstd = p.stats[((long long)t.n * p.G + g0 + i / sub) * 2 + 1];
      st[(i / sub) * 2] = rstd * (a / m);
      st[(i / sub) * 2 + 1] = rstd * rstd * (q / m);
    }
  }
  __syncthreads();
  const int lane = threadIdx.x & (p.lanes - 1), rl = threadIdx.x / p.lanes, RL = GN_T / p.lanes;
  if (lane * V >= t.ct) return;
  const int c = t.c0 + lane * V;
  GnCh<V> h;
  gn_channels<V, Q8>(p, t.n, c, h);
  float m1[V], m2[V];  // dx = sc dz - m1 - d m2
  GnGroup cg(c, p.Cg);
#pragma unroll
  for (int i = 0; i < V; ++i, cg.next(p.Cg)) {
    m1[i] = (float)st[(cg.g - g0) * 2];
    m2[i] = (float)st[(cg.g - g0) * 2 + 1];
  }
  const int r1 = min(p.S, min((t.k + 1) * p.crows, t.k * p.crows + (piece + 1) * p.arows));
  int r = t.k * p.crows + piece * p.arows + rl;
  GnAt<E, V, Q8> at(p, t.n, r, c);
  typename E::type *dx = reinterpret_cast<typename E::type *>(p.y) + ((long long)t.n * p.S + r) * p.C + c;
  const auto write = [&](const GnRow<E, V, Q8> &w) {
    float d[V], dz[V];
    gn_row<E, V, ACT, Q8>(w, h, d, dz);
#pragma unroll
    for (int i = 0; i < V; ++i) dz[i] = fmaf(-d[i], m2[i], fmaf(dz[i], h.sc[i], -m1[i]));
    st_pack<E, V>(dx, put_pack<E, V>(dz));
    dx += (long long)RL * p.C;
  };
  for (; r + (U - 1) * RL < r1; r += U * RL) {
    GnRow<E, V, Q8> w[U];
#pragma unroll
    for (int u = 0; u < U; ++u) w[u] = at.next(p, RL);
#pragma unroll
    for (int u = 0; u < U; ++u) write(w[u]);
  }
  for (; r < r1; r += RL) write(at.next(p, RL));
}

// ---- host side
// What a call runs is a function of the descriptor and the pointers' alignment.  The workspace holds for either alignment.
static bool gn_desc_ok(const tbg_gn_desc *d) {
  return d && d->N >= 1 && d->S >= 1 && d->C >= 1 && d->G >= 1 && d->C % d->G == 0 && dt_valid(d->dtype) && d->act >= TBG_ACT_LINEAR &&
         d->act <= TBG_ACT_SILU && (d->per_sample == 0 || d->per_sample == 1) && d->eps > 0.f && d->xs >= d->C && d->xn >= 0 && d->ds >= d->C && d->dn >= 0;
}
// Row ranges: the sums launch has at most 32 a tile (64 where the samples and tiles are few), each joined by every block of the second
// launch that needs it; that launch cuts them into pieces for about 8 blocks a CU, of 8 rows a lane or more.
static int gn_geometry(const tbg_gn_desc *d, bool vec, bool backward, GnP &p) {
  if (d->S > (1 << 30) || d->C > (1 << 24)) return TBG_ERANGE;
  const int V = vec ? 8 : 1;
  p.N = d->N; p.S = d->S; p.C = d->C; p.G = d->G; p.Cg = d->C / d->G; p.affn = d->per_sample ? d->C : 0;
  p.nb = (d->C + A8_BLOCK - 1) / A8_BLOCK;
  p.xn = d->xn; p.xs = d->xs; p.dn = d->dn; p.ds = d->ds; p.eps = d->eps;
  // the tile (a power of two; a row's 8-bit block never spans two) that leaves the fewest lanes without channels
  const int padded = p.nb * A8_BLOCK;
  p.CT = 0;
  for (int ct = vec ? GN_CT : 64, best = 0; ct >= 32; ct >>= 1) {
    const int used = (int)(1000LL * padded / ((long long)(padded + ct - 1) / ct * ct));
    if (used > best && (ct > 32 || padded == 32 || !p.CT)) { best = used; p.CT = ct; }
  }
  p.ntile = (d->C + p.CT - 1) / p.CT;
  p.lanes = p.CT / V;
  p.nslot = p.ntile + p.G - 1;
  const int RL = (backward ? GN_TB : GN_TS) / p.lanes, RA = GN_T / p.lanes;
  const long long tiles = (long long)p.N * p.ntile;
  long long want = 512 / tiles;
  const long long cap = tiles < 8 ? 64 : 32, most = (p.S + 4LL * RL - 1) / (4LL * RL);
  want = want > cap ? cap : want;
  want = want > most ? most : want;
  if (want >= 8) want &= ~7LL;
  if (want < 1) want = 1;
  long long rows = (p.S + want - 1) / want;
  p.crows = (int)((rows + RL - 1) / RL * RL);
  p.nchunk = (int)((p.S + p.crows - 1LL) / p.crows);
  long long split = GN_BLOCKS / (tiles * p.nchunk);
  const long long least = p.crows / (8LL * RA);
  split = split > least ? least : split;
  if (split < 1) split = 1;
  p.arows = (int)(((p.crows + split - 1) / split + RA - 1) / RA * RA);
  p.split = (p.crows + p.arows - 1) / p.arows;
  const long long count = d->per_sample ? (long long)d->N * d->C : d->C;
  if (tiles * p.nchunk * p.split > 0x3fffffffLL || count > 0x3fffffffLL) return TBG_ERANGE;
  p.pblocks = (int)((count + GN_T / 8 - 1) / (GN_T / 8));
  return TBG_OK;
}
static long long gn_part_bytes(const GnP &p) { return (long long)p.N * p.nchunk * p.nslot * 2 * (long long)sizeof(double); }
static long long gn_pch_bytes(const GnP &p) { return (long long)p.N * p.nchunk * p.C * 2 * (long long)sizeof(float); }

extern "C" long long tbg_group_norm_workspace_bytes(const tbg_gn_desc *d, int backward) {
  if (!gn_desc_ok(d)) return TBG_EINVAL;
  long long most = 0;
  for (int vec = 0; vec < 2; ++vec) {
    GnP p{};
    if (const int rc = gn_geometry(d, vec != 0, backward != 0, p)) return rc;
    const long long b = gn_part_bytes(p) + (backward ? gn_pch_bytes(p) : 0);
    if (b > most) most = b;
  }
  return most;
}

template <class E, int V, int ACT>
static int gn_run_fwd(const GnP &p, hipStream_t st) {
  const auto sums = V == 1 || p.Cg % 8 == 0 ? gn_sums_kernel<E, V, 1>
                    : p.Cg % 4 == 0 ? gn_sums_kernel<E, V, V == 8 ? 2 : 1>
                    : p.Cg % 2 == 0 ? gn_sums_kernel<E, V, V == 8 ? 4 : 1> : gn_sums_kernel<E, V, V>;
  const auto apply = p.q || p.yq ? gn_apply_kernel<E, V, ACT, true> : gn_apply_kernel<E, V, ACT, false>;
  hipLaunchKernelGGL(sums, dim3(p.N * p.ntile * p.nchunk), dim3(GN_TS), 0, st, p);
  TBG_LAUNCH_CHECK();
  hipLaunchKernelGGL(apply, dim3(p.N * p.ntile * p.nchunk * p.split), dim3(GN_T), 0, st, p);
  TBG_LAUNCH_CHECK();
  return TBG_OK;
}
template <class E, int V, int ACT, bool Q8>
static int gn_run_bwd(const GnP &p, hipStream_t st) {
  hipLaunchKernelGGL((gn_bwd_sums_kernel<E, V, ACT, Q8>), dim3(p.N * p.ntile * p.nchunk), dim3(GN_TB), 0, st, p);
  TBG_LAUNCH_CHECK();
  hipLaunchKernelGGL((gn_bwd_dx_kernel<E, V, ACT, Q8>), dim3(p.pblocks + p.N * p.ntile * p.nchunk * p.split), dim3(GN_T), 0, st, p);
  TBG_LAUNCH_CHECK();
  return TBG_OK;
}
template <class E, int V, int ACT>
static int gn_run(const GnP &p, bool backward, hipStream_t st) {
  if (!backward) return gn_run_fwd<E, V, ACT>(p, st);
  return p.q ? gn_run_bwd<E, V, ACT, true>(p, st) : gn_run_bwd<E, V, ACT, false>(p, st);
}
template <class E>
static int gn_run_type(const GnP &p, bool vec, int act, bool backward, hipStream_t st) {
  if (vec)
    return act == TBG_ACT_LINEAR ? gn_run<E, 8, TBG_ACT_LINEAR>(p, backward, st)
           : act == TBG_ACT_LRELU ? gn_run<E, 8, TBG_ACT_LRELU>(p, backward, st)
                                  : gn_run<E, 8, TBG_ACT_SILU>(p, backward, st);
  return act == TBG_ACT_LINEAR ? gn_run<E, 1, TBG_ACT_LINEAR>(p, backward, st)
         : act == TBG_ACT_LRELU ? gn_run<E, 1, TBG_ACT_LRELU>(p, backward, st)
                                : gn_run<E, 1, TBG_ACT_SILU>(p, backward, st);
}
static int gn_dispatch(const tbg_gn_desc *d, const GnP &p, bool vec, bool backward, void *stream) {
  hipStream_t st = tbg_stream(stream);
  return d->dtype == TBG_DT_F32 ? gn_run_type<ElF32>(p, vec, d->act, backward, st)
         : d->dtype == TBG_DT_BF16 ? gn_run_type<ElBf16>(p, vec, d->act, backward, st)
                                   : gn_run_type<ElF16>(p, vec, d->act, backward, st);
}
static bool gn_misaligned(const void *a, const void *b) { return ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b)) & 15) != 0; }

extern "C" int tbg_group_norm_fwd(const tbg_gn_desc *d, const void *x, const float *gamma, const float *beta, void *y, double *stats,
                                  void *q, void *e, void *yq, void *ye, void *workspace, long long workspace_bytes, void *stream) {
  if (!gn_desc_ok(d) || !x || !gamma || !beta || !y || !workspace || (q == nullptr) != (e == nullptr) || (yq == nullptr) != (ye == nullptr))
    return TBG_EINVAL;
  if (gn_misaligned(q, yq) || gn_misaligned(workspace, stats)) return TBG_EINVAL;
  const bool vec = d->C % 8 == 0 && vec8_ok(x, d->dtype, d->xs, d->xn) && vec8_ok(y, d->dtype, d->C);
  GnP p{};
  if (const int rc = gn_geometry(d, vec, false, p)) return rc;
  if (gn_part_bytes(p) > workspace_bytes) return TBG_EINVAL;
  p.x = x; p.gamma = gamma; p.beta = beta; p.y = y; p.stats = stats; p.part = reinterpret_cast<double *>(workspace);
  p.q = reinterpret_cast<unsigned char *>(q); p.e = reinterpret_cast<unsigned char *>(e);
  p.yq = reinterpret_cast<unsigned char *>(yq); p.ye = reinterpret_cast<unsigned char *>(ye);
  return gn_dispatch(d, p, vec, false, stream);
}

extern "C" int tbg_group_norm_bwd(const tbg_gn_desc *d, const void *x, const void *q, const void *e, const void *dy, const float *gamma,
                                  const float *beta, const double *stats, void *dx, float *dgamma, float *dbeta, void *workspace,
                                  long long workspace_bytes, void *stream) {
  if (!gn_desc_ok(d) || !dy || !gamma || !beta || !stats || !dx || !dgamma || !dbeta || !workspace || (q == nullptr) != (e == nullptr) ||
      (x == nullptr) == (q == nullptr))
    return TBG_EINVAL;
  if (gn_misaligned(q, workspace) || gn_misaligned(stats, nullptr)) return TBG_EINVAL;
  const bool vec = d->C % 8 == 0 && (!x || vec8_ok(x, d->dtype, d->xs, d->xn)) && vec8_ok(dy, d->dtype, d->ds, d->dn) && vec8_ok(dx, d->dtype, d->C);
  GnP p{};
  if (const int rc = gn_geometry(d, vec, true, p)) return rc;
  if (gn_part_bytes(p) + gn_pch_bytes(p) > workspace_bytes) return TBG_EINVAL;
  p.x = x; p.dy = dy; p.gamma = gamma; p.beta = beta; p.y = dx; p.stats = const_cast<double *>(stats);
  p.q = const_cast<unsigned char *>(reinterpret_cast<const unsigned char *>(q));
  p.e = const_cast<unsigned char *>(reinterpret_cast<const unsigned char *>(e));
  p.part = reinterpret_cast<double *>(workspace);
  p.pch = reinterpret_cast<float *>(reinterpret_cast<char *>(workspace) + gn_part_bytes(p));
  p.dgamma = dgamma; p.dbeta = dbeta;
  return gn_dispatch(d, p, vec, true, stream);
}
