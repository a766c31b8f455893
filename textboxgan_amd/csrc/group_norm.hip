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
// The statistics are 64-bit sums of x and x^2 (fp64 adds run at half the fp32 rate here, far from the bound of a streaming pass): one pass,
// and mean(x^2) - mean^2 loses nothing that matters even for |mean| = 10^5 standard deviations.  The mean is used as fp32 + its remainder.
#include "act8.h"

struct GnP {
  const void *x, *dy;
  const float *gamma, *beta;
  void *y;                             // forward: output; backward: dx
  unsigned char *q, *e;                // checkpoint of x - mean (written forward, read backward), or null
  unsigned char *yq, *ye;              // forward: checkpoint of y, or null
  double *stats;                       // [N][G][2] mean, rstd
  double *part;                        // forward: [N][nchunk][nslot][2] sum x, sum x^2; backward: sum gamma dz, sum gamma dz xh
  float *pch;                          // backward: [N][nchunk][Cp][2] sum dz, sum dz xh of a channel
  float *dgamma, *dbeta;
  long long xn, xs, dn, ds;            // sample / row pitches of x and dy in elements (y, dx: contiguous)
  int N, S, C, G, Cg, affn, nb;        // affn: affine parameters' sample pitch (0 or C); nb: 8-bit blocks a row
  int CT, ntile, lanes, RL;            // channels a tile, tiles, lanes a row, rows a pass
  int nchunk, crows, nslot;            // row ranges of the sums launch
  int achunk, arows;                   // row ranges of the second launch
  int pblocks;                         // backward: first blocks of the second launch that sum dgamma / dbeta
  float eps;
};

constexpr int GN_T = 256, GN_CT = 128;  // threads a block, most channels a tile

template <int ACT>
__device__ __forceinline__ float gn_act(float z) {
  if constexpr (ACT == TBG_ACT_LRELU) return 1.41421356237309515f * (z > 0.f ? z : 0.2f * z);
  if constexpr (ACT == TBG_ACT_SILU) return z / (1.f + __expf(-z));
  return z;
}
// dy act'(z).  z64: LeakyReLU's side of the kink is decided in 64 bits, so that it does not hang on the last bit of a 32-bit product
template <int ACT>
__device__ __forceinline__ float gn_dact(float dy, float z, bool positive) {
  if constexpr (ACT == TBG_ACT_LRELU) return dy * (positive ? 1.41421356237309515f : 0.282842712474619f);
  if constexpr (ACT == TBG_ACT_SILU) {
    const float s = 1.f / (1.f + __expf(-z));
    return dy * (s * (1.f + z * (1.f - s)));
  }
  return dy;
}

// sums of one group's partial pairs over its tiles and the row ranges, by `sub` neighbouring lanes (a power of two), all of which get it
__device__ __forceinline__ void gn_join(const GnP &p, int n, int g, int lane, int sub, double &a, double &b) {
  const int t0 = g * p.Cg / p.CT, t1 = ((g + 1) * p.Cg - 1) / p.CT, nt = t1 - t0 + 1;
  a = b = 0.0;
  const double *base = p.part + (long long)n * p.nchunk * p.nslot * 2;
  for (int i = lane; i < nt * p.nchunk; i += sub) {
    const int k = i / nt, t = t0 + i - k * nt;
    const double *s = base + ((long long)k * p.nslot + t + g) * 2;
    a += s[0];
    b += s[1];
  }
  for (int off = sub >> 1; off > 0; off >>= 1) {
    a += __shfl_xor(a, off, 64);
    b += __shfl_xor(b, off, 64);
  }
}

// ---- forward, first launch: sums of x and x^2
template <class E, int V>
__global__ __launch_bounds__(GN_T) void gn_sums_kernel(GnP p) {
  __shared__ double red[GN_T * V * 2];
  int b = blockIdx.x;
  const int k = b % p.nchunk; b /= p.nchunk;
  const int tile = b % p.ntile, n = b / p.ntile;
  const int c0 = tile * p.CT, ct = min(p.CT, p.C - c0);
  const int lane = threadIdx.x % p.lanes, rl = threadIdx.x / p.lanes;
  const int r0 = k * p.crows, r1 = min(p.S, r0 + p.crows);
  double s1[V], s2[V];
#pragma unroll
  for (int i = 0; i < V; ++i) s1[i] = s2[i] = 0.0;
  if (rl < p.RL && lane * V < ct) {
    const typename E::type *x = reinterpret_cast<const typename E::type *>(p.x) + n * p.xn + c0 + lane * V;
#pragma unroll 4
    for (int r = r0 + rl; r < r1; r += p.RL) {
      const Pack<E, V> v = ld_pack<E, V>(x + r * p.xs);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const double d = E::get(v.v[i]);
        s1[i] += d;
        s2[i] = fma(d, d, s2[i]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < V; ++i) {
    red[(threadIdx.x * V + i) * 2] = s1[i];
    red[(threadIdx.x * V + i) * 2 + 1] = s2[i];
  }
  __syncthreads();
  const int row = p.lanes * V;  // channels of one row lane in `red`
  for (int c = threadIdx.x; c < ct; c += GN_T) {
    double a = red[c * 2], q = red[c * 2 + 1];
    for (int j = 1; j < p.RL; ++j) {
      a += red[(j * row + c) * 2];
      q += red[(j * row + c) * 2 + 1];
    }
    red[c * 2] = a;
    red[c * 2 + 1] = q;
  }
  __syncthreads();
  const int g0 = c0 / p.Cg, g1 = (c0 + ct - 1) / p.Cg;
  for (int g = g0 + threadIdx.x; g <= g1; g += GN_T) {
    const int a0 = max(g * p.Cg - c0, 0), a1 = min((g + 1) * p.Cg - c0, ct);
    double a = 0.0, q = 0.0;
    for (int c = a0; c < a1; ++c) {
      a += red[c * 2];
      q += red[c * 2 + 1];
    }
    double *o = p.part + (((long long)n * p.nchunk + k) * p.nslot + tile + g) * 2;
    o[0] = a;
    o[1] = q;
  }
}

// ---- forward, second launch
template <class E, int V, int ACT>
__global__ __launch_bounds__(GN_T) void gn_apply_kernel(GnP p) {
  __shared__ double st[2 * GN_CT];  // mean, rstd of the tile's groups
  int b = blockIdx.x;
  const int k = b % p.achunk; b /= p.achunk;
  const int tile = b % p.ntile, n = b / p.ntile;
  const int c0 = tile * p.CT, ct = min(p.CT, p.C - c0);
  const int g0 = c0 / p.Cg, ng = (c0 + ct - 1) / p.Cg - g0 + 1;
  int sub = 64;
  while (sub > 1 && ng * sub > GN_T) sub >>= 1;
  for (int i = threadIdx.x; i < ng * sub; i += GN_T) {
    const int g = g0 + i / sub;
    double a, q;
    gn_join(p, n, g, i % sub, sub, a, q);
    const double m = (double)p.S * p.Cg, mean = a / m, var = q / m - mean * mean;
    const double rstd = 1.0 / sqrt((var < 0.0 ? 0.0 : var) + (double)p.eps);  // (a NaN stays one)
    if (i % sub == 0) {
      st[(g - g0) * 2] = mean;
      st[(g - g0) * 2 + 1] = rstd;
      if (p.stats && k == 0 && g * p.Cg >= c0) {  // the tile in which the group begins
        p.stats[((long long)n * p.G + g) * 2] = mean;
        p.stats[((long long)n * p.G + g) * 2 + 1] = rstd;
      }
    }
  }
  __syncthreads();
  const int lane = threadIdx.x % p.lanes, rl = threadIdx.x / p.lanes;
  const int c = c0 + lane * V;
  if (rl >= p.RL || c >= p.nb * A8_BLOCK) return;  // whole 8-bit blocks leave together
  const bool in = lane * V < ct;                   // the others of the last block write the checkpoints' padding
  float mu[V], sc[V], sh[V];
  double sc64[V], be64[V];  // LeakyReLU's kink in 64 bits, as the backward pass has it
#pragma unroll
  for (int i = 0; i < V; ++i) {
    mu[i] = sc[i] = sh[i] = 0.f;
    sc64[i] = be64[i] = 0.0;
    if (in) {
      const int g = (c + i) / p.Cg - g0;
      const double mean = st[g * 2], rstd = st[g * 2 + 1];
      const float ga = p.gamma[(long long)n * p.affn + c + i], be = p.beta[(long long)n * p.affn + c + i];
      mu[i] = (float)mean;
      sc[i] = ga * (float)rstd;
      sh[i] = (float)((double)be - (mean - (double)mu[i]) * rstd * (double)ga);
      sc64[i] = rstd * (double)ga;
      be64[i] = be;
    }
  }
  const typename E::type *x = reinterpret_cast<const typename E::type *>(p.x) + n * p.xn + c;
  typename E::type *y = reinterpret_cast<typename E::type *>(p.y) + (long long)n * p.S * p.C + c;
  const int r1 = min(p.S, (k + 1) * p.arows);
#pragma unroll 2
  for (int r = k * p.arows + rl; r < r1; r += p.RL) {
    float d[V], o[V];
#pragma unroll
    for (int i = 0; i < V; ++i) d[i] = o[i] = 0.f;
    if (in) {
      const Pack<E, V> v = ld_pack<E, V>(x + r * p.xs);
      Pack<E, V> w;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        d[i] = E::get(v.v[i]) - mu[i];
        w.v[i] = E::put(gn_act<ACT>(fmaf(d[i], sc[i], sh[i])));
        o[i] = E::get(w.v[i]);
      }
      st_pack<E, V>(y + (long long)r * p.C, w);
    }
    const long long row = (long long)n * p.S + r;
    if (p.q) {
      const unsigned code = a8_code(a8_block_max<V>(d));
      float t[V];
      a8_round<V>(d, code, t);
      if constexpr (ACT == TBG_ACT_LRELU) {  // one step back where rounding has crossed the kink: the backward pass takes the value's own slope
        const float scale = a8_scale(code);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float kept = t[i] * scale;
          if ((fma((double)d[i], sc64[i], be64[i]) > 0.0) != (fma((double)kept, sc64[i], be64[i]) > 0.0))
            t[i] = fminf(fmaxf(t[i] + (d[i] > kept ? 1.f : -1.f), -127.f), 127.f);
        }
      }
      a8_store<V>(p.q + row * p.nb * A8_BLOCK + c, t);
      if ((c & (A8_BLOCK - 1)) == 0) p.e[row * p.nb + c / A8_BLOCK] = (unsigned char)code;
    }
    if (p.yq) {
      const unsigned code = a8_code(a8_block_max<V>(o));
      float t[V];
      a8_round<V>(o, code, t);
      a8_store<V>(p.yq + row * p.nb * A8_BLOCK + c, t);
      if ((c & (A8_BLOCK - 1)) == 0) p.ye[row * p.nb + c / A8_BLOCK] = (unsigned char)code;
    }
  }
}

// ---- backward: what a lane knows of its V channels
template <int V>
struct GnCh {
  float mu[V], lo[V], rstd[V], ga[V], be[V];
  double sc64[V];
};
template <int V, bool Q8>
__device__ __forceinline__ void gn_channels(const GnP &p, int n, int c, bool in, GnCh<V> &h) {
#pragma unroll
  for (int i = 0; i < V; ++i) {
    h.mu[i] = h.lo[i] = h.rstd[i] = h.ga[i] = h.be[i] = 0.f;
    h.sc64[i] = 0.0;
    if (in) {
      const double *s = p.stats + ((long long)n * p.G + (c + i) / p.Cg) * 2;
      h.mu[i] = Q8 ? 0.f : (float)s[0];
      h.lo[i] = Q8 ? 0.f : (float)(s[0] - (double)(float)s[0]);
      h.rstd[i] = (float)s[1];
      h.ga[i] = p.gamma[(long long)n * p.affn + c + i];
      h.be[i] = p.beta[(long long)n * p.affn + c + i];
      h.sc64[i] = s[1] * (double)h.ga[i];
    }
  }
}
// xh and dz of one row
template <class E, int V, int ACT, bool Q8>
__device__ __forceinline__ void gn_row(const GnP &p, const GnCh<V> &h, int n, int r, int c, float (&xh)[V], float (&dz)[V]) {
  float d[V];
  if constexpr (Q8) {
    const long long row = (long long)n * p.S + r;
    a8_load<V>(p.q + row * p.nb * A8_BLOCK + c, a8_scale(p.e[row * p.nb + c / A8_BLOCK]), d);
  } else {
    const Pack<E, V> v = ld_pack<E, V>(reinterpret_cast<const typename E::type *>(p.x) + n * p.xn + r * p.xs + c);
#pragma unroll
    for (int i = 0; i < V; ++i) d[i] = (E::get(v.v[i]) - h.mu[i]) - h.lo[i];
  }
  const Pack<E, V> g = ld_pack<E, V>(reinterpret_cast<const typename E::type *>(p.dy) + n * p.dn + r * p.ds + c);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    xh[i] = d[i] * h.rstd[i];
    const float z = fmaf(xh[i], h.ga[i], h.be[i]);
    const bool pos = ACT == TBG_ACT_LRELU ? fma((double)d[i], h.sc64[i], (double)h.be[i]) > 0.0 : false;
    dz[i] = gn_dact<ACT>(E::get(g.v[i]), z, pos);
  }
}

// ---- backward, first launch: sums of dz and dz xh of every channel, and of gamma dz and gamma dz xh of every group
template <class E, int V, int ACT, bool Q8>
__global__ __launch_bounds__(GN_T) void gn_bwd_sums_kernel(GnP p) {
  __shared__ float red[GN_T * V * 2];
  int b = blockIdx.x;
  const int k = b % p.nchunk; b /= p.nchunk;
  const int tile = b % p.ntile, n = b / p.ntile;
  const int c0 = tile * p.CT, ct = min(p.CT, p.C - c0);
  const int lane = threadIdx.x % p.lanes, rl = threadIdx.x / p.lanes;
  const int r1 = min(p.S, (k + 1) * p.crows), c = c0 + lane * V;
  float s1[V], s2[V];
#pragma unroll
  for (int i = 0; i < V; ++i) s1[i] = s2[i] = 0.f;
  if (rl < p.RL && lane * V < ct) {
    GnCh<V> h;
    gn_channels<V, Q8>(p, n, c, true, h);
#pragma unroll 2
    for (int r = k * p.crows + rl; r < r1; r += p.RL) {
      float xh[V], dz[V];
      gn_row<E, V, ACT, Q8>(p, h, n, r, c, xh, dz);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        s1[i] += dz[i];
        s2[i] = fmaf(dz[i], xh[i], s2[i]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < V; ++i) {
    red[(threadIdx.x * V + i) * 2] = s1[i];
    red[(threadIdx.x * V + i) * 2 + 1] = s2[i];
  }
  __syncthreads();
  const int row = p.lanes * V;
  for (int j = threadIdx.x; j < ct; j += GN_T) {
    float a = red[j * 2], q = red[j * 2 + 1];
    for (int l = 1; l < p.RL; ++l) {
      a += red[(l * row + j) * 2];
      q += red[(l * row + j) * 2 + 1];
    }
    red[j * 2] = a;
    red[j * 2 + 1] = q;
    float *o = p.pch + (((long long)n * p.nchunk + k) * p.C + c0 + j) * 2;
    o[0] = a;
    o[1] = q;
  }
  __syncthreads();
  const int g0 = c0 / p.Cg, g1 = (c0 + ct - 1) / p.Cg;
  for (int g = g0 + threadIdx.x; g <= g1; g += GN_T) {
    const int a0 = max(g * p.Cg - c0, 0), a1 = min((g + 1) * p.Cg - c0, ct);
    double a = 0.0, q = 0.0;
    for (int j = a0; j < a1; ++j) {
      const double ga = p.gamma[(long long)n * p.affn + c0 + j];
      a = fma(ga, (double)red[j * 2], a);
      q = fma(ga, (double)red[j * 2 + 1], q);
    }
    double *o = p.part + (((long long)n * p.nchunk + k) * p.nslot + tile + g) * 2;
    o[0] = a;
    o[1] = q;
  }
}

// ---- backward, second launch: dx, and in its first blocks dgamma / dbeta
template <class E, int V, int ACT, bool Q8>
__global__ __launch_bounds__(GN_T) void gn_bwd_dx_kernel(GnP p) {
  __shared__ double st[2 * GN_CT];  // means of gamma dz and gamma dz xh over the tile's groups
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
        const float *s = p.pch + (((long long)n * p.nchunk + i) * p.C + c) * 2;
        a += s[0];
        q += s[1];
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
  const int k = b % p.achunk; b /= p.achunk;
  const int tile = b % p.ntile, n = b / p.ntile;
  const int c0 = tile * p.CT, ct = min(p.CT, p.C - c0);
  const int g0 = c0 / p.Cg, ng = (c0 + ct - 1) / p.Cg - g0 + 1;
  int sub = 64;
  while (sub > 1 && ng * sub > GN_T) sub >>= 1;
  for (int i = threadIdx.x; i < ng * sub; i += GN_T) {
    double a, q;
    gn_join(p, n, g0 + i / sub, i % sub, sub, a, q);
    const double m = (double)p.S * p.Cg;
    if (i % sub == 0) {
      st[(i / sub) * 2] = a / m;
      st[(i / sub) * 2 + 1] = q / m;
    }
  }
  __syncthreads();
  const int lane = threadIdx.x % p.lanes, rl = threadIdx.x / p.lanes;
  if (rl >= p.RL || lane * V >= ct) return;
  const int c = c0 + lane * V;
  GnCh<V> h;
  gn_channels<V, Q8>(p, n, c, true, h);
  float m1[V], m2[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int g = (c + i) / p.Cg - g0;
    m1[i] = (float)st[g * 2];
    m2[i] = (float)st[g * 2 + 1];
  }
  typename E::type *dx = reinterpret_cast<typename E::type *>(p.y) + (long long)n * p.S * p.C + c;
  const int r1 = min(p.S, (k + 1) * p.arows);
#pragma unroll 2
  for (int r = k * p.arows + rl; r < r1; r += p.RL) {
    float xh[V], dz[V];
    gn_row<E, V, ACT, Q8>(p, h, n, r, c, xh, dz);
    Pack<E, V> w;
#pragma unroll
    for (int i = 0; i < V; ++i) w.v[i] = E::put(h.rstd[i] * ((h.ga[i] * dz[i] - m1[i]) - xh[i] * m2[i]));
    st_pack<E, V>(dx + (long long)r * p.C, w);
  }
}

// ---- host side
// What a call runs is a function of the descriptor and the pointers' alignment.  The workspace holds for either alignment.
static bool gn_desc_ok(const tbg_gn_desc *d) {
  return d && d->N >= 1 && d->S >= 1 && d->C >= 1 && d->G >= 1 && d->C % d->G == 0 && dt_valid(d->dtype) && d->act >= TBG_ACT_LINEAR &&
         d->act <= TBG_ACT_SILU && (d->per_sample == 0 || d->per_sample == 1) && d->eps > 0.f && d->xs >= d->C && d->xn >= 0 && d->ds >= d->C && d->dn >= 0;
}
static int gn_geometry(const tbg_gn_desc *d, bool vec, GnP &p) {
  if (d->S > (1 << 30) || d->C > (1 << 24)) return TBG_ERANGE;
  const int V = vec ? 8 : 1;
  p.N = d->N; p.S = d->S; p.C = d->C; p.G = d->G; p.Cg = d->C / d->G; p.affn = d->per_sample ? d->C : 0;
  p.nb = (d->C + A8_BLOCK - 1) / A8_BLOCK;
  p.xn = d->xn; p.xs = d->xs; p.dn = d->dn; p.ds = d->ds; p.eps = d->eps;
  const int padded = p.nb * A8_BLOCK, most = vec ? GN_CT : 64;
  p.CT = padded < most ? padded : most;  // (a multiple of 32: a row's 8-bit block never spans two tiles)
  p.ntile = (d->C + p.CT - 1) / p.CT;
  p.lanes = p.CT / V;
  p.RL = GN_T / p.lanes;
  p.nslot = p.ntile + p.G - 1;
  const auto ranges = [&](int target, int least, int &count, int &rows) {  // row ranges: about `target` blocks, `least` passes each
    long long want = target / ((long long)p.N * p.ntile);
    if (want < 1) want = 1;
    const long long most_c = (p.S + (long long)p.RL * least - 1) / ((long long)p.RL * least);
    if (want > most_c) want = most_c;
    rows = (int)((p.S + want - 1) / want);
    rows = (rows + p.RL - 1) / p.RL * p.RL;
    count = (p.S + rows - 1) / rows;
  };
  ranges(1024, 4, p.nchunk, p.crows);
  ranges(2048, 4, p.achunk, p.arows);
  const long long count = d->per_sample ? (long long)d->N * d->C : d->C;
  if ((long long)p.N * p.ntile * p.achunk > 0x3fffffffLL || count > 0x3fffffffLL) return TBG_ERANGE;
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
    if (const int rc = gn_geometry(d, vec != 0, p)) return rc;
    const long long b = gn_part_bytes(p) + (backward ? gn_pch_bytes(p) : 0);
    if (b > most) most = b;
  }
  return most;
}

template <class E, int V, int ACT>
static int gn_run_fwd(const GnP &p, hipStream_t st) {
  hipLaunchKernelGGL((gn_sums_kernel<E, V>), dim3(p.N * p.ntile * p.nchunk), dim3(GN_T), 0, st, p);
  TBG_LAUNCH_CHECK();
  hipLaunchKernelGGL((gn_apply_kernel<E, V, ACT>), dim3(p.N * p.ntile * p.achunk), dim3(GN_T), 0, st, p);
  TBG_LAUNCH_CHECK();
  return TBG_OK;
}
template <class E, int V, int ACT, bool Q8>
static int gn_run_bwd(const GnP &p, hipStream_t st) {
  hipLaunchKernelGGL((gn_bwd_sums_kernel<E, V, ACT, Q8>), dim3(p.N * p.ntile * p.nchunk), dim3(GN_T), 0, st, p);
  TBG_LAUNCH_CHECK();
  hipLaunchKernelGGL((gn_bwd_dx_kernel<E, V, ACT, Q8>), dim3(p.pblocks + p.N * p.ntile * p.achunk), dim3(GN_T), 0, st, p);
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
  if (gn_misaligned(q, yq) || gn_misaligned(workspace, nullptr)) return TBG_EINVAL;
  const bool vec = d->C % 8 == 0 && vec8_ok(x, d->dtype, d->xs, d->xn) && vec8_ok(y, d->dtype, d->C);
  GnP p{};
  if (const int rc = gn_geometry(d, vec, p)) return rc;
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
  if (gn_misaligned(q, workspace)) return TBG_EINVAL;
  const bool vec = d->C % 8 == 0 && (!x || vec8_ok(x, d->dtype, d->xs, d->xn)) && vec8_ok(dy, d->dtype, d->ds, d->dn) && vec8_ok(dx, d->dtype, d->C);
  GnP p{};
  if (const int rc = gn_geometry(d, vec, p)) return rc;
  if (gn_part_bytes(p) + gn_pch_bytes(p) > workspace_bytes) return TBG_EINVAL;
  p.x = x; p.dy = dy; p.gamma = gamma; p.beta = beta; p.y = dx; p.stats = const_cast<double *>(stats);
  p.q = const_cast<unsigned char *>(reinterpret_cast<const unsigned char *>(q));
  p.e = const_cast<unsigned char *>(reinterpret_cast<const unsigned char *>(e));
  p.part = reinterpret_cast<double *>(workspace);
  p.pch = reinterpret_cast<float *>(reinterpret_cast<char *>(workspace) + gn_part_bytes(p));
  p.dgamma = dgamma; p.dbeta = dbeta;
  return gn_dispatch(d, p, vec, true, stream);
}
