// Group norm with an activation over channels-last tensors (tbg.h "GROUP NORM"): x [N][S][C], statistics over the S x C/G values of a
// (sample, group), forward and backward, with the input kept whole or as an 8-bit checkpoint of x - mean.
//
//   xh = (x - mean) rstd,  z = gamma xh + beta,  y = act(z)
//   dz = dy act'(z),  dbeta = sum dz,  dgamma = sum dz xh,  dx = rstd (gamma dz - mean(gamma dz) - xh mean(gamma dz xh))
//
// HBM-bound.  A block works on a tile of CT channels (every lane has 8 fixed neighbouring ones) and a range of rows, so all accesses are
// whole 16-byte pieces of rows whatever the group width: groups need not line up with tiles.  Direction forward / backward: a sums launch
// leaves partial sums per (sample, row range, tile, group), the second launch joins those of its groups in a fixed order (no atomics) and
// writes the result.
//
// The statistics are 64-bit sums of x and x^2 (the card adds fp64 about as fast as unpacked fp32, so a streaming pass hardly notices): one pass,
// mean(x^2) - mean^2 loses nothing that matters even where |mean| is 10^5 standard deviations, and no value of any type overflows.  The mean
// is used as fp32 + its remainder.
//
// Measured (us): 32 x 16384 x 128 bf16, SiLU, 8-bit checkpoint: sums 27 (5.0 TB/s), second launch 54-58 (337 MB: 5.8-6.2), backward sums 48-52
// and second launch 56 (203 and 337 MB: 3.9-4.2, 6.0), whose two quarter-rate instructions a value are 34 us of vector time; 16 x 16384 x 128 forward 14 + 26.
#include "act8.h"

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
  bool past;                           // second launches write past the caches (rows of whole 8 channels)
  int team;                            // one launch: lanes that share a tile of a sample (0: two launches)
  int nteam, ng, per, slots;           // teams of a block; most groups of a tile; backward: samples a team takes in turn, blocks' partial sums a channel
  int pblocks;                         // backward: first blocks of the second launch (one launch: blocks of one behind it) that sum dgamma / dbeta
  float eps;
};

// threads a block: second launches, forward sums, backward sums, one-launch forward; most channels a tile of two launches
constexpr int GN_T = 256, GN_TS = 1024, GN_TB = 512, GN_TW = 512, GN_CT = 128;
// rows that a lane of the one-launch forms keeps in registers, forward and backward
constexpr int GN_R = 8, GN_RB = 4;

template <int ACT>
__device__ __forceinline__ float gn_act(float z) {
  if constexpr (ACT == TBG_ACT_LRELU) return 1.41421356237309515f * (z > 0.f ? z : 0.2f * z);
  if constexpr (ACT == TBG_ACT_SILU) return z * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.44269504088896341f * z));
  return z;
}
// LeakyReLU's slope where z = scale d + be > 0, scale = sc + lo.  The side of the kink is decided as in 64 bits, so that it does not hang on the
// last bit of a 32-bit product: that one, off by 2^-24 (|be| + 3 |z|) at most, says it unless |z| <= 2^-22 |be|.
__device__ __forceinline__ void gn_slope(const float (&d)[8], const float (&sc)[8], const float (&lo)[8], const float (&be)[8], float (&f)[8]) {
  bool close = false;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float z = fmaf(d[i], sc[i], be[i]);
    close |= fabsf(z) * 4194304.f <= fabsf(be[i]);
    f[i] = z > 0.f ? 1.41421356237309515f : 0.282842712474619f;
  }
  if (close) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float s = sc[i], l = lo[i], b = be[i];
      asm volatile("" : "+v"(s), "+v"(l), "+v"(b));  // (their 64-bit forms are not worth keeping in registers over the rows)
      f[i] = fma((double)d[i], (double)s + (double)l, (double)b) > 0.0 ? 1.41421356237309515f : 0.282842712474619f;
    }
  }
}
// dy act'(z), LeakyReLU apart
template <int ACT>
__device__ __forceinline__ float gn_dact(float dy, float z) {
  if constexpr (ACT == TBG_ACT_SILU) {  // z comes times -log2(e): s = 1 / (1 + e^-z), act' = s + z s (1 - s)
    const float s = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(z)), u = z * s;
    return dy * fmaf(fmaf(-u, s, u), -0.693147180559945309f, s);
  }
  return dy;
}

// groups of a lane's 8 channels (of the last channel for those that do not exist)
__device__ __forceinline__ void gn_groups(const GnP &p, int c, int (&g)[8]) {
  int at = min(c, p.C - 1) / p.Cg, left = (at + 1) * p.Cg - c;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    g[i] = min(at, p.G - 1);
    --left;
    at += left <= 0;
    left = left <= 0 ? p.Cg : left;
  }
}

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
  const double *base = p.part + ((long long)n * p.nchunk * p.nslot + t0 + g) * 2;
  if (nt == 1) {
#pragma unroll 8
    for (int k = lane; k < p.nchunk; k += sub) {  // (the loads of all ranges under way at once)
      const double2 s = *reinterpret_cast<const double2 *>(base + (long long)k * p.nslot * 2);
      a += s.x;
      b += s.y;
    }
  } else {
    for (int i = lane; i < nt * p.nchunk; i += sub) {
      const int k = i / nt;
      const double2 s = *reinterpret_cast<const double2 *>(base + ((long long)k * p.nslot + i - k * nt) * 2);
      a += s.x;
      b += s.y;
    }
  }
  for (int off = sub >> 1; off > 0; off >>= 1) {
    a += __shfl_xor(a, off, 64);
    b += __shfl_xor(b, off, 64);
  }
}

// ---- forward: sums of x and x^2, in fp64 from the first addition on.  8 / A neighbouring channels share a group (A accumulators a lane)
template <class E, int A>
__device__ __forceinline__ void gn_add(const Pack8<E> &v, double (&s1)[A], double (&s2)[A]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const double d = E::get(v.v[i]);
    s1[i * A / 8] += d;
    s2[i * A / 8] = fma(d, d, s2[i * A / 8]);
  }
}
// a block's sums of each 8 / A channels of the tile, in red[2 c], red[2 c + 1]: rows of a wave by lane exchanges, the waves through LDS
template <int A, int T>
__device__ __forceinline__ void gn_block_sums(const GnP &p, double (&s1)[A], double (&s2)[A], double *red) {
  constexpr int NW = T / 64;
  const int lane = threadIdx.x & (p.lanes - 1), wave = threadIdx.x >> 6, cols = p.lanes * A;
  for (int off = p.lanes; off < 64; off <<= 1)
#pragma unroll
    for (int i = 0; i < A; ++i) {
      s1[i] += __shfl_xor(s1[i], off, 64);
      s2[i] += __shfl_xor(s2[i], off, 64);
    }
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
}
// sums over the part of each of the tile's ng groups (from g0 on) that lies in it, of red's pairs (one for each `step` channels), by as many
// lanes a group as the block has; done(group - g0, sum) in one lane of each
template <int T, class F>
__device__ __forceinline__ void gn_group_sums(const GnP &p, const GnTile &t, int g0, int ng, int step, const double *red, F done) {
  int sub = 64;
  while (sub > 1 && ng * sub > T) sub >>= 1;
  const int i = threadIdx.x / sub, l = threadIdx.x & (sub - 1);
  if (i < ng) {
    const int g = g0 + i, a0 = max(g * p.Cg - t.c0, 0) / step, a1 = min((g + 1) * p.Cg - t.c0, t.ct) / step;
    double2 o = {0.0, 0.0};
    for (int c = a0 + l; c < a1; c += sub) {
      o.x += red[c * 2];
      o.y += red[c * 2 + 1];
    }
    for (int off = sub >> 1; off > 0; off >>= 1) {
      o.x += __shfl_xor(o.x, off, 64);
      o.y += __shfl_xor(o.y, off, 64);
    }
    if (l == 0) done(i, o);
  }
}
__device__ __forceinline__ double2 gn_stats(const GnP &p, double a, double q) {  // mean, rstd
  const double m = (double)p.S * p.Cg, mean = a / m, var = q / m - mean * mean;
  return {mean, 1.0 / sqrt((var < 0.0 ? 0.0 : var) + (double)p.eps)};  // (a NaN stays one)
}

template <class E, int A, bool TAIL>
__global__ __launch_bounds__(GN_TS) void gn_sums_kernel(GnP p) {
  constexpr int U = 4;  // rows under way
  __shared__ double red[GN_TS / 64 * (GN_CT / 8) * A * 2];
  const GnTile t = gn_tile(p, blockIdx.x);
  const int lane = threadIdx.x & (p.lanes - 1), rl = threadIdx.x / p.lanes, RL = GN_TS / p.lanes;
  const int r1 = min(p.S, (t.k + 1) * p.crows);
  double s1[A], s2[A];
#pragma unroll
  for (int i = 0; i < A; ++i) s1[i] = s2[i] = 0.0;
  if (lane * 8 < t.ct) {
    int r = t.k * p.crows + rl;
    const Row8<E, TAIL> row(t.c0 + lane * 8, p.C);
    const typename E::type *x = reinterpret_cast<const typename E::type *>(p.x) + t.n * p.xn + r * p.xs;
    const long long step = RL * p.xs;
    for (; r + (U - 1) * RL < r1; r += U * RL) {
      Pack8<E> v[U];
#pragma unroll
      for (int u = 0; u < U; ++u, x += step) v[u] = row.load(x);
#pragma unroll
      for (int u = 0; u < U; ++u) gn_add<E, A>(v[u], s1, s2);
    }
    for (; r < r1; r += RL, x += step) gn_add<E, A>(row.load(x), s1, s2);
  }
  gn_block_sums<A, GN_TS>(p, s1, s2, red);
  const int g0 = t.c0 / p.Cg, ng = (t.c0 + t.ct - 1) / p.Cg - g0 + 1;
  gn_group_sums<GN_TS>(p, t, g0, ng, 8 / A, red, [&](int i, const double2 &o) {
    *reinterpret_cast<double2 *>(p.part + (((long long)t.n * p.nchunk + t.k) * p.nslot + t.tile + g0 + i) * 2) = o;
  });
}

// gamma and beta of a lane's channels, zeros beyond the last
template <bool TAIL>
__device__ __forceinline__ void gn_affine(const GnP &p, int n, int c, float (&ga)[8], float (&be)[8]) {
  const Row8<ElF32, TAIL> row(c, p.C);
  const Pack8<ElF32> a = row.load(p.gamma + (long long)n * p.affn), b = row.load(p.beta + (long long)n * p.affn);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    ga[i] = a.v[i];
    be[i] = b.v[i];
  }
}

// ---- forward: what a lane does to a row.  Q: checkpoints are written
template <class E, int ACT, bool Q, bool TAIL, bool PAST = false>
struct GnOut {
  const GnP &p;
  Row8<E, TAIL> row;
  int c;
  bool in;
  float mu[8], sc[8], sh[8];
  float lo[8], be[8];  // LeakyReLU's kink: the scale's remainder, beta

  __device__ __forceinline__ GnOut(const GnP &p_, int c_) : p(p_), row(c_, p_.C), c(c_), in(c_ < p_.C) {}
  // affine parameters, 0 where there is no channel (loaded before the statistics are waited for)
  __device__ __forceinline__ void affine(int n) {
    if (in) gn_affine<TAIL>(p, n, c, sc, sh);
  }
  // st: mean, rstd of the groups from g0 on
  __device__ __forceinline__ void stats(const double *st, int g0) {
    int g[8];
    gn_groups(p, c, g);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const bool real = !TAIL || c + i < p.C;
      const double2 s = *reinterpret_cast<const double2 *>(st + (g[i] - g0) * 2);
      const double b = sh[i], scale = s.y * (double)sc[i];
      mu[i] = real ? (float)s.x : 0.f;
      be[i] = (float)b;
      sc[i] = (float)scale;
      lo[i] = (float)(scale - (double)sc[i]);
      sh[i] = (float)(b - (s.x - (double)(float)s.x) * scale);
    }
  }
  __device__ __forceinline__ void keep(const float (&v)[8], unsigned char *q, unsigned char *e, long long r, bool kink) const {
    const unsigned code = a8_code(a8_block_max(v));
    float k[8];
    a8_round(v, code, k);
    if (ACT == TBG_ACT_LRELU && kink) {  // one step back where rounding has crossed the kink: the backward pass takes the value's own slope
      const float scale = a8_scale(code);
      float kept[8], f[8], g[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) kept[i] = (k[i] - A8_MAGIC) * scale;
      gn_slope(v, sc, lo, be, f);
      gn_slope(kept, sc, lo, be, g);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (f[i] != g[i]) k[i] = fminf(fmaxf(k[i] + (v[i] > kept[i] ? 1.f : -1.f), A8_MAGIC - 127.f), A8_MAGIC + 127.f);
    }
    a8_store<PAST>(q + r * p.nb * A8_BLOCK + c, code, k);
    if ((c & (A8_BLOCK - 1)) == 0) e[r * p.nb + c / A8_BLOCK] = (unsigned char)code;
  }
  // v: channels of row r (of all samples' rows; zeros where there are none), y: where the row goes
  __device__ __forceinline__ void write(const Pack8<E> &v, typename E::type *y, long long r) const {
    float d[8], o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      d[i] = E::get(v.v[i]) - mu[i];
      o[i] = gn_act<ACT>(fmaf(d[i], sc[i], sh[i]));
    }
    const Pack8<E> w = put8<E>(o);
    if (!Q || in) row.template store<PAST>(y, w);
    if constexpr (Q) {
      if (p.q) {
        if (!in) {
#pragma unroll
          for (int i = 0; i < 8; ++i) d[i] = 0.f;
        }
        keep(d, p.q, p.e, r, true);
      }
      if (p.yq) {
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = in && (!TAIL || c + i < p.C) ? E::get(w.v[i]) : 0.f;
        keep(o, p.yq, p.ye, r, false);
      }
    }
  }
};

template <class E, int ACT, bool Q, bool TAIL, bool PAST>
__global__ __launch_bounds__(GN_T) void gn_apply_kernel(GnP p) {
  constexpr int U = 4;
  __shared__ double2 st[GN_CT];  // mean, rstd of the tile's groups
  const int piece = blockIdx.x / p.nchunk % p.split;
  const GnTile t = gn_tile(p, blockIdx.x / p.nchunk / p.split * p.nchunk + blockIdx.x % p.nchunk);
  const int lane = threadIdx.x & (p.lanes - 1), rl = threadIdx.x / p.lanes, RL = GN_T / p.lanes;
  GnOut<E, ACT, Q, TAIL, PAST> out(p, t.c0 + lane * 8);
  out.affine(t.n);
  const int g0 = t.c0 / p.Cg, ng = (t.c0 + t.ct - 1) / p.Cg - g0 + 1;
  int sub = 64;
  while (sub > 1 && ng * sub > GN_T) sub >>= 1;
  if (threadIdx.x < ng * sub) {
    const int i = threadIdx.x / sub, g = g0 + i;
    double a, q;
    gn_join(p, t.n, g, threadIdx.x & (sub - 1), sub, a, q);
    if ((threadIdx.x & (sub - 1)) == 0) {
      st[i] = gn_stats(p, a, q);
      if (p.stats && t.k == 0 && piece == 0 && g * p.Cg >= t.c0)  // the tile in which the group begins
        *reinterpret_cast<double2 *>(p.stats + ((long long)t.n * p.G + g) * 2) = st[i];
    }
  }
  __syncthreads();
  if (out.c >= p.nb * A8_BLOCK || (!Q && !out.in)) return;  // whole 8-bit blocks leave together; those beyond the last channel write the padding
  out.stats(reinterpret_cast<const double *>(st), g0);
  const int r1 = min(p.S, min((t.k + 1) * p.crows, t.k * p.crows + (piece + 1) * p.arows));
  int r = t.k * p.crows + piece * p.arows + rl;
  const typename E::type *x = reinterpret_cast<const typename E::type *>(p.x) + t.n * p.xn + r * p.xs;
  const long long row0 = (long long)t.n * p.S, xstep = RL * p.xs, ystep = (long long)RL * p.C;
  typename E::type *y = reinterpret_cast<typename E::type *>(p.y) + (row0 + r) * p.C;
  const Pack8<E> zero = {};
  for (; r + (U - 1) * RL < r1; r += U * RL) {
    Pack8<E> v[U];
#pragma unroll
    for (int u = 0; u < U; ++u, x += xstep) v[u] = out.in ? out.row.template load<PAST>(x) : zero;
#pragma unroll
    for (int u = 0; u < U; ++u, y += ystep) out.write(v[u], y, row0 + r + u * RL);
  }
  for (; r < r1; r += RL, x += xstep, y += ystep) out.write(out.in ? out.row.load(x) : zero, y, row0 + r);
}

// ---- one launch, where the rows of a tile of whole groups fit the registers of a team of lanes (a power of two, those of a row or more).  A
// block's teams have the same tile of neighbouring samples, so that small samples leave no lanes idle and large ones get a whole block
struct GnTeam {
  int id, l, lane, rl, RL;         // team; lane of the team; of the row; row, rows at a time
  int width, part, nparts;         // lanes that exchange rows' sums; then there are `nparts` sums of a channel left, this lane's among them
  bool first;                      // has its part's sum
  __device__ __forceinline__ GnTeam(const GnP &p) {
    id = threadIdx.x / p.team;
    l = threadIdx.x & (p.team - 1);
    lane = l & (p.lanes - 1);
    rl = l / p.lanes;
    RL = p.team / p.lanes;
    width = min(p.team, 64);
    const int span = max(p.lanes, 64);
    nparts = max(p.team / span, 1);
    part = nparts > 1 ? l / span : 0;
    first = (l & (width - 1)) < p.lanes;
  }
  // sums over a tile's groups of pairs (one for each `step` channels), done(group of the tile, sum) in one lane of each
  template <class T, class F>
  __device__ __forceinline__ void groups(const GnP &p, int ct, int ng, int step, const T *pairs, F done) const {
    int sub = width;
    while (sub > 1 && ng * sub > p.team) sub >>= 1;
    const int k = l & (sub - 1);
    for (int i = l / sub; i < ng; i += p.team / sub) {  // (more than one trip only where sub is 1)
      const int a0 = i * p.Cg / step, a1 = min((i + 1) * p.Cg, ct) / step;
      double2 o = {0.0, 0.0};
      for (int c = a0 + k; c < a1; c += sub) {
        o.x += pairs[c * 2];
        o.y += pairs[c * 2 + 1];
      }
      for (int off = sub >> 1; off > 0; off >>= 1) {
        o.x += __shfl_xor(o.x, off, 64);
        o.y += __shfl_xor(o.y, off, 64);
      }
      if (k == 0) done(i, o);
    }
  }
};

// x is read once
template <class E, int A, int ACT, bool Q, bool TAIL>
__global__ __launch_bounds__(GN_TW) void gn_whole_kernel(GnP p) {
  extern __shared__ __align__(16) char smem[];
  const GnTeam w(p);
  const int tile = blockIdx.x % p.ntile, n = blockIdx.x / p.ntile * p.nteam + w.id, c0 = tile * p.CT, ct = min(p.CT, p.C - c0), cols = p.lanes * A;
  double *red = reinterpret_cast<double *>(smem) + w.id * w.nparts * cols * 2;  // [nparts][cols][2]
  double2 *st = reinterpret_cast<double2 *>(smem) + p.nteam * w.nparts * cols + w.id * p.ng;
  const bool live = n < p.N;
  GnOut<E, ACT, Q, TAIL> out(p, c0 + w.lane * 8);
  const typename E::type *x = reinterpret_cast<const typename E::type *>(p.x) + n * p.xn;
  Pack8<E> v[GN_R] = {};
  double s1[A], s2[A];
#pragma unroll
  for (int i = 0; i < A; ++i) s1[i] = s2[i] = 0.0;
  if (live && out.in) {
#pragma unroll
    for (int u = 0; u < GN_R; ++u)
      if (w.rl + u * w.RL < p.S) v[u] = out.row.load(x + (w.rl + u * w.RL) * p.xs);
  }
  if (live) out.affine(n);
  if (live && out.in) {
#pragma unroll
    for (int u = 0; u < GN_R; ++u) gn_add<E, A>(v[u], s1, s2);  // (rows that do not exist are zeros)
  }
  for (int off = p.lanes; off < w.width; off <<= 1)
#pragma unroll
    for (int i = 0; i < A; ++i) {
      s1[i] += __shfl_xor(s1[i], off, 64);
      s2[i] += __shfl_xor(s2[i], off, 64);
    }
  if (w.first)
#pragma unroll
    for (int i = 0; i < A; ++i) {
      red[(w.part * cols + w.lane * A + i) * 2] = s1[i];
      red[(w.part * cols + w.lane * A + i) * 2 + 1] = s2[i];
    }
  __syncthreads();
  if (w.nparts > 1) {
    for (int j = w.l; j < 2 * cols; j += p.team) {
      double a = red[j];
      for (int k = 1; k < w.nparts; ++k) a += red[k * 2 * cols + j];
      red[j] = a;
    }
    __syncthreads();
  }
  const int g0 = c0 / p.Cg;
  w.groups(p, ct, (ct + p.Cg - 1) / p.Cg, 8 / A, red, [&](int i, const double2 &o) {
    st[i] = gn_stats(p, o.x, o.y);
    if (live && p.stats) *reinterpret_cast<double2 *>(p.stats + ((long long)n * p.G + g0 + i) * 2) = st[i];
  });
  __syncthreads();
  if (!live || out.c >= p.nb * A8_BLOCK || (!Q && !out.in)) return;
  out.stats(reinterpret_cast<const double *>(st), g0);
  const long long row0 = (long long)n * p.S;
  typename E::type *y = reinterpret_cast<typename E::type *>(p.y) + row0 * p.C;
#pragma unroll
  for (int u = 0; u < GN_R; ++u)
    if (w.rl + u * w.RL < p.S) out.write(v[u], y + (long long)(w.rl + u * w.RL) * p.C, row0 + w.rl + u * w.RL);
}

// ---- backward.  With d = x - mean (or its checkpoint), xh = d rstd and z = sc d + be.  Sums and dx take d times the power of two next to rstd (an
// exact product): xh but for a factor of 1 to 2, so that neither dz d nor rstd^2 leaves the range that x and dx themselves are in.
__device__ __forceinline__ float gn_power(double rstd) { return fmaxf(__uint_as_float(__float_as_uint((float)rstd) & 0x7f800000u), 0x1p-126f); }
__device__ __forceinline__ double gn_factor(double rstd, float power) { return rstd * (double)__uint_as_float(0x7f000000u - __float_as_uint(power)); }
// Two launches do without it where rstd is within 2^+-32, whose loops have no registers left (LeakyReLU from a whole input with a channel tail keeps 8-12
// of them in scratch as it is); in one launch it costs 0-8 % (512 x 32 x 512 bf16 SiLU 26.6 -> 28.7 us, linear 23.9 -> 24.4).
__device__ __forceinline__ bool gn_far(double rstd) { return (unsigned)__double2hiint(rstd) - ((1023u - 32u) << 20) > 64u << 20; }
__device__ __forceinline__ float gn_far_power(double rstd) { return gn_far(rstd) ? gn_power(rstd) : 1.f; }
struct GnCh {
  float mu[8], mlo[8], sc[8], lo[8], be[8], za[8], zb[8];  // mean, scale: and their remainders; za, zb: sc, be times -log2(e), for the exponential
  bool far;                                                // one of the wave's rstd is beyond 2^+-32
};
// st: mean, rstd of the groups from g0 on; sc, be come as gamma, beta
template <bool Q8>
__device__ __forceinline__ void gn_channels(const GnP &p, int c, const double2 *st, int g0, GnCh &h) {
  int g[8];
  gn_groups(p, c, g);
  bool far = false;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const double2 s = st[g[i] - g0];
    h.mu[i] = Q8 ? 0.f : (float)s.x;
    h.mlo[i] = Q8 ? 0.f : (float)(s.x - (double)(float)s.x);
    far |= gn_far(s.y);
    const double scale = s.y * (double)h.sc[i];
    h.sc[i] = (float)scale;
    h.lo[i] = (float)(scale - (double)h.sc[i]);
    h.za[i] = (float)(-1.44269504088896341 * scale);
    h.zb[i] = (float)(-1.44269504088896341 * (double)h.be[i]);
  }
  h.far = __any(far);
}
// the channels' powers of two
template <bool ALL>
__device__ __forceinline__ void gn_powers(const GnP &p, int c, const double2 *st, int g0, float (&pw)[8]) {
  int g[8];
  gn_groups(p, c, g);
#pragma unroll
  for (int i = 0; i < 8; ++i) pw[i] = ALL ? gn_power(st[g[i] - g0].y) : gn_far_power(st[g[i] - g0].y);
}
// a row's operands as they lie in memory
template <class E, bool Q8>
struct GnRow {
  Pack8<E> g, x;
  u32x2 q;
  unsigned e;
};
// (what is made of the operands before and after is made twice: it would fill the registers)
template <class T>
__device__ __forceinline__ void gn_opaque(T &v) {
  static_assert(sizeof(T) % 4 == 0, "whole registers");
  unsigned w[sizeof(T) / 4];
  __builtin_memcpy(w, &v, sizeof(T));
#pragma unroll
  for (unsigned i = 0; i < sizeof(T) / 4; ++i) asm volatile("" : "+v"(w[i]));
  __builtin_memcpy(&v, w, sizeof(T));
}
// where a lane stands, and a step of `rows` rows
template <class E, bool Q8, bool TAIL>
struct GnAt {
  Row8<E, TAIL> row;
  const typename E::type *x, *g;
  const unsigned char *q, *e;
  __device__ __forceinline__ GnAt(const GnP &p, int n, int r, int c) : row(c, p.C) {
    const long long at = (long long)n * p.S + r;
    x = reinterpret_cast<const typename E::type *>(p.x) + n * p.xn + r * p.xs;
    g = reinterpret_cast<const typename E::type *>(p.dy) + n * p.dn + r * p.ds;
    q = p.q + at * p.nb * A8_BLOCK + c;
    e = p.e + at * p.nb + c / A8_BLOCK;
  }
  template <bool PAST = false>
  __device__ __forceinline__ GnRow<E, Q8> next(const GnP &p, int rows) {
    GnRow<E, Q8> w;
    if constexpr (Q8) {
      w.e = *e;
      w.q = ld_vec<PAST>(reinterpret_cast<const u32x2 *>(q));
      q += (long long)rows * p.nb * A8_BLOCK;
      e += (long long)rows * p.nb;
    } else {
      w.x = row.template load<PAST>(x);
      x += rows * p.xs;
    }
    w.g = row.template load<PAST>(g);
    g += rows * p.ds;
    return w;
  }
};
// d and dz of a row
template <class E, int ACT, bool Q8>
__device__ __forceinline__ void gn_row(const GnRow<E, Q8> &w, const GnCh &h, float (&d)[8], float (&dz)[8]) {
  const float scale = Q8 ? a8_scale(w.e) : 1.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if constexpr (Q8) d[i] = a8_value(w.q, i) * scale;
    else d[i] = (E::get(w.x.v[i]) - h.mu[i]) - h.mlo[i];
  }
  if constexpr (ACT == TBG_ACT_LRELU) {
    gn_slope(d, h.sc, h.lo, h.be, dz);
#pragma unroll
    for (int i = 0; i < 8; ++i) dz[i] *= E::get(w.g.v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) dz[i] = gn_dact<ACT>(E::get(w.g.v[i]), ACT == TBG_ACT_SILU ? fmaf(d[i], h.za[i], h.zb[i]) : 0.f);
  }
}

// ---- backward, first launch: sums of dz and dz xh of every channel, and of gamma dz and gamma dz xh of every group
template <class E, int ACT, bool Q8, bool TAIL>
__global__ __launch_bounds__(GN_TB, 4) void gn_bwd_sums_kernel(GnP p) {
  constexpr int U = 2, NW = GN_TB / 64;
  __shared__ float red[NW * GN_CT * 2];
  __shared__ double gred[GN_CT * 2];  // times gamma
  __shared__ double2 st[GN_CT];  // mean, rstd of the tile's groups
  const GnTile t = gn_tile(p, blockIdx.x);
  const int g0 = t.c0 / p.Cg, g1 = (t.c0 + t.ct - 1) / p.Cg;
  if (threadIdx.x <= g1 - g0) st[threadIdx.x] = *reinterpret_cast<const double2 *>(p.stats + ((long long)t.n * p.G + g0 + threadIdx.x) * 2);
  const int lane = threadIdx.x & (p.lanes - 1), rl = threadIdx.x / p.lanes, RL = GN_TB / p.lanes;
  const int r1 = min(p.S, (t.k + 1) * p.crows), c = t.c0 + lane * 8;
  float s1[8], s2[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) s1[i] = s2[i] = 0.f;
  GnCh h;
  if (lane * 8 < t.ct) gn_affine<TAIL>(p, t.n, c, h.sc, h.be);
  __syncthreads();
  if (lane * 8 < t.ct) {
    gn_channels<Q8>(p, c, st, g0, h);
    const auto add = [&](const GnRow<E, Q8> &w, auto pw) {
      float d[8], dz[8];
      gn_row<E, ACT, Q8>(w, h, d, dz);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        s1[i] += dz[i];
        s2[i] = fmaf(dz[i], pw(d[i], i), s2[i]);
      }
    };
    int r = t.k * p.crows + rl;
    GnAt<E, Q8, TAIL> at(p, t.n, r, c);
    if (h.far) {  // (a loop of its own: that of ordinary values does without the registers)
      float pw[8];
      gn_powers<false>(p, c, st, g0, pw);
      for (; r < r1; r += RL) add(at.next(p, RL), [&](float d, int i) { return d * pw[i]; });
    } else {
      const auto one = [](float d, int) { return d; };
      for (; r + (U - 1) * RL < r1; r += U * RL) {
        GnRow<E, Q8> w[U];
#pragma unroll
        for (int u = 0; u < U; ++u) w[u] = at.next(p, RL);
#pragma unroll
        for (int u = 0; u < U; ++u) add(w[u], one);
      }
      for (; r < r1; r += RL) add(at.next(p, RL), one);
    }
  }
  for (int off = p.lanes; off < 64; off <<= 1)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      s1[i] += __shfl_xor(s1[i], off, 64);
      s2[i] += __shfl_xor(s2[i], off, 64);
    }
  const int wave = threadIdx.x >> 6;
  if ((threadIdx.x & 63) < p.lanes)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      red[(wave * p.CT + lane * 8 + i) * 2] = s1[i];
      red[(wave * p.CT + lane * 8 + i) * 2 + 1] = s2[i];
    }
  __syncthreads();
  if (threadIdx.x < 2 * t.ct) {
    float a = red[threadIdx.x];
#pragma unroll
    for (int w = 1; w < NW; ++w) a += red[w * 2 * p.CT + threadIdx.x];
    const int j = threadIdx.x >> 1;
    if (threadIdx.x & 1) {  // -> xh
      const double rstd = st[(t.c0 + j) / p.Cg - g0].y;
      a *= (float)gn_factor(rstd, gn_far_power(rstd));
    }
    p.pch[(((long long)t.n * p.nchunk + t.k) * p.C + t.c0) * 2 + threadIdx.x] = a;
    gred[threadIdx.x] = (double)p.gamma[(long long)t.n * p.affn + t.c0 + j] * (double)a;
  }
  __syncthreads();
  gn_group_sums<GN_TB>(p, t, g0, g1 - g0 + 1, 1, gred, [&](int i, const double2 &o) {
    *reinterpret_cast<double2 *>(p.part + (((long long)t.n * p.nchunk + t.k) * p.nslot + t.tile + g0 + i) * 2) = o;
  });
}

// dgamma, dbeta of 32 channels from partial sums, by 8 lanes each of a block of GN_T: the row ranges (or blocks of the one-launch form, and the
// samples, where the parameters are shared) in a fixed order
__device__ __forceinline__ void gn_param_sums(const GnP &p, int b, double2 *sh) {
  static_assert(GN_T == 256 && 2 * GN_CT == GN_T, "a lane's sums in sh");
  const int sub = threadIdx.x >> 5;
  const long long idx = (long long)b * 32 + (threadIdx.x & 31), count = p.affn ? (long long)p.N * p.C : p.C;
  double2 o = {0.0, 0.0};
  if (idx < count) {
    const int n = p.affn ? (int)(idx / p.C) : 0, c = (int)(idx % p.C);
    const long long len = p.team ? p.slots : (long long)(p.affn ? 1 : p.N) * p.nchunk;
    const float *src = p.pch + ((long long)n * p.nchunk * p.C + c) * 2;
#pragma unroll 8
    for (long long i = sub; i < len; i += 8) {
      const float2 s = *reinterpret_cast<const float2 *>(src + i * p.C * 2);
      o.x += s.x;
      o.y += s.y;
    }
  }
  sh[threadIdx.x] = o;
  __syncthreads();
  if (threadIdx.x < 32 && idx < count) {
#pragma unroll
    for (int l = 1; l < 8; ++l) {
      o.x += sh[l * 32 + threadIdx.x].x;
      o.y += sh[l * 32 + threadIdx.x].y;
    }
    p.dbeta[idx] = (float)o.x;
    p.dgamma[idx] = (float)o.y;
  }
}
__global__ __launch_bounds__(GN_T) void gn_params_kernel(GnP p) {
  __shared__ double2 sh[GN_T];
  gn_param_sums(p, blockIdx.x, sh);
}

// ---- backward, second launch: dx, and in its first blocks dgamma / dbeta
template <class E, int ACT, bool Q8, bool TAIL, bool PAST>
__global__ __launch_bounds__(GN_T, 4) void gn_bwd_dx_kernel(GnP p) {
  constexpr int U = 2;
  __shared__ double2 sh[2 * GN_CT];
  double2 *st = sh, *stats = sh + GN_CT;  // of the tile's groups: rstd mean(gamma dz), rstd (times its factor) mean(gamma dz xh); mean, rstd
  int b = blockIdx.x;
  if (b < p.pblocks) {
    gn_param_sums(p, b, sh);
    return;
  }
  b -= p.pblocks;
  const int piece = b / p.nchunk % p.split;
  const GnTile t = gn_tile(p, b / p.nchunk / p.split * p.nchunk + b % p.nchunk);
  const int lane = threadIdx.x & (p.lanes - 1), rl = threadIdx.x / p.lanes, RL = GN_T / p.lanes, c = t.c0 + lane * 8;
  GnCh h;
  if (lane * 8 < t.ct) gn_affine<TAIL>(p, t.n, c, h.sc, h.be);
  const int g0 = t.c0 / p.Cg, ng = (t.c0 + t.ct - 1) / p.Cg - g0 + 1;
  int sub = 64;
  while (sub > 1 && ng * sub > GN_T) sub >>= 1;
  if (threadIdx.x < ng * sub) {
    const int i = threadIdx.x / sub;
    double a, q;
    gn_join(p, t.n, g0 + i, threadIdx.x & (sub - 1), sub, a, q);
    const double m = (double)p.S * p.Cg;
    if ((threadIdx.x & (sub - 1)) == 0) {
      stats[i] = *reinterpret_cast<const double2 *>(p.stats + ((long long)t.n * p.G + g0 + i) * 2);
      const double rstd = stats[i].y;
      st[i] = {rstd * (a / m), rstd * gn_factor(rstd, gn_far_power(rstd)) * (q / m)};
    }
  }
  __syncthreads();
  if (lane * 8 >= t.ct) return;
  gn_channels<Q8>(p, c, stats, g0, h);
  float m1[8], m2[8];  // dx = sc dz - m1 - d m2
  {
    int g[8];
    gn_groups(p, c, g);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const double2 s = st[g[i] - g0];
      m1[i] = (float)s.x;
      m2[i] = (float)s.y;
    }
  }
  const int r1 = min(p.S, min((t.k + 1) * p.crows, t.k * p.crows + (piece + 1) * p.arows));
  int r = t.k * p.crows + piece * p.arows + rl;
  GnAt<E, Q8, TAIL> at(p, t.n, r, c);
  typename E::type *dx = reinterpret_cast<typename E::type *>(p.y) + ((long long)t.n * p.S + r) * p.C;
  const auto write = [&](const GnRow<E, Q8> &w, auto pw) {
    float d[8], dz[8];
    gn_row<E, ACT, Q8>(w, h, d, dz);
#pragma unroll
    for (int i = 0; i < 8; ++i) dz[i] = fmaf(-pw(d[i], i), m2[i], fmaf(dz[i], h.sc[i], -m1[i]));
    at.row.template store<PAST>(dx, put8<E>(dz));
    dx += (long long)RL * p.C;
  };
  if (h.far) {
    float pw[8];
    gn_powers<false>(p, c, stats, g0, pw);
    for (; r < r1; r += RL) write(at.template next<PAST>(p, RL), [&](float d, int i) { return d * pw[i]; });
    return;
  }
  const auto one = [](float d, int) { return d; };
  for (; r + (U - 1) * RL < r1; r += U * RL) {
    GnRow<E, Q8> w[U];
#pragma unroll
    for (int u = 0; u < U; ++u) w[u] = at.template next<PAST>(p, RL);
#pragma unroll
    for (int u = 0; u < U; ++u) write(w[u], one);
  }
  for (; r < r1; r += RL) write(at.next(p, RL), one);
}

// ---- backward in one launch (teams as in the forward one): x (or its checkpoint) and dy are read once.  The parameters' gradients are summed
// over the `per` samples that a team takes in turn and the teams of the block; one block a tile: that is all of them, else a launch joins the blocks
template <class E, int ACT, bool Q8, bool TAIL>
__global__ __launch_bounds__(GN_T, 2) void gn_bwd_whole_kernel(GnP p) {
  constexpr int R = GN_RB;
  extern __shared__ __align__(16) char smem[];
  const GnTeam w(p);
  const int tile = blockIdx.x % p.ntile, chunk = blockIdx.x / p.ntile, c0 = tile * p.CT, ct = min(p.CT, p.C - c0), c = c0 + w.lane * 8, g0 = c0 / p.Cg;
  double2 *st = reinterpret_cast<double2 *>(smem) + w.id * p.ng;  // of the tile's groups: mean(sc dz), mean(sc dz d) times rstd's factor squared
  float *reds = reinterpret_cast<float *>(reinterpret_cast<double2 *>(smem) + p.nteam * p.ng);
  float *red = reds + w.id * w.nparts * p.CT * 2;  // [nparts][CT][2]
  const bool in = w.lane * 8 < ct;
  float a1[8], a2[8];  // sums of dz, dz xh over the samples
#pragma unroll
  for (int i = 0; i < 8; ++i) a1[i] = a2[i] = 0.f;
  for (int k = 0; k < p.per; ++k) {
    const long long at = ((long long)chunk * p.per + k) * p.nteam + w.id;
    const bool live = at < p.N && in;
    const int n = at < p.N ? (int)at : 0;
    GnRow<E, Q8> row[R];
    GnCh h;
    float pw[8], s1[8], s2[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) s1[i] = s2[i] = 0.f;
    if (live) {
      GnAt<E, Q8, TAIL> from(p, n, w.rl, c);
#pragma unroll
      for (int u = 0; u < R; ++u)
        if (w.rl + u * w.RL < p.S) row[u] = from.next(p, w.RL);
      gn_affine<TAIL>(p, n, c, h.sc, h.be);
      gn_channels<Q8>(p, c, reinterpret_cast<const double2 *>(p.stats) + (long long)n * p.G, 0, h);
      gn_powers<true>(p, c, reinterpret_cast<const double2 *>(p.stats) + (long long)n * p.G, 0, pw);
#pragma unroll
      for (int u = 0; u < R; ++u)
        if (w.rl + u * w.RL < p.S) {
          float d[8], dz[8];
          gn_row<E, ACT, Q8>(row[u], h, d, dz);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            s1[i] += dz[i];
            s2[i] = fmaf(dz[i], pw[i] * d[i], s2[i]);
          }
        }
    }
    for (int off = p.lanes; off < w.width; off <<= 1)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        s1[i] += __shfl_xor(s1[i], off, 64);
        s2[i] += __shfl_xor(s2[i], off, 64);
      }
    if (w.nparts > 1) {
      if (w.first)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          red[(w.part * p.CT + w.lane * 8 + i) * 2] = s1[i];
          red[(w.part * p.CT + w.lane * 8 + i) * 2 + 1] = s2[i];
        }
      __syncthreads();
      if (w.rl == 0)
#pragma unroll
        for (int i = 0; i < 8; ++i)
          for (int o = 1; o < w.nparts; ++o) {
            s1[i] += red[(o * p.CT + w.lane * 8 + i) * 2];
            s2[i] += red[(o * p.CT + w.lane * 8 + i) * 2 + 1];
          }
    }
    if (w.rl == 0 && live) {  // the channels' sums: for the parameters, and times the scale for the groups
      int g[8];
      gn_groups(p, c, g);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float xh = s2[i] * (float)gn_factor(p.stats[((long long)n * p.G + g[i]) * 2 + 1], pw[i]);
        if (p.affn) {
          if (!TAIL || c + i < p.C) {
            p.dbeta[(long long)n * p.C + c + i] = s1[i];
            p.dgamma[(long long)n * p.C + c + i] = xh;
          }
        } else {
          a1[i] += s1[i];
          a2[i] += xh;
        }
        red[(w.lane * 8 + i) * 2] = h.sc[i] * s1[i];
        red[(w.lane * 8 + i) * 2 + 1] = h.sc[i] * s2[i];
      }
    }
    __syncthreads();
    w.groups(p, ct, (ct + p.Cg - 1) / p.Cg, 1, red, [&](int i, const double2 &o) {
      const double rstd = p.stats[((long long)n * p.G + g0 + i) * 2 + 1], f = gn_factor(rstd, gn_power(rstd)), m = (double)p.S * p.Cg;
      st[i] = {o.x / m, f * f * (o.y / m)};
    });
    __syncthreads();
    if (live) {
      float m1[8], m2[8];  // dx = sc dz - m1 - d m2
      int g[8];
      gn_groups(p, c, g);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const double2 m = st[g[i] - g0];
        m1[i] = (float)m.x;
        m2[i] = (float)m.y;
      }
      const Row8<E, TAIL> to(c, p.C);
      typename E::type *dx = reinterpret_cast<typename E::type *>(p.y) + (long long)n * p.S * p.C;
#pragma unroll
      for (int u = 0; u < R; ++u)
        if (w.rl + u * w.RL < p.S) {
          float d[8], dz[8];
          gn_opaque(row[u].g);
          if constexpr (Q8) gn_opaque(row[u].q);
          else gn_opaque(row[u].x);
          gn_row<E, ACT, Q8>(row[u], h, d, dz);
#pragma unroll
          for (int i = 0; i < 8; ++i) dz[i] = fmaf(-pw[i] * d[i], m2[i], fmaf(dz[i], h.sc[i], -m1[i]));
          to.store(dx + (long long)(w.rl + u * w.RL) * p.C, put8<E>(dz));
        }
    }
  }
  if (p.affn) return;
  // (all reads of `reds` are before the last barrier)
  if (w.rl == 0)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      reds[(w.id * p.CT + w.lane * 8 + i) * 2] = a1[i];
      reds[(w.id * p.CT + w.lane * 8 + i) * 2 + 1] = a2[i];
    }
  __syncthreads();
  for (int j = threadIdx.x; j < 2 * ct; j += GN_T) {
    float a = reds[j];
    for (int t = 1; t < p.nteam; ++t) a += reds[t * 2 * p.CT + j];
    if (p.slots > 1) p.pch[((long long)chunk * p.C + c0) * 2 + j] = a;
    else (j & 1 ? p.dgamma : p.dbeta)[c0 + (j >> 1)] = a;
  }
}

// ---- host side
static bool gn_desc_ok(const tbg_gn_desc *d) {
  return d && d->N >= 1 && d->S >= 1 && d->C >= 1 && d->G >= 1 && d->C % d->G == 0 && dt_valid(d->dtype) && d->act >= TBG_ACT_LINEAR &&
         d->act <= TBG_ACT_SILU && (d->per_sample == 0 || d->per_sample == 1) && d->eps > 0.f && d->xs >= d->C && d->xn >= 0 && d->ds >= d->C && d->dn >= 0;
}
static void gn_tiles(GnP &p, int CT) {
  p.CT = CT;
  p.ntile = (p.C + CT - 1) / CT;
  p.lanes = CT / 8;
  p.nslot = p.ntile + p.G - 1;
}
// channels in runs of 8, 4, 2 or 1 within a group (of the forward sums: 8 / run accumulators a lane)
static int gn_run_length(const GnP &p) { return p.C % 8 == 0 && p.Cg % 8 == 0 ? 8 : p.Cg % 4 == 0 ? 4 : p.Cg % 2 == 0 ? 2 : 1; }
static size_t gn_team_lds(const GnP &p, bool backward) {
  const int span = p.lanes > 64 ? p.lanes : 64, nparts = p.team > span ? p.team / span : 1;
  return (size_t)p.nteam * (nparts * p.lanes * (backward ? 64 : 16 * (8 / gn_run_length(p))) + p.ng * 16);
}
// One launch: a tile of whole groups whose rows fit the registers of a block's lanes.  Few samples: the narrowest such tile and all of the
// block's lanes.  Samples for more than the card's threads: tiles of up to GN_CT channels, as few lanes a sample as its rows need.
// Forward (bf16, SiLU, us of kernels, one launch / two): 1 x 64 x 256 channels 8.4 / 10.0, 32 x 16 x 64 7.0 / 9.8, 128 x 64 x 512 14.5 / 17.6, 512 x 32
// x 512 18 / 37, 65536 x 1 x 256 55 / 4800; a few blocks of full registers 11.1 / 9.6 (1 x 1024 x 32), where the launch saved is worth the rest.
// Backward: one launch where it makes the parameters' gradients whole as well (1 x 64 x 256 9.0 / 12.7) or where samples are many (512 x 32 x 512 29 / 43,
// 65536 x 1 x 256 84 / 1390); between, a second launch would join them (32 x 64 x 512 14.4 / 13.4, 4 x 128 x 256 13.3 / 11.5).
static bool gn_one_launch(GnP &p, int least_ct, bool backward) {
  const int T = backward ? GN_T : GN_TW, R = backward ? GN_RB : GN_R;
  constexpr long long FULL = 256 * 1024;
  constexpr size_t LDS = 40960;  // four blocks a CU
  const GnP two = p;
  const auto fits = [&](int ct, int team) {
    if ((ct % p.Cg && ct < p.C) || ct / 8 > team || p.S > (long long)R * (team / (ct / 8))) return false;
    gn_tiles(p, ct);
    p.team = team;
    p.nteam = T / team;
    p.ng = p.G < ct / p.Cg ? p.G : ct / p.Cg;
    return gn_team_lds(p, backward) <= LDS;
  };
  int ct = least_ct;
  while (!fits(ct, T)) {
    if (ct >= p.C || ct >= 8 * T) {
      p = two;
      return false;
    }
    ct <<= 1;
  }
  if (backward && !p.affn && p.N > 1 && (long long)p.N * p.ntile * T < 4 * FULL) {
    p = two;
    return false;
  }
  while (ct < GN_CT && ct < p.C && (long long)p.N * p.ntile * T > FULL && fits(2 * ct, T)) ct <<= 1;
  fits(ct, T);
  int team = T;
  while ((long long)p.N * p.ntile * team > FULL && fits(ct, team / 2)) team >>= 1;
  fits(ct, team);
  p.nchunk = p.split = 1;
  p.crows = p.arows = p.S;
  const long long blocks = (long long)p.N * p.ntile / p.nteam;
  p.per = 1;
  if (backward && blocks > 1024) p.per = (int)(blocks / 1024 < 64 ? blocks / 1024 : 64);
  p.slots = (int)((p.N + (long long)p.nteam * p.per - 1) / (p.nteam * p.per));
  return true;
}
// Two launches.  Row ranges: the sums launch has at most 32 a tile (256 where samples and tiles are few), each joined by every block of the
// second launch that needs it; of 4 rows a lane or more, fewer where that leaves CUs idle.  The second launch cuts them into pieces for about
// 8 blocks a CU, of 8 rows a lane or more, fewer for 2 blocks a CU.
static int gn_geometry(const tbg_gn_desc *d, bool backward, bool writes8, GnP &p) {
  if (d->S > (1 << 30) || d->C > (1 << 24)) return TBG_ERANGE;
  p.N = d->N; p.S = d->S; p.C = d->C; p.G = d->G; p.Cg = d->C / d->G; p.affn = d->per_sample ? d->C : 0;
  p.nb = (d->C + A8_BLOCK - 1) / A8_BLOCK;
  p.xn = d->xn; p.xs = d->xs; p.dn = d->dn; p.ds = d->ds; p.eps = d->eps;
  const long long count = d->per_sample ? (long long)d->N * d->C : d->C;
  if (count > 0x3fffffffLL) return TBG_ERANGE;
  p.pblocks = (int)((count + 31) / 32);
  // the tile (a power of two; where 8-bit blocks are written, none spans two) that leaves the fewest lanes without channels
  const int padded = p.nb * A8_BLOCK, least_ct = p.C > 16 || writes8 ? A8_BLOCK : p.C > 8 ? 16 : 8;
  int best = 0, tile = least_ct;
  for (int ct = GN_CT; ct > A8_BLOCK && p.C > A8_BLOCK; ct >>= 1) {
    const int used = (int)(1000LL * padded / ((long long)(padded + ct - 1) / ct * ct));
    if (used > best) { best = used; tile = ct; }
  }
  gn_tiles(p, tile);
  const int RL = (backward ? GN_TB : GN_TS) / p.lanes, RA = GN_T / p.lanes;
  const long long tiles = (long long)p.N * p.ntile;
  long long want = 512 / tiles;
  const long long cap = tiles < 8 ? 256 : 32, fill = 128 / tiles, rows_each = (p.S + RL - 1) / RL;
  long long most = (p.S + 4LL * RL - 1) / (4LL * RL);
  most = most > fill ? most : (rows_each < fill ? rows_each : fill);
  if (most < 1) most = 1;
  want = want > cap ? cap : want;
  want = want > most ? most : want;
  if (want >= 8) want &= ~7LL;
  if (want < 1) want = 1;
  long long rows = (p.S + want - 1) / want;
  p.crows = (int)((rows + RL - 1) / RL * RL);
  p.nchunk = (int)((p.S + p.crows - 1LL) / p.crows);
  long long split = 2048 / (tiles * p.nchunk);
  long long least = p.crows / (8LL * RA);
  const long long filled = 512 / (tiles * p.nchunk), pieces = p.crows / RA;
  least = least > filled ? least : (pieces < filled ? pieces : filled);
  split = split > least ? least : split;
  if (split < 1) split = 1;
  p.arows = (int)(((p.crows + split - 1) / split + RA - 1) / RA * RA);
  p.split = (p.crows + p.arows - 1) / p.arows;
  const bool one = gn_one_launch(p, least_ct, backward);
  // a grid holds less than 2^32 threads
  const long long blocks = (long long)(one ? p.slots : p.N) * p.ntile * p.nchunk, threads = (1LL << 32) - 1;
  if (blocks > threads / (backward ? (one ? GN_T : GN_TB) : one ? GN_TW : GN_TS) || blocks * p.split + (backward ? p.pblocks : 0) > threads / GN_T)
    return TBG_ERANGE;
  return TBG_OK;
}
static long long gn_part_bytes(const GnP &p) { return p.team ? 0 : (long long)p.N * p.nchunk * p.nslot * 2 * (long long)sizeof(double); }
static long long gn_pch_bytes(const GnP &p) {
  if (p.team) return p.affn || p.slots == 1 ? 0 : (long long)p.slots * p.C * 2 * (long long)sizeof(float);
  return (long long)p.N * p.nchunk * p.C * 2 * (long long)sizeof(float);
}

extern "C" long long tbg_group_norm_workspace_bytes(const tbg_gn_desc *d, int backward) {
  if (!gn_desc_ok(d)) return TBG_EINVAL;
  GnP p{}, w{};
  if (const int rc = gn_geometry(d, backward != 0, false, p)) return rc;
  if (backward) return gn_part_bytes(p) + gn_pch_bytes(p);
  if (const int rc = gn_geometry(d, false, true, w)) return rc;  // (the form that writes checkpoints has wider tiles for few channels)
  return gn_part_bytes(p) > gn_part_bytes(w) ? gn_part_bytes(p) : gn_part_bytes(w);
}

template <class E, int ACT, bool Q, bool TAIL>
static int gn_run_fwd(const GnP &p, hipStream_t st) {
  const int run = gn_run_length(p);
  constexpr int A8 = TAIL ? 2 : 1;
  if (p.team) {
    const auto whole = run == 8 ? gn_whole_kernel<E, A8, ACT, Q, TAIL> : run == 4 ? gn_whole_kernel<E, 2, ACT, Q, TAIL>
                       : run == 2 ? gn_whole_kernel<E, 4, ACT, Q, TAIL> : gn_whole_kernel<E, 8, ACT, Q, TAIL>;
    hipLaunchKernelGGL(whole, dim3(p.slots * p.ntile), dim3(GN_TW), gn_team_lds(p, false), st, p);
    TBG_LAUNCH_CHECK();
    return TBG_OK;
  }
  const auto sums = run == 8 ? gn_sums_kernel<E, A8, TAIL> : run == 4 ? gn_sums_kernel<E, 2, TAIL>
                    : run == 2 ? gn_sums_kernel<E, 4, TAIL> : gn_sums_kernel<E, 8, TAIL>;
  hipLaunchKernelGGL(sums, dim3(p.N * p.ntile * p.nchunk), dim3(GN_TS), 0, st, p);
  TBG_LAUNCH_CHECK();
  const auto apply = !TAIL && p.past ? gn_apply_kernel<E, ACT, Q, TAIL, !TAIL> : gn_apply_kernel<E, ACT, Q, TAIL, false>;
  hipLaunchKernelGGL(apply, dim3(p.N * p.ntile * p.nchunk * p.split), dim3(GN_T), 0, st, p);
  TBG_LAUNCH_CHECK();
  return TBG_OK;
}
template <class E, int ACT, bool Q8, bool TAIL>
static int gn_run_bwd(const GnP &p, hipStream_t st) {
  if (p.team) {
    hipLaunchKernelGGL((gn_bwd_whole_kernel<E, ACT, Q8, TAIL>), dim3(p.slots * p.ntile), dim3(GN_T), gn_team_lds(p, true), st, p);
    TBG_LAUNCH_CHECK();
    if (!p.affn && p.slots > 1) {
      hipLaunchKernelGGL(gn_params_kernel, dim3(p.pblocks), dim3(GN_T), 0, st, p);
      TBG_LAUNCH_CHECK();
    }
    return TBG_OK;
  }
  hipLaunchKernelGGL((gn_bwd_sums_kernel<E, ACT, Q8, TAIL>), dim3(p.N * p.ntile * p.nchunk), dim3(GN_TB), 0, st, p);
  TBG_LAUNCH_CHECK();
  const auto second = !TAIL && p.past ? gn_bwd_dx_kernel<E, ACT, Q8, TAIL, !TAIL> : gn_bwd_dx_kernel<E, ACT, Q8, TAIL, false>;
  hipLaunchKernelGGL(second, dim3(p.pblocks + p.N * p.ntile * p.nchunk * p.split), dim3(GN_T), 0, st, p);
  TBG_LAUNCH_CHECK();
  return TBG_OK;
}
template <class E, int ACT, bool TAIL>
static int gn_run(const GnP &p, bool backward, hipStream_t st) {
  if (backward) return p.q ? gn_run_bwd<E, ACT, true, TAIL>(p, st) : gn_run_bwd<E, ACT, false, TAIL>(p, st);
  return p.q || p.yq ? gn_run_fwd<E, ACT, true, TAIL>(p, st) : gn_run_fwd<E, ACT, false, TAIL>(p, st);
}
template <class E, bool TAIL>
static int gn_run_act(const GnP &p, int act, bool backward, hipStream_t st) {
  return act == TBG_ACT_LINEAR ? gn_run<E, TBG_ACT_LINEAR, TAIL>(p, backward, st)
         : act == TBG_ACT_LRELU ? gn_run<E, TBG_ACT_LRELU, TAIL>(p, backward, st)
                                : gn_run<E, TBG_ACT_SILU, TAIL>(p, backward, st);
}
template <class E>
static int gn_run_type(const GnP &p, int act, bool backward, hipStream_t st) {
  return p.C % 8 ? gn_run_act<E, true>(p, act, backward, st) : gn_run_act<E, false>(p, act, backward, st);
}
static int gn_dispatch(const tbg_gn_desc *d, const GnP &p, bool backward, void *stream) {
  hipStream_t st = tbg_stream(stream);
  return d->dtype == TBG_DT_F32 ? gn_run_type<ElF32>(p, d->act, backward, st)
         : d->dtype == TBG_DT_BF16 ? gn_run_type<ElBf16>(p, d->act, backward, st)
                                   : gn_run_type<ElF16>(p, d->act, backward, st);
}
// Calls that move more than the 256 MB of the card's memory-side cache read (for the second and last time) and write past the caches: lines that
// are left to be written back slow the next launch's reads, and what the first launch has read stays for the second.  32 x 16384 x 128 bf16 with 8-bit
// checkpoint (337 MB a direction): sums 33.8 -> 27.1, second launch 66 -> 54, backward sums 55.9 -> 48, second launch 63 -> 56 us.  Smaller calls
// leave their results to the next reader (unpacking a 69 MB checkpoint takes 17.4 us, 19.3 if it was written past them).  Rows of other than whole 8
// channels have no such form: their last lanes move single elements.
static bool gn_past(const tbg_gn_desc *d, int bytes) {
  return (double)d->N * d->S * d->C * bytes > 256e6;
}
static bool gn_misaligned(const void *a, const void *b) { return ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b)) & 15) != 0; }

extern "C" int tbg_group_norm_fwd(const tbg_gn_desc *d, const void *x, const float *gamma, const float *beta, void *y, double *stats,
                                  void *q, void *e, void *yq, void *ye, void *workspace, long long workspace_bytes, void *stream) {
  if (!gn_desc_ok(d) || !x || !gamma || !beta || !y || (q == nullptr) != (e == nullptr) || (yq == nullptr) != (ye == nullptr))
    return TBG_EINVAL;
  if (gn_misaligned(q, yq) || gn_misaligned(workspace, stats)) return TBG_EINVAL;
  GnP p{};
  if (const int rc = gn_geometry(d, false, q || yq, p)) return rc;
  if (gn_part_bytes(p) > (workspace ? workspace_bytes : 0)) return TBG_EINVAL;
  p.past = gn_past(d, 2 * dt_bytes(d->dtype) + (q != nullptr) + (yq != nullptr));
  p.x = x; p.gamma = gamma; p.beta = beta; p.y = y; p.stats = stats; p.part = reinterpret_cast<double *>(workspace);
  p.q = reinterpret_cast<unsigned char *>(q); p.e = reinterpret_cast<unsigned char *>(e);
  p.yq = reinterpret_cast<unsigned char *>(yq); p.ye = reinterpret_cast<unsigned char *>(ye);
  return gn_dispatch(d, p, false, stream);
}

extern "C" int tbg_group_norm_bwd(const tbg_gn_desc *d, const void *x, const void *q, const void *e, const void *dy, const float *gamma,
                                  const float *beta, const double *stats, void *dx, float *dgamma, float *dbeta, void *workspace,
                                  long long workspace_bytes, void *stream) {
  if (!gn_desc_ok(d) || !dy || !gamma || !beta || !stats || !dx || !dgamma || !dbeta || (q == nullptr) != (e == nullptr) ||
      (x == nullptr) == (q == nullptr))
    return TBG_EINVAL;
  if (gn_misaligned(q, workspace) || gn_misaligned(stats, nullptr)) return TBG_EINVAL;
  GnP p{};
  if (const int rc = gn_geometry(d, true, false, p)) return rc;
  if (gn_part_bytes(p) + gn_pch_bytes(p) > (workspace ? workspace_bytes : 0)) return TBG_EINVAL;
  p.past = gn_past(d, 2 * dt_bytes(d->dtype) + (q ? 1 : dt_bytes(d->dtype)));
  p.x = x; p.dy = dy; p.gamma = gamma; p.beta = beta; p.y = dx; p.stats = const_cast<double *>(stats);
  p.q = const_cast<unsigned char *>(reinterpret_cast<const unsigned char *>(q));
  p.e = const_cast<unsigned char *>(reinterpret_cast<const unsigned char *>(e));
  p.part = reinterpret_cast<double *>(workspace);
  p.pch = reinterpret_cast<float *>(reinterpret_cast<char *>(workspace) + gn_part_bytes(p));
  p.dgamma = dgamma; p.dbeta = dbeta;
  return gn_dispatch(d, p, true, stream);
}
