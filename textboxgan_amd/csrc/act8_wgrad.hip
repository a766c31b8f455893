// Weight and bias gradient of a dense (1x1) layer from the 8-bit checkpoint of its input (tbg.h "tbg_act8_wgrad"):
//   dw[k][n] = coef sum_r x[r][k] dy[r][n],   db[n] = sum_r dy[r][n],   x = q 2^e.
//
// x has 7 significant bits, so it is EXACT in bf16 and the product runs on the bf16 matrix pipe without rounding either operand: dy is one
// bf16 term (bf16), two (fp16: 11 bits = 8 + 3) or three (fp32: 24 = 8 + 8 + 8), accumulated in fp32.
//
// Both operands are stored with the reduction axis (rows) outermost.  A block stages RB rows of both tiles in LDS as they lie -- the
// checkpoint scaled and converted on the way, dy split into its terms -- and the transposing LDS read (ds_read_b64_tr_b16) hands each lane
// 4 rows of its channel: no transposition pass over either tensor.  The rows are split over blocks; partial products are joined by a second
// launch in a fixed order.
#include "act8.h"

#include <type_traits>

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

struct A8wP {
  const unsigned char *q, *e;
  const void *dy;
  float *out, *dbout;  // partial sums [split][cin][cout], [split][cout]; one split: dw, db themselves
  long long rows, ldy, rsplit;  // rsplit: rows a split (a multiple of RB)
  int cin, cout, pitch, nsplit, tk, tn;
  float coef;
  int want_db;
};

constexpr int A8W_RB = 32, A8W_PAD = 32;  // rows a stage; elements between two LDS rows (the 4 rows x 64 B of two transposing reads: all 64 banks)

// the bf16 terms of 8 values of dy, largest first, by truncation: every remainder is exact and nothing overflows (an infinity leaves NaN behind)
template <int NP>
__device__ __forceinline__ void a8w_terms(const float (&v)[8], Pack8<ElBf16> (&w)[NP]) {
  float rest[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) rest[j] = v[j];
#pragma unroll
  for (int m = 0; m < NP; ++m) {
    unsigned u[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) u[j] = __builtin_amdgcn_perm(__float_as_uint(rest[2 * j + 1]), __float_as_uint(rest[2 * j]), 0x07060302u);
    __builtin_memcpy(&w[m], u, 16);
    if (m + 1 < NP) {
#pragma unroll
      for (int j = 0; j < 8; ++j) rest[j] -= __uint_as_float(__float_as_uint(rest[j]) & 0xffff0000u);
    }
  }
}

// a wave's products: entry (8 (r / 4) + 4 (lane / 32) + r % 4, lane % 32) of each 32 x 32 in register r
template <int WM, int WN>
__device__ __forceinline__ void a8w_store(const A8wP &p, const f32x16 (&acc)[WM][WN], int z, int k, int n, bool whole, int lane) {
  float *out = p.out + (long long)z * p.cin * p.cout;
  const float f = p.nsplit == 1 ? p.coef : 1.f;
  const int kl = k + 4 * (lane >> 5), nl = n + (lane & 31);
#pragma unroll
  for (int i = 0; i < WM; ++i)
#pragma unroll
    for (int j = 0; j < WN; ++j) {
      float *o = out + (long long)(kl + 32 * i) * p.cout + nl + 32 * j;
      if (whole) {
#pragma unroll
        for (int r = 0; r < 16; ++r) o[(8 * (r >> 2) + (r & 3)) * (long long)p.cout] = f * acc[i][j][r];
      } else {
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (kl + 32 * i + 8 * (r >> 2) + (r & 3) < p.cin && nl + 32 * j < p.cout) o[(8 * (r >> 2) + (r & 3)) * (long long)p.cout] = f * acc[i][j][r];
      }
    }
}

// KW x NW waves of WM x WN products of 32 x 32.  Three LDS buffers and one barrier a stage: while the block multiplies stage t it writes stage
// t + 2, which its registers hold, and reads the first operands of stage t + 1, so that the matrix pipe has work right behind the barrier; the
// loads of stage t + 4 go into the registers that this frees.  Whole stages only; rows left over go through stages of their own at the end.
template <class E, int NP, int WM, int WN, int KW, int NW, bool VEC>
__global__ __launch_bounds__(64 * KW * NW, 2) void act8_wgrad_kernel(A8wP p) {
  constexpr int T = 64 * KW * NW, TK = 32 * WM * KW, TN = 32 * WN * NW, PK = TK + A8W_PAD, PN = TN + A8W_PAD;
  constexpr int BUF = A8W_RB * (PK + NP * PN);  // elements of one buffer: the checkpoint's tile, then dy's terms
  // a lane stages the same column of every stage: 8 channels of XN rows of the checkpoint, 8 columns of DN rows of dy
  constexpr int XR = T / (TK / 8), DR = T / (TN / 8), XN = A8W_RB / XR, DN = A8W_RB / DR;
  static_assert(XN * XR == A8W_RB && DN * DR == A8W_RB && XR * (TK / 8) == T && DR * (TN / 8) == T, "pieces of a stage");
  extern __shared__ __align__(16) char smem[];
  unsigned short *lds = reinterpret_cast<unsigned short *>(smem);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wk = wave % KW, wn = wave / KW;
  // (split, tile) pairs, a split's tiles together, in 8 equal runs: blocks go round the 8 XCDs, so that the tiles that share a split's rows share an L2,
  // and all XCDs have the same work whatever the number of splits
  const int tiles = p.tk * p.tn, pairs = p.nsplit * tiles;
  int b = (blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3);
  if (b >= pairs) return;
  const int z = b / tiles;
  b -= z * tiles;
  const int k0 = (b / p.tn) * TK, n0 = (b % p.tn) * TN;
  const long long r0 = z * p.rsplit, rend = min(p.rows, r0 + p.rsplit);
  const bool do_db = p.want_db && k0 == 0;

  const int i16 = lane & 15, grp = lane >> 4, jj = i16 >> 2, cq = i16 & 3, chblk = grp & 1, khalf = grp >> 1;
  const int a_off = (8 * khalf + jj) * PK + wk * 32 * WM + chblk * 16 + cq * 4;
  const int b_off = A8W_RB * PK + (8 * khalf + jj) * PN + wn * 32 * WN + chblk * 16 + cq * 4;
  auto rd = [](const unsigned short *ptr, int pitch) -> bf16x8 {  // 8 rows of this lane's channel
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)(ptr));
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)(ptr + 4 * pitch));
    return __builtin_bit_cast(bf16x8, s16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]});
  };

  f32x16 acc[WM][WN];
#pragma unroll
  for (int i = 0; i < WM; ++i)
#pragma unroll
    for (int j = 0; j < WN; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
  float dbs[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) dbs[i] = 0.f;

  struct Regs {
    u32x2 xq[XN];
    unsigned xe[XN];
    Pack8<E> dv[DN];
  };
  const int xrow = tid / (TK / 8), xc = (tid % (TK / 8)) * 8, drow = tid / (TN / 8), dc = (tid % (TN / 8)) * 8, epitch = p.pitch / A8_BLOCK;
  // pieces beyond the last channel read one that exists (their products are not stored)
  const int xat = min(k0 + xc, p.pitch - 8), dat = VEC ? min(n0 + dc, p.cout - 8) : min(n0 + dc, p.cout - 1);
  const typename E::type *dy = reinterpret_cast<const typename E::type *>(p.dy);
  const unsigned qoff = xrow * p.pitch + xat, eoff = xrow * epitch + xat / A8_BLOCK, doff = drow * (unsigned)p.ldy + dat;
  auto fetch = [&](Regs &g, long long r) {  // a whole stage, rows r .. r + 31
    const unsigned char *qp = p.q + r * p.pitch, *ep = p.e + r * epitch;
    const typename E::type *dp = dy + r * p.ldy;
#pragma unroll
    for (int i = 0; i < XN; ++i) {
      g.xq[i] = *reinterpret_cast<const u32x2 *>(qp + (size_t)XR * i * p.pitch + qoff);
      g.xe[i] = (ep + (size_t)XR * i * epitch)[eoff];
    }
#pragma unroll
    for (int i = 0; i < DN; ++i) g.dv[i] = ld8<E>(dp + (size_t)DR * i * p.ldy + doff);
  };
  auto fetch_some = [&](Regs &g, long long r) {  // fewer rows, the others zero; dy by elements
#pragma unroll
    for (int i = 0; i < XN; ++i) {
      g.xq[i] = u32x2{0, 0};
      g.xe[i] = 0;
      if (r + xrow + XR * i < rend) {
        g.xq[i] = *reinterpret_cast<const u32x2 *>(p.q + (r + XR * i) * p.pitch + qoff);
        g.xe[i] = p.e[(r + XR * i) * epitch + eoff];
      }
    }
#pragma unroll
    for (int i = 0; i < DN; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        g.dv[i].v[j] = 0;
        if (r + drow + DR * i < rend && n0 + dc + j < p.cout) g.dv[i].v[j] = dy[(r + drow + DR * i) * p.ldy + n0 + dc + j];
      }
  };
  auto stage = [&](unsigned short *buf, const Regs &g) {
#pragma unroll
    for (int i = 0; i < XN; ++i) {
      const float s = a8_scale(g.xe[i]);
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = a8_value(g.xq[i], j) * s;
      st8_lds(buf + (xrow + XR * i) * PK + xc, put8<ElBf16>(v));
    }
#pragma unroll
    for (int i = 0; i < DN; ++i) {
      Pack8<ElBf16> w[NP];
      if constexpr (NP == 1) {
        __builtin_memcpy(&w[0], &g.dv[i], 16);
      } else {
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = E::get(g.dv[i].v[j]);
        a8w_terms<NP>(v, w);
      }
#pragma unroll
      for (int m = 0; m < NP; ++m) st8_lds(buf + A8W_RB * PK + (m * A8W_RB + drow + DR * i) * PN + dc, w[m]);
    }
  };
  auto column_sums = [&](const Regs &g) {
#pragma unroll
    for (int i = 0; i < DN; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) dbs[j] += E::get(g.dv[i].v[j]);
  };
  struct Ops {  // 16 rows' operands
    bf16x8 a[WM], d[WN][NP];
  };
  auto operands = [&](const unsigned short *buf, int s) {
    Ops o;
#pragma unroll
    for (int i = 0; i < WM; ++i) o.a[i] = rd(buf + a_off + 16 * s * PK + 32 * i, PK);
#pragma unroll
    for (int j = 0; j < WN; ++j)
#pragma unroll
      for (int m = 0; m < NP; ++m) o.d[j][m] = rd(buf + b_off + (m * A8W_RB + 16 * s) * PN + 32 * j, PN);
    return o;
  };
  auto multiply = [&](const Ops &o) {
#pragma unroll
    for (int j = 0; j < WN; ++j)
#pragma unroll
      for (int m = NP - 1; m >= 0; --m)  // smallest terms first
#pragma unroll
        for (int i = 0; i < WM; ++i) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(o.a[i], o.d[j][m], acc[i][j], 0, 0, 0);
  };
  // whole stages.  Where the columns are not a multiple of 8, a load of 8 may pass a row's end by 7: the last rows, whose loads would pass the
  // tensor's end, are left to the masked stages
  const long long margin = VEC ? 0 : (6 + p.ldy) / p.ldy;
  const int full = (int)max((min(rend, p.rows - margin) - r0) / A8W_RB, 0LL);
  unsigned short *cur = lds, *next = lds + BUF, *last = lds + 2 * BUF;
  auto whole_stages = [&](auto sums) {
    Regs g[2];
    const auto load = [&](Regs &to, int t) { fetch(to, r0 + (long long)min(t, full - 1) * A8W_RB); };  // (behind the last stage: that one again)
    const auto put = [&](unsigned short *buf, const Regs &from, bool counts) {
      stage(buf, from);
      if (sums.value) {  // branch-free, as the whole loop body is
#pragma unroll
        for (int i = 0; i < DN; ++i)
#pragma unroll
          for (int j = 0; j < 8; ++j) dbs[j] += counts ? E::get(from.dv[i].v[j]) : 0.f;
      }
    };
    load(g[0], 0);
    load(g[1], 1);
    put(cur, g[0], true);
    load(g[0], 2);
    put(next, g[1], 1 < full);
    load(g[1], 3);
    __syncthreads();
    Ops lo = operands(cur, 0);
    for (int t = 0; t < full; t += 2) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        if (t + u < full) {
          const Ops hi = operands(cur, 1);
          multiply(lo);
          lo = operands(next, 0);
          put(last, g[u], t + u + 2 < full);
          load(g[u], t + u + 4);
          multiply(hi);
          __syncthreads();
          unsigned short *x = cur; cur = next; next = last; last = x;
        }
      }
    }
  };
  if (full > 0) {
    if (do_db) whole_stages(std::true_type());
    else whole_stages(std::false_type());
  }
  for (long long r = r0 + (long long)full * A8W_RB; r < rend; r += A8W_RB) {  // (nobody reads this buffer any more: the barriers above, below)
    Regs g;
    fetch_some(g, r);
    stage(cur, g);
    if (do_db) column_sums(g);
    __syncthreads();
    multiply(operands(cur, 0));
    multiply(operands(cur, 1));
    __syncthreads();
  }

  a8w_store<WM, WN>(p, acc, z, k0 + wk * 32 * WM, n0 + wn * 32 * WN, k0 + TK <= p.cin && n0 + TN <= p.cout, lane);
  if (do_db) {
    float *red = reinterpret_cast<float *>(smem);  // [T][8]; every wave is past its last operand read
#pragma unroll
    for (int j = 0; j < 8; ++j) red[tid * 8 + j] = dbs[j];
    __syncthreads();
    if (tid < TN && n0 + tid < p.cout) {
      float a = 0.f;
      for (int l = 0; l < DR; ++l) a += red[(l * (TN / 8) + tid / 8) * 8 + (tid & 7)];
      p.dbout[(long long)z * p.cout + n0 + tid] = a;
    }
  }
}

// dw = coef sum of the splits' products, db = sum of theirs.  A lane takes V neighbouring entries; `ranks` lanes (4 to 64) take every ranks-th
// split of the same entries each, joined through LDS: the loads are what there is to wait for, and small products have few entries.
template <int V>
__global__ __launch_bounds__(256) void act8_wgrad_join_kernel(const float *ws, const float *dbws, float *dw, float *db, long long kn, int cout,
                                                              int nsplit, int ranks, float coef) {
  typedef float vec __attribute__((ext_vector_type(V)));
  __shared__ vec red[256];
  const int wide = 256 / ranks, lane = threadIdx.x & (wide - 1), rank = threadIdx.x / wide;
  long long i = ((long long)blockIdx.x * wide + lane) * V;
  const bool bias = i >= kn;
  if (bias) i -= kn;
  const bool live = !bias || (db && i < cout);
  const long long len = bias ? cout : kn;
  const float *src = (bias ? dbws : ws) + i;
  vec a;
#pragma unroll
  for (int j = 0; j < V; ++j) a[j] = 0.f;
  if (live) {
#pragma unroll 8
    for (int z = rank; z < nsplit; z += ranks) a += *reinterpret_cast<const vec *>(src + z * len);
  }
  red[threadIdx.x] = a;
  for (int half = ranks >> 1; half > 0; half >>= 1) {
    __syncthreads();
    if (rank < half) red[threadIdx.x] += red[threadIdx.x + half * wide];
  }
  if (rank == 0 && live) *reinterpret_cast<vec *>((bias ? db : dw) + i) = (bias ? 1.f : coef) * red[threadIdx.x];
}

// Tile and row splits.  The tile: the largest that the channels fill (fewer re-reads of both operands, fewer operand reads an MFMA), made
// smaller while splits of 256 rows would leave a quarter of the CUs without a block; the splits then fill the card once: as many blocks a CU as its
// registers and its 160 KB of LDS hold (the three buffers take 60 KB for 128 x 128 of one term, 120 KB of three).  Calls, us, with the splits of one
// round of blocks / of two: fp32 65536 x 256 x 256 44 / 50, 262144 x 64 x 64 24 / 30, 20000 x 1024 x 512 89 / 93; fp16 36 / 43, 21 / 27, 69 / 72, but
// 262144 x 512 x 512 407 / 391.  Measured, us of kernels:
// 262144 x 512 x 512 bf16 158 + 12 (join) with 256 x 256 tiles, 200 with 128 x 128; fp32 (three terms: 256 x 256 tiles do not fit the registers)
// 16384 x 256 x 256 20 + 4 with 128 x 128 tiles.
// Up to 512 rows are not split: a second launch and its partial sums cost the host 4 us (a call 12.3 / 16.4 us, whichever of the two is longer), and the
// GPU more than the split saves where the product is wide.  Us of the GPU alone, whole / split:
//   64 x 64      bf16 256 rows 5.5 / 6.5, 512 8.0 / 6.6, 768 10.6 / 6.7; fp16 256 6.4 / 7.0, 512 9.7 / 7.1; fp32 256 7.0 / 7.4, 512 10.9 / 7.5
//   512 x 512    bf16 256 5.6 / 7.4, 512 8.2 / 8.5, 768 10.7 / 10.3; fp16 256 6.5 / 7.9, 512 9.9 / 9.2; fp32 256 7.2 / 8.4, 512 11.3 / 9.6
//   1024 x 1024  bf16 256 6.0 / 13.0, 512 8.7 / 20.4, 640 14.2 / 16.7; fp16 512 10.4 / 15.5, 640 18.8 / 18.1; fp32 512 11.5 / 16.6, 640 23.9 / 20.3
// (narrow products in a captured graph, which has no host, lose up to 3.4 us).
struct A8wGeo {
  int form, tk, tn, nsplit;
  long long rsplit;
};
struct A8wForm {
  int tk, tn, per_cu;  // blocks a CU, as far as the registers go
};
static constexpr A8wForm A8W_FORMS[] = {{256, 256, 1}, {128, 128, 2}, {128, 64, 2}, {64, 128, 2}, {64, 64, 4}};
static constexpr long long a8w_lds(int tk, int tn, int terms) { return 3LL * A8W_RB * (tk + A8W_PAD + terms * (tn + A8W_PAD)) * 2; }
static A8wGeo a8w_geometry(long long rows, int cin, int cout, int dtype) {
  A8wGeo g;
  const long long most = (rows + 8 * A8W_RB - 1) / (8 * A8W_RB);
  for (g.form = cin > 128 && cout > 128 && dtype == TBG_DT_BF16 ? 0 : cin > 64 ? (cout > 64 ? 1 : 2) : (cout > 64 ? 3 : 4);; g.form = g.form == 0 ? 1 : 4) {
    g.tk = (cin + A8W_FORMS[g.form].tk - 1) / A8W_FORMS[g.form].tk;
    g.tn = (cout + A8W_FORMS[g.form].tn - 1) / A8W_FORMS[g.form].tn;
    if ((long long)g.tk * g.tn * most >= 192 || g.form == 4) break;
  }
  const A8wForm &f = A8W_FORMS[g.form];
  const long long fits = 160 * 1024 / a8w_lds(f.tk, f.tn, dtype == TBG_DT_F32 ? 3 : dtype == TBG_DT_F16 ? 2 : 1);
  long long want = 256LL * (f.per_cu < fits ? f.per_cu : fits) / ((long long)g.tk * g.tn);
  const long long cap = rows <= 512 ? 1 : g.form == 4 ? (rows + 4 * A8W_RB - 1) / (4 * A8W_RB) : most;
  if (want > cap) want = cap;
  if (want < 1) want = 1;
  g.rsplit = ((rows + want - 1) / want + A8W_RB - 1) / A8W_RB * A8W_RB;
  g.nsplit = (int)((rows + g.rsplit - 1) / g.rsplit);
  return g;
}

static int a8w_args(long long rows, int cin, int cout, int dtype) {
  if (rows < 1 || cin < 1 || cout < 1 || !dt_valid(dtype)) return TBG_EINVAL;
  if (cin > (1 << 20) || cout > (1 << 20) || (long long)cin * cout > (1LL << 31) || rows > (1LL << 40)) return TBG_ERANGE;
  return TBG_OK;
}

// partial sums: products of every split, then column sums of every split
static long long a8w_workspace(const A8wGeo &g, int cin, int cout) {
  return g.nsplit == 1 ? 0 : (long long)g.nsplit * ((long long)cin * cout + cout) * (long long)sizeof(float);
}

extern "C" long long tbg_act8_wgrad_workspace_bytes(long long rows, int cin, int cout, int dtype) {
  if (const int rc = a8w_args(rows, cin, cout, dtype)) return rc;
  const A8wGeo g = a8w_geometry(rows, cin, cout, dtype);
  return a8w_workspace(g, cin, cout);
}

template <class E, int NP, int WM, int WN, int KW, int NW>
static int a8w_launch(const A8wP &p, bool vec, hipStream_t st) {
  constexpr size_t lds = a8w_lds(32 * WM * KW, 32 * WN * NW, NP);
  const unsigned blocks = (unsigned)((p.nsplit * p.tk * p.tn + 7) / 8 * 8);
  const auto kern = vec ? act8_wgrad_kernel<E, NP, WM, WN, KW, NW, true> : act8_wgrad_kernel<E, NP, WM, WN, KW, NW, false>;
  if (lds > 65536 && hipFuncSetAttribute(reinterpret_cast<const void *>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds) != hipSuccess)
    return TBG_EHIP;
  hipLaunchKernelGGL(kern, dim3(blocks), dim3(64 * KW * NW), lds, st, p);
  TBG_LAUNCH_CHECK();
  return TBG_OK;
}
template <class E, int NP>
static int a8w_tiles(const A8wP &p, const A8wGeo &g, bool vec, hipStream_t st) {
  switch (g.form) {
    case 0:
      if constexpr (NP == 1) return a8w_launch<E, NP, 4, 2, 2, 4>(p, vec, st);
      return TBG_EINVAL;
    case 1: return a8w_launch<E, NP, 2, 2, 2, 2>(p, vec, st);
    case 2: return a8w_launch<E, NP, 2, 1, 2, 2>(p, vec, st);
    case 3: return a8w_launch<E, NP, 1, 2, 2, 2>(p, vec, st);
    default: return a8w_launch<E, NP, 1, 1, 2, 2>(p, vec, st);
  }
}

// joins the splits' partial sums of dw (kn entries) and db
static int a8w_join(const float *ws, const float *dbws, float *dw, float *db, long long kn, int cout, int nsplit, float coef, hipStream_t st) {
  const bool v4 = cout % 4 == 0 && ((reinterpret_cast<uintptr_t>(dw) | reinterpret_cast<uintptr_t>(db)) & 15) == 0;
  const long long lanes = (kn + (db ? cout : 0) + (v4 ? 3 : 0)) / (v4 ? 4 : 1);
  int ranks = 4;  // more while the launch has less than a block a CU
  while (ranks < 64 && ranks < nsplit && lanes * ranks < 256 * 256) ranks <<= 1;
  hipLaunchKernelGGL(v4 ? act8_wgrad_join_kernel<4> : act8_wgrad_join_kernel<1>, dim3((unsigned)((lanes * ranks + 255) / 256)), dim3(256), 0, st, ws,
                     dbws, dw, db, kn, cout, nsplit, ranks, coef);
  TBG_LAUNCH_CHECK();
  return TBG_OK;
}

extern "C" int tbg_act8_wgrad(const void *q, const void *e, const void *dy, int dtype, long long rows, int cin, int cout, long long ldy,
                              float coef, float *dw, float *db, void *workspace, long long workspace_bytes, void *stream) {
  if (!q || !e || !dy || !dw || ldy < cout || (reinterpret_cast<uintptr_t>(q) & 15) != 0) return TBG_EINVAL;
  if (const int rc = a8w_args(rows, cin, cout, dtype)) return rc;
  if (ldy > (1LL << 26)) return TBG_ERANGE;
  const A8wGeo g = a8w_geometry(rows, cin, cout, dtype);
  if ((long long)(g.nsplit + 7) * g.tk * g.tn >= 1LL << 23) return TBG_ERANGE;  // a grid holds less than 2^32 threads
  const long long kn = (long long)cin * cout, need = a8w_workspace(g, cin, cout);
  if (need > workspace_bytes || (need && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15) != 0))) return TBG_EINVAL;
  A8wP p{};
  p.q = reinterpret_cast<const unsigned char *>(q); p.e = reinterpret_cast<const unsigned char *>(e); p.dy = dy;
  p.rows = rows; p.ldy = ldy; p.rsplit = g.rsplit; p.cin = cin; p.cout = cout; p.pitch = (cin + A8_BLOCK - 1) / A8_BLOCK * A8_BLOCK;
  p.nsplit = g.nsplit; p.tk = g.tk; p.tn = g.tn; p.coef = coef; p.want_db = db != nullptr;
  float *ws = reinterpret_cast<float *>(workspace);
  p.out = g.nsplit == 1 ? dw : ws;
  p.dbout = g.nsplit == 1 ? db : ws + g.nsplit * kn;
  const bool vec = cout % 8 == 0;
  hipStream_t st = tbg_stream(stream);
  const int rc = dtype == TBG_DT_F32 ? a8w_tiles<ElF32, 3>(p, g, vec, st)
                 : dtype == TBG_DT_BF16 ? a8w_tiles<ElBf16, 1>(p, g, vec, st)
                                        : a8w_tiles<ElF16, 2>(p, g, vec, st);
  if (rc || g.nsplit == 1) return rc;
  return a8w_join(ws, ws + g.nsplit * kn, dw, db, kn, cout, g.nsplit, coef, st);
}

// ---- bias gradient alone (the weight is frozen: no checkpoint): db[n] = sum_r dy[r][n].  Memory-bound; a lane sums 8 neighbouring columns of every
// RL-th row of its split in fp32, the block's lanes join through LDS, the splits in the join launch, all in a fixed order.
// Measured, a call: 262144 x 512 bf16 43 us (268 MB: 6.2 TB/s), x 128 15 us, 100000 x 72 fp32 11.5 us (kernels 9.1), 512 x 512 bf16 7.2 us (6.0).
template <class E, bool TAIL>
__global__ __launch_bounds__(256) void column_sums_kernel(const typename E::type *__restrict__ x, long long rows, int cols, long long ldx, long long rsplit,
                                                          int lanes, int tiles, float *__restrict__ out) {
  constexpr int U = 4;  // rows under way
  __shared__ float red[256 * 8];
  const int lane = threadIdx.x & (lanes - 1), rl = threadIdx.x / lanes, RL = 256 / lanes;
  const int c0 = blockIdx.x % tiles * lanes * 8, c = c0 + lane * 8;
  const long long z = blockIdx.x / tiles, r1 = min(rows, (z + 1) * rsplit);
  float s[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) s[i] = 0.f;
  if (c < cols) {
    const auto add = [&](const Pack8<E> &v) {
#pragma unroll
      for (int i = 0; i < 8; ++i) s[i] += E::get(v.v[i]);
    };
    const Row8<E, TAIL> row(c, cols);
    long long r = z * rsplit + rl;
    const typename E::type *p = x + r * ldx;
    const long long step = RL * ldx;
    for (; r + (U - 1) * RL < r1; r += U * RL) {
      Pack8<E> v[U];
#pragma unroll
      for (int u = 0; u < U; ++u, p += step) v[u] = row.load(p);
#pragma unroll
      for (int u = 0; u < U; ++u) add(v[u]);
    }
    for (; r < r1; r += RL, p += step) add(row.load(p));
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) red[threadIdx.x * 8 + i] = s[i];
  __syncthreads();
  const int j = threadIdx.x;
  if (j < lanes * 8 && c0 + j < cols) {
    float a = 0.f;
    for (int k = 0; k < RL; ++k) a += red[k * lanes * 8 + j];
    out[z * cols + c0 + j] = a;
  }
}

struct ColumnGeo {
  int lanes, tiles, nsplit;
  long long rsplit;
};
// Up to 256 columns a block; one split up to 64 rows a lane, else splits for two blocks a CU of 16 rows a lane or more.  Bf16, us of the GPU (of a call),
// one split / splits of 16 rows a lane: 256 x 512 4.3 (7.2) / 5.5 (11.3), 512 x 512 6.0 (7.2) / 5.6 (11.3), 2048 x 64 6.1 (7.2) / 5.5 (11.6), 1024 x 512
// 9.7 (10.2) / 5.8 (11.3), 2048 x 512 17 (17) / 6.0 (11.2); 16384 x 512 with splits of 4, 16, 64 rows a lane 7.2, 7.6, 8.8.
static ColumnGeo column_geometry(long long rows, int cols) {
  ColumnGeo g;
  g.lanes = 1;
  while (g.lanes < 32 && g.lanes * 8 < cols) g.lanes <<= 1;
  g.tiles = (cols + g.lanes * 8 - 1) / (g.lanes * 8);
  const long long lines = 256 / g.lanes, cap = rows <= 64 * lines ? 1 : (rows + 16 * lines - 1) / (16 * lines);
  long long want = 512 / g.tiles;
  if (want > cap) want = cap;
  if (want < 1) want = 1;
  g.rsplit = (rows + want - 1) / want;
  g.nsplit = (int)((rows + g.rsplit - 1) / g.rsplit);
  return g;
}
static long long column_workspace(const ColumnGeo &g, int cols) { return g.nsplit == 1 ? 0 : (long long)g.nsplit * cols * (long long)sizeof(float); }
static int column_args(long long rows, int cols, int dtype) {
  if (rows < 1 || cols < 1 || !dt_valid(dtype)) return TBG_EINVAL;
  return cols > (1 << 30) || rows > (1LL << 40) ? TBG_ERANGE : TBG_OK;
}

extern "C" long long tbg_column_sums_workspace_bytes(long long rows, int cols, int dtype) {
  if (const int rc = column_args(rows, cols, dtype)) return rc;
  return column_workspace(column_geometry(rows, cols), cols);
}

template <class E>
static int column_launch(const void *x, long long rows, int cols, long long ldx, const ColumnGeo &g, float *out, hipStream_t st) {
  hipLaunchKernelGGL((cols % 8 ? column_sums_kernel<E, true> : column_sums_kernel<E, false>), dim3((unsigned)(g.nsplit * g.tiles)), dim3(256), 0, st,
                     reinterpret_cast<const typename E::type *>(x), rows, cols, ldx, g.rsplit, g.lanes, g.tiles, out);
  TBG_LAUNCH_CHECK();
  return TBG_OK;
}

extern "C" int tbg_column_sums(const void *x, int dtype, long long rows, int cols, long long ldx, float *out, void *workspace, long long workspace_bytes,
                               void *stream) {
  if (!x || !out || ldx < cols) return TBG_EINVAL;
  if (const int rc = column_args(rows, cols, dtype)) return rc;
  const ColumnGeo g = column_geometry(rows, cols);
  const long long need = column_workspace(g, cols);
  if (need > workspace_bytes || (need && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15) != 0))) return TBG_EINVAL;
  float *part = need ? reinterpret_cast<float *>(workspace) : out;
  hipStream_t st = tbg_stream(stream);
  const int rc = dtype == TBG_DT_F32 ? column_launch<ElF32>(x, rows, cols, ldx, g, part, st)
                 : dtype == TBG_DT_BF16 ? column_launch<ElBf16>(x, rows, cols, ldx, g, part, st)
                                        : column_launch<ElF16>(x, rows, cols, ldx, g, part, st);
  return rc || !need ? rc : a8w_join(nullptr, part, nullptr, out, 0, cols, g.nsplit, 1.f, st);
}
