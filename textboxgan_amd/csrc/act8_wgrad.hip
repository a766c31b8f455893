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

constexpr int A8W_RB = 32, A8W_PAD = 16;  // rows a stage; elements between two LDS rows (4 rows x 32 B of one transposing read: 4 bank groups)

// the bf16 terms of dy, largest first, by truncation: every remainder is exact and nothing overflows
template <int NP>
__device__ __forceinline__ void a8w_terms(float v, unsigned short (&t)[NP]) {
  const bool fine = (__float_as_uint(v) & 0x7f800000u) != 0x7f800000u;
  float rest = v;
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const unsigned hi = __float_as_uint(rest) & 0xffff0000u;
    t[i] = fine ? (unsigned short)(hi >> 16) : (i == 0 ? ElBf16::put(v) : (unsigned short)0);
    rest -= __uint_as_float(hi);
  }
}

// One barrier a stage: the block multiplies stage t out of one LDS buffer, writes stage t + 1 (loaded into registers a stage ago) to the other
// and issues the loads of stage t + 2, so a global load has a whole stage to land.  2 blocks a CU cover each other's waits.
template <class E, int NP, int WM, int WN, bool VEC>
__global__ __launch_bounds__(256, 2) void act8_wgrad_kernel(A8wP p) {
  constexpr int TK = 64 * WM, TN = 64 * WN, PK = TK + A8W_PAD, PN = TN + A8W_PAD;
  constexpr int BUF = A8W_RB * (PK + NP * PN);  // elements of one buffer: the checkpoint's tile, then dy's terms
  extern __shared__ __align__(16) char smem[];
  unsigned short *lds = reinterpret_cast<unsigned short *>(smem);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wk = wave & 1, wn = wave >> 1;
  // 8 neighbouring splits x all tiles of a split: blocks go round the 8 XCDs, so the tiles that share a split's rows share an L2
  const int tiles = p.tk * p.tn;
  int b = blockIdx.x;
  const int z = b / (8 * tiles) * 8 + (b & 7);
  b = b % (8 * tiles) / 8;
  if (z >= p.nsplit) return;
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

  // a lane stages the same column of every stage: 8 channels of WM rows of the checkpoint and 8 columns of WN rows of dy
  constexpr int XR = 256 / (TK / 8), DR = 256 / (TN / 8);  // rows between a lane's pieces
  const int xrow = tid / (TK / 8), xc = (tid % (TK / 8)) * 8, drow = tid / (TN / 8), dc = (tid % (TN / 8)) * 8;
  const bool xin = k0 + xc < p.pitch, din = n0 + dc < p.cout;
  const int epitch = p.pitch / A8_BLOCK;
  const unsigned char *qp = p.q + (r0 + xrow) * p.pitch + k0 + xc;
  const unsigned char *ep = p.e + (r0 + xrow) * epitch + (k0 + xc) / A8_BLOCK;
  const typename E::type *dp = reinterpret_cast<const typename E::type *>(p.dy) + (r0 + drow) * p.ldy + n0 + dc;
  u32x2 xq[WM];
  unsigned xe[WM];
  Pack<E, 8> dv[WN];
#pragma unroll
  for (int i = 0; i < WM; ++i) { xq[i] = u32x2{0, 0}; xe[i] = 0; }
#pragma unroll
  for (int i = 0; i < WN; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) dv[i].v[j] = 0;
  auto fetch_dy = [&](Pack<E, 8> &v, const typename E::type *src) {
    if constexpr (VEC) {
      if (din) v = ld_pack<E, 8>(src);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (n0 + dc + j < p.cout) v.v[j] = src[j];
    }
  };
  auto fetch = [&](long long r) {  // the next stage, rows r .. r + 31; rows and columns that do not exist are zeros
    if (r + A8W_RB <= rend) {
      if (xin) {
#pragma unroll
        for (int i = 0; i < WM; ++i) {
          xq[i] = *reinterpret_cast<const u32x2 *>(qp + XR * i * p.pitch);
          xe[i] = ep[XR * i * epitch];
        }
      }
#pragma unroll
      for (int i = 0; i < WN; ++i) fetch_dy(dv[i], dp + DR * i * p.ldy);
    } else {
#pragma unroll
      for (int i = 0; i < WM; ++i) {
        xq[i] = u32x2{0, 0};
        xe[i] = 0;
        if (xin && r + xrow + XR * i < rend) {
          xq[i] = *reinterpret_cast<const u32x2 *>(qp + XR * i * p.pitch);
          xe[i] = ep[XR * i * epitch];
        }
      }
#pragma unroll
      for (int i = 0; i < WN; ++i) {
#pragma unroll
        for (int j = 0; j < 8; ++j) dv[i].v[j] = 0;
        if (r + drow + DR * i < rend) fetch_dy(dv[i], dp + DR * i * p.ldy);
      }
    }
    qp += A8W_RB * p.pitch;
    ep += A8W_RB * epitch;
    dp += A8W_RB * p.ldy;
  };
  auto stage = [&](unsigned short *buf) {
#pragma unroll
    for (int i = 0; i < WM; ++i) {
      const float s = a8_scale(xe[i]);
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = (float)(int)(signed char)(xq[i][j >> 2] >> (8 * (j & 3)) & 0xff) * s;
      st_pack<ElBf16, 8>(buf + (xrow + XR * i) * PK + xc, put_pack<ElBf16, 8>(v));
    }
#pragma unroll
    for (int i = 0; i < WN; ++i) {
      Pack<ElBf16, 8> w[NP];
      if constexpr (NP == 1) {
        __builtin_memcpy(&w[0], &dv[i], 16);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          unsigned short t[NP];
          a8w_terms<NP>(E::get(dv[i].v[j]), t);
#pragma unroll
          for (int m = 0; m < NP; ++m) w[m].v[j] = t[m];
        }
      }
      if (do_db) {
#pragma unroll
        for (int j = 0; j < 8; ++j) dbs[j] += E::get(dv[i].v[j]);
      }
#pragma unroll
      for (int m = 0; m < NP; ++m) st_pack<ElBf16, 8>(buf + A8W_RB * PK + (m * A8W_RB + drow + DR * i) * PN + dc, w[m]);
    }
  };

  fetch(r0);
  stage(lds);
  fetch(r0 + A8W_RB);
  __syncthreads();
  int cur = 0;
  for (long long r = r0; r < rend; r += A8W_RB) {
    const unsigned short *buf = lds + cur * BUF;
#pragma unroll
    for (int s = 0; s < A8W_RB / 16; ++s) {
      bf16x8 a[WM];
#pragma unroll
      for (int i = 0; i < WM; ++i) a[i] = rd(buf + a_off + 16 * s * PK + 32 * i, PK);
#pragma unroll
      for (int j = 0; j < WN; ++j)
#pragma unroll
        for (int m = NP - 1; m >= 0; --m) {  // smallest terms first
          const bf16x8 d = rd(buf + b_off + (m * A8W_RB + 16 * s) * PN + 32 * j, PN);
#pragma unroll
          for (int i = 0; i < WM; ++i) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[i], d, acc[i][j], 0, 0, 0);
        }
    }
    cur ^= 1;
    stage(lds + cur * BUF);
    fetch(r + 2 * A8W_RB);
    __syncthreads();
  }

  float *out = p.out + (long long)z * p.cin * p.cout;
  const float f = p.nsplit == 1 ? p.coef : 1.f;
#pragma unroll
  for (int i = 0; i < WM; ++i)
#pragma unroll
    for (int j = 0; j < WN; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int k = k0 + wk * 32 * WM + 32 * i + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3), n = n0 + wn * 32 * WN + 32 * j + (lane & 31);
        if (k < p.cin && n < p.cout) out[(long long)k * p.cout + n] = f * acc[i][j][r];
      }
  if (do_db) {
    float *red = reinterpret_cast<float *>(smem);  // [256][8]; every wave is past its last operand read
#pragma unroll
    for (int j = 0; j < 8; ++j) red[tid * 8 + j] = dbs[j];
    __syncthreads();
    if (tid < TN && n0 + tid < p.cout) {
      float a = 0.f;
      for (int l = 0; l < 256 / (TN / 8); ++l) a += red[(l * (TN / 8) + tid / 8) * 8 + (tid & 7)];
      p.dbout[(long long)z * p.cout + n0 + tid] = a;
    }
  }
}

// dw = coef sum of the splits' products, db = sum of theirs.  A lane takes V neighbouring entries; the 4 waves of a block every fourth split of
// the same entries each, joined through LDS: the loads are what there is to wait for, and small products have few entries.
template <int V>
__global__ __launch_bounds__(256) void act8_wgrad_join_kernel(const float *ws, const float *dbws, float *dw, float *db, long long kn, int cout,
                                                              int nsplit, float coef) {
  typedef float vec __attribute__((ext_vector_type(V)));
  __shared__ vec red[256];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  long long i = ((long long)blockIdx.x * 64 + lane) * V;
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
    for (int z = wave; z < nsplit; z += 4) a += *reinterpret_cast<const vec *>(src + z * len);
  }
  red[threadIdx.x] = a;
  __syncthreads();
  if (wave == 0 && live)
    *reinterpret_cast<vec *>((bias ? db : dw) + i) = (bias ? 1.f : coef) * ((red[lane] + red[64 + lane]) + (red[128 + lane] + red[192 + lane]));
}

struct A8wGeo {
  int wm, wn, tk, tn, nsplit;
  long long rsplit;
};
// Tile 64 wm x 64 wn and row splits: the largest tile that the channels fill (fewer re-reads of both operands and fewer operand reads an
// MFMA), made smaller while the launch has less than a block a CU; splits of 128 rows or more, for 2 blocks a CU.
static A8wGeo a8w_geometry(long long rows, int cin, int cout, int dtype) {
  A8wGeo g;
  g.wm = cin > 64 ? 2 : 1;
  g.wn = cout > 128 && dtype == TBG_DT_BF16 ? 4 : cout > 64 ? 2 : 1;
  const long long most = (rows + 4 * A8W_RB - 1) / (4 * A8W_RB);
  for (;;) {
    g.tk = (cin + 64 * g.wm - 1) / (64 * g.wm);
    g.tn = (cout + 64 * g.wn - 1) / (64 * g.wn);
    if ((long long)g.tk * g.tn * most >= 256 || (g.wm == 1 && g.wn == 1)) break;
    if (g.wn > g.wm || g.wm == 1) g.wn >>= 1;
    else g.wm >>= 1;
  }
  long long want = 512 / ((long long)g.tk * g.tn);
  if (want > most) want = most;
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

extern "C" long long tbg_act8_wgrad_workspace_bytes(long long rows, int cin, int cout, int dtype) {
  if (const int rc = a8w_args(rows, cin, cout, dtype)) return rc;
  const A8wGeo g = a8w_geometry(rows, cin, cout, dtype);
  return g.nsplit == 1 ? 0 : (long long)g.nsplit * ((long long)cin * cout + cout) * (long long)sizeof(float);
}

template <class E, int NP, int WM, int WN>
static int a8w_launch(const A8wP &p, bool vec, hipStream_t st) {
  constexpr size_t lds = 2 * (size_t)A8W_RB * (64 * WM + A8W_PAD + NP * (64 * WN + A8W_PAD)) * 2;
  const unsigned blocks = (unsigned)((p.nsplit + 7) / 8 * 8 * p.tk * p.tn);
  const auto kern = vec ? act8_wgrad_kernel<E, NP, WM, WN, true> : act8_wgrad_kernel<E, NP, WM, WN, false>;
  if (lds > 65536 && hipFuncSetAttribute(reinterpret_cast<const void *>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds) != hipSuccess)
    return TBG_EHIP;
  hipLaunchKernelGGL(kern, dim3(blocks), dim3(256), lds, st, p);
  TBG_LAUNCH_CHECK();
  return TBG_OK;
}
template <class E, int NP>
static int a8w_tiles(const A8wP &p, const A8wGeo &g, bool vec, hipStream_t st) {
  if constexpr (NP == 1)
    if (g.wn == 4) return g.wm == 2 ? a8w_launch<E, NP, 2, 4>(p, vec, st) : a8w_launch<E, NP, 1, 4>(p, vec, st);
  if (g.wm == 2) return g.wn == 2 ? a8w_launch<E, NP, 2, 2>(p, vec, st) : a8w_launch<E, NP, 2, 1>(p, vec, st);
  return g.wn == 2 ? a8w_launch<E, NP, 1, 2>(p, vec, st) : a8w_launch<E, NP, 1, 1>(p, vec, st);
}

extern "C" int tbg_act8_wgrad(const void *q, const void *e, const void *dy, int dtype, long long rows, int cin, int cout, long long ldy,
                              float coef, float *dw, float *db, void *workspace, long long workspace_bytes, void *stream) {
  if (!q || !e || !dy || !dw || ldy < cout || (reinterpret_cast<uintptr_t>(q) & 15) != 0) return TBG_EINVAL;
  if (const int rc = a8w_args(rows, cin, cout, dtype)) return rc;
  const A8wGeo g = a8w_geometry(rows, cin, cout, dtype);
  if ((long long)(g.nsplit + 7) * g.tk * g.tn > 0x7fffffffLL) return TBG_ERANGE;
  const long long kn = (long long)cin * cout, need = g.nsplit == 1 ? 0 : g.nsplit * (kn + cout) * (long long)sizeof(float);
  if (need > workspace_bytes || (need && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15) != 0))) return TBG_EINVAL;
  A8wP p{};
  p.q = reinterpret_cast<const unsigned char *>(q); p.e = reinterpret_cast<const unsigned char *>(e); p.dy = dy;
  p.rows = rows; p.ldy = ldy; p.rsplit = g.rsplit; p.cin = cin; p.cout = cout; p.pitch = (cin + A8_BLOCK - 1) / A8_BLOCK * A8_BLOCK;
  p.nsplit = g.nsplit; p.tk = g.tk; p.tn = g.tn; p.coef = coef; p.want_db = db != nullptr;
  float *ws = reinterpret_cast<float *>(workspace);
  p.out = g.nsplit == 1 ? dw : ws;
  p.dbout = g.nsplit == 1 ? db : ws + g.nsplit * kn;
  const bool vec = cout % 8 == 0 && vec8_ok(dy, dtype, ldy);
  hipStream_t st = tbg_stream(stream);
  const int rc = dtype == TBG_DT_F32 ? a8w_tiles<ElF32, 3>(p, g, vec, st)
                 : dtype == TBG_DT_BF16 ? a8w_tiles<ElBf16, 1>(p, g, vec, st)
                                        : a8w_tiles<ElF16, 2>(p, g, vec, st);
  if (rc || g.nsplit == 1) return rc;
  const bool v4 = cout % 4 == 0 && ((reinterpret_cast<uintptr_t>(dw) | reinterpret_cast<uintptr_t>(db)) & 15) == 0;
  const long long lanes = (kn + (db ? cout : 0) + (v4 ? 3 : 0)) / (v4 ? 4 : 1);
  hipLaunchKernelGGL(v4 ? act8_wgrad_join_kernel<4> : act8_wgrad_join_kernel<1>, dim3((unsigned)((lanes + 63) / 64)), dim3(256), 0, st, ws,
                     ws + g.nsplit * kn, dw, db, kn, cout, g.nsplit, coef);
  TBG_LAUNCH_CHECK();
  return TBG_OK;
}
