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
template <class E, int NP>
__device__ __forceinline__ void a8w_terms(float v, unsigned short (&t)[NP]) {
  if constexpr (NP == 1) {
    t[0] = ElBf16::put(v);
  } else {
    const bool fine = (__float_as_uint(v) & 0x7f800000u) != 0x7f800000u;
    float rest = v;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const unsigned hi = __float_as_uint(rest) & 0xffff0000u;
      t[i] = fine ? (unsigned short)(hi >> 16) : (i == 0 ? ElBf16::put(v) : (unsigned short)0);
      rest -= __uint_as_float(hi);
    }
  }
}

template <class E, int NP, int WM, int WN, bool VEC>
__global__ __launch_bounds__(256) void act8_wgrad_kernel(A8wP p) {
  constexpr int TK = 64 * WM, TN = 64 * WN, PK = TK + A8W_PAD, PN = TN + A8W_PAD;
  extern __shared__ __align__(16) char smem[];
  unsigned short *Xs = reinterpret_cast<unsigned short *>(smem), *Ds = Xs + A8W_RB * PK;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wk = wave & 1, wn = wave >> 1;
  int b = blockIdx.x;
  const int z = b / (p.tk * p.tn); b -= z * (p.tk * p.tn);
  const int k0 = (b / p.tn) * TK, n0 = (b % p.tn) * TN;
  const long long r0 = z * p.rsplit, rend = min(p.rows, r0 + p.rsplit);
  const bool do_db = p.want_db && k0 == 0;

  const int i16 = lane & 15, grp = lane >> 4, jj = i16 >> 2, cq = i16 & 3, chblk = grp & 1, khalf = grp >> 1;
  const int a_off = (8 * khalf + jj) * PK + wk * 32 * WM + chblk * 16 + cq * 4;
  const int b_off = (8 * khalf + jj) * PN + wn * 32 * WN + chblk * 16 + cq * 4;
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

  for (long long r = r0; r < rend; r += A8W_RB) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < WM; ++i) {
      const int id = tid + 256 * i, row = id / (TK / 8), c = (id % (TK / 8)) * 8;
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = 0.f;
      if (r + row < rend && k0 + c < p.pitch)
        a8_load<8>(p.q + (r + row) * p.pitch + k0 + c, a8_scale(p.e[(r + row) * (p.pitch / A8_BLOCK) + (k0 + c) / A8_BLOCK]), v);
      Pack<ElBf16, 8> w;
#pragma unroll
      for (int j = 0; j < 8; ++j) w.v[j] = ElBf16::put(v[j]);
      st_pack<ElBf16, 8>(Xs + row * PK + c, w);
    }
#pragma unroll
    for (int i = 0; i < WN; ++i) {
      const int id = tid + 256 * i, row = id / (TN / 8), c = (id % (TN / 8)) * 8;
      const typename E::type *src = reinterpret_cast<const typename E::type *>(p.dy) + (r + row) * p.ldy + n0 + c;
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = 0.f;
      if (r + row < rend) {
        if constexpr (VEC) {
          if (n0 + c < p.cout) {
            const Pack<E, 8> d = ld_pack<E, 8>(src);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = E::get(d.v[j]);
          }
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (n0 + c + j < p.cout) v[j] = E::get(src[j]);
        }
      }
      Pack<ElBf16, 8> w[NP];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        unsigned short t[NP];
        a8w_terms<E, NP>(v[j], t);
#pragma unroll
        for (int m = 0; m < NP; ++m) w[m].v[j] = t[m];
        dbs[j] += v[j];
      }
#pragma unroll
      for (int m = 0; m < NP; ++m) st_pack<ElBf16, 8>(Ds + (m * A8W_RB + row) * PN + c, w[m]);
    }
    __syncthreads();
#pragma unroll
    for (int s = 0; s < A8W_RB / 16; ++s) {
      bf16x8 a[WM];
#pragma unroll
      for (int i = 0; i < WM; ++i) a[i] = rd(Xs + a_off + 16 * s * PK + 32 * i, PK);
#pragma unroll
      for (int j = 0; j < WN; ++j)
#pragma unroll
        for (int m = NP - 1; m >= 0; --m) {  // smallest terms first
          const bf16x8 d = rd(Ds + b_off + (m * A8W_RB + 16 * s) * PN + 32 * j, PN);
#pragma unroll
          for (int i = 0; i < WM; ++i) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[i], d, acc[i][j], 0, 0, 0);
        }
    }
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
    float *red = reinterpret_cast<float *>(smem);  // [256][8]
    __syncthreads();
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

// dw = coef sum of the splits' products, db = sum of theirs
__global__ __launch_bounds__(256) void act8_wgrad_join_kernel(const float *ws, const float *dbws, float *dw, float *db, long long kn, int cout,
                                                              int nsplit, float coef) {
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i < kn) {
    float a = 0.f;
    for (int z = 0; z < nsplit; ++z) a += ws[z * kn + i];
    dw[i] = coef * a;
  } else if (db && i - kn < cout) {
    float a = 0.f;
    for (int z = 0; z < nsplit; ++z) a += dbws[(long long)z * cout + (i - kn)];
    db[i - kn] = a;
  }
}

struct A8wGeo {
  int wm, wn, tk, tn, nsplit;
  long long rsplit;
};
static A8wGeo a8w_geometry(long long rows, int cin, int cout) {
  A8wGeo g;
  g.wm = cin > 64 ? 2 : 1;
  g.wn = cout > 64 ? 2 : 1;
  g.tk = (cin + 64 * g.wm - 1) / (64 * g.wm);
  g.tn = (cout + 64 * g.wn - 1) / (64 * g.wn);
  long long want = 512 / ((long long)g.tk * g.tn);
  const long long most = (rows + 4 * A8W_RB - 1) / (4 * A8W_RB);
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
  const A8wGeo g = a8w_geometry(rows, cin, cout);
  return g.nsplit == 1 ? 0 : (long long)g.nsplit * ((long long)cin * cout + cout) * (long long)sizeof(float);
}

template <class E, int NP, int WM, int WN>
static int a8w_launch(const A8wP &p, bool vec, hipStream_t st) {
  const size_t lds = (size_t)A8W_RB * (64 * WM + A8W_PAD + NP * (64 * WN + A8W_PAD)) * 2;
  const unsigned blocks = (unsigned)(p.nsplit * p.tk * p.tn);
  if (vec) hipLaunchKernelGGL((act8_wgrad_kernel<E, NP, WM, WN, true>), dim3(blocks), dim3(256), lds, st, p);
  else hipLaunchKernelGGL((act8_wgrad_kernel<E, NP, WM, WN, false>), dim3(blocks), dim3(256), lds, st, p);
  TBG_LAUNCH_CHECK();
  return TBG_OK;
}
template <class E, int NP>
static int a8w_tiles(const A8wP &p, const A8wGeo &g, bool vec, hipStream_t st) {
  if (g.wm == 2) return g.wn == 2 ? a8w_launch<E, NP, 2, 2>(p, vec, st) : a8w_launch<E, NP, 2, 1>(p, vec, st);
  return g.wn == 2 ? a8w_launch<E, NP, 1, 2>(p, vec, st) : a8w_launch<E, NP, 1, 1>(p, vec, st);
}

extern "C" int tbg_act8_wgrad(const void *q, const void *e, const void *dy, int dtype, long long rows, int cin, int cout, long long ldy,
                              float coef, float *dw, float *db, void *workspace, long long workspace_bytes, void *stream) {
  if (!q || !e || !dy || !dw || ldy < cout || (reinterpret_cast<uintptr_t>(q) & 15) != 0) return TBG_EINVAL;
  if (const int rc = a8w_args(rows, cin, cout, dtype)) return rc;
  const A8wGeo g = a8w_geometry(rows, cin, cout);
  if ((long long)g.nsplit * g.tk * g.tn > 0x7fffffffLL) return TBG_ERANGE;
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
  const long long total = kn + (db ? cout : 0);
  hipLaunchKernelGGL(act8_wgrad_join_kernel, dim3((unsigned)((total + 255) / 256)), dim3(256), 0, st, ws, ws + g.nsplit * kn, dw, db, kn, cout,
                     g.nsplit, coef);
  TBG_LAUNCH_CHECK();
  return TBG_OK;
}
