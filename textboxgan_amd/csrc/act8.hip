// 8-bit activation checkpoints (tbg.h "ACT8"): packing rows of channels and reading them back.
//
// HBM-bound both ways: es + 1 + 1/32 bytes an element.  A lane holds 8 channels of one row (16-byte loads, 8-byte stores of q), the four
// lanes of a block find its largest magnitude with two DPP exchanges, so a value is touched once.  Items (row, group of 8 channels) are
// laid end to end over the lanes whatever the row length, so that short and odd rows waste no lanes, and rows that begin anywhere are read in
// 16-byte pieces all the same.
// Measured: 262144 rows x 128 bf16 packed in 19 us, unpacked in 17 (101 MB each: 5.3, 5.9 TB/s), 10007 x 250 fp32 in 3.8 and 5.2 us, a launch's own
// time (17.8 together while rows that do not begin at multiples of 16 bytes went by elements).
#include "act8.h"

template <class E, bool TAIL>
__global__ __launch_bounds__(256) void act8_pack_kernel(const typename E::type *__restrict__ x, long long rows, int ch, long long ldx,
                                                        unsigned char *__restrict__ q, unsigned char *__restrict__ e, unsigned cols) {
  // cols = 8-channel groups of a padded row (a multiple of 4)
  const long long base = (long long)blockIdx.x * 256;
  const long long row0 = base / cols;
  const unsigned local = (unsigned)(base - row0 * cols) + threadIdx.x;
  const long long row = row0 + local / cols;
  const int c = (int)(local % cols) * 8;
  if (row >= rows) return;  // whole blocks of 32 channels leave together: cols and 256 are multiples of a block's lanes
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = 0.f;
  if (c < ch) {
    const Pack8<E> p = Row8<E, TAIL>(c, ch).load(x + row * ldx);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = E::get(p.v[i]);
  }
  const unsigned code = a8_code(a8_block_max(v));
  float t[8];
  a8_round(v, code, t);
  a8_store(q + row * ((long long)cols * 8) + c, code, t);
  if ((c & (A8_BLOCK - 1)) == 0) e[row * (cols / 4) + c / A8_BLOCK] = (unsigned char)code;
}

template <class E, bool TAIL>
__global__ __launch_bounds__(256) void act8_unpack_kernel(const unsigned char *__restrict__ q, const unsigned char *__restrict__ e,
                                                          long long rows, int ch, typename E::type *__restrict__ x, long long ldx,
                                                          unsigned cols, unsigned pitch) {
  // cols = 8-channel groups of an unpadded row
  const long long base = (long long)blockIdx.x * 256;
  const long long row0 = base / cols;
  const unsigned local = (unsigned)(base - row0 * cols) + threadIdx.x;
  const long long row = row0 + local / cols;
  const int c = (int)(local % cols) * 8;
  if (row >= rows) return;
  const u32x2 w = *reinterpret_cast<const u32x2 *>(q + row * pitch + c);
  const float scale = a8_scale(e[row * (pitch / A8_BLOCK) + c / A8_BLOCK]);
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = a8_value(w, i) * scale;
  if constexpr (__is_same(E, ElF16)) {
    // the largest values of fp16 itself (65280 .. 65504) are kept as 64 2^10 = 65536, which the type does not hold: a value that lies within half
    // a step of the type's range is its end, values further out round to infinities (a NaN's comparison is false)
    const float most = 65504.f + 0.5f * scale;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = fabsf(v[i]) <= most ? fminf(fmaxf(v[i], -65504.f), 65504.f) : v[i];
  }
  Row8<E, TAIL>(c, ch).store(x + row * ldx, put8<E>(v));
}

static int act8_args(const void *x, const void *q, const void *e, int dtype, long long rows, int ch, long long ldx) {
  if (!x || !q || !e || !dt_valid(dtype) || rows < 1 || ch < 1 || ldx < ch) return TBG_EINVAL;
  if ((reinterpret_cast<uintptr_t>(q) & 15) != 0) return TBG_EINVAL;
  if (ch > (1 << 24) || rows > (1LL << 39) / ((ch + A8_BLOCK - 1) / A8_BLOCK * A8_BLOCK)) return TBG_ERANGE;
  return TBG_OK;
}

// rows a launch: a grid holds less than 2^32 threads
static long long act8_rows(unsigned cols) { return (1LL << 31) / cols; }

template <class E>
static int launch_pack(const void *x, long long rows, int ch, long long ldx, void *q, void *e, hipStream_t st) {
  const unsigned cols = (unsigned)((ch + A8_BLOCK - 1) / A8_BLOCK * (A8_BLOCK / 8));
  const long long most = act8_rows(cols);
  for (long long r = 0; r < rows; r += most) {
    const long long n = rows - r < most ? rows - r : most;
    auto *xp = reinterpret_cast<const typename E::type *>(x) + r * ldx;
    auto *qp = reinterpret_cast<unsigned char *>(q) + r * cols * 8, *ep = reinterpret_cast<unsigned char *>(e) + r * (cols / 4);
    hipLaunchKernelGGL((ch % 8 ? act8_pack_kernel<E, true> : act8_pack_kernel<E, false>), dim3((unsigned)((n * cols + 255) / 256)), dim3(256), 0, st, xp,
                       n, ch, ldx, qp, ep, cols);
    TBG_LAUNCH_CHECK();
  }
  return TBG_OK;
}

template <class E>
static int launch_unpack(const void *q, const void *e, long long rows, int ch, void *x, long long ldx, hipStream_t st) {
  const unsigned padded = (unsigned)((ch + A8_BLOCK - 1) / A8_BLOCK * A8_BLOCK);
  const unsigned cols = (ch + 7) / 8;
  const long long most = act8_rows(cols);
  for (long long r = 0; r < rows; r += most) {
    const long long n = rows - r < most ? rows - r : most;
    auto *xp = reinterpret_cast<typename E::type *>(x) + r * ldx;
    auto *qp = reinterpret_cast<const unsigned char *>(q) + r * padded, *ep = reinterpret_cast<const unsigned char *>(e) + r * (padded / A8_BLOCK);
    hipLaunchKernelGGL((ch % 8 ? act8_unpack_kernel<E, true> : act8_unpack_kernel<E, false>), dim3((unsigned)((n * cols + 255) / 256)), dim3(256), 0, st,
                       qp, ep, n, ch, xp, ldx, cols, padded);
    TBG_LAUNCH_CHECK();
  }
  return TBG_OK;
}

extern "C" int tbg_act8_pack(const void *x, int dtype, long long rows, int ch, long long ldx, void *q, void *e, void *stream) {
  if (const int rc = act8_args(x, q, e, dtype, rows, ch, ldx)) return rc;
  hipStream_t st = tbg_stream(stream);
  return dtype == TBG_DT_F32 ? launch_pack<ElF32>(x, rows, ch, ldx, q, e, st)
         : dtype == TBG_DT_BF16 ? launch_pack<ElBf16>(x, rows, ch, ldx, q, e, st)
                                : launch_pack<ElF16>(x, rows, ch, ldx, q, e, st);
}

extern "C" int tbg_act8_unpack(const void *q, const void *e, long long rows, int ch, void *x, int dtype, long long ldx, void *stream) {
  if (const int rc = act8_args(x, q, e, dtype, rows, ch, ldx)) return rc;
  hipStream_t st = tbg_stream(stream);
  return dtype == TBG_DT_F32 ? launch_unpack<ElF32>(q, e, rows, ch, x, ldx, st)
         : dtype == TBG_DT_BF16 ? launch_unpack<ElBf16>(q, e, rows, ch, x, ldx, st)
                                : launch_unpack<ElF16>(q, e, rows, ch, x, ldx, st);
}
