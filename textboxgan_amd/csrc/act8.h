// Device helpers of the channels-last kernels (group_norm.hip, act8.hip): element types, 8-channel loads and stores, and the 8-bit
// activation format of tbg.h "ACT8" (blocks of 32 channels, one power-of-two scale, int8 values).
#pragma once
#include "common.h"

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

// ---- element types: how a value is read to and rounded from fp32 (round to nearest, ties to even)
struct ElF32 {
  typedef float type;
  static constexpr int BYTES = 4;
  static __device__ __forceinline__ float get(float v) { return v; }
  static __device__ __forceinline__ float put(float v) { return v; }
};
struct ElBf16 {
  typedef unsigned short type;
  static constexpr int BYTES = 2;
  static __device__ __forceinline__ float get(unsigned short v) { return __uint_as_float((unsigned)v << 16); }
  static __device__ __forceinline__ unsigned short put(float v) { return __builtin_bit_cast(unsigned short, (__bf16)v); }
};
struct ElF16 {
  typedef unsigned short type;
  static constexpr int BYTES = 2;
  static __device__ __forceinline__ float get(unsigned short v) { return (float)__builtin_bit_cast(_Float16, v); }
  static __device__ __forceinline__ unsigned short put(float v) {
    asm("" : "+v"(v));  // v is rounded to fp32 first in every kernel: without this some products become mixed-precision ones that round once
    return __builtin_bit_cast(unsigned short, (_Float16)v);
  }
};

// 8 neighbouring channels of a row, moved in 16-byte pieces wherever the row begins: the card takes them at any address.  The alignment belongs to
// the typedef and not to the vector type, so a template's deduced parameter would lose it: the functions below name their pointers' types.
typedef u32x4 u32x4_any __attribute__((aligned(2)));
typedef f32x4 f32x4_any __attribute__((aligned(4)));

template <class E>
struct Pack8 {
  typename E::type v[8];
};
// PAST: read past the caches, which keep other lines
template <bool PAST>
__device__ __forceinline__ u32x4 ld_vec(const u32x4_any *p) {
  if constexpr (PAST) return __builtin_nontemporal_load(p);
  else return *p;
}
template <bool PAST>
__device__ __forceinline__ f32x4 ld_vec(const f32x4_any *p) {
  if constexpr (PAST) return __builtin_nontemporal_load(p);
  else return *p;
}
template <bool PAST>
__device__ __forceinline__ u32x2 ld_vec(const u32x2 *p) {
  if constexpr (PAST) return __builtin_nontemporal_load(p);
  else return *p;
}
template <class E, bool PAST = false>
__device__ __forceinline__ Pack8<E> ld8(const typename E::type *p) {
  Pack8<E> r;
  if constexpr (E::BYTES == 2) {
    const u32x4 w = ld_vec<PAST>(reinterpret_cast<const u32x4_any *>(p));
    __builtin_memcpy(&r, &w, 16);
  } else {
    const f32x4 a = ld_vec<PAST>(reinterpret_cast<const f32x4_any *>(p)), b = ld_vec<PAST>(reinterpret_cast<const f32x4_any *>(p + 4));
#pragma unroll
    for (int i = 0; i < 4; ++i) { r.v[i] = a[i]; r.v[4 + i] = b[i]; }
  }
  return r;
}
// PAST: written past the caches, whose other lines stay
template <bool PAST>
__device__ __forceinline__ void st_vec(u32x4_any *p, u32x4 v) {
  if constexpr (PAST) __builtin_nontemporal_store(v, p);
  else *p = v;
}
template <bool PAST>
__device__ __forceinline__ void st_vec(f32x4_any *p, f32x4 v) {
  if constexpr (PAST) __builtin_nontemporal_store(v, p);
  else *p = v;
}
template <bool PAST>
__device__ __forceinline__ void st_vec(u32x2 *p, u32x2 v) {
  if constexpr (PAST) __builtin_nontemporal_store(v, p);
  else *p = v;
}
template <class E, bool PAST = false>
__device__ __forceinline__ void st8(typename E::type *p, const Pack8<E> &r) {
  if constexpr (E::BYTES == 2) {
    u32x4 w;
    __builtin_memcpy(&w, &r, 16);
    st_vec<PAST>(reinterpret_cast<u32x4_any *>(p), w);
  } else {
    st_vec<PAST>(reinterpret_cast<f32x4_any *>(p), f32x4{r.v[0], r.v[1], r.v[2], r.v[3]});
    st_vec<PAST>(reinterpret_cast<f32x4_any *>(p + 4), f32x4{r.v[4], r.v[5], r.v[6], r.v[7]});
  }
}
// 8 bf16 values to LDS, at a multiple of 16 bytes
__device__ __forceinline__ void st8_lds(unsigned short *p, const Pack8<ElBf16> &r) {
  u32x4 w;
  __builtin_memcpy(&w, &r, 16);
  *reinterpret_cast<u32x4 *>(p) = w;
}
// moved down by k elements (k the same in all lanes), zeros above
template <class E>
__device__ __forceinline__ Pack8<E> shift_down(const Pack8<E> &r, int k) {
  if constexpr (E::BYTES == 2) {
    unsigned w[4];
    __builtin_memcpy(w, &r, 16);
    if (k & 4) { w[0] = w[2]; w[1] = w[3]; w[2] = w[3] = 0; }
    if (k & 2) { w[0] = w[1]; w[1] = w[2]; w[2] = w[3]; w[3] = 0; }
    if (k & 1) {
#pragma unroll
      for (int i = 0; i < 3; ++i) w[i] = __builtin_amdgcn_alignbit(w[i + 1], w[i], 16);
      w[3] >>= 16;
    }
    Pack8<E> o;
    __builtin_memcpy(&o, w, 16);
    return o;
  } else {
    Pack8<E> o = r;
#pragma unroll
    for (int step = 4; step > 0; step >>= 1)
      if (k & step) {
#pragma unroll
        for (int i = 0; i < 8; ++i) o.v[i] = i + step < 8 ? o.v[i + step] : (typename E::type)0;
      }
    return o;
  }
}
// A lane's channels c .. c + 7 of rows of C.  TAIL (C % 8 != 0): the lane that holds the last C % 8 channels reads the row's last 8 and moves
// them down, so that nothing beyond the row is touched; its other values are zeros and are not stored.  Rows of fewer than 8 go by elements.
template <class E, bool TAIL>
struct Row8 {
  int off, left;  // where the lane reads; channels of the lane (8, fewer in the last one)
  int C;
  __device__ __forceinline__ Row8(int c, int C_) : off(c), left(8), C(C_) {
    if (TAIL && c + 8 > C) {
      left = C - c;
      off = C >= 8 ? C - 8 : 0;
    }
  }
  template <bool PAST = false>
  __device__ __forceinline__ Pack8<E> load(const typename E::type *row) const {
    if constexpr (!TAIL) return ld8<E, PAST>(row + off);
    Pack8<E> r;
    if (C >= 8) {
      r = ld8<E>(row + off);
      const Pack8<E> low = shift_down(r, 8 - (C & 7));
#pragma unroll
      for (int i = 0; i < 8; ++i) r.v[i] = left < 8 ? low.v[i] : r.v[i];
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) r.v[i] = i < C ? row[i] : (typename E::type)0;
    }
    return r;
  }
  template <bool PAST = false>
  __device__ __forceinline__ void store(typename E::type *row, const Pack8<E> &r) const {
    if (!TAIL || left == 8) {
      st8<E, PAST>(row + off, r);
    } else {
      typename E::type *to = row + (C & ~7);
#pragma unroll
      for (int i = 0; i < 7; ++i)
        if (i < (C & 7)) to[i] = r.v[i];
    }
  }
};

// 8 values rounded to the type, two conversions an instruction where the type has one
template <class E>
__device__ __forceinline__ Pack8<E> put8(const float (&v)[8]) {
  Pack8<E> r;
  if constexpr (__is_same(E, ElBf16)) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    unsigned w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __builtin_bit_cast(unsigned, __builtin_convertvector(f32x2{v[2 * i], v[2 * i + 1]}, bf16x2));
    __builtin_memcpy(&r, w, 16);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) r.v[i] = E::put(v[i]);
  }
  return r;
}

// ---- ACT8.  A lane holds 8 channels of a block of 32, neighbouring lanes its other 24
constexpr int A8_BLOCK = 32;
constexpr unsigned A8_NAN = 255u;

// largest bit pattern of |x| in the block.  Bit patterns of non-negative floats order like the floats, infinities and NaN on top.
__device__ __forceinline__ unsigned a8_block_max(const float (&x)[8]) {
  unsigned m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(x[i]) & 0x7fffffffu);
  m = max(m, (unsigned)__builtin_amdgcn_mov_dpp((int)m, 0xB1, 0xf, 0xf, true));  // quad_perm [1,0,3,2]
  m = max(m, (unsigned)__builtin_amdgcn_mov_dpp((int)m, 0x4E, 0xf, 0xf, true));  // quad_perm [2,3,0,1]
  return m;
}
// scale code of a block: e + 127 with e = floor(log2 amax) - 6, one more where amax 2^-e would round to 128 (mantissa >= 127.5 / 64,
// i.e. bits >= 0x7f0000: adding 0x10000 carries into the exponent exactly then), held in [1, 248]; 255 for a block that is not finite.
__device__ __forceinline__ unsigned a8_code(unsigned amax_bits) {
  if (amax_bits >= 0x7f800000u) return A8_NAN;
  const int e = (int)((amax_bits + 0x10000u) >> 23) - 6;
  return (unsigned)min(max(e, 1), 248);
}
// x in steps of its block's scale, rounded to the nearest integer (ties to even) within +-127, as 1.5 2^23 + that integer: x 2^-e is exact, so
// the one rounding is that of the sum, and the low byte of the result is the integer in two's complement.  Only a block of code 248 may hold
// values beyond 127.5 steps (up to 128).  Values of a block that is not finite are of no account (a8_store writes zeros).
constexpr float A8_MAGIC = 12582912.f;
__device__ __forceinline__ void a8_round(const float (&x)[8], unsigned code, float (&t)[8]) {
  const float inv = __uint_as_float((254u - code) << 23);
#pragma unroll
  for (int i = 0; i < 8; ++i) t[i] = fmaf(x[i], inv, A8_MAGIC);
  if (code == 248u) {
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = fminf(fmaxf(t[i], A8_MAGIC - 127.f), A8_MAGIC + 127.f);
  }
}
__device__ __forceinline__ float a8_scale(unsigned code) { return __uint_as_float(code == A8_NAN ? 0x7fc00000u : code << 23); }
// what a8_round has left -> bytes
template <bool PAST = false>
__device__ __forceinline__ void a8_store(unsigned char *q, unsigned code, const float (&t)[8]) {
  u32x2 w;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const unsigned lo = __builtin_amdgcn_perm(__float_as_uint(t[4 * k + 1]), __float_as_uint(t[4 * k]), 0x0c0c0400u);
    const unsigned hi = __builtin_amdgcn_perm(__float_as_uint(t[4 * k + 3]), __float_as_uint(t[4 * k + 2]), 0x04000c0cu);
    w[k] = code == A8_NAN ? 0u : lo | hi;
  }
  st_vec<PAST>(reinterpret_cast<u32x2 *>(q), w);
}
// one value of eight packed bytes, in steps
__device__ __forceinline__ float a8_value(const u32x2 &w, int i) { return (float)(int)(signed char)(w[i >> 2] >> (8 * (i & 3)) & 0xff); }

// ---- dispatch
#define TBG_DT_F32 0
#define TBG_DT_BF16 1
#define TBG_DT_F16 2
static inline int dt_bytes(int dtype) { return dtype == TBG_DT_F32 ? 4 : 2; }
static inline bool dt_valid(int dtype) { return dtype >= TBG_DT_F32 && dtype <= TBG_DT_F16; }
