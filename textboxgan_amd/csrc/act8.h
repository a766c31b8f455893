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

// 16-byte accesses to elements of a row wherever the row begins: the card takes them at any address
typedef u32x4 u32x4_any __attribute__((aligned(2)));
typedef f32x4 f32x4_any __attribute__((aligned(4)));

// V consecutive elements of a row.  V = 8: 16-byte accesses; V = 1: one element.
template <class E, int V>
struct Pack {
  typename E::type v[V];
};
template <class E, int V>
__device__ __forceinline__ Pack<E, V> ld_pack(const typename E::type *p) {
  Pack<E, V> r;
  if constexpr (V == 8 && E::BYTES == 2) {
    const u32x4 w = *reinterpret_cast<const u32x4_any *>(p);
    __builtin_memcpy(&r, &w, 16);
  } else if constexpr (V == 8) {
    const f32x4 a = reinterpret_cast<const f32x4_any *>(p)[0], b = reinterpret_cast<const f32x4_any *>(p)[1];
#pragma unroll
    for (int i = 0; i < 4; ++i) { r.v[i] = a[i]; r.v[4 + i] = b[i]; }
  } else {
    r.v[0] = *p;
  }
  return r;
}
template <class E, int V>
__device__ __forceinline__ void st_pack(typename E::type *p, const Pack<E, V> &r) {
  if constexpr (V == 8 && E::BYTES == 2) {
    u32x4 w;
    __builtin_memcpy(&w, &r, 16);
    *reinterpret_cast<u32x4 *>(p) = w;
  } else if constexpr (V == 8) {
    reinterpret_cast<f32x4 *>(p)[0] = f32x4{r.v[0], r.v[1], r.v[2], r.v[3]};
    reinterpret_cast<f32x4 *>(p)[1] = f32x4{r.v[4], r.v[5], r.v[6], r.v[7]};
  } else {
    *p = r.v[0];
  }
}

// V values rounded to the type, two conversions an instruction where the type has one
template <class E, int V>
__device__ __forceinline__ Pack<E, V> put_pack(const float (&v)[V]) {
  Pack<E, V> r;
  if constexpr (V == 8 && __is_same(E, ElBf16)) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    unsigned w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __builtin_bit_cast(unsigned, __builtin_convertvector(f32x2{v[2 * i], v[2 * i + 1]}, bf16x2));
    __builtin_memcpy(&r, w, 16);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) r.v[i] = E::put(v[i]);
  }
  return r;
}

// ---- ACT8.  The lanes that hold one block of 32 channels are neighbours: 4 lanes of 8 channels or 32 lanes of one.
constexpr int A8_BLOCK = 32;
constexpr unsigned A8_NAN = 255u;

// largest bit pattern of |x| in the block.  Bit patterns of non-negative floats order like the floats, infinities and NaN on top.
template <int V>
__device__ __forceinline__ unsigned a8_block_max(const float (&x)[V]) {
  unsigned m = 0;
#pragma unroll
  for (int i = 0; i < V; ++i) m = max(m, __float_as_uint(x[i]) & 0x7fffffffu);
  if constexpr (V == 8) {
    m = max(m, (unsigned)__builtin_amdgcn_mov_dpp((int)m, 0xB1, 0xf, 0xf, true));  // quad_perm [1,0,3,2]
    m = max(m, (unsigned)__builtin_amdgcn_mov_dpp((int)m, 0x4E, 0xf, 0xf, true));  // quad_perm [2,3,0,1]
  } else {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) m = max(m, (unsigned)__shfl_xor((int)m, off, 64));
  }
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
template <int V>
__device__ __forceinline__ void a8_round(const float (&x)[V], unsigned code, float (&t)[V]) {
  const float inv = __uint_as_float((254u - code) << 23);
#pragma unroll
  for (int i = 0; i < V; ++i) t[i] = fmaf(x[i], inv, A8_MAGIC);
  if (code == 248u) {
#pragma unroll
    for (int i = 0; i < V; ++i) t[i] = fminf(fmaxf(t[i], A8_MAGIC - 127.f), A8_MAGIC + 127.f);
  }
}
__device__ __forceinline__ float a8_scale(unsigned code) { return __uint_as_float(code == A8_NAN ? 0x7fc00000u : code << 23); }
// what a8_round has left -> bytes
template <int V>
__device__ __forceinline__ void a8_store(unsigned char *q, unsigned code, const float (&t)[V]) {
  if constexpr (V == 8) {
    u32x2 w;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const unsigned lo = __builtin_amdgcn_perm(__float_as_uint(t[4 * k + 1]), __float_as_uint(t[4 * k]), 0x0c0c0400u);
      const unsigned hi = __builtin_amdgcn_perm(__float_as_uint(t[4 * k + 3]), __float_as_uint(t[4 * k + 2]), 0x04000c0cu);
      w[k] = code == A8_NAN ? 0u : lo | hi;
    }
    *reinterpret_cast<u32x2 *>(q) = w;
  } else {
    *q = code == A8_NAN ? 0 : (unsigned char)(__float_as_uint(t[0]) & 0xffu);
  }
}
template <int V>
__device__ __forceinline__ void a8_load(const unsigned char *q, float scale, float (&x)[V]) {
  if constexpr (V == 8) {
    const u32x2 w = *reinterpret_cast<const u32x2 *>(q);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = (float)(int)(signed char)(w[i >> 2] >> (8 * (i & 3)) & 0xff) * scale;
  } else {
    x[0] = (float)(int)(signed char)*q * scale;
  }
}

// ---- dispatch
#define TBG_DT_F32 0
#define TBG_DT_BF16 1
#define TBG_DT_F16 2
static inline int dt_bytes(int dtype) { return dtype == TBG_DT_F32 ? 4 : 2; }
static inline bool dt_valid(int dtype) { return dtype >= TBG_DT_F32 && dtype <= TBG_DT_F16; }
// 16-byte accesses of 8 channels: base and row / sample pitches (elements) allow them
static inline bool vec8_ok(const void *p, int dtype, long long pitch_a, long long pitch_b = 0) {
  const long long unit = 16 / dt_bytes(dtype);
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && pitch_a % unit == 0 && pitch_b % unit == 0;
}
