// rows_kernel.hpp -- device helpers of the row operators (norm_kernel.hpp, act8.hip).
//
// Every lane owns 8 consecutive elements of a row (16 bytes of a 16-bit type, two 16-byte loads of
// float), so 16 consecutive lanes own one checkpoint block of 128 columns and its maximum is a
// reduction inside a DPP row. The vector types carry the alignment of their element alone: the
// same global_load_dwordx4 then serves every base address and row stride (this part splits what
// crosses a line), and only a row's last vector is loaded element by element.
#ifndef EMAC_ROWS_KERNEL_HPP_
#define EMAC_ROWS_KERNEL_HPP_

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "rows.h"

namespace emac_rows {

typedef __bf16 bf16;
typedef _Float16 half;

template <class T>
using v8 = T __attribute__((ext_vector_type(8)));
template <class T>
struct packed { // 8 elements in memory, at any element's address
  typedef T type __attribute__((ext_vector_type(8), aligned(sizeof(T))));
};
typedef v8<float> f8;
typedef unsigned short us8 __attribute__((ext_vector_type(8)));
typedef unsigned short us2 __attribute__((ext_vector_type(2)));
typedef unsigned u2 __attribute__((ext_vector_type(2)));
typedef unsigned u2_any __attribute__((ext_vector_type(2), aligned(1)));

// `n` (clamped) of the 8 elements at p, zeros in the place of the others
template <class T>
__device__ inline v8<T> load8(const T *p, long n) {
  if (n >= 8) return *(const typename packed<T>::type *)p;
  v8<T> r = (v8<T>)(T)0;
#pragma unroll
  for (int j = 0; j < 8; j++)
    if (j < n) r[j] = p[j];
  return r;
}

template <class T>
__device__ inline void store8(T *p, v8<T> v, long n) {
  if (n >= 8) {
    *(typename packed<T>::type *)p = v;
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; j++)
    if (j < n) p[j] = v[j];
}

__device__ inline u2 load8q(const signed char *p, long n) {
  if (n >= 8) return *(const u2_any *)p;
  u2 r = {0, 0};
#pragma unroll
  for (int j = 0; j < 8; j++)
    if (j < n) r[j / 4] |= (unsigned)(unsigned char)p[j] << 8 * (j % 4);
  return r;
}

__device__ inline void store8q(signed char *p, u2 v, long n) {
  if (n >= 8) {
    *(u2_any *)p = v;
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; j++)
    if (j < n) p[j] = (signed char)(v[j / 4] >> 8 * (j % 4));
}

template <class T>
__device__ inline f8 widen(v8<T> v) {
  return __builtin_convertvector(v, f8);
}
template <class T>
__device__ inline v8<T> round_to(f8 v) {
  return __builtin_convertvector(v, v8<T>);
}

// ---- reductions inside a wave: DPP row rotations (16 lanes), then the four rows by readlane.
// Every step adds the same two values on both sides, so all lanes hold the same bits. ----
template <int N>
__device__ inline unsigned row_ror(unsigned v) {
  return (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x120 + N, 0xf, 0xf, true);
}
template <int N>
__device__ inline float row_ror(float v) {
  return __uint_as_float(row_ror<N>(__float_as_uint(v)));
}
__device__ inline float sum16(float v) {
  v += row_ror<8>(v);
  v += row_ror<4>(v);
  v += row_ror<2>(v);
  v += row_ror<1>(v);
  return v;
}
__device__ inline unsigned max16(unsigned v) {
  v = max(v, row_ror<8>(v));
  v = max(v, row_ror<4>(v));
  v = max(v, row_ror<2>(v));
  v = max(v, row_ror<1>(v));
  return v;
}
__device__ inline float lane_of(float v, int lane) {
  return __uint_as_float((unsigned)__builtin_amdgcn_readlane((int)__float_as_uint(v), lane));
}
__device__ inline float sum64(float v) {
  v = sum16(v);
  return (lane_of(v, 0) + lane_of(v, 16)) + (lane_of(v, 32) + lane_of(v, 48));
}

// ---- checkpoints: 8 bits and a float scale for each 128 columns ----

// the bits of max |x| as a float's: integer order, in which an infinity and every NaN lie above
// all finite values, so neither is lost in the maximum
__device__ inline unsigned abs_bits(v8<float> x) {
  unsigned m = 0;
#pragma unroll
  for (int j = 0; j < 8; j++) m = max(m, __float_as_uint(x[j]) & 0x7fffffffu);
  return m;
}
template <class T>
__device__ inline unsigned abs_bits(v8<T> x) { // 16-bit types: their own bits
  us8 u = __builtin_bit_cast(us8, x) & (us8)(unsigned short)0x7fff;
  us2 a = __builtin_elementwise_max(u.s01, u.s23), b = __builtin_elementwise_max(u.s45, u.s67);
  a = __builtin_elementwise_max(a, b);
  return max((unsigned)a.x, (unsigned)a.y);
}
template <class T>
__device__ inline float of_bits(unsigned m);
template <>
__device__ inline float of_bits<float>(unsigned m) {
  return __uint_as_float(m);
}
template <>
__device__ inline float of_bits<bf16>(unsigned m) {
  return __uint_as_float(m << 16);
}
template <>
__device__ inline float of_bits<half>(unsigned m) {
  return (float)__builtin_bit_cast(half, (unsigned short)m);
}

struct block8 {
  u2 q;        // this lane's 8 bytes
  float scale; // the block's
};

// The checkpoint of the block that 16 lanes hold. Each operation is rounded to 32 bits on its own
// (no contraction), so the bytes are the definition's on every path. 1.5 * 2^23 added to a value
// of magnitude <= 128 leaves its integer, ties to even, in the low byte of the sum.
template <class T>
__device__ inline block8 quantise(v8<T> x) {
#pragma clang fp contract(off)
  const float a = of_bits<T>(max16(abs_bits(x)));
  const bool finite = a <= 3.4028234663852886e38f;
  const float am = fmaxf(a, 0x1p-100f);
  const float inv = finite ? 127.0f / am : 0.0f;
  const f8 f = widen<T>(x);
  unsigned b[8];
#pragma unroll
  for (int j = 0; j < 8; j++) {
    const float p = f[j] * inv;
    b[j] = __float_as_uint(p + 12582912.0f);
  }
  block8 r;
#pragma unroll
  for (int k = 0; k < 2; k++) { // v_perm: byte 0 of each of four words
    const unsigned lo = __builtin_amdgcn_perm(b[4 * k + 1], b[4 * k], 0x0c0c0400u);
    const unsigned hi = __builtin_amdgcn_perm(b[4 * k + 3], b[4 * k + 2], 0x04000c0cu);
    r.q[k] = finite ? lo | hi : 0u;
  }
  r.scale = finite ? am * (1.0f / 127.0f) : __uint_as_float(0x7fc00000u);
  return r;
}

__device__ inline f8 restore(u2 q, float scale) {
#pragma clang fp contract(off)
  f8 r;
#pragma unroll
  for (int j = 0; j < 8; j++) r[j] = (float)(int)(signed char)(q[j / 4] >> 8 * (j % 4)) * scale;
  return r;
}

// ---- launch helper: the grid must not be empty, and a launch error is the caller's ----
inline int launched() { return hipGetLastError() == hipSuccess ? 0 : EMAC_ERR_DEVICE; }

} // namespace emac_rows
#endif
