// rows_kernel.hpp -- device helpers of the row operators (norm_kernel.hpp, act8.hip).
//
// Every lane owns 8 consecutive elements of a row (16 bytes of a 16-bit type, two 16-byte loads of
// float), so 16 consecutive lanes own one checkpoint block of 128 columns and its maximum is a
// reduction inside a DPP row. The vector types carry the alignment of their element alone: the
// same global_load_dwordx4 then serves every base address and row stride (this part splits what
// crosses a line); a row's last vector is taken in one of three ways (WHOLE, SHIFT, PIECES below).
#ifndef EMAC_ROWS_KERNEL_HPP_
#define EMAC_ROWS_KERNEL_HPP_

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "rows.h"

namespace emac_rows {

typedef __bf16 bf16;
typedef _Float16 half;

typedef float f8 __attribute__((ext_vector_type(8)));
typedef float f2 __attribute__((ext_vector_type(2)));
typedef unsigned u2 __attribute__((ext_vector_type(2)));
typedef unsigned u4 __attribute__((ext_vector_type(4)));
typedef unsigned u8x __attribute__((ext_vector_type(8)));
typedef unsigned short us2 __attribute__((ext_vector_type(2)));

// 8 elements as loaded, in dwords (vectors of 16-bit types end up an element to a register where
// they cross a branch): two elements of a 16-bit type to a dword, four bytes of a checkpoint
template <int ESIZE>
struct dwords;
template <>
struct dwords<4> { typedef u8x type; };
template <>
struct dwords<2> { typedef u4 type; };
template <>
struct dwords<1> { typedef u2 type; };
template <class T>
using raw8 = typename dwords<sizeof(T)>::type;
template <class V, int ALIGN>
struct any { // V in memory at any element's address
  typedef V type __attribute__((aligned(ALIGN)));
};

// a value that the compiler takes to be new here
template <class V>
__device__ inline void hold(V &v) {
#pragma unroll
  for (unsigned k = 0; k < sizeof(V) / 4; k++) {
    unsigned t = v[k];
    asm volatile("" : "+v"(t));
    v[k] = t;
  }
}

// How a row's last vector of n < 8 elements is taken. WHOLE (cols >= 8): its lane takes 8 elements
// like every other, the row's last, of which its own are the last n: it keeps the others out of sums,
// and stores them too, as the same bits that the lane before it stores. No load or store has a branch
// around it, and no two ways of one that would have to wait for each other's registers (a 8192 x 4099
// gradient of bf16 72 us against 118). SHIFT: loaded like that, but its own elements moved to the front
// where they are used, and stored alone: where a checkpoint's last block has fewer than 8 columns, so
// that the others have another scale. PIECES: its n elements alone, in pieces of 1, 2 and 4, where there
// are no 8, or where the others may have been replaced already (in place, in another wave).
enum { WHOLE = 0, SHIFT = 1, PIECES = 2 };
inline int tail_of(long cols, bool saved) {
  return cols < 8 ? PIECES : saved && cols % EMAC_BLOCK8 > 0 && cols % EMAC_BLOCK8 < 8 ? SHIFT : WHOLE;
}

// 8 elements at column c of a row (a row that all lanes share is a scalar base, and c a 32-bit offset
// from it). Matrices pass through once: nontemporal (a 4096 x 8192 norm of bf16 56 us against 65, a
// checkpoint of 8192 x 16384 71 against 90); what is read again soon is loaded with `again`.
template <class T, bool again = false>
__device__ inline raw8<T> load8(const T *row, unsigned c) {
  typedef typename any<raw8<T>, sizeof(T)>::type RA;
  const RA *p = (const RA *)((const char *)row + c * (unsigned)sizeof(T));
  if (again) return *p;
  return __builtin_nontemporal_load(p);
}

// n (clamped) of 8 elements, zeros behind them: pieces of 1, 2 and 4 from its end, each moving up
// what it precedes
template <class T>
__device__ inline raw8<T> load_pieces(const T *row, int n) {
  constexpr int E = sizeof(T);
  const char *p = (const char *)row;
  if (n >= 8) return load8(row, 0u);
  raw8<T> r = (raw8<T>)0u;
  if (n <= 0) return r;
  if constexpr (E == 4) {
    if (n & 1) r[0] = *(const unsigned *)(p + 4 * (n & 6));
    if (n & 2) {
      const u2 v = *(const typename any<u2, 4>::type *)(p + 4 * (n & 4));
      r[2] = r[0];
      r[0] = v[0];
      r[1] = v[1];
    }
    if (n & 4) {
      r.hi = r.lo;
      r.lo = *(const typename any<u4, 4>::type *)p;
    }
  } else if constexpr (E == 2) {
    if (n & 1) r[0] = *(const unsigned short *)(p + 2 * (n & 6));
    if (n & 2) {
      r[1] = r[0];
      r[0] = *(const typename any<unsigned, 2>::type *)(p + 2 * (n & 4));
    }
    if (n & 4) {
      r.hi = r.lo;
      r.lo = *(const typename any<u2, 2>::type *)p;
    }
  } else {
    if (n & 1) r[0] = *(const unsigned char *)(p + (n & 6));
    if (n & 2) r[0] = r[0] << 16 | *(const typename any<unsigned short, 1>::type *)(p + (n & 4));
    if (n & 4) {
      r[1] = r[0];
      r[0] = *(const typename any<unsigned, 1>::type *)p;
    }
  }
  return r;
}

// the last n of 8 elements (none if n <= 0) moved to the front, zeros behind them
template <class T>
__device__ inline raw8<T> last8(raw8<T> r, int n) {
  constexpr int E = sizeof(T);
  asm volatile("" : "+v"(n)); // as in slot::sums
  if (n >= 8) return r;
  const int k = n > 0 ? 8 - n : 0;
  if constexpr (E == 4) {
    if (k & 4) {
      r.lo = r.hi;
      r.hi = (u4)0u;
    }
    if (k & 2) r = __builtin_shufflevector(r, (u8x)0u, 2, 3, 4, 5, 6, 7, 8, 9);
    if (k & 1) r = __builtin_shufflevector(r, (u8x)0u, 1, 2, 3, 4, 5, 6, 7, 8);
  } else if constexpr (E == 2) {
    if (k & 4) {
      r.lo = r.hi;
      r.hi = (u2)0u;
    }
    if (k & 2) r = __builtin_shufflevector(r, (u4)0u, 1, 2, 3, 4);
    if (k & 1) {
      r[0] = __builtin_amdgcn_alignbit(r[1], r[0], 16);
      r[1] = __builtin_amdgcn_alignbit(r[2], r[1], 16);
      r[2] = __builtin_amdgcn_alignbit(r[3], r[2], 16);
      r[3] >>= 16;
    }
  } else {
    r = __builtin_bit_cast(u2, __builtin_bit_cast(unsigned long, r) >> 8 * k);
  }
  return n > 0 ? r : (raw8<T>)0u;
}

// the first n (clamped) of 8 elements to column c of a row
template <class T, bool again = false>
__device__ inline void store8(T *row, unsigned c, raw8<T> v, int n) {
  constexpr int E = sizeof(T);
  char *p = (char *)row + c * (unsigned)E;
  if (!__builtin_constant_p(n)) asm volatile("" : "+v"(n)); // as in slot::sums
  if (n >= 8) {
    typedef typename any<raw8<T>, E>::type RA;
    if (again) *(RA *)p = v;
    else __builtin_nontemporal_store((RA)v, (RA *)p);
    return;
  }
  if (n <= 0) return;
  if constexpr (E == 4) {
    if (n & 4) {
      *(typename any<u4, 4>::type *)p = v.lo;
      v.lo = v.hi;
    }
    if (n & 2) {
      *(typename any<u2, 4>::type *)(p + 4 * (n & 4)) = v.lo.lo;
      v[0] = v[2];
    }
    if (n & 1) *(unsigned *)(p + 4 * (n & 6)) = v[0];
  } else if constexpr (E == 2) {
    if (n & 4) {
      *(typename any<u2, 2>::type *)p = v.lo;
      v.lo = v.hi;
    }
    if (n & 2) {
      *(typename any<unsigned, 2>::type *)(p + 2 * (n & 4)) = v[0];
      v[0] = v[1];
    }
    if (n & 1) *(unsigned short *)(p + 2 * (n & 6)) = (unsigned short)v[0];
  } else {
    if (n & 4) {
      *(typename any<unsigned, 1>::type *)p = v[0];
      v[0] = v[1];
    }
    if (n & 2) {
      *(typename any<unsigned short, 1>::type *)(p + (n & 4)) = (unsigned short)v[0];
      v[0] >>= 16;
    }
    if (n & 1) *(unsigned char *)(p + (n & 6)) = (unsigned char)v[0];
  }
}

// between dwords and 32-bit floats; round_to rounds to nearest, ties to even
template <class T>
__device__ inline f8 widen(raw8<T> v) {
  f8 r;
  if constexpr (sizeof(T) == 4) {
    r = __builtin_bit_cast(f8, v);
  } else {
#pragma unroll
    for (int k = 0; k < 4; k++) {
      if constexpr (__is_same(T, bf16)) {
        r[2 * k] = __uint_as_float(v[k] << 16);
        r[2 * k + 1] = __uint_as_float(v[k] & 0xffff0000u);
      } else {
        typedef half h2 __attribute__((ext_vector_type(2)));
        const h2 h = __builtin_bit_cast(h2, (unsigned)v[k]);
        r[2 * k] = (float)h.x;
        r[2 * k + 1] = (float)h.y;
      }
    }
  }
  return r;
}
template <class T>
__device__ inline raw8<T> round_to(f8 v) {
  raw8<T> r;
  if constexpr (sizeof(T) == 4) {
    r = __builtin_bit_cast(u8x, v);
  } else {
    typedef T t2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const f2 f = {v[2 * k], v[2 * k + 1]};
      r[k] = __builtin_bit_cast(unsigned, __builtin_convertvector(f, t2));
    }
  }
  return r;
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
__device__ inline float sum8(float v) { // of lanes that hold the same eight values every eight lanes
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

// the bits of max |x| in its own type: integer order, in which an infinity and every NaN lie above
// all finite values, so neither is lost in the maximum
template <class T>
__device__ inline unsigned abs_bits(raw8<T> x) {
  if constexpr (sizeof(T) == 4) {
    unsigned m = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) m = max(m, x[j] & 0x7fffffffu);
    return m;
  } else {
    us2 m = {0, 0};
#pragma unroll
    for (int k = 0; k < 4; k++) m = __builtin_elementwise_max(m, __builtin_bit_cast(us2, (unsigned)x[k] & 0x7fff7fffu));
    return max((unsigned)m.x, (unsigned)m.y);
  }
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
__device__ inline block8 quantise(raw8<T> x) {
#pragma clang fp contract(off)
  const float a = of_bits<T>(max16(abs_bits<T>(x)));
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

// eight signed bytes as floats
__device__ inline f8 bytes(u2 q) {
  f8 r;
#pragma unroll
  for (int j = 0; j < 8; j++) r[j] = (float)(int)(signed char)(q[j / 4] >> 8 * (j % 4));
  return r;
}
// what a checkpoint restores to, to the bit: the product is rounded on its own
__device__ inline f8 restore(u2 q, float scale) {
#pragma clang fp contract(off)
  return bytes(q) * scale;
}

// A launch, with its own error and not one that an earlier call of the program left behind.
template <class... A, class... V>
int launch(void (*kernel)(A...), dim3 grid, int block, hipStream_t stream, V... values) {
  return [&](A... a) {
    void *args[] = {(void *)&a...};
    return hipLaunchKernel((const void *)kernel, grid, dim3(block), args, 0, stream) == hipSuccess ? 0 : EMAC_ERR_DEVICE;
  }(values...);
}

} // namespace emac_rows
#endif
