// act8.hip -- activations with 8-bit checkpoints of their inputs, their gradient from the
// checkpoints, and the checkpoints alone.
//
// Everything here is one pass over HBM: a 16-lane group owns one checkpoint block (128 columns of
// one row), U groups' loads are issued before the first is used, and a block's maximum is a
// reduction inside the group, so nothing is read twice and no barrier is needed. Blocks are
// numbered row by row; a workgroup divides once (scalars) and a lane only where a row holds fewer
// blocks than a workgroup takes. Bound by HBM; the arithmetic is about 30 lane operations per
// element, of the 50 or so that fit beside 8 bytes of traffic. Measured: a gated SiLU of 8192 x 12288
// bf16 with both checkpoints and its gradient from them, 1.62 GB in 279 us (5.8 TB/s); save and
// restore of 8192 x 16384 bf16, 814 MB in 132 us (6.1 TB/s).
#include "rows_kernel.hpp"

namespace {

using namespace emac_rows;

constexpr int kGroups = 16; // lane groups in a workgroup
constexpr int kGridX = 23;  // a launch's lanes in one dimension stay under 2^32: from 2^23 workgroups on there are two

// ---- activations: value and slope, in 32 bits ----
// 16-bit types take the native exp2 (of x log2 e rounded) and reciprocal, 1 ulp each. Float adds what
// the rounded product lost, |x| ulp in the exponential's far tails, and one Newton step: the library's
// exponential and an IEEE division make a gated SiLU of 8192 x 4096 floats 156 us instead of 94.
template <class T>
__device__ inline float exp_of(float x) {
  const float log2e = 1.44269504088896340736f;
  if constexpr (sizeof(T) == 4) {
    x = __builtin_amdgcn_fmed3f(x, -104.0f, 88.5f); // 0 and its reciprocal's reach: finite
    const float y = x * log2e, lost = fmaf(x, log2e, -y) + x * 1.92596299e-8f; // log2 e - log2e
    const float e = __builtin_amdgcn_exp2f(y);
    return fmaf(e, lost * 0.693147181f, e);
  }
  return __builtin_amdgcn_exp2f(x * log2e);
}
template <class T>
__device__ inline float recip(float x) {
  const float r = __builtin_amdgcn_rcpf(x);
  if constexpr (sizeof(T) == 4) return fmaf(fmaf(-x, r, 1.0f), r, r);
  return r;
}

// the normal distribution's tail beyond |a|, with e = exp(-a^2/2): e erfcx(|a| / sqrt 2) / 2, the latter as
// EMAC_GELU_TAIL's polynomial, which is off by 1.6e-7 of it at most (4.4e-7 as evaluated in 32 bits)
template <class T>
__device__ inline float normal_tail(float a, float e) {
  constexpr float c[] = EMAC_GELU_TAIL;
  const float t = recip<T>(1.0f + EMAC_GELU_TAIL_AT * fminf(fabsf(a), 64.0f)); // beyond, e is 0
  float p = c[0];
#pragma unroll
  for (int k = 1; k < 8; k++) p = p * t + c[k];
  return p * t * e;
}

template <class T, int KIND>
__device__ inline float act_value(float a) {
  if constexpr (KIND == EXT_MPI_AMD_SILU) {
    return a * recip<T>(1.0f + exp_of<T>(-a));
  } else if constexpr (KIND == EXT_MPI_AMD_GELU_TANH) {
    // (1 + tanh u) / 2 = 1 / (1 + exp(-2u)); beyond |a| = 64 it is 0 or 1 in 32 bits
    const float c = __builtin_amdgcn_fmed3f(a, -64.0f, 64.0f);
    const float u = 1.5957691216057308f * c * (1.0f + 0.044715f * c * c);
    return a * recip<T>(1.0f + exp_of<T>(-u));
  } else {
    const float p = normal_tail<T>(a, exp_of<T>(-0.5f * a * a));
    return a * (a > 0.0f ? 1.0f - p : p);
  }
}

template <class T, int KIND>
__device__ inline void act_both(float a, float &value, float &slope) {
  if constexpr (KIND == EXT_MPI_AMD_SILU) {
    const float s = recip<T>(1.0f + exp_of<T>(-a));
    value = a * s;
    slope = s * (1.0f + a * (1.0f - s));
  } else if constexpr (KIND == EXT_MPI_AMD_GELU_TANH) {
    const float c = __builtin_amdgcn_fmed3f(a, -64.0f, 64.0f), c2 = 0.044715f * c * c;
    const float s = recip<T>(1.0f + exp_of<T>(-1.5957691216057308f * c * (1.0f + c2)));
    value = a * s;
    slope = s + value * (1.0f - s) * (1.5957691216057308f * (1.0f + 3.0f * c2));
  } else {
    const float e = exp_of<T>(-0.5f * a * a), p = normal_tail<T>(a, e);
    const float phi = a > 0.0f ? 1.0f - p : p;
    value = a * phi;
    slope = phi + a * e * 0.3989422804014327f;
  }
}

// where a lane's 8 elements of block `u` (0 .. U - 1) of its group lie
template <int TAIL>
struct place {
  long row, from; // its row, the row loaded from (the last one again past it)
  int blk, own, c; // block of the row, first column of the lane, the column loaded from
  int n;           // elements from there to the row's end, 0 or less if none
  template <class T>
  __device__ raw8<T> load(const void *p, long stride) const {
    const T *r = (const T *)p + from * stride;
    if constexpr (TAIL == WHOLE) return load8(r, (unsigned)c);
    else return load_pieces(r + own, n);
  }
  template <class T>
  __device__ void store(void *p, long stride, raw8<T> v) const {
    if (n > 0) store8<T>((T *)p + row * stride, (unsigned)(TAIL == WHOLE ? c : own), v, TAIL == WHOLE ? 8 : n);
  }
};
template <int U, int TAIL>
struct span8 {
  long row0;
  unsigned blk0, nblk;
  long rows;
  int cols;
  __device__ span8(long rows_, long cols_, unsigned nblk_) : nblk(nblk_), rows(rows_), cols((int)cols_) {
    const unsigned first = (blockIdx.y << kGridX | blockIdx.x) * (unsigned)(U * kGroups);
    row0 = first / nblk;
    blk0 = first - (unsigned)row0 * nblk;
  }
  __device__ place<TAIL> at(int u) const {
    const unsigned x = blk0 + u * kGroups + threadIdx.x / 16;
    place<TAIL> p;
    unsigned k;
    if (nblk >= (unsigned)(U * kGroups)) k = x >= nblk ? 1u : 0u;
    else k = x / nblk;
    p.row = row0 + k;
    p.from = p.row < rows ? p.row : rows - 1;
    p.blk = (int)(x - k * nblk);
    p.own = p.blk * EMAC_BLOCK8 + (int)(threadIdx.x % 16) * 8;
    p.n = p.row < rows ? cols - p.own : 0;
    p.c = min(p.own, cols - 8); // with PIECES not used
    return p;
  }
};

template <class T, int TAIL>
__device__ inline void put8(const place<TAIL> &p, raw8<T> x, signed char *q, long q_stride, float *scale, unsigned nblk) {
  const block8 b = quantise<T>(x); // what a lane holds of another's is of the same block
  p.template store<signed char>(q, q_stride, b.q);
  if (p.n > 0 && threadIdx.x % 16 == 0) scale[p.row * nblk + p.blk] = b.scale;
}

template <class T, int KIND, bool GATE, int U, int TAIL>
__global__ __launch_bounds__(256) void act_kernel(const ext_mpi_amd_act d, unsigned nblk) {
  const span8<U, TAIL> s(d.rows, d.cols, nblk);
  raw8<T> a[U], b[GATE ? U : 1];
#pragma unroll
  for (int u = 0; u < U; u++) {
    const place<TAIL> p = s.at(u);
    a[u] = p.template load<T>(d.a, d.a_stride);
    if (GATE) b[GATE ? u : 0] = p.template load<T>(d.b, d.b_stride);
  }
#pragma unroll
  for (int u = 0; u < U; u++) {
    const place<TAIL> p = s.at(u);
    if constexpr (KIND != EMAC_SAVE8) {
      if (d.h) {
        const f8 f = widen<T>(a[u]);
        f8 v;
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = act_value<T, KIND>(f[j]);
        if (GATE) v *= widen<T>(b[GATE ? u : 0]);
        p.template store<T>(d.h, d.h_stride, round_to<T>(v));
      }
    }
    if (d.qa) {
      put8<T>(p, a[u], d.qa, d.q_stride, d.sa, nblk);
      if (GATE) put8<T>(p, b[GATE ? u : 0], d.qb, d.q_stride, d.sb, nblk);
    }
  }
}

template <class T, int KIND, bool GATE, int U, int TAIL>
__global__ __launch_bounds__(256) void act_grad_kernel(const ext_mpi_amd_act_grad d, unsigned nblk) {
  const span8<U, TAIL> s(d.rows, d.cols, nblk);
  raw8<T> g[U];
  u2 qa[U], qb[GATE ? U : 1];
  float sa[U], sb[GATE ? U : 1];
#pragma unroll
  for (int u = 0; u < U; u++) {
    const place<TAIL> p = s.at(u);
    g[u] = p.template load<T>(d.dh, d.dh_stride);
    qa[u] = p.template load<signed char>(d.qa, d.q_stride);
    sa[u] = d.sa[p.from * nblk + p.blk];
    if (GATE) {
      qb[GATE ? u : 0] = p.template load<signed char>(d.qb, d.q_stride);
      sb[GATE ? u : 0] = d.sb[p.from * nblk + p.blk];
    }
  }
#pragma unroll
  for (int u = 0; u < U; u++) {
    const place<TAIL> p = s.at(u);
    const f8 a = restore(qa[u], sa[u]), dh = widen<T>(g[u]);
    f8 value, slope;
#pragma unroll
    for (int j = 0; j < 8; j++) {
      float v, w;
      act_both<T, KIND>(a[j], v, w);
      value[j] = v;
      slope[j] = w;
    }
    slope *= dh;
    if (GATE) {
      const f8 b = restore(qb[GATE ? u : 0], sb[GATE ? u : 0]);
      p.template store<T>(d.da, d.da_stride, round_to<T>(slope * b));
      p.template store<T>(d.db, d.db_stride, round_to<T>(dh * value));
      value *= b;
    } else {
      p.template store<T>(d.da, d.da_stride, round_to<T>(slope));
    }
    if (d.h) p.template store<T>(d.h, d.h_stride, round_to<T>(value));
  }
}

template <class T, int U, int TAIL>
__global__ __launch_bounds__(256) void restore8_kernel(long rows, long cols, const signed char *q, long q_stride,
                                                       const float *scale, T *x, long x_stride, unsigned nblk) {
  const span8<U, TAIL> s(rows, cols, nblk);
  u2 w[U];
  float sc[U];
#pragma unroll
  for (int u = 0; u < U; u++) {
    const place<TAIL> p = s.at(u);
    w[u] = p.template load<signed char>(q, q_stride);
    sc[u] = scale[p.from * nblk + p.blk];
  }
#pragma unroll
  for (int u = 0; u < U; u++) {
    const place<TAIL> p = s.at(u);
    p.template store<T>(x, x_stride, round_to<T>(restore(w[u], sc[u])));
  }
}

// ---- launches ----

struct grid8 {
  unsigned nblk;
  dim3 grid;
  int u, tail;
};
// blocks, workgroups and blocks per lane group (engine_rows.c holds rows * blocks under 2^31): 4
// blocks' loads in flight where that leaves 8 workgroups to a CU, else as many workgroups as can be
grid8 grid_of(long rows, long cols, bool in_place) {
  grid8 g;
  g.nblk = (unsigned)((cols + EMAC_BLOCK8 - 1) / EMAC_BLOCK8);
  // an odd width that a checkpoint's scale crosses is faster in pieces than shifted here (8192 x 4099
  // gated SiLU of bf16 52 us against 62)
  g.tail = tail_of(cols, true) != WHOLE || (in_place && cols % 8) ? PIECES : WHOLE;
  g.u = g.tail != PIECES && rows * g.nblk >= 4L * kGroups * 2048 ? 4 : 1;
  const long n = (rows * g.nblk + g.u * kGroups - 1) / (g.u * kGroups), x = 1L << kGridX;
  g.grid = n < x ? dim3((unsigned)n) : dim3((unsigned)x, (unsigned)((n + x - 1) / x));
  return g;
}

template <int V>
struct num {
  static constexpr int v = V;
};
// calls go with the kernel's U and TAIL
template <class F>
int shaped(const grid8 &g, F go) {
  if (g.tail == PIECES) return go(num<1>(), num<PIECES>());
  if (g.u == 4) return go(num<4>(), num<WHOLE>());
  return go(num<1>(), num<WHOLE>());
}

template <class T, int KIND, bool GATE>
int act_go(const ext_mpi_amd_act &d, hipStream_t st) {
  const grid8 g = grid_of(d.rows, d.cols, d.h && (d.h == d.a || d.h == d.b));
  return shaped(g, [&](auto u, auto tail) { return launch(act_kernel<T, KIND, GATE, u.v, tail.v>, g.grid, 256, st, d, g.nblk); });
}

template <class T, int KIND>
int act_k(const ext_mpi_amd_act &d, hipStream_t st) {
  return d.b ? act_go<T, KIND, true>(d, st) : act_go<T, KIND, false>(d, st);
}

template <class T>
int act_t(const ext_mpi_amd_act &d, hipStream_t st) {
  switch (d.kind) {
  case EMAC_SAVE8: return act_go<T, EMAC_SAVE8, false>(d, st);
  case EXT_MPI_AMD_SILU: return act_k<T, EXT_MPI_AMD_SILU>(d, st);
  case EXT_MPI_AMD_GELU: return act_k<T, EXT_MPI_AMD_GELU>(d, st);
  case EXT_MPI_AMD_GELU_TANH: return act_k<T, EXT_MPI_AMD_GELU_TANH>(d, st);
  }
  return EMAC_ERR_ARG;
}

template <class T, int KIND, bool GATE>
int act_grad_go(const ext_mpi_amd_act_grad &d, hipStream_t st) {
  const grid8 g = grid_of(d.rows, d.cols, d.da == d.dh || d.db == d.dh || d.h == d.dh);
  return shaped(g, [&](auto u, auto tail) {
    return launch(act_grad_kernel<T, KIND, GATE, u.v, tail.v>, g.grid, 256, st, d, g.nblk);
  });
}

template <class T, int KIND>
int act_grad_k(const ext_mpi_amd_act_grad &d, hipStream_t st) {
  return d.qb ? act_grad_go<T, KIND, true>(d, st) : act_grad_go<T, KIND, false>(d, st);
}

template <class T>
int act_grad_t(const ext_mpi_amd_act_grad &d, hipStream_t st) {
  switch (d.kind) {
  case EXT_MPI_AMD_SILU: return act_grad_k<T, EXT_MPI_AMD_SILU>(d, st);
  case EXT_MPI_AMD_GELU: return act_grad_k<T, EXT_MPI_AMD_GELU>(d, st);
  case EXT_MPI_AMD_GELU_TANH: return act_grad_k<T, EXT_MPI_AMD_GELU_TANH>(d, st);
  }
  return EMAC_ERR_ARG;
}

template <class T>
int restore_t(long rows, long cols, const signed char *q, long q_stride, const float *scale, void *x, long x_stride,
              hipStream_t st) {
  const grid8 g = grid_of(rows, cols, false);
  return shaped(g, [&](auto u, auto tail) {
    return launch(restore8_kernel<T, u.v, tail.v>, g.grid, 256, st, rows, cols, q, q_stride, scale, (T *)x, x_stride, g.nblk);
  });
}

} // namespace

extern "C" {

int emac_gpu_act(const ext_mpi_amd_act *d, void *stream) {
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (d->rows <= 0) return 0;
  switch (d->dtype) {
  case EXT_MPI_AMD_FLOAT: return act_t<float>(*d, st);
  case EXT_MPI_AMD_BF16: return act_t<bf16>(*d, st);
  case EXT_MPI_AMD_HALF: return act_t<half>(*d, st);
  }
  return EMAC_ERR_UNSUPPORTED;
}

int emac_gpu_act_grad(const ext_mpi_amd_act_grad *d, void *stream) {
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (d->rows <= 0) return 0;
  switch (d->dtype) {
  case EXT_MPI_AMD_FLOAT: return act_grad_t<float>(*d, st);
  case EXT_MPI_AMD_BF16: return act_grad_t<bf16>(*d, st);
  case EXT_MPI_AMD_HALF: return act_grad_t<half>(*d, st);
  }
  return EMAC_ERR_UNSUPPORTED;
}

int emac_gpu_restore8(long rows, long cols, int dtype, const signed char *q, long q_stride, const float *scale, void *x,
                      long x_stride, void *stream) {
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (rows <= 0) return 0;
  switch (dtype) {
  case EXT_MPI_AMD_FLOAT: return restore_t<float>(rows, cols, q, q_stride, scale, x, x_stride, st);
  case EXT_MPI_AMD_BF16: return restore_t<bf16>(rows, cols, q, q_stride, scale, x, x_stride, st);
  case EXT_MPI_AMD_HALF: return restore_t<half>(rows, cols, q, q_stride, scale, x, x_stride, st);
  }
  return EMAC_ERR_UNSUPPORTED;
}

} // extern "C"
