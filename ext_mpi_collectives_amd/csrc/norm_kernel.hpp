// norm_kernel.hpp -- layer norm over the folded partials of the ranks, and its gradient.
//
// Forward: a row lives in the registers of its lanes (NV vectors of 8 elements each) from the
// leaves' loads to y's stores, so each input is read once and each output written once; the mean
// and then the sum of squared differences are two reductions over those registers (never E[x^2] -
// mean^2). x is rounded to its type before its statistics, so a gradient that reads x (or the
// checkpoint, taken from the same registers) sees the values that were normalised.
// Gradient: the same layout; each lane owns the same columns in every row its workgroup takes, so
// the two column sums (dweight, dbias) stay in its registers over all of them, and leave as one
// partial row per workgroup, which a second kernel adds in order: no atomics, the same bits every
// time. Both directions are bound by HBM at large sizes and by launch latency at small ones: 4096 x
// 8192 bf16 with a residual added and the sum stored, 268 MB in 45.8 us (5.9 TB/s); the gradient of
// 16384 x 4096 bf16 with dsum, 537 MB in 89 us (6.0 TB/s); one row of 4096 from 8 leaves 4.1 us.
#ifndef EMAC_NORM_KERNEL_HPP_
#define EMAC_NORM_KERNEL_HPP_

#include "rows_kernel.hpp"

namespace emac_rows {

// How the lanes of a workgroup share out rows: MODE 16 or 64 lanes to a row, 256 lanes in all, or all
// of a workgroup of as many waves as the row needs at NV vectors to a lane, at most 8 (MODE 512) or 16
// (MODE 1024). With many rows, few waves with many registers (up to 256) and the next row's loads in
// flight hide the latency; more waves only repeat what every wave does once a row. With a row or less
// for each CU they shorten it: 32 rows of 8192 bf16 from 8 leaves 7.4 us with 16 waves, 7.8 with 8.
template <int MODE>
struct lanes {
  static constexpr bool kOneRow = MODE >= 512;             // a workgroup takes one row at a time
  static constexpr int kBlock = kOneRow ? MODE : 256;      // at most
  static constexpr int kWaves = MODE == 512 ? 2 : 4;       // waves to a SIMD that the registers allow
  static constexpr int kRows = kOneRow ? 1 : 256 / MODE;
  static constexpr int kSlots = MODE == 1024 ? 16 : 8;     // waves that share a row, at most
  int per, l, sub; // lanes to a row, this lane's place in it, its row in the workgroup
  __device__ lanes() {
    per = kOneRow ? (int)blockDim.x : MODE;
    l = kOneRow ? threadIdx.x : threadIdx.x % MODE;
    sub = kOneRow ? 0 : threadIdx.x / MODE;
    if (MODE == 64) sub = __builtin_amdgcn_readfirstlane(sub);
  }
};

// A lane's vector i of a row. A lane past the row's end loads the row's last 8 elements and keeps
// them out of every sum and store.
template <int TAIL>
struct slot {
  static constexpr int kTail = TAIL;
  int own, c, n; // first column of its own, of those it loads; its own elements (0 or less: none)
  __device__ slot(int i, int per, int l, int cols, bool live) {
    own = (l + i * per) * 8;
    n = live ? cols - own : 0;
    c = TAIL != PIECES ? min(own, cols - 8) : own;
  }
  __device__ bool in() const { return n > 0; }
  // whether the lane's element j is its own
  __device__ bool mine(int j) const { return TAIL == WHOLE ? j >= 8 - n : j < n; }
  template <class T, bool again = false>
  __device__ raw8<T> load(const void *row) const {
    if constexpr (TAIL != PIECES) return load8<T, again>((const T *)row, (unsigned)c);
    else return load_pieces((const T *)row + c, n);
  }
  // what was loaded, where it is used
  template <class T>
  __device__ raw8<T> put(raw8<T> v) const {
    if constexpr (TAIL == SHIFT) return last8<T>(v, n);
    else return v;
  }
  __device__ f8 put(f8 v) const {
    if constexpr (TAIL == SHIFT) return __builtin_bit_cast(f8, last8<float>(__builtin_bit_cast(u8x, v), n));
    else return v;
  }
  template <class T, bool again = false>
  __device__ void store(void *row, raw8<T> v) const {
    if (in()) store8<T, again>((T *)row, (unsigned)(TAIL == WHOLE ? c : own), v, TAIL == WHOLE ? 8 : n);
  }
  // f's, and f h's, own elements added to s0 and s1, each vector's first among themselves: short chains
  __device__ void sums(f8 f, f8 h, float &s0, float &s1) const {
    int m = n;
    asm volatile("" : "+v"(m)); // or the branches of several vectors are threaded together, and their registers
    float t0, t1;
    if (m >= 8) {
      t0 = f[0];
      t1 = f[0] * h[0];
#pragma unroll
      for (int j = 1; j < 8; j++) {
        t0 += f[j];
        t1 += f[j] * h[j];
      }
    } else {
      t0 = t1 = 0.0f;
#pragma unroll
      for (int j = 0; j < 8; j++) {
        t0 += mine(j) ? f[j] : 0.0f;
        t1 += mine(j) ? f[j] * h[j] : 0.0f;
      }
    }
    s0 += t0;
    s1 += t1;
  }
};
template <class T>
__device__ inline const T *row_of(const void *p, long row, long stride) {
  return (const T *)p + row * stride;
}

// Sums over a row's lanes. Between waves they go through LDS: each wave leaves its own, and after
// one barrier 8 or 16 lanes of every wave add as many of them; the two slots are used in turn, so
// a slot's last read and its next write have a barrier between them.
template <int MODE, int NS>
struct row_sum {
  static constexpr int kSlots = lanes<MODE>::kSlots;
  float (*red)[kSlots][NS];
  int turn;
  __device__ row_sum(float (*r)[kSlots][NS]) : red(r), turn(0) {
    if (lanes<MODE>::kOneRow) { // the places of waves that are not there
      const int nw = blockDim.x / 64, t = threadIdx.x;
      if (t < 2 * kSlots && t % kSlots >= nw) {
#pragma unroll
        for (int k = 0; k < NS; k++) r[t / kSlots][t % kSlots][k] = 0.0f;
      }
    }
  }
  __device__ void operator()(float (&v)[NS]) {
#pragma unroll
    for (int k = 0; k < NS; k++) v[k] = MODE == 16 ? sum16(v[k]) : sum64(v[k]);
    if constexpr (lanes<MODE>::kOneRow) {
      if (threadIdx.x % 64 == 0) {
#pragma unroll
        for (int k = 0; k < NS; k++) red[turn][threadIdx.x / 64][k] = v[k];
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < NS; k++) {
        const float t = red[turn][threadIdx.x % kSlots][k];
        v[k] = kSlots == 8 ? sum8(t) : sum16(t);
      }
      turn ^= 1;
    }
  }
};

// ((leaf 0 + leaf 1) + ...) of a lane's NV vectors of a row, in 32 bits. The loads of a batch of leaves
// are in flight together, for all vectors: as many as 32 registers hold, 64 with several vectors (one
// row of 8832 floats from 4 leaves 6.7 us against 10.3 vector by vector).
template <class T, int NV, int TAIL>
__device__ inline void fold_rows(f8 (&s)[NV], const void *const *src, int nsrc, long row, long stride, int per, int l, int cols) {
  constexpr int fit = (NV == 1 ? 16 : 32) / (NV * (int)sizeof(T)), B = fit < 1 ? 1 : fit;
  for (int t0 = 0; t0 < nsrc; t0 += B) {
    raw8<T> raw[B][NV];
#pragma unroll
    for (int k = 0; k < B; k++)
      if (t0 + k < nsrc) {
        const T *p = row_of<T>(src[t0 + k], row, stride);
#pragma unroll
        for (int i = 0; i < NV; i++) raw[k][i] = slot<TAIL>(i, per, l, cols, true).template load<T>(p);
      }
#pragma unroll
    for (int k = 0; k < B; k++)
      if (t0 + k < nsrc) {
#pragma unroll
        for (int i = 0; i < NV; i++) s[i] = t0 + k ? s[i] + widen<T>(raw[k][i]) : widen<T>(raw[k][i]);
      }
  }
}

// A row's weights (`none` without any), in registers over all rows of a workgroup. A load of them
// among the next row's would be worse than its own latency: loads return in order, so waiting for it
// is waiting for the next row. At up to two vectors to a lane they are held as floats; as loaded at
// more, and by the forms that do not load ahead, which would wait for them before their first row's
// loads. The widest of those load them at their use.
template <class W, int NV, int TAIL, bool AHEAD>
struct weights {
  static constexpr bool kFloats = NV <= 2 && AHEAD, kRaw = !kFloats && (AHEAD || NV <= 2);
  f8 v[kFloats ? NV : 1];
  raw8<W> r[kRaw ? NV : 1];
  const W *p;
  float none;
  __device__ weights(const void *p_, float none_, int per, int l, int cols) : p((const W *)p_), none(none_) {
#pragma unroll
    for (int i = 0; i < NV; i++) {
      const slot<TAIL> at(i, per, l, cols, true);
      if (kFloats) v[kFloats ? i : 0] = floats(p ? at.template load<W, true>(p) : (raw8<W>)0u, at);
      if (kRaw && p) r[kRaw ? i : 0] = at.template load<W, true>(p);
    }
  }
  __device__ f8 floats(raw8<W> w, const slot<TAIL> &at) const {
    return p ? widen<W>(at.template put<W>(w)) : (f8)none;
  }
  __device__ f8 at(int i, const slot<TAIL> &s) const {
    if (kFloats) return v[kFloats ? i : 0];
    raw8<W> w = (raw8<W>)0u;
    if (kRaw) {
      w = r[kRaw ? i : 0];
      hold(w); // widened at each use: the floats would stay in twice the registers
    } else if (p) {
      w = s.template load<W, true>(p);
    }
    return floats(w, s);
  }
};

template <class T, class W, int MODE, int NV, bool MULTI, int TAIL>
__global__ __launch_bounds__(lanes<MODE>::kBlock, lanes<MODE>::kWaves) void layernorm_kernel(const ext_mpi_amd_layernorm d) {
  constexpr bool AHEAD = !MULTI && NV * sizeof(T) <= 12; // the next row's loads are issued before this row's sums
  constexpr bool EACH = MULTI && MODE == 1024 && NV > 1; // wide rows, folded vector by vector: x alone stays in registers
  const lanes<MODE> ln;
  const int l = ln.l, per = ln.per, cols = (int)d.cols;
  const int nblk = (cols + EMAC_BLOCK8 - 1) / EMAC_BLOCK8;
  const float inv = 1.0f / (float)cols;
  __shared__ float red[2][lanes<MODE>::kSlots][1];
  row_sum<MODE, 1> sum_row(red);
  const weights<W, NV, TAIL, AHEAD> w(d.weight, 1.0f, per, l, cols), b(d.bias, 0.0f, per, l, cols);
  const long step = (long)gridDim.x * ln.kRows;
  raw8<T> nx[MULTI ? 1 : NV], nr[NV];
  const auto load = [&](long row) {
#pragma unroll
    for (int i = 0; i < NV; i++) {
      const slot<TAIL> at(i, per, l, cols, true);
      if (!MULTI) nx[MULTI ? 0 : i] = at.template load<T>(row_of<T>(d.src[0], row, d.src_stride));
      if (d.residual) nr[i] = at.template load<T>(row_of<T>(d.residual, row, d.residual_stride));
    }
  };
  // past the last row the last one is loaded again: no branch around the loads
  const auto within = [&](long row) { return row < d.rows ? row : d.rows - 1; };
  long r0 = (long)blockIdx.x * ln.kRows;
  if (AHEAD) load(within(r0 + ln.sub));
  for (; r0 < d.rows; r0 += step) {
    const long row = r0 + ln.sub;
    const bool live = ln.kOneRow || row < d.rows;
    raw8<T> x[NV];
    float s[1] = {0.0f};
    if (!AHEAD && !EACH) load(within(row));
    f8 sum[MULTI && !EACH ? NV : 1];
    if constexpr (MULTI && !EACH) fold_rows<T, NV, TAIL>(sum, d.src, d.nsrc, within(row), d.src_stride, per, l, cols);
#pragma unroll
    for (int i = 0; i < NV; i++) {
      const slot<TAIL> at(i, per, l, cols, true);
      if constexpr (EACH) {
        if (d.residual) nr[i] = at.template load<T>(row_of<T>(d.residual, row, d.residual_stride));
        f8 one[1];
        fold_rows<T, 1, TAIL>(one, d.src, d.nsrc, row, d.src_stride, per, l + i * per, cols);
        sum[0] = one[0];
      }
      if (MULTI || d.residual) {
        f8 f;
        if (MULTI) f = sum[MULTI && !EACH ? i : 0];
        else f = widen<T>(nx[MULTI ? 0 : i]);
        if (d.residual) f += widen<T>(nr[i]);
        x[i] = round_to<T>(f);
      } else {
        x[i] = nx[MULTI ? 0 : i];
      }
      x[i] = at.template put<T>(x[i]);
      if (EACH && NV > 4 && i % 2) { // two vectors' loads in flight: all of them would spill
        hold(x[i - (NV > 4)]);
        hold(x[i]);
        asm volatile("" ::: "memory");
      }
    }
    if (AHEAD) load(within(row + step));
#pragma unroll
    for (int i = 0; i < NV; i++) {
      float none = 0.0f;
      slot<TAIL>(i, per, l, cols, true).sums(widen<T>(x[i]), (f8)0.0f, s[0], none);
    }
    if (d.y || d.mean || d.rstd) {
      sum_row(s);
      const float mean = s[0] * inv;
      s[0] = 0.0f;
#pragma unroll
      for (int i = 0; i < NV; i++) {
        const slot<TAIL> at(i, per, l, cols, true);
        if (EACH) hold(x[i]); // or its floats, and then the differences, stay in registers beside x
        const f8 f = widen<T>(x[i]) - mean;
        float none = 0.0f;
        at.sums(f * f, (f8)0.0f, s[0], none);
      }
      sum_row(s);
      const float rstd = 1.0f / sqrtf(s[0] * inv + (float)d.eps);
      if (l == 0 && live) {
        if (d.mean) d.mean[row] = mean;
        if (d.rstd) d.rstd[row] = rstd;
      }
#pragma unroll
      for (int i = 0; i < NV; i++) {
        const slot<TAIL> at(i, per, l, cols, live);
        if (!d.y) continue;
        if (EACH) hold(x[i]);
        const f8 f = (widen<T>(x[i]) - mean) * rstd * w.at(i, at) + b.at(i, at);
        at.template store<T>((T *)d.y + row * d.y_stride, round_to<T>(f));
      }
    } else if (ln.kOneRow && TAIL != PIECES) {
      __syncthreads(); // sum may replace the residual: the row's last lane has read what the one before it owns
    }
#pragma unroll
    for (int i = 0; i < NV; i++) {
      const slot<TAIL> at(i, per, l, cols, live);
      if (d.sum) at.template store<T>((T *)d.sum + row * d.sum_stride, x[i]);
      if (d.q) { // every lane of a block takes part; what a lane holds of another's is of the same block
        const block8 k = quantise<T>(x[i]);
        at.template store<signed char>(d.q + row * d.q_stride, k.q);
        if (at.in() && at.own % EMAC_BLOCK8 == 0) d.scale[row * nblk + at.own / EMAC_BLOCK8] = k.scale;
      }
    }
  }
}

// a finished column sum into dweight / dbias
__device__ inline void put_grad(void *out, int gdtype, int accumulate, long c, float v) {
  if (gdtype == EXT_MPI_AMD_FLOAT) {
    float *p = (float *)out + c;
    *p = accumulate ? *p + v : v;
  } else if (gdtype == EXT_MPI_AMD_BF16) {
    bf16 *p = (bf16 *)out + c;
    *p = (bf16)(accumulate ? (float)*p + v : v);
  } else {
    half *p = (half *)out + c;
    *p = (half)(accumulate ? (float)*p + v : v);
  }
}

// Column sums that a workgroup has finished, 8 of each, into its partial row
template <int TAIL>
__device__ inline void put_cols(float *part, int slice, long cols, const slot<TAIL> &at, f8 w, f8 b) {
  float *p = part + (long)slice * 2 * cols;
  at.template store<float, true>(p, round_to<float>(w));
  at.template store<float, true>(p + cols, round_to<float>(b));
}

// x of a row, or its checkpoint, as loaded
template <class T, bool Q8, int TAIL>
struct row8 {
  raw8<T> x;
  u2 q;
  float scale;
  __device__ void load(const ext_mpi_amd_layernorm_grad &d, long row, const slot<TAIL> &at, int nblk) {
    if (Q8) {
      q = at.template load<signed char>(d.q + row * d.q_stride);
      scale = d.scale[row * nblk + min(at.own / EMAC_BLOCK8, nblk - 1)];
    } else {
      x = at.template load<T>(row_of<T>(d.x, row, d.x_stride));
    }
  }
  // (x - mean) * rstd, the difference first: x * rstd - mean * rstd would be one operation, but off by half
  // a step of mean * rstd, which is far more than xh in rows whose mean is large against their deviation (both
  // at HBM's rate: 16384 x 4096 bf16 90.0 us, from a checkpoint 8192 x 5120 54.5; 65536 x 256 34 against 32.5)
  __device__ f8 normed(float mean, float rstd, const slot<TAIL> &at) const {
    if constexpr (Q8) return (restore(at.template put<signed char>(q), scale) - mean) * rstd;
    else return (widen<T>(at.template put<T>(x)) - mean) * rstd;
  }
};

// The rows of workgroup `block` of `blocks`: dx, y, and with ACC the two column sums.
template <class T, class W, int MODE, int NV, bool Q8, bool MULTI, int TAIL, bool ACC>
__device__ inline void grad_rows(const ext_mpi_amd_layernorm_grad &d, int block, int blocks, float *part) {
  // one leaf: the next row's loads are issued before this row's sums, as far as registers go
  constexpr bool AHEAD = !MULTI && (NV <= 2 || NV * sizeof(T) <= 6);
  // y has kernels of its own (the ones for any number of leaves and any width): a load of the bias
  // among the next row's, even where no y is asked for, makes every row wait for the next
  constexpr bool Y = MULTI;
  const lanes<MODE> ln;
  const int l = ln.l, per = ln.per, cols = (int)d.cols;
  const int nblk = (cols + EMAC_BLOCK8 - 1) / EMAC_BLOCK8;
  const float inv = 1.0f / (float)cols;
  __shared__ float red[2][lanes<MODE>::kSlots][2];
  row_sum<MODE, 2> sum_row(red);
  const weights<W, NV, TAIL, AHEAD> w(d.weight, 1.0f, per, l, cols);
  const long step = (long)blocks * ln.kRows;
  const bool more = d.dsum && d.dx;
  f8 aw[ACC ? NV : 1] = {}, ab[ACC ? NV : 1] = {};
  raw8<T> ng[MULTI ? 1 : NV], nd[NV];
  row8<T, Q8, TAIL> nx[NV];
  float nmean, nrstd;
  const auto load = [&](long row) {
    nmean = d.mean[row];
    nrstd = d.rstd[row];
#pragma unroll
    for (int i = 0; i < NV; i++) {
      const slot<TAIL> at(i, per, l, cols, true);
      if (!MULTI) ng[MULTI ? 0 : i] = at.template load<T>(row_of<T>(d.dy[0], row, d.dy_stride));
      nx[i].load(d, row, at, nblk);
      if (more) nd[i] = at.template load<T>(row_of<T>(d.dsum, row, d.dsum_stride));
    }
  };
  const auto within = [&](long row) { return row < d.rows ? row : d.rows - 1; };
  long r0 = (long)block * ln.kRows;
  if (AHEAD) load(within(r0 + ln.sub));
  for (; r0 < d.rows; r0 += step) {
    const long row = r0 + ln.sub;
    const bool live = ln.kOneRow || row < d.rows;
    if (!AHEAD) load(within(row));
    const float rstd = nrstd, mean = nmean;
    f8 g[NV], xh[NV];
    raw8<T> dsum[NV];
    float s[2] = {0.0f, 0.0f};
    if constexpr (MULTI) fold_rows<T, NV, TAIL>(g, d.dy, d.nsrc, within(row), d.dy_stride, per, l, cols);
#pragma unroll
    for (int i = 0; i < NV; i++) {
      const slot<TAIL> at(i, per, l, cols, true);
      if (!MULTI) g[i] = widen<T>(ng[MULTI ? 0 : i]);
      g[i] = at.put(g[i]);
      xh[i] = nx[i].normed(mean, rstd, at);
      dsum[i] = nd[i];
      // a row past the last, for which the last one was loaded: nothing of it counts, for its values may
      // be infinite, or be replaced by dx in another wave at this time
      if (!ln.kOneRow && !live) g[i] = xh[i] = (f8)0.0f;
    }
    if (AHEAD) load(within(row + step));
#pragma unroll
    for (int i = 0; i < NV; i++) {
      const slot<TAIL> at(i, per, l, cols, live);
      const f8 ww = w.at(i, at);
      if (ACC) {
        aw[ACC ? i : 0] += g[i] * xh[i];
        ab[ACC ? i : 0] += g[i];
      }
      if (Y && d.y) {
        f8 y = xh[i] * ww;
        if (d.bias) y += widen<W>(at.template put<W>(at.template load<W, true>(d.bias)));
        at.template store<T>((T *)d.y + row * d.y_stride, round_to<T>(y));
      }
      g[i] *= ww;
      at.sums(g[i], xh[i], s[0], s[1]);
    }
    if (!d.dx) continue;
    sum_row(s);
    const float c1 = -s[0] * inv * rstd, c2 = -s[1] * inv * rstd;
#pragma unroll
    for (int i = 0; i < NV; i++) {
      const slot<TAIL> at(i, per, l, cols, live);
      f8 dx = xh[i] * c2 + c1;
      dx += g[i] * rstd;
      if (more) dx += widen<T>(at.template put<T>(dsum[i]));
      at.template store<T>((T *)d.dx + row * d.dx_stride, round_to<T>(dx));
    }
  }
  if constexpr (ACC) {
    if (!part) return; // no column sums are asked for
    if constexpr (!lanes<MODE>::kOneRow) { // the rows of a workgroup taken side by side, added in order
      __shared__ f8 comb[2][MODE * NV];
      for (int k = 1; k < ln.kRows; k++) {
        __syncthreads();
        if (ln.sub == k) {
#pragma unroll
          for (int i = 0; i < NV; i++) {
            comb[0][l + i * per] = aw[i];
            comb[1][l + i * per] = ab[i];
          }
        }
        __syncthreads();
        if (ln.sub == 0) {
#pragma unroll
          for (int i = 0; i < NV; i++) {
            aw[i] += comb[0][l + i * per];
            ab[i] += comb[1][l + i * per];
          }
        }
      }
      if (ln.sub) return;
    }
#pragma unroll
    for (int i = 0; i < NV; i++) put_cols(part, block, d.cols, slot<TAIL>(i, per, l, cols, true), aw[i], ab[i]);
  }
}

template <class T, class W, int MODE, int NV, bool Q8, bool MULTI, int TAIL>
__global__ __launch_bounds__(lanes<MODE>::kBlock, lanes<MODE>::kWaves) void layernorm_grad_kernel(
    const ext_mpi_amd_layernorm_grad d, float *part) {
  grad_rows<T, W, MODE, NV, Q8, MULTI, TAIL, true>(d, blockIdx.x, gridDim.x, part);
}

// the sums of up to 512 lanes, by row taken and column
template <int LANES>
using lanes_sums = float[512 / LANES][8 * LANES];

// The column sums alone: a workgroup takes 8 * LANES columns of every slices'th group of rows, as
// many rows at a time as it has lanes for. They go into its slice's partial row, or (no partial rows) into
// the gradients.
template <class T, int LANES, bool Q8, bool MULTI, int TAIL>
__device__ inline void cols_tile(const ext_mpi_amd_layernorm_grad &d, int tile, int slice, int slices, float *part,
                                 lanes_sums<LANES> *comb) {
  constexpr int C = 8 * LANES;
  const int l = threadIdx.x % LANES, k0 = threadIdx.x / LANES, R = blockDim.x / LANES;
  const int cols = (int)d.cols, nblk = (cols + EMAC_BLOCK8 - 1) / EMAC_BLOCK8;
  const slot<TAIL> at(0, 0, tile * LANES + l, cols, true);
  f8 aw = {}, ab = {};
#pragma unroll 4
  for (long row = (long)slice * R + k0; row < d.rows; row += (long)slices * R) {
    row8<T, Q8, TAIL> x;
    x.load(d, row, at, nblk);
    const float rstd = d.rstd[row], mean = d.mean[row];
    f8 gs[1];
    if (MULTI) fold_rows<T, 1, TAIL>(gs, d.dy, d.nsrc, row, d.dy_stride, 0, tile * LANES + l, cols);
    else gs[0] = widen<T>(at.template load<T>(row_of<T>(d.dy[0], row, d.dy_stride)));
    const f8 g = gs[0];
    aw += g * x.normed(mean, rstd, at);
    ab += g;
  }
#pragma unroll
  for (int j = 0; j < 8; j++)
    if (at.mine(j)) {
      comb[0][k0][at.c - tile * C + j] = aw[j];
      comb[1][k0][at.c - tile * C + j] = ab[j];
    }
  __syncthreads();
  for (int o = threadIdx.x; o < 2 * C; o += blockDim.x) {
    const int which = o / C, c = o % C, col = tile * C + c;
    if (col >= cols) continue;
    float s = 0.0f;
    for (int k = 0; k < R; k += 4) // R is a multiple of 4
      s += (comb[which][k][c] + comb[which][k + 1][c]) + (comb[which][k + 2][c] + comb[which][k + 3][c]);
    void *out = which ? d.dbias : d.dweight;
    if (part) part[(long)slice * 2 * cols + (long)which * cols + col] = s;
    else if (out) put_grad(out, d.gdtype, d.accumulate, col, s);
  }
}

// For rows too wide to keep the sums in registers beside the row: a wave takes 512 columns.
// grid: slices (x), column tiles (y).
template <class T, bool Q8>
__global__ __launch_bounds__(256) void layernorm_cols_kernel(const ext_mpi_amd_layernorm_grad d, float *part) {
  __shared__ lanes_sums<64> comb[2];
  cols_tile<T, 64, Q8, true, WHOLE>(d, blockIdx.y, blockIdx.x, gridDim.x, part, comb);
}

// Rows without column sums, and in the workgroups behind theirs (from `blocks` on) the column sums of
// 32 columns each over all rows: the rows are read twice, but nothing waits for anything. Fewer columns
// to a workgroup, more rows at a time (256 x 2048 bf16 6.9 us against 8.6 with 64 columns).
template <class T, class W, int MODE, int NV, bool Q8, int TAIL>
__global__ __launch_bounds__(lanes<MODE>::kBlock, lanes<MODE>::kWaves) void layernorm_grad_apart_kernel(
    const ext_mpi_amd_layernorm_grad d, int blocks) {
  __shared__ lanes_sums<4> comb[2]; // one for all forms below
  if ((int)blockIdx.x < blocks) grad_rows<T, W, MODE, NV, Q8, true, TAIL, false>(d, blockIdx.x, blocks, nullptr);
  else if (TAIL == PIECES) cols_tile<T, 4, Q8, true, PIECES>(d, blockIdx.x - blocks, 0, 1, nullptr, comb);
  else if (d.nsrc == 1) cols_tile<T, 4, Q8, false, WHOLE>(d, blockIdx.x - blocks, 0, 1, nullptr, comb);
  else cols_tile<T, 4, Q8, true, WHOLE>(d, blockIdx.x - blocks, 0, 1, nullptr, comb);
}

// Rows of more than 16384 columns. Held in registers they spill: a workgroup reads its row twice, for
// the sums and for dx, the second time from the caches. The workgroups behind `blocks` as above.
template <class T, class W, bool Q8>
__global__ __launch_bounds__(512) void layernorm_grad_wide_kernel(const ext_mpi_amd_layernorm_grad d, int blocks) {
  __shared__ lanes_sums<4> comb[2];
  if ((int)blockIdx.x >= blocks) return cols_tile<T, 4, Q8, true, WHOLE>(d, blockIdx.x - blocks, 0, 1, nullptr, comb);
  const int cols = (int)d.cols, full = cols / 8, nblk = (cols + EMAC_BLOCK8 - 1) / EMAC_BLOCK8;
  const float inv = 1.0f / (float)cols;
  __shared__ float red[2][lanes<512>::kSlots][2];
  row_sum<512, 2> sum_row(red);
  for (long row = blockIdx.x; row < d.rows; row += blocks) {
    const float rstd = d.rstd[row], mean = d.mean[row];
    float s[2] = {0.0f, 0.0f}, c1, c2;
    // vector v of the row: into the sums (and y), or into dx. Each lane loads its own elements alone,
    // which dx may replace.
    const auto take = [&](auto at, bool sums, int v) {
      typedef decltype(at) slot_t;
      row8<T, Q8, slot_t::kTail> x;
      x.load(d, row, at, nblk);
      raw8<T> more;
      if (!sums && d.dsum) more = at.template load<T>(row_of<T>(d.dsum, row, d.dsum_stride));
      f8 g[1], ww = 1.0f;
      if (d.weight) ww = widen<W>(at.template load<W, true>(d.weight));
      fold_rows<T, 1, slot_t::kTail>(g, d.dy, d.nsrc, row, d.dy_stride, 0, v, cols);
      const f8 xh = x.normed(mean, rstd, at);
      if (sums) {
        if (d.y) {
          f8 y = xh * ww;
          if (d.bias) y += widen<W>(at.template load<W, true>(d.bias));
          at.template store<T>((T *)d.y + row * d.y_stride, round_to<T>(y));
        }
        at.sums(g[0] * ww, xh, s[0], s[1]);
      } else {
        f8 dx = xh * c2 + c1;
        dx += g[0] * ww * rstd;
        if (d.dsum) dx += widen<T>(more);
        at.template store<T>((T *)d.dx + row * d.dx_stride, round_to<T>(dx));
      }
    };
    const auto pass = [&](bool sums) {
      for (int v = threadIdx.x; v < full; v += 512) take(slot<WHOLE>(0, 0, v, cols, true), sums, v);
      if (cols % 8 && (int)threadIdx.x == full % 512) take(slot<PIECES>(0, 0, full, cols, true), sums, full);
    };
    if (d.dx || d.y) pass(true);
    if (!d.dx) continue;
    sum_row(s);
    c1 = -s[0] * inv * rstd;
    c2 = -s[1] * inv * rstd;
    pass(false);
  }
}

// ---- launches ----

#define EMAC_NORM_CUS 256 // compute units of the part

// The launch of a norm of `cols` columns: lanes to a row, vectors to a lane, lanes of a workgroup.
struct row_shape {
  int mode, nv, block;
};
inline row_shape row_shape_of(long cols) {
  const long v = (cols + 7) / 8; // vectors in a row
  row_shape s;
  s.mode = v <= 16 ? 16 : v <= 64 ? 64 : v <= 2048 ? 512 : 1024;
  s.nv = v <= 512 ? 1 : v <= 1024 ? 2 : v <= 1536 ? 3 : v <= 4096 ? 4 : 8;
  s.block = s.mode < 512 ? 256 : (int)((v + s.nv - 1) / s.nv + 63) / 64 * 64;
  return s;
}

// Workgroups to a CU, as few as keep enough loads in flight: 8 KB of rows of each matrix (65536 x 256
// bf16 norm: 2 to a CU, 4 KB, 35 us, 4 27 us; 65536 x 512: 2, 8 KB, 46 us, 4 50 us), and 8 waves. More
// of them cost more than they hide, the gradient (not `most`) above all: each leaves a partial row.
inline int per_cu(const row_shape &s, long cols, int dtype, bool most) {
  const long bytes = (s.mode < 512 ? 256 / s.mode : 1) * cols * (dtype == EXT_MPI_AMD_FLOAT ? 4 : 2);
  const long by_bytes = (8192 + bytes / 2) / bytes;
  const long by_waves = most ? (512 + s.block - 1) / s.block : s.block > 256 ? 1 : 512 / s.block;
  const long cap = most ? 8 : 5;
  return (int)(by_bytes > cap ? cap : by_bytes > by_waves ? by_bytes : by_waves);
}

template <class T, class W, int MODE, int NV, bool MULTI, int TAIL>
int norm_go(const ext_mpi_amd_layernorm &d, const row_shape &s, hipStream_t st) {
  constexpr int rows = lanes<MODE>::kRows;
  const long want = (d.rows + rows - 1) / rows;
  long wgs = per_cu(s, d.cols, d.dtype, true);
  if (MULTI && MODE == 512) {
    // nothing is loaded ahead: 32 KB of leaves in flight to a CU, and with one vector to a lane two
    // workgroups, as far as 16 waves go (bf16, 2 leaves: 16384 x 1024 26.2 us against 34.2 by the rule of
    // the one-leaf kernels, 8192 x 4096 49.7 against 69.5; float 8192 x 4096 112 against 125)
    const long bytes = d.nsrc * d.cols * (long)sizeof(T), fit = 1024 / s.block, least = NV == 1 ? 2 : 1;
    const long fill = (32768 + bytes - 1) / bytes > least ? (32768 + bytes - 1) / bytes : least;
    wgs = wgs > fill ? wgs : fill > fit ? fit : fill;
  }
  const long most = EMAC_NORM_CUS * wgs;
  const int grid = (int)(want < most ? want : most);
  return launch(layernorm_kernel<T, W, MODE, NV, MULTI, TAIL>, grid, s.block, st, d);
}

// Rows of 16 to 32 KB from one leaf: a workgroup of up to 16 waves with 32 bytes of the row to a lane,
// where row_shape_of gives fewer waves more of it (float, 8192 x 5120 with residual, sum and checkpoint
// 131 us against 168, 4096 x 8192 112 against 129; bf16 with float weights 4096 x 8200 27.5 against 35.8,
// 4096 x 10240 37.0 against 40.2, 4096 x 16384 49.4 against 50.1). Not in 16 bits with weights of the rows'
// type, or none: that kernel's widened rows and weights take more than the 128 registers, and it spills (bf16
// 4096 x 8200 118 us against 36.5, 4096 x 16384 227 against 49). Shorter rows are slower with more waves
// (bf16 4096 x 8192 38.3 against 25.1), and longer ones do not fit the registers (float 4096 x 12288 90
// against 79).
template <class T, class W, int NV>
constexpr bool sixteen() {
  return sizeof(T) == 4 ? NV == 2 : sizeof(W) == 4 && (NV == 3 || NV == 4);
}
inline int sixteen_block(long cols, int esize) { return (int)((cols * esize + 31) / 32 + 63) / 64 * 64; }

template <class T, class W, int MODE, int NV>
int norm_nv(const ext_mpi_amd_layernorm &d, const row_shape &s, hipStream_t st) {
  if (tail_of(d.cols, d.q) == SHIFT) return norm_go<T, W, MODE, NV, true, SHIFT>(d, s, st);
  if (d.nsrc > 1) return norm_go<T, W, MODE, NV, true, WHOLE>(d, s, st);
  if constexpr (sixteen<T, W, NV>()) {
    const int block = sixteen_block(d.cols, sizeof(T));
    return norm_go<T, W, 1024, 4 / sizeof(T), false, WHOLE>(d, row_shape{1024, 4 / (int)sizeof(T), block}, st);
  } else {
    return norm_go<T, W, MODE, NV, false, WHOLE>(d, s, st);
  }
}

template <class T, class W>
int norm_w(const ext_mpi_amd_layernorm &d, hipStream_t st) {
  row_shape s = row_shape_of(d.cols);
  const int tail = tail_of(d.cols, d.q);
  if (tail == PIECES) return norm_go<T, W, 16, 1, true, PIECES>(d, s, st);
  if (s.nv == 2 && d.rows <= EMAC_NORM_CUS) { // few rows: one vector to a lane (two of them spill at 16 waves)
    s.mode = 1024;
    s.nv = 1;
    s.block = (int)((d.cols + 7) / 8 + 63) / 64 * 64;
    return tail == SHIFT ? norm_go<T, W, 1024, 1, true, SHIFT>(d, s, st) : norm_go<T, W, 1024, 1, true, WHOLE>(d, s, st);
  }
  if (s.mode == 16) return norm_nv<T, W, 16, 1>(d, s, st);
  if (s.mode == 64) return norm_nv<T, W, 64, 1>(d, s, st);
  if (s.nv == 1) return norm_nv<T, W, 512, 1>(d, s, st);
  if (s.nv == 2) return norm_nv<T, W, 512, 2>(d, s, st);
  if (s.nv == 3) return norm_nv<T, W, 512, 3>(d, s, st);
  if (s.mode == 512) return norm_nv<T, W, 512, 4>(d, s, st);
  // wider: the forms that take any number of leaves
  if (s.nv == 4) return tail == WHOLE ? norm_go<T, W, 1024, 4, true, WHOLE>(d, s, st) : norm_go<T, W, 1024, 4, true, SHIFT>(d, s, st);
  return tail == WHOLE ? norm_go<T, W, 1024, 8, true, WHOLE>(d, s, st) : norm_go<T, W, 1024, 8, true, SHIFT>(d, s, st);
}

// the gradient's launch: `grid` workgroups take the rows, and each leaves a partial row of column sums
// (of wide rows: each slice of the rows does, in a launch of its own); or (apart) `tiles` more take the
// column sums, in a launch before the rows' where dx replaces what they read (the same sums either way)
struct grad_shape {
  row_shape r;
  int grid, tiles, parts; // parts: partial rows
  bool apart, before;
  bool wide; // two column sums beside a row's values no longer fit in registers
};
inline grad_shape grad_shape_of(const ext_mpi_amd_layernorm_grad &d) {
  grad_shape s;
  s.r = row_shape_of(d.cols);
  s.wide = s.r.mode == 1024;
  if (s.wide) s.r.block = 512;
  const bool sums = d.dweight || d.dbias;
  const long rows = s.r.mode < 512 ? 256 / s.r.mode : 1, want = (d.rows + rows - 1) / rows;
  // few rows: the second launch, which adds the partial rows, costs more than reading the rows twice
  // (bf16, one leaf: 32 x 4096 4.5 us against 6.3, 200 x 1024 5.9 against 7.5, 256 x 2048 6.9 against
  // 8.9, but 512 x 4096 13.8 against 11.5; float, 4 leaves: 64 x 1024 5.0 against 6.5, but 200 x 1024
  // 10.2 against 7.1)
  s.before = d.dx && d.dx == d.x;
  for (int i = 0; i < d.nsrc; i++) s.before = s.before || (d.dx && d.dx == d.dy[i]);
  const long twice = d.rows * d.cols * (d.nsrc + 1) * (d.dtype == EXT_MPI_AMD_FLOAT ? 4 : 2);
  const int lanes = s.r.block < 256 ? 256 : s.r.block; // more rows at a time for the column sums
  s.apart = sums && d.rows <= (d.nsrc > 1 && lanes == 256 ? 128 : 256) && twice <= 16L << 20;
  s.tiles = s.apart ? (int)((d.cols + 31) / 32) : 0;
  if (s.apart) s.r.block = lanes;
  const long most = s.apart ? 2048 : (long)EMAC_NORM_CUS * (s.wide ? 2 : per_cu(s.r, d.cols, d.dtype, false));
  s.grid = (int)(want < most ? want : most);
  if (!s.apart && !s.wide && want > 0) {
    // no more of them than the longest one's rows ask for: fewer partial rows (300 x 8192 bf16 13.3 us with
    // 150 workgroups of 2 rows, 16.0 with 256 of 1 or 2)
    const long each = (want + most - 1) / most;
    s.grid = (int)((want + each - 1) / each);
  }
  s.parts = s.grid;
  if (s.wide) { // 8 workgroups to a CU for the column sums
    const int slices = 2048 / (int)((d.cols + 511) / 512);
    s.parts = s.parts < slices ? s.parts : slices;
  }
  if (s.apart && !d.dx && !d.y) s.grid = 0;
  return s;
}

typedef void apart_kernel(const ext_mpi_amd_layernorm_grad, int);
inline int apart_go(apart_kernel *k, const ext_mpi_amd_layernorm_grad &d, const grad_shape &s, hipStream_t st) {
  if (!s.before || !s.tiles || !s.grid) return launch(k, s.grid + s.tiles, s.r.block, st, d, s.grid);
  const int rc = launch(k, s.tiles, s.r.block, st, d, 0);
  return rc ? rc : launch(k, s.grid, s.r.block, st, d, s.grid);
}

template <class T, class W, int MODE, int NV, int TAIL>
int apart_t(const ext_mpi_amd_layernorm_grad &d, const grad_shape &s, hipStream_t st) {
  if (d.q) return apart_go(layernorm_grad_apart_kernel<T, W, MODE, NV, true, TAIL>, d, s, st);
  return apart_go(layernorm_grad_apart_kernel<T, W, MODE, NV, false, TAIL>, d, s, st);
}

template <class T, class W, int MODE, int NV, bool MULTI, int TAIL>
int grad_go(const ext_mpi_amd_layernorm_grad &d, const grad_shape &s, float *part, hipStream_t st) {
  if (d.q) return launch(layernorm_grad_kernel<T, W, MODE, NV, true, MULTI, TAIL>, s.grid, s.r.block, st, d, part);
  return launch(layernorm_grad_kernel<T, W, MODE, NV, false, MULTI, TAIL>, s.grid, s.r.block, st, d, part);
}

template <class T, class W, int MODE, int NV>
int grad_nv(const ext_mpi_amd_layernorm_grad &d, const grad_shape &s, float *part, hipStream_t st) {
  if (tail_of(d.cols, d.q) == SHIFT)
    return s.apart ? apart_t<T, W, MODE, NV, SHIFT>(d, s, st) : grad_go<T, W, MODE, NV, true, SHIFT>(d, s, part, st);
  if (s.apart) return apart_t<T, W, MODE, NV, WHOLE>(d, s, st);
  if (d.nsrc > 1 || d.y) return grad_go<T, W, MODE, NV, true, WHOLE>(d, s, part, st);
  if constexpr (sizeof(T) == 4 && NV == 2) {
    // as in sixteen (float 8192 x 5120 127 us against 131); 16-bit types' two vectors and their column
    // sums would not fit the registers
    grad_shape z = s;
    z.r = row_shape{1024, 1, sixteen_block(d.cols, 4)};
    return grad_go<T, W, 1024, 1, false, WHOLE>(d, z, part, st);
  } else {
    return grad_go<T, W, MODE, NV, false, WHOLE>(d, s, part, st);
  }
}

template <class T, class W>
int grad_w(const ext_mpi_amd_layernorm_grad &d, const grad_shape &s, float *part, hipStream_t st) {
  const int tail = tail_of(d.cols, d.q);
  if (tail == PIECES)
    return s.apart ? apart_t<T, W, 16, 1, PIECES>(d, s, st) : grad_go<T, W, 16, 1, true, PIECES>(d, s, part, st);
  if (s.wide) { // the column sums, if not apart, have a launch of their own before this one
    if (d.q) return apart_go(layernorm_grad_wide_kernel<T, W, true>, d, s, st);
    return apart_go(layernorm_grad_wide_kernel<T, W, false>, d, s, st);
  }
  if (s.r.mode == 16) return grad_nv<T, W, 16, 1>(d, s, part, st);
  if (s.r.mode == 64) return grad_nv<T, W, 64, 1>(d, s, part, st);
  if (s.r.nv == 1) return grad_nv<T, W, 512, 1>(d, s, part, st);
  if (s.r.nv == 2) return grad_nv<T, W, 512, 2>(d, s, part, st);
  if (s.r.nv == 3) return grad_nv<T, W, 512, 3>(d, s, part, st);
  return grad_nv<T, W, 512, 4>(d, s, part, st);
}

template <class T>
int grad_cols(const ext_mpi_amd_layernorm_grad &d, int slices, float *part, hipStream_t st) {
  const dim3 grid(slices, (unsigned)((d.cols + 511) / 512));
  if (d.q) return launch(layernorm_cols_kernel<T, true>, grid, 256, st, d, part);
  return launch(layernorm_cols_kernel<T, false>, grid, 256, st, d, part);
}

// whether weights of their own type need their own kernels
inline bool own_weights(int dtype, int wdtype, const void *w, const void *b) { return (w || b) && wdtype != dtype; }

} // namespace emac_rows
#endif
