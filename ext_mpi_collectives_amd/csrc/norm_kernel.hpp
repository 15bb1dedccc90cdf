// norm_kernel.hpp -- layer norm over the folded partials of the ranks, and its gradient.
//
// Forward: a row lives in the registers of TPR lanes (NV vectors of 8 elements each) from the
// leaves' loads to y's stores, so each input is read once and each output written once; the mean
// and then the sum of squared differences are two reductions over those registers (never E[x^2] -
// mean^2). x is rounded to its type before its statistics, so a gradient that reads x (or the
// checkpoint, taken from the same registers) sees the values that were normalised.
// Gradient: the same layout; each lane owns the same columns in every row its workgroup takes, so
// the two column sums (dweight, dbias) stay in its registers over all of them, and leave as one
// partial row per workgroup, which a second kernel adds in order: no atomics, the same bits every
// time. Both directions are bound by HBM at large sizes and by launch latency at small ones.
#ifndef EMAC_NORM_KERNEL_HPP_
#define EMAC_NORM_KERNEL_HPP_

#include "rows_kernel.hpp"

namespace emac_rows {

// the sum over a row's TPR lanes; `red` holds two slots per wave, used in turn (`turn` flips with
// each call), so one barrier separates a slot's last read from its next write
template <int TPR, int BLOCK, int NS>
struct row_sum {
  static constexpr int kWaves = BLOCK / 64, kPer = TPR / 64;
  __device__ static void run(float (&v)[NS], float (*red)[kWaves][NS], int &turn) {
    if constexpr (TPR == 16) {
#pragma unroll
      for (int k = 0; k < NS; k++) v[k] = sum16(v[k]);
      return;
    }
#pragma unroll
    for (int k = 0; k < NS; k++) v[k] = sum64(v[k]);
    if constexpr (TPR > 64) {
      const int wave = threadIdx.x / 64, first = wave / kPer * kPer;
      if (threadIdx.x % 64 == 0) {
#pragma unroll
        for (int k = 0; k < NS; k++) red[turn][wave][k] = v[k];
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < NS; k++) {
        float s = red[turn][first][k];
#pragma unroll
        for (int w = 1; w < kPer; w++) s += red[turn][first + w][k];
        v[k] = s;
      }
      turn ^= 1;
    }
  }
};

// ((leaf 0 + leaf 1) + ...) of 8 elements in 32 bits; four leaves' loads in flight at a time
template <class T>
__device__ inline f8 fold8(const void *const *src, int nsrc, long at, long n) {
  f8 s = {};
  for (int t0 = 0; t0 < nsrc; t0 += 4) {
    v8<T> raw[4];
#pragma unroll
    for (int k = 0; k < 4; k++)
      if (t0 + k < nsrc) raw[k] = load8((const T *)src[t0 + k] + at, n);
#pragma unroll
    for (int k = 0; k < 4; k++)
      if (t0 + k < nsrc) s = t0 + k ? s + widen<T>(raw[k]) : widen<T>(raw[k]);
  }
  return s;
}

template <class T, class W, int NV, int TPR, int BLOCK, bool MULTI>
__global__ __launch_bounds__(BLOCK) void layernorm_kernel(const ext_mpi_amd_layernorm d) {
  constexpr int RPB = BLOCK / TPR;
  __shared__ float red[2][BLOCK / 64][1];
  int turn = 0;
  const int l = threadIdx.x % TPR;
  int sub = threadIdx.x / TPR;
  if constexpr (TPR >= 64) sub = __builtin_amdgcn_readfirstlane(sub);
  const int cols = (int)d.cols;
  const int nblk = (cols + EMAC_BLOCK8 - 1) / EMAC_BLOCK8;
  for (long r0 = (long)blockIdx.x * RPB; r0 < d.rows; r0 += (long)gridDim.x * RPB) {
    const long row = r0 + sub;
    const bool live = row < d.rows;
    v8<T> x[NV];
    float s[1] = {0.0f};
#pragma unroll
    for (int i = 0; i < NV; i++) {
      const int c = (l + i * TPR) * 8;
      const long n = live ? cols - c : 0;
      if (n > 0) {
        if (!MULTI && !d.residual) {
          x[i] = load8((const T *)d.src[0] + row * d.src_stride + c, n);
        } else {
          f8 f;
          v8<T> res;
          if (d.residual) res = load8((const T *)d.residual + row * d.residual_stride + c, n);
          if constexpr (MULTI)
            f = fold8<T>(d.src, d.nsrc, row * d.src_stride + c, n);
          else
            f = widen<T>(load8((const T *)d.src[0] + row * d.src_stride + c, n));
          if (d.residual) f += widen<T>(res);
          x[i] = round_to<T>(f);
        }
      } else {
        x[i] = (v8<T>)(T)0;
      }
      const f8 f = widen<T>(x[i]);
#pragma unroll
      for (int j = 0; j < 8; j++) s[0] += f[j];
    }
#pragma unroll
    for (int i = 0; i < NV; i++) {
      const int c = (l + i * TPR) * 8;
      const long n = live ? cols - c : 0;
      if (d.sum && n > 0) store8((T *)d.sum + row * d.sum_stride + c, x[i], n);
      if (d.q) { // every lane of a block takes part; lanes past the row hold zeros
        const block8 b = quantise<T>(x[i]);
        if (n > 0) {
          store8q(d.q + row * d.q_stride + c, b.q, n);
          if (c % EMAC_BLOCK8 == 0) d.scale[row * nblk + c / EMAC_BLOCK8] = b.scale;
        }
      }
    }
    if (!d.y && !d.mean && !d.rstd) continue;
    row_sum<TPR, BLOCK, 1>::run(s, red, turn);
    const float mean = s[0] / (float)cols;
    s[0] = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; i++) {
      const int c = (l + i * TPR) * 8, n = cols - c;
      const f8 f = widen<T>(x[i]);
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const float t = f[j] - mean;
        s[0] += j < n ? t * t : 0.0f;
      }
    }
    row_sum<TPR, BLOCK, 1>::run(s, red, turn);
    const float rstd = 1.0f / sqrtf(s[0] / (float)cols + (float)d.eps);
    if (l == 0 && live) {
      if (d.mean) d.mean[row] = mean;
      if (d.rstd) d.rstd[row] = rstd;
    }
    if (!d.y) continue;
#pragma unroll
    for (int i = 0; i < NV; i++) {
      const int c = (l + i * TPR) * 8;
      const long n = live ? cols - c : 0;
      if (n <= 0) continue;
      f8 f = (widen<T>(x[i]) - mean) * rstd;
      if (d.weight) f *= widen<W>(load8((const W *)d.weight + c, n));
      if (d.bias) f += widen<W>(load8((const W *)d.bias + c, n));
      store8((T *)d.y + row * d.y_stride + c, round_to<T>(f), n);
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

// a workgroup's column sums of 8 columns: into its partial row, or (one workgroup) the gradients
__device__ inline void put_cols(const ext_mpi_amd_layernorm_grad &d, float *part, int c, f8 w, f8 b) {
  const int cols = (int)d.cols, n = cols - c;
  if (n <= 0) return;
  if (part) {
    float *p = part + (long)blockIdx.x * 2 * cols;
    store8(p + c, w, n);
    store8(p + cols + c, b, n);
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; j++)
    if (j < n) {
      if (d.dweight) put_grad(d.dweight, d.gdtype, d.accumulate, c + j, w[j]);
      if (d.dbias) put_grad(d.dbias, d.gdtype, d.accumulate, c + j, b[j]);
    }
}

// xh = (x - mean) * rstd of 8 elements, from x or its checkpoint
template <class T, bool Q8>
__device__ inline f8 load_x(const ext_mpi_amd_layernorm_grad &d, long row, int c, long n, int nblk) {
  if constexpr (Q8)
    return restore(load8q(d.q + row * d.q_stride + c, n), d.scale[row * nblk + c / EMAC_BLOCK8]);
  else
    return widen<T>(load8((const T *)d.x + row * d.x_stride + c, n));
}
template <class T, bool MULTI>
__device__ inline f8 load_g(const ext_mpi_amd_layernorm_grad &d, long row, int c, long n) {
  if constexpr (MULTI)
    return fold8<T>(d.dy, d.nsrc, row * d.dy_stride + c, n);
  else
    return widen<T>(load8((const T *)d.dy[0] + row * d.dy_stride + c, n));
}

template <class T, class W, int NV, int TPR, int BLOCK, bool Q8, bool MULTI, bool ACC>
__global__ __launch_bounds__(BLOCK) void layernorm_grad_kernel(const ext_mpi_amd_layernorm_grad d, float *part) {
  constexpr int RPB = BLOCK / TPR;
  __shared__ float red[2][BLOCK / 64][2];
  int turn = 0;
  const int l = threadIdx.x % TPR;
  int sub = threadIdx.x / TPR;
  if constexpr (TPR >= 64) sub = __builtin_amdgcn_readfirstlane(sub);
  const int cols = (int)d.cols;
  const int nblk = (cols + EMAC_BLOCK8 - 1) / EMAC_BLOCK8;
  f8 aw[ACC ? NV : 1] = {}, ab[ACC ? NV : 1] = {};
  for (long r0 = (long)blockIdx.x * RPB; r0 < d.rows; r0 += (long)gridDim.x * RPB) {
    const long row = r0 + sub;
    const bool live = row < d.rows;
    const float mean = live ? d.mean[row] : 0.0f, rstd = live ? d.rstd[row] : 0.0f;
    f8 g[NV], xh[NV]; // g w after the sums
    float s[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < NV; i++) {
      const int c = (l + i * TPR) * 8;
      const long n = live ? cols - c : 0;
      if (n > 0) {
        g[i] = load_g<T, MULTI>(d, row, c, n);
        xh[i] = (load_x<T, Q8>(d, row, c, n, nblk) - mean) * rstd;
      } else {
        g[i] = xh[i] = (f8)0.0f;
      }
    }
#pragma unroll
    for (int i = 0; i < NV; i++) {
      const int c = (l + i * TPR) * 8;
      const long n = live ? cols - c : 0;
      if (n <= 0) continue;
      if (ACC) {
        aw[ACC ? i : 0] += g[i] * xh[i];
        ab[ACC ? i : 0] += g[i];
      }
      f8 w = (f8)1.0f;
      if (d.weight) w = widen<W>(load8((const W *)d.weight + c, n));
      if (d.y) {
        f8 y = xh[i] * w;
        if (d.bias) y += widen<W>(load8((const W *)d.bias + c, n));
        store8((T *)d.y + row * d.y_stride + c, round_to<T>(y), n);
      }
      g[i] *= w;
#pragma unroll
      for (int j = 0; j < 8; j++) {
        s[0] += j < n ? g[i][j] : 0.0f;
        s[1] += j < n ? g[i][j] * xh[i][j] : 0.0f;
      }
    }
    if (!d.dx) continue;
    row_sum<TPR, BLOCK, 2>::run(s, red, turn);
    const float c1 = s[0] / (float)cols, c2 = s[1] / (float)cols;
#pragma unroll
    for (int i = 0; i < NV; i++) {
      const int c = (l + i * TPR) * 8;
      const long n = live ? cols - c : 0;
      if (n <= 0) continue;
      f8 dx = rstd * (g[i] - c1 - xh[i] * c2);
      if (d.dsum) dx += widen<T>(load8((const T *)d.dsum + row * d.dsum_stride + c, n));
      store8((T *)d.dx + row * d.dx_stride + c, round_to<T>(dx), n);
    }
  }
  if constexpr (ACC) {
    if (!d.dweight && !d.dbias) return;
    if constexpr (RPB > 1) { // the rows of a workgroup taken side by side, added in order
      __shared__ f8 comb[2][TPR * NV];
      for (int k = 1; k < RPB; k++) {
        __syncthreads();
        if (sub == k) {
#pragma unroll
          for (int i = 0; i < NV; i++) {
            comb[0][l + i * TPR] = aw[i];
            comb[1][l + i * TPR] = ab[i];
          }
        }
        __syncthreads();
        if (sub == 0) {
#pragma unroll
          for (int i = 0; i < NV; i++) {
            aw[i] += comb[0][l + i * TPR];
            ab[i] += comb[1][l + i * TPR];
          }
        }
      }
      if (sub) return;
    }
#pragma unroll
    for (int i = 0; i < NV; i++) put_cols(d, part, (l + i * TPR) * 8, aw[i], ab[i]);
  }
}

// The column sums alone, for rows too wide to keep them in registers beside the row: a wave takes
// 512 columns of every fourth of its slice's rows. grid: slices (x), column tiles (y).
template <class T, bool Q8, bool MULTI>
__global__ __launch_bounds__(256) void layernorm_cols_kernel(const ext_mpi_amd_layernorm_grad d, float *part) {
  __shared__ f8 comb[2][4][64];
  const int l = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int cols = (int)d.cols, c = ((int)blockIdx.y * 64 + l) * 8;
  const int nblk = (cols + EMAC_BLOCK8 - 1) / EMAC_BLOCK8;
  f8 aw = {}, ab = {};
  if (c < cols)
    for (long row = (long)blockIdx.x * 4 + wave; row < d.rows; row += (long)gridDim.x * 4) {
      const f8 g = load_g<T, MULTI>(d, row, c, cols - c);
      const f8 xh = (load_x<T, Q8>(d, row, c, cols - c, nblk) - d.mean[row]) * d.rstd[row];
      aw += g * xh;
      ab += g;
    }
  comb[0][wave][l] = aw;
  comb[1][wave][l] = ab;
  __syncthreads();
  if (wave) return;
  for (int k = 1; k < 4; k++) {
    aw += comb[0][k][l];
    ab += comb[1][k][l];
  }
  put_cols(d, part, c, aw, ab);
}

// ---- launches ----

#define EMAC_NORM_CUS 256 // compute units of the part

template <class T, class W, int NV, int TPR, int BLOCK>
int norm_go(const ext_mpi_amd_layernorm &d, hipStream_t st) {
  const long want = (d.rows + BLOCK / TPR - 1) / (BLOCK / TPR), most = 2048L * EMAC_NORM_CUS / BLOCK * 2;
  const int grid = (int)(want < most ? want : most);
  if (d.nsrc > 1)
    layernorm_kernel<T, W, NV, TPR, BLOCK, true><<<grid, BLOCK, 0, st>>>(d);
  else
    layernorm_kernel<T, W, NV, TPR, BLOCK, false><<<grid, BLOCK, 0, st>>>(d);
  return launched();
}

template <class T, class W>
int norm_w(const ext_mpi_amd_layernorm &d, hipStream_t st) {
  const long v = (d.cols + 7) / 8; // vectors in a row
  const bool few = d.rows < 2 * EMAC_NORM_CUS;
  if (v <= 16) return norm_go<T, W, 1, 16, 256>(d, st);
  if (v <= 64) return norm_go<T, W, 1, 64, 256>(d, st);
  if (v <= 128 && !few) return norm_go<T, W, 2, 64, 256>(d, st);
  if (v <= 256) return norm_go<T, W, 1, 256, 256>(d, st);
  if (v <= 512 && !few) return norm_go<T, W, 2, 256, 256>(d, st);
  if (v <= 1024 && !few) return norm_go<T, W, 4, 256, 256>(d, st);
  if (v <= 1024) return norm_go<T, W, 1, 1024, 1024>(d, st);
  if (v <= 2048) return norm_go<T, W, 2, 1024, 1024>(d, st);
  if (v <= 4096) return norm_go<T, W, 4, 1024, 1024>(d, st);
  return norm_go<T, W, 8, 1024, 1024>(d, st);
}

template <class T>
int norm_launch(const ext_mpi_amd_layernorm &d, hipStream_t st) {
  if (d.wdtype == d.dtype || !(d.weight || d.bias)) return norm_w<T, T>(d, st);
  return norm_w<T, float>(d, st);
}

// workgroups of the gradient, each of which leaves one partial row
struct grad_shape {
  int tpr, nv, block, grid;
  bool wide;
};
inline grad_shape grad_shape_of(const ext_mpi_amd_layernorm_grad &d) {
  const long v = (d.cols + 7) / 8;
  grad_shape s = {1024, 2, 1024, 0, false};
  if (v <= 16) s = {16, 1, 256, 0, false};
  else if (v <= 64) s = {64, 1, 256, 0, false};
  else if (v <= 128) s = {64, 2, 256, 0, false};
  else if (v <= 256) s = {256, 1, 256, 0, false};
  else if (v <= 512) s = {512, 1, 512, 0, false};
  else if (v <= 1024) s = {1024, 1, 1024, 0, false};
  else if (v > 2048) s = {1024, v <= 4096 ? 4 : 8, 1024, 0, true};
  const long want = (d.rows + s.block / s.tpr - 1) / (s.block / s.tpr), most = 1024L * EMAC_NORM_CUS / s.block;
  s.grid = (int)(want < most ? want : most);
  return s;
}

template <class T, class W, int NV, int TPR, int BLOCK, bool ACC>
int grad_go(const ext_mpi_amd_layernorm_grad &d, int grid, float *part, hipStream_t st) {
  if (d.q && d.nsrc > 1)
    layernorm_grad_kernel<T, W, NV, TPR, BLOCK, true, true, ACC><<<grid, BLOCK, 0, st>>>(d, part);
  else if (d.q)
    layernorm_grad_kernel<T, W, NV, TPR, BLOCK, true, false, ACC><<<grid, BLOCK, 0, st>>>(d, part);
  else if (d.nsrc > 1)
    layernorm_grad_kernel<T, W, NV, TPR, BLOCK, false, true, ACC><<<grid, BLOCK, 0, st>>>(d, part);
  else
    layernorm_grad_kernel<T, W, NV, TPR, BLOCK, false, false, ACC><<<grid, BLOCK, 0, st>>>(d, part);
  return launched();
}

template <class T, class W>
int grad_w(const ext_mpi_amd_layernorm_grad &d, const grad_shape &s, float *part, hipStream_t st) {
  if (s.wide) return s.nv == 4 ? grad_go<T, W, 4, 1024, 1024, false>(d, s.grid, part, st)
                               : grad_go<T, W, 8, 1024, 1024, false>(d, s.grid, part, st);
  if (s.tpr == 16) return grad_go<T, W, 1, 16, 256, true>(d, s.grid, part, st);
  if (s.tpr == 64) return s.nv == 1 ? grad_go<T, W, 1, 64, 256, true>(d, s.grid, part, st)
                                    : grad_go<T, W, 2, 64, 256, true>(d, s.grid, part, st);
  if (s.tpr == 256) return grad_go<T, W, 1, 256, 256, true>(d, s.grid, part, st);
  if (s.tpr == 512) return grad_go<T, W, 1, 512, 512, true>(d, s.grid, part, st);
  return s.nv == 1 ? grad_go<T, W, 1, 1024, 1024, true>(d, s.grid, part, st)
                   : grad_go<T, W, 2, 1024, 1024, true>(d, s.grid, part, st);
}

template <class T>
int grad_cols(const ext_mpi_amd_layernorm_grad &d, int slices, float *part, hipStream_t st) {
  const dim3 grid(slices, (unsigned)((d.cols + 511) / 512));
  if (d.q && d.nsrc > 1)
    layernorm_cols_kernel<T, true, true><<<grid, 256, 0, st>>>(d, part);
  else if (d.q)
    layernorm_cols_kernel<T, true, false><<<grid, 256, 0, st>>>(d, part);
  else if (d.nsrc > 1)
    layernorm_cols_kernel<T, false, true><<<grid, 256, 0, st>>>(d, part);
  else
    layernorm_cols_kernel<T, false, false><<<grid, 256, 0, st>>>(d, part);
  return launched();
}

template <class T>
int grad_launch(const ext_mpi_amd_layernorm_grad &d, const grad_shape &s, float *part, hipStream_t st) {
  int rc;
  if (s.wide) {
    // the column sums first: dx may overwrite what they read
    if ((d.dweight || d.dbias) && (rc = grad_cols<T>(d, s.grid, part, st))) return rc;
    if (!d.dx && !d.y) return 0;
  }
  if (d.wdtype == d.dtype || !(d.weight || d.bias)) return grad_w<T, T>(d, s, part, st);
  return grad_w<T, float>(d, s, part, st);
}

} // namespace emac_rows
#endif
