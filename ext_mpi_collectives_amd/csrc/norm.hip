// norm.hip -- layer norm's dispatch by element type, and the end of its gradient's column sums.
#include "norm_kernel.hpp"

using namespace emac_rows;

namespace {

// The partial rows (one per workgroup of the gradient, dweight's columns then dbias's) added in a
// fixed order: 32 threads of a workgroup take every 32nd partial row of one column, 8 of them in
// flight, and their sums are added in order. 32 neighbouring columns make a 128-byte access.
__global__ __launch_bounds__(1024) void colsum_kernel(const float *part, int nparts, long cols, void *dweight, void *dbias,
                                                      int gdtype, int accumulate) {
  __shared__ float red[32][33];
  const int col = threadIdx.x % 32, slice = threadIdx.x / 32;
  const long c = (long)blockIdx.x * 32 + col;
  void *out = blockIdx.y ? dbias : dweight;
  if (!out) return;
  float s = 0.0f;
  if (c < cols) {
    const float *p = part + (long)blockIdx.y * cols + c;
    for (int g0 = slice; g0 < nparts; g0 += 256) {
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; k++) v[k] = g0 + 32 * k < nparts ? p[(long)(g0 + 32 * k) * 2 * cols] : 0.0f;
#pragma unroll
      for (int k = 0; k < 8; k++) s += v[k];
    }
  }
  red[slice][col] = s;
  __syncthreads();
  if (slice || c >= cols) return;
  for (int k = 1; k < 32; k++) s += red[k][col];
  put_grad(out, gdtype, accumulate, c, s);
}

} // namespace

extern "C" {

#define EMAC_DECL(n)                                                   \
  int emac_norm_launch_##n(const ext_mpi_amd_layernorm *d, void *st); \
  int emac_grad_launch_##n(const ext_mpi_amd_layernorm_grad *d, float *part, void *st);
EMAC_DECL(f32)
EMAC_DECL(bf16)
EMAC_DECL(bf16_w32)
EMAC_DECL(f16)
EMAC_DECL(f16_w32)
#undef EMAC_DECL

int emac_gpu_layernorm(const ext_mpi_amd_layernorm *d, void *stream) {
  const bool w32 = own_weights(d->dtype, d->wdtype, d->weight, d->bias);
  if (d->rows <= 0) return 0;
  switch (d->dtype) {
  case EXT_MPI_AMD_FLOAT: return emac_norm_launch_f32(d, stream);
  case EXT_MPI_AMD_BF16: return w32 ? emac_norm_launch_bf16_w32(d, stream) : emac_norm_launch_bf16(d, stream);
  case EXT_MPI_AMD_HALF: return w32 ? emac_norm_launch_f16_w32(d, stream) : emac_norm_launch_f16(d, stream);
  }
  return EMAC_ERR_UNSUPPORTED;
}

size_t emac_gpu_layernorm_grad_ws(const ext_mpi_amd_layernorm_grad *d) {
  const grad_shape s = grad_shape_of(*d);
  if (s.apart || !(d->dweight || d->dbias)) return 0;
  return sizeof(float) * 2 * (size_t)d->cols * (size_t)s.parts;
}

int emac_gpu_layernorm_grad(const ext_mpi_amd_layernorm_grad *d, float *part, void *stream) {
  const grad_shape s = grad_shape_of(*d);
  const bool w32 = own_weights(d->dtype, d->wdtype, d->weight, d->bias), sums = d->dweight || d->dbias;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  int rc = 0;
  if (d->rows > 0) {
    if (s.wide && sums && !s.apart) { // the column sums first: dx may overwrite what they read
      switch (d->dtype) {
      case EXT_MPI_AMD_FLOAT: rc = grad_cols<float>(*d, s.parts, part, st); break;
      case EXT_MPI_AMD_BF16: rc = grad_cols<bf16>(*d, s.parts, part, st); break;
      case EXT_MPI_AMD_HALF: rc = grad_cols<half>(*d, s.parts, part, st); break;
      }
      if (rc) return rc;
    }
    if (!s.wide || s.apart || d->dx || d->y) {
      switch (d->dtype) {
      case EXT_MPI_AMD_FLOAT: rc = emac_grad_launch_f32(d, part, stream); break;
      case EXT_MPI_AMD_BF16: rc = w32 ? emac_grad_launch_bf16_w32(d, part, stream) : emac_grad_launch_bf16(d, part, stream); break;
      case EXT_MPI_AMD_HALF: rc = w32 ? emac_grad_launch_f16_w32(d, part, stream) : emac_grad_launch_f16(d, part, stream); break;
      default: rc = EMAC_ERR_UNSUPPORTED;
      }
    }
    if (rc || !part) return rc; // no workspace: no column sums, or the apart form wrote them
  }
  if (!sums) return 0;
  // no rows: the sums are zeros
  return launch(colsum_kernel, dim3((unsigned)((d->cols + 31) / 32), 2), 1024, st, part, d->rows > 0 ? s.parts : 0, d->cols,
                d->dweight, d->dbias, d->gdtype, d->accumulate);
}

} // extern "C"
