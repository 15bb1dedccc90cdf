// norm.hip -- layer norm's dispatch by element type, and the end of its gradient's column sums.
#include "norm_kernel.hpp"

namespace {

using namespace emac_rows;

// The partial rows (one per workgroup of the gradient, dweight's columns then dbias's) added in a
// fixed order: 8 threads of a workgroup take every 8th partial row of one column, 4 of them in
// flight, and their sums are added in order. 32 neighbouring columns make a 128-byte access.
__global__ __launch_bounds__(256) void colsum_kernel(const float *part, int nparts, long cols, void *dweight, void *dbias,
                                                     int gdtype, int accumulate) {
  __shared__ float red[8][32];
  const int col = threadIdx.x % 32, slice = threadIdx.x / 32;
  const long c = (long)blockIdx.x * 32 + col;
  void *out = blockIdx.y ? dbias : dweight;
  if (!out) return;
  float s = 0.0f;
  if (c < cols) {
    const float *p = part + (long)blockIdx.y * cols + c;
    int g = slice;
    for (; g + 24 < nparts; g += 32) {
      const float a = p[(long)g * 2 * cols], b = p[(long)(g + 8) * 2 * cols];
      const float e = p[(long)(g + 16) * 2 * cols], f = p[(long)(g + 24) * 2 * cols];
      s += (a + b) + (e + f);
    }
    for (; g < nparts; g += 8) s += p[(long)g * 2 * cols];
  }
  red[slice][col] = s;
  __syncthreads();
  if (slice || c >= cols) return;
  for (int k = 1; k < 8; k++) s += red[k][col];
  put_grad(out, gdtype, accumulate, c, s);
}

} // namespace

extern "C" {

#define EMAC_DECL(n)                                                   \
  int emac_norm_launch_##n(const ext_mpi_amd_layernorm *d, void *st); \
  int emac_grad_launch_##n(const ext_mpi_amd_layernorm_grad *d, float *part, void *st);
EMAC_DECL(f32)
EMAC_DECL(bf16)
EMAC_DECL(f16)
#undef EMAC_DECL

int emac_gpu_layernorm(const ext_mpi_amd_layernorm *d, void *stream) {
  if (d->rows <= 0) return 0;
  switch (d->dtype) {
  case EXT_MPI_AMD_FLOAT: return emac_norm_launch_f32(d, stream);
  case EXT_MPI_AMD_BF16: return emac_norm_launch_bf16(d, stream);
  case EXT_MPI_AMD_HALF: return emac_norm_launch_f16(d, stream);
  }
  return EMAC_ERR_UNSUPPORTED;
}

size_t emac_gpu_layernorm_grad_ws(const ext_mpi_amd_layernorm_grad *d) {
  const emac_rows::grad_shape s = emac_rows::grad_shape_of(*d);
  if (s.grid <= 1 || !(d->dweight || d->dbias)) return 0;
  return sizeof(float) * 2 * (size_t)d->cols * (size_t)s.grid;
}

int emac_gpu_layernorm_grad(const ext_mpi_amd_layernorm_grad *d, float *part, void *stream) {
  const emac_rows::grad_shape s = emac_rows::grad_shape_of(*d);
  int rc = EMAC_ERR_UNSUPPORTED;
  if (d->rows > 0) {
    switch (d->dtype) {
    case EXT_MPI_AMD_FLOAT: rc = emac_grad_launch_f32(d, part, stream); break;
    case EXT_MPI_AMD_BF16: rc = emac_grad_launch_bf16(d, part, stream); break;
    case EXT_MPI_AMD_HALF: rc = emac_grad_launch_f16(d, part, stream); break;
    }
    if (rc || !part) return rc; // no workspace: no column sums, or one workgroup wrote them
  }
  if (!(d->dweight || d->dbias)) return 0;
  // no rows: the sums are zeros
  colsum_kernel<<<dim3((unsigned)((d->cols + 31) / 32), 2), 256, 0, static_cast<hipStream_t>(stream)>>>(
      part, d->rows > 0 ? s.grid : 0, d->cols, d->dweight, d->dbias, d->gdtype, d->accumulate);
  return launched();
}

} // extern "C"
