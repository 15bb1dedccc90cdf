// norm_grad_bf16.hip -- layer norm's gradient, bf16 rows and weights of the same type (one translation unit per
// combination, so that they compile in parallel). See norm_kernel.hpp.
#include "norm_kernel.hpp"

extern "C" int emac_grad_launch_bf16(const ext_mpi_amd_layernorm_grad *d, float *part, void *st) {
  return emac_rows::grad_w<emac_rows::bf16, emac_rows::bf16>(*d, emac_rows::grad_shape_of(*d), part, static_cast<hipStream_t>(st));
}
