// norm_grad_f16_w32.hip -- layer norm's gradient, half rows and float weights (one translation unit per
// combination, so that they compile in parallel). See norm_kernel.hpp.
#include "norm_kernel.hpp"

extern "C" int emac_grad_launch_f16_w32(const ext_mpi_amd_layernorm_grad *d, float *part, void *st) {
  return emac_rows::grad_w<emac_rows::half, float>(*d, emac_rows::grad_shape_of(*d), part, static_cast<hipStream_t>(st));
}
