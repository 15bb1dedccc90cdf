// norm_grad_f16.hip -- layer norm's gradient, half rows and weights of the same type (one translation unit per
// combination, so that they compile in parallel). See norm_kernel.hpp.
#include "norm_kernel.hpp"

extern "C" int emac_grad_launch_f16(const ext_mpi_amd_layernorm_grad *d, float *part, void *st) {
  return emac_rows::grad_w<emac_rows::half, emac_rows::half>(*d, emac_rows::grad_shape_of(*d), part, static_cast<hipStream_t>(st));
}
