// norm_grad_f32.hip -- layer norm's gradient, float rows and weights of the same type (one translation unit per
// combination, so that they compile in parallel). See norm_kernel.hpp.
#include "norm_kernel.hpp"

extern "C" int emac_grad_launch_f32(const ext_mpi_amd_layernorm_grad *d, float *part, void *st) {
  return emac_rows::grad_w<float, float>(*d, emac_rows::grad_shape_of(*d), part, static_cast<hipStream_t>(st));
}
