// norm_f32.hip -- float instantiations of the layer norm kernels (one translation unit per element
// type so that they compile in parallel). See norm_kernel.hpp.
#include "norm_kernel.hpp"

extern "C" int emac_norm_launch_f32(const ext_mpi_amd_layernorm *d, void *st) {
  return emac_rows::norm_launch<float>(*d, static_cast<hipStream_t>(st));
}

extern "C" int emac_grad_launch_f32(const ext_mpi_amd_layernorm_grad *d, float *part, void *st) {
  return emac_rows::grad_launch<float>(*d, emac_rows::grad_shape_of(*d), part, static_cast<hipStream_t>(st));
}
