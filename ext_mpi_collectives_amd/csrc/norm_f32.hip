// norm_f32.hip -- layer norm, float rows and weights of the same type (one translation unit per
// combination, so that they compile in parallel). See norm_kernel.hpp.
#include "norm_kernel.hpp"

extern "C" int emac_norm_launch_f32(const ext_mpi_amd_layernorm *d, void *st) {
  return emac_rows::norm_w<float, float>(*d, static_cast<hipStream_t>(st));
}
