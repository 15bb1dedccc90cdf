// norm_f16_w32.hip -- layer norm, half rows and float weights (one translation unit per
// combination, so that they compile in parallel). See norm_kernel.hpp.
#include "norm_kernel.hpp"

extern "C" int emac_norm_launch_f16_w32(const ext_mpi_amd_layernorm *d, void *st) {
  return emac_rows::norm_w<emac_rows::half, float>(*d, static_cast<hipStream_t>(st));
}
