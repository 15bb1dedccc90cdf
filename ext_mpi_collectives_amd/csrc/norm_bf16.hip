// norm_bf16.hip -- layer norm, bf16 rows and weights of the same type (one translation unit per
// combination, so that they compile in parallel). See norm_kernel.hpp.
#include "norm_kernel.hpp"

extern "C" int emac_norm_launch_bf16(const ext_mpi_amd_layernorm *d, void *st) {
  return emac_rows::norm_w<emac_rows::bf16, emac_rows::bf16>(*d, static_cast<hipStream_t>(st));
}
