/*
 * rows.h -- internal C ABI between the row operators' host code (engine_rows.c) and their kernels
 * (norm_kernel.hpp, act8.hip). The descriptors are the public ones (include/ext_mpi_amd.h), checked
 * and with every stride filled in by engine_rows.c.
 */
#ifndef EMAC_ROWS_H_
#define EMAC_ROWS_H_

#include "ext_mpi_amd.h"
#include "plan.h"

#ifdef __cplusplus
extern "C" {
#endif

#define EMAC_BLOCK8 EXT_MPI_AMD_BLOCK8

/* erfcx(z) / 2 for z = |a| / sqrt 2 as a polynomial of degree 8 in t = 1 / (1 + 0.4348731 z) = 1 / (1 + AT |a|)
   without a constant term, the highest power first; fitted for the least relative error on 0 <= z <= 12 */
#define EMAC_GELU_TAIL_AT 0.30750170f
#define EMAC_GELU_TAIL                                                                                      \
  {0.036300003528594971f, -0.14733710885047913f, 0.1701858937740326f, -0.026046559214591980f,             \
   0.1153081208467484f,   0.1056915521621704f,   0.1232480555772781f, 0.1226501166820526f}

/* layer norm, forward: one launch */
int emac_gpu_layernorm(const ext_mpi_amd_layernorm *d, void *stream);
/* its gradient: one to three launches; `part` is the workspace of emac_gpu_layernorm_grad_ws bytes */
size_t emac_gpu_layernorm_grad_ws(const ext_mpi_amd_layernorm_grad *d);
int emac_gpu_layernorm_grad(const ext_mpi_amd_layernorm_grad *d, float *part, void *stream);
/* activations and checkpoints: one launch each */
int emac_gpu_act(const ext_mpi_amd_act *d, void *stream); /* kind EMAC_SAVE8: checkpoints alone */
int emac_gpu_act_grad(const ext_mpi_amd_act_grad *d, void *stream);
#define EMAC_SAVE8 (-1)
int emac_gpu_restore8(long rows, long cols, int dtype, const signed char *q, long q_stride, const float *scale, void *x,
                      long x_stride, void *stream);

#ifdef __cplusplus
}
#endif
#endif
