/* The row operators' host code over a runtime that only keeps books: two devices, one current, memory whose
 * device is its address' first digit, streams that say which device was current when they were used. Built by
 * tests/test_rows_cpu.py from the engine's own sources (what is not called here stays unresolved). */
#include <stdio.h>
#include <stdlib.h>

#include "engine_int.h"
#include "rows.h"

static int current, synced, queried, launched, live_streams;

int emac_gpu_device_count(void) { return 2; }
int emac_gpu_get_device(int *d) { *d = current; return 0; }
int emac_gpu_set_device(int d) { current = d; return 0; }
int emac_gpu_is_device_pointer(const void *p) { return p != NULL; }
int ext_mpi_amd_gpu_device_of(const void *p) { return (int)((size_t)p >> 28); }
int emac_gpu_malloc(void **p, size_t n) { *p = malloc(n); return 0; }
int emac_gpu_free(void *p) { free(p); return 0; }
int emac_gpu_stream_create(void **s) { *s = malloc(1); live_streams++; return 0; }
int emac_gpu_stream_destroy(void *s) { free(s); live_streams--; return 0; }
int emac_gpu_stream_sync(void *s) { synced = s ? 100 : current; return 0; }
int emac_gpu_stream_query(void *s) { queried = s ? 100 : current; return 0; }
int emac_gpu_stream_device(void *s, int *d) { *d = s ? (int)((size_t)s >> 28) : current; return 0; }
int emac_gpu_event_destroy(void *e) { return 0; }
int emac_gpu_graph_destroy(void *g) { return 0; }
int emac_gpu_act(const ext_mpi_amd_act *d, void *s) { launched = current; return 0; }
int emac_gpu_layernorm(const ext_mpi_amd_layernorm *d, void *s) { launched = current; return 0; }
size_t emac_gpu_layernorm_grad_ws(const ext_mpi_amd_layernorm_grad *d) { return 64; }
int emac_gpu_layernorm_grad(const ext_mpi_amd_layernorm_grad *d, float *w, void *s) { launched = current; return 0; }

#define CHECK(x)                                              \
  do {                                                        \
    if (!(x)) {                                               \
      printf("%s:%d: %s\n", __FILE__, __LINE__, #x);          \
      exit(1);                                                \
    }                                                         \
  } while (0)

#define ON(dev, k) ((void *)(((size_t)(dev) << 28) + (size_t)(k) * 4096))

static int save8(int dev) {
  int h = -1;
  CHECK(ext_mpi_amd_save8_init(2, 8, EXT_MPI_AMD_FLOAT, ON(dev, 1), 0, ON(dev, 2), 0, ON(dev, 3), &h) == 0);
  return h;
}

/* a handle of device 1 on the default stream, used while device 0 is current */
static void default_stream_of_another_device(void) {
  int h = save8(1);
  CHECK(current == 0);
  CHECK(ext_mpi_amd_set_stream(h, NULL) == 0);
  launched = synced = queried = -1;
  CHECK(ext_mpi_amd_start(h) == 0 && launched == 1 && current == 0);
  CHECK(ext_mpi_amd_test(h) == 0 && queried == 1 && current == 0);
  CHECK(ext_mpi_amd_wait(h) == 0 && synced == 1 && current == 0);
  synced = -1;
  CHECK(ext_mpi_amd_start(h) == 0);
  CHECK(ext_mpi_amd_set_stream(h, NULL) == 0 && synced == 1 && current == 0); /* a pending Start is waited for */
  synced = -1;
  CHECK(ext_mpi_amd_start(h) == 0);
  CHECK(ext_mpi_amd_done(h) == 0 && synced == 1 && current == 0);
}

/* memory and stream of one device, whichever is current */
static void stream_of_another_device(void) {
  int h = save8(1);
  synced = -1;
  CHECK(ext_mpi_amd_set_stream(h, ON(1, 7)) == 0);
  CHECK(ext_mpi_amd_start(h) == 0 && launched == 1);
  CHECK(ext_mpi_amd_set_stream(h, ON(0, 7)) == EXT_MPI_AMD_ERROR_ARG && synced == -1);
  CHECK(ext_mpi_amd_stream(h) == ON(1, 7)); /* as before */
  CHECK(ext_mpi_amd_set_stream(h, NULL) == 0 && current == 0);
  CHECK(ext_mpi_amd_done(h) == 0);
  CHECK(ext_mpi_amd_save8_init(0, 8, EXT_MPI_AMD_FLOAT, NULL, 0, NULL, 0, NULL, &h) == 0); /* no rows, no memory */
  CHECK(ext_mpi_amd_set_stream(h, ON(1, 7)) == 0 && ext_mpi_amd_start(h) == 0 && ext_mpi_amd_done(h) == 0);
}

/* eps is added as a float: 0, or what a float holds */
static void eps_range(void) {
  const double in[] = {0.0, 1.5e-45, 1e-38, 1e-5, 3.4e38}, out[] = {-1.0, -1e-60, 1e-60, 7e-46, 3.5e38, 1e300, 1.0 / 0.0, 0.0 / 0.0};
  ext_mpi_amd_layernorm d = {0};
  unsigned k;
  int h;
  d.rows = 2;
  d.cols = 8;
  d.dtype = EXT_MPI_AMD_FLOAT;
  d.nsrc = 1;
  d.src[0] = ON(0, 1);
  d.y = ON(0, 2);
  for (k = 0; k < sizeof(in) / sizeof(*in); k++) {
    d.eps = in[k];
    CHECK(ext_mpi_amd_layernorm_init(&d, &h) == 0 && ext_mpi_amd_done(h) == 0);
  }
  for (k = 0; k < sizeof(out) / sizeof(*out); k++) {
    d.eps = out[k];
    CHECK(ext_mpi_amd_layernorm_init(&d, &h) == EXT_MPI_AMD_ERROR_ARG);
  }
}

int main(int argc, char **argv) {
  const char *what = argc > 1 ? argv[1] : "";
  if (!strcmp(what, "default_stream")) default_stream_of_another_device();
  else if (!strcmp(what, "other_stream")) stream_of_another_device();
  else if (!strcmp(what, "eps")) eps_range();
  else return 2;
  CHECK(live_streams == 0);
  return 0;
}
