/*
 * engine_rows.c -- handles of the row operators (include/ext_mpi_amd.h "row operators"): checks of
 * the descriptors, workspaces, Start. The launches are rows.h's (norm.hip, act8.hip).
 *
 * A handle keeps a copy of its descriptor with every stride filled in, and its workspace; Start is
 * one to three kernel launches on the handle's stream and nothing else, so it can be captured. The
 * handle's own stream is created by the first Start or ext_mpi_amd_stream that needs it: a caller
 * that supplies one (ext_mpi_amd_set_stream) never pays for a stream it does not use.
 */
#include <limits.h>
#include <math.h>
#include <stdint.h>

#include "engine_int.h"
#include "ext_mpi_amd_gpu.h"
#include "rows.h"

enum { ROWS_NORM = 1, ROWS_NORM_GRAD, ROWS_ACT, ROWS_ACT_GRAD, ROWS_RESTORE8 };

struct emac_rows {
  int what;
  union {
    ext_mpi_amd_layernorm norm;
    ext_mpi_amd_layernorm_grad grad;
    ext_mpi_amd_act act;
    ext_mpi_amd_act_grad agrad;
  } d;
  void *ws;       /* the gradient's partial rows */
  int stream_set; /* the caller's stream, which may be NULL (the default stream) */
  int anywhere;   /* no memory (no rows): any device will do */
};

/* ---- the memory a descriptor names ---- */

/* rows of `len` bytes, `ld` bytes apart */
typedef struct {
  const char *p;
  long rows, len, ld;
  int out;
  int type; /* element type of a matrix that an output may replace in place, -1: none */
} region;

#define MAX_REGIONS (2 * EMAC_MAX_RANKS)
typedef struct {
  region r[MAX_REGIONS];
  int n;
  int device;
  int rc;
} memory;

static int elem_size(int dtype) { return dtype == EXT_MPI_AMD_FLOAT ? 4 : 2; }

static int type_check(int dtype) {
  if (dtype == EXT_MPI_AMD_FLOAT || dtype == EXT_MPI_AMD_BF16 || dtype == EXT_MPI_AMD_HALF) return 0;
  return emac_type_size(dtype) > 0 ? EMAC_ERR_UNSUPPORTED : EMAC_ERR_ARG;
}

/* the type of a vector beside matrices of `dtype`: the same, or FLOAT */
static int type2_check(int t, int dtype) {
  const int rc = type_check(t);
  return rc || t == dtype || t == EXT_MPI_AMD_FLOAT ? rc : EMAC_ERR_UNSUPPORTED;
}

static void fail(memory *m, int rc) {
  if (!m->rc) m->rc = rc;
}

/* one matrix or vector: present unless `optional` (or without rows), its stride filled in (NULL
   for a vector), aligned to its element, in memory of one device */
static void add(memory *m, const void *p, long rows, long cols, long *stride, int esize, int type, int out, int optional) {
  region *r;
  int dev;
  long ld = cols;
  if (stride) {
    if (*stride < 0 || (*stride > 0 && *stride < cols)) {
      if (p) fail(m, EMAC_ERR_ARG);
      return;
    }
    if (!*stride) *stride = cols;
    ld = *stride;
  }
  if (rows <= 0 || cols <= 0) return; /* nothing is touched */
  if (!p) {
    if (!optional) fail(m, EMAC_ERR_ARG);
    return;
  }
  /* byte offsets of the last row stay below 2^62 */
  if (rows > 1 && ld > (LONG_MAX / 4 / esize - cols) / (rows - 1)) {
    fail(m, EMAC_ERR_ARG);
    return;
  }
  if ((uintptr_t)p % (uintptr_t)esize) {
    fail(m, EMAC_ERR_ARG);
    return;
  }
  dev = emac_gpu_is_device_pointer(p) ? ext_mpi_amd_gpu_device_of(p) : -1;
  if (dev < 0 || (m->device >= 0 && dev != m->device) || m->n == MAX_REGIONS) {
    fail(m, EMAC_ERR_ARG);
    return;
  }
  m->device = dev;
  r = &m->r[m->n++];
  r->p = (const char *)p;
  r->rows = rows;
  r->len = cols * esize;
  r->ld = ld * esize;
  r->out = out;
  r->type = type;
}

static long span(const region *r) { return (r->rows - 1) * r->ld + r->len; }

/* whether two regions share a byte. Rows of one stride that interleave (the halves of one
   product's rows) are told apart by their columns; ranges of different strides that cross count
   as shared. */
static int share(const region *a, const region *b) {
  long d, w;
  if (a->p + span(a) <= b->p || b->p + span(b) <= a->p) return 0;
  if (a->rows == 1 && b->rows == 1) return 1;
  w = a->rows == 1 ? b->ld : a->ld;
  if (a->rows > 1 && b->rows > 1 && a->ld != b->ld) return 1;
  d = (long)(b->p - a->p) % w;
  if (d < 0) d += w; /* b's columns start d bytes into a's rows */
  return d < a->len || d + b->len > w;
}

/* the same for tests (host only): rows of `len` bytes, `ld` bytes apart, at addresses a and b */
int ext_mpi_amd_check_rows_share(long a, long rows_a, long len_a, long ld_a, long b, long rows_b, long len_b, long ld_b) {
  const region x = {(const char *)a, rows_a, len_a, ld_a, 0, -1}, y = {(const char *)b, rows_b, len_b, ld_b, 0, -1};
  return share(&x, &y);
}

/* the polynomial of the normal distribution's tail for tests (host only): its argument's factor, its coefficients */
double ext_mpi_amd_check_gelu_tail(int k) {
  static const float c[8] = EMAC_GELU_TAIL;
  return k ? c[(k - 1) & 7] : EMAC_GELU_TAIL_AT;
}

static int settle(memory *m) {
  int i, k;
  for (i = 0; i < m->n && !m->rc; i++)
    for (k = i + 1; k < m->n && !m->rc; k++) {
      const region *a = &m->r[i], *b = &m->r[k];
      if (!a->out && !b->out) continue;
      if (a->out != b->out && a->type >= 0 && a->type == b->type && a->p == b->p && (a->ld == b->ld || a->rows == 1) &&
          a->len == b->len)
        continue; /* in place */
      if (share(a, b)) fail(m, EMAC_ERR_ARG);
    }
  return m->rc;
}

/* The kernels of act8.hip number columns and checkpoint blocks in 32 bits (narrow matrices of a device's
   memory can have more blocks: 2^31 of one bf16 column are 15 GB with their checkpoint); the last 4096 of
   them are left for a launch's own rounding up. */
static int fits8(long rows, long cols) {
  if (cols < 1 || cols > EXT_MPI_AMD_COLS8_MAX) return 0;
  return rows <= EXT_MPI_AMD_BLOCKS8_MAX / ((cols + EMAC_BLOCK8 - 1) / EMAC_BLOCK8);
}

static int begin(memory *m, long rows, long cols, int fits, int dtype, int *handle) {
  int rc;
  memset(m, 0, sizeof(*m));
  m->device = -1;
  *handle = -1;
  if (rows < 0 || cols < 1) return EMAC_ERR_ARG;
  if ((rc = type_check(dtype))) return rc;
  if (!fits) return EMAC_ERR_UNSUPPORTED;
  if (emac_gpu_device_count() <= 0) return EMAC_ERR_DEVICE;
  return 0;
}

static void add_saved(memory *m, long rows, long cols, const signed char *q, long *q_stride, const float *scale, int out,
                      int optional) {
  const long nblk = (cols + EMAC_BLOCK8 - 1) / EMAC_BLOCK8;
  if (optional && !q != !scale && rows > 0) fail(m, EMAC_ERR_ARG); /* both or neither */
  add(m, q, rows, cols, q_stride, 1, -1, out, optional);
  add(m, scale, rows, nblk, NULL, 4, -1, out, optional);
}

static int finish(const memory *m, int what, const void *d, size_t bytes, size_t ws, int *handle) {
  emac_handle *h = (emac_handle *)calloc(1, sizeof(emac_handle));
  int rc = 0, cur = -1;
  if (!h) return EMAC_ERR_MALLOC;
  h->kind = KIND_ROWS;
  h->rows = (struct emac_rows *)calloc(1, sizeof(struct emac_rows));
  if (!h->rows) {
    handle_release(h);
    return EMAC_ERR_MALLOC;
  }
  h->rows->what = what;
  memcpy(&h->rows->d, d, bytes);
  emac_gpu_get_device(&cur);
  h->rows->anywhere = m->device < 0;
  h->device = h->rows->anywhere ? cur : m->device;
  if (ws) {
    rc = emac_gpu_set_device(h->device);
    if (!rc) rc = emac_gpu_malloc(&h->rows->ws, ws);
    if (cur >= 0 && cur != h->device) emac_gpu_set_device(cur);
  }
  if (!rc) rc = finish_init(h, handle);
  if (rc) handle_release(h);
  return rc;
}

/* ---- the operators ---- */

int ext_mpi_amd_layernorm_init(const ext_mpi_amd_layernorm *desc, int *handle) {
  ext_mpi_amd_layernorm d;
  memory m;
  int rc, i, es;
  if (!desc || !handle) return EMAC_ERR_ARG;
  d = *desc;
  if ((rc = begin(&m, d.rows, d.cols, d.cols <= EXT_MPI_AMD_ROW_COLS_MAX, d.dtype, handle))) return rc;
  if (d.nsrc < 1 || d.nsrc > EMAC_MAX_RANKS) return EMAC_ERR_ARG;
  /* the kernels add it as a float: 0 in place of a smaller eps would make a row of one value NaN */
  if (!(d.eps >= 0.0) || isinf((float)d.eps) || (d.eps > 0.0 && (float)d.eps == 0.0f)) return EMAC_ERR_ARG;
  if (!d.y && !d.sum && !d.q && d.rows > 0) return EMAC_ERR_ARG;
  if ((d.weight || d.bias) && (rc = type2_check(d.wdtype, d.dtype))) return rc;
  es = elem_size(d.dtype);
  for (i = 0; i < d.nsrc; i++) add(&m, d.src[i], d.rows, d.cols, &d.src_stride, es, d.dtype, 0, 0);
  add(&m, d.residual, d.rows, d.cols, &d.residual_stride, es, d.dtype, 0, 1);
  add(&m, d.weight, 1, d.cols, NULL, elem_size(d.wdtype), -1, 0, 1);
  add(&m, d.bias, 1, d.cols, NULL, elem_size(d.wdtype), -1, 0, 1);
  add(&m, d.y, d.rows, d.cols, &d.y_stride, es, d.dtype, 1, 1);
  add(&m, d.sum, d.rows, d.cols, &d.sum_stride, es, d.dtype, 1, 1);
  add(&m, d.mean, 1, d.rows, NULL, 4, -1, 1, 1);
  add(&m, d.rstd, 1, d.rows, NULL, 4, -1, 1, 1);
  add_saved(&m, d.rows, d.cols, d.q, &d.q_stride, d.scale, 1, 1);
  if ((rc = settle(&m))) return rc;
  return finish(&m, ROWS_NORM, &d, sizeof(d), 0, handle);
}

int ext_mpi_amd_layernorm_grad_init(const ext_mpi_amd_layernorm_grad *desc, int *handle) {
  ext_mpi_amd_layernorm_grad d;
  memory m;
  int rc, i, es;
  if (!desc || !handle) return EMAC_ERR_ARG;
  d = *desc;
  if ((rc = begin(&m, d.rows, d.cols, d.cols <= EXT_MPI_AMD_ROW_COLS_MAX, d.dtype, handle))) return rc;
  if (d.nsrc < 1 || d.nsrc > EMAC_MAX_RANKS) return EMAC_ERR_ARG;
  if (!d.dx && !d.dweight && !d.dbias && d.rows > 0) return EMAC_ERR_ARG;
  if (d.rows > 0 && !d.x == !d.q) return EMAC_ERR_ARG; /* exactly one */
  if ((d.weight || d.bias) && (rc = type2_check(d.wdtype, d.dtype))) return rc;
  if ((d.dweight || d.dbias) && (rc = type2_check(d.gdtype, d.dtype))) return rc;
  es = elem_size(d.dtype);
  for (i = 0; i < d.nsrc; i++) add(&m, d.dy[i], d.rows, d.cols, &d.dy_stride, es, d.dtype, 0, 0);
  add(&m, d.x, d.rows, d.cols, &d.x_stride, es, d.dtype, 0, 1);
  add_saved(&m, d.rows, d.cols, d.q, &d.q_stride, d.scale, 0, 1);
  add(&m, d.mean, 1, d.rows, NULL, 4, -1, 0, 0);
  add(&m, d.rstd, 1, d.rows, NULL, 4, -1, 0, 0);
  add(&m, d.weight, 1, d.cols, NULL, elem_size(d.wdtype), -1, 0, 1);
  add(&m, d.bias, 1, d.cols, NULL, elem_size(d.wdtype), -1, 0, 1);
  add(&m, d.dsum, d.rows, d.cols, &d.dsum_stride, es, d.dtype, 0, 1);
  add(&m, d.dx, d.rows, d.cols, &d.dx_stride, es, d.dtype, 1, 1);
  add(&m, d.dweight, 1, d.cols, NULL, elem_size(d.gdtype), -1, 1, 1);
  add(&m, d.dbias, 1, d.cols, NULL, elem_size(d.gdtype), -1, 1, 1);
  add(&m, d.y, d.rows, d.cols, &d.y_stride, es, -1, 1, 1); /* stored before dsum is read */
  if ((rc = settle(&m))) return rc;
  d.accumulate = d.accumulate != 0;
  return finish(&m, ROWS_NORM_GRAD, &d, sizeof(d), emac_gpu_layernorm_grad_ws(&d), handle);
}

int ext_mpi_amd_save8_init(long rows, long cols, int dtype, const void *x, long x_stride, signed char *q, long q_stride,
                           float *scale, int *handle) {
  ext_mpi_amd_act d;
  memory m;
  int rc;
  if (!handle) return EMAC_ERR_ARG;
  if ((rc = begin(&m, rows, cols, fits8(rows, cols), dtype, handle))) return rc;
  add(&m, x, rows, cols, &x_stride, elem_size(dtype), -1, 0, 0);
  add_saved(&m, rows, cols, q, &q_stride, scale, 1, 0);
  if ((rc = settle(&m))) return rc;
  memset(&d, 0, sizeof(d));
  d.rows = rows;
  d.cols = cols;
  d.dtype = dtype;
  d.kind = EMAC_SAVE8;
  d.a = x;
  d.a_stride = x_stride;
  d.qa = q;
  d.q_stride = q_stride;
  d.sa = scale;
  return finish(&m, ROWS_ACT, &d, sizeof(d), 0, handle);
}

int ext_mpi_amd_restore8_init(long rows, long cols, int dtype, const signed char *q, long q_stride, const float *scale,
                              void *x, long x_stride, int *handle) {
  ext_mpi_amd_act_grad d; /* qa, sa and da alone */
  memory m;
  int rc;
  if (!handle) return EMAC_ERR_ARG;
  if ((rc = begin(&m, rows, cols, fits8(rows, cols), dtype, handle))) return rc;
  add_saved(&m, rows, cols, q, &q_stride, scale, 0, 0);
  add(&m, x, rows, cols, &x_stride, elem_size(dtype), -1, 1, 0);
  if ((rc = settle(&m))) return rc;
  memset(&d, 0, sizeof(d));
  d.rows = rows;
  d.cols = cols;
  d.dtype = dtype;
  d.qa = q;
  d.q_stride = q_stride;
  d.sa = scale;
  d.da = x;
  d.da_stride = x_stride;
  return finish(&m, ROWS_RESTORE8, &d, sizeof(d), 0, handle);
}

int ext_mpi_amd_act_init(const ext_mpi_amd_act *desc, int *handle) {
  ext_mpi_amd_act d;
  memory m;
  int rc, es;
  if (!desc || !handle) return EMAC_ERR_ARG;
  d = *desc;
  if ((rc = begin(&m, d.rows, d.cols, fits8(d.rows, d.cols), d.dtype, handle))) return rc;
  if (d.kind < EXT_MPI_AMD_SILU || d.kind > EXT_MPI_AMD_GELU_TANH) return EMAC_ERR_ARG;
  if (!d.h && !d.qa && d.rows > 0) return EMAC_ERR_ARG;
  /* the gate's checkpoint goes with the gate's and the other's */
  if (d.rows > 0 && !d.qb != !(d.b && d.qa)) return EMAC_ERR_ARG;
  es = elem_size(d.dtype);
  add(&m, d.a, d.rows, d.cols, &d.a_stride, es, d.dtype, 0, 0);
  add(&m, d.b, d.rows, d.cols, &d.b_stride, es, d.dtype, 0, 1);
  add(&m, d.h, d.rows, d.cols, &d.h_stride, es, d.dtype, 1, 1);
  add_saved(&m, d.rows, d.cols, d.qa, &d.q_stride, d.sa, 1, 1);
  add_saved(&m, d.rows, d.cols, d.qb, &d.q_stride, d.sb, 1, 1);
  if ((rc = settle(&m))) return rc;
  return finish(&m, ROWS_ACT, &d, sizeof(d), 0, handle);
}

int ext_mpi_amd_act_grad_init(const ext_mpi_amd_act_grad *desc, int *handle) {
  ext_mpi_amd_act_grad d;
  memory m;
  int rc, es;
  if (!desc || !handle) return EMAC_ERR_ARG;
  d = *desc;
  if ((rc = begin(&m, d.rows, d.cols, fits8(d.rows, d.cols), d.dtype, handle))) return rc;
  if (d.kind < EXT_MPI_AMD_SILU || d.kind > EXT_MPI_AMD_GELU_TANH) return EMAC_ERR_ARG;
  if (d.rows > 0 && !d.qb != !d.db) return EMAC_ERR_ARG; /* a gate and its gradient */
  es = elem_size(d.dtype);
  add(&m, d.dh, d.rows, d.cols, &d.dh_stride, es, d.dtype, 0, 0);
  add_saved(&m, d.rows, d.cols, d.qa, &d.q_stride, d.sa, 0, 0);
  add_saved(&m, d.rows, d.cols, d.qb, &d.q_stride, d.sb, 0, 1);
  add(&m, d.da, d.rows, d.cols, &d.da_stride, es, d.dtype, 1, 0);
  add(&m, d.db, d.rows, d.cols, &d.db_stride, es, d.dtype, 1, 1);
  add(&m, d.h, d.rows, d.cols, &d.h_stride, es, d.dtype, 1, 1);
  if ((rc = settle(&m))) return rc;
  return finish(&m, ROWS_ACT_GRAD, &d, sizeof(d), 0, handle);
}

/* ---- life cycle (engine.c's entry points come here for KIND_ROWS) ---- */

/* the handle's own stream, on its device, if the caller has not supplied one */
int rows_stream(emac_handle *h) {
  int cur = -1, rc;
  if (h->stream || h->rows->stream_set) return 0;
  emac_gpu_get_device(&cur);
  if ((rc = emac_gpu_set_device(h->device))) return rc;
  rc = emac_gpu_stream_create(&h->stream);
  if (cur >= 0 && cur != h->device) emac_gpu_set_device(cur);
  return rc;
}

/* f of a stream with the handle's device current: the default stream is the current device's */
static int on_device(const emac_handle *h, void *stream, int (*f)(void *)) {
  int cur = -1, rc;
  emac_gpu_get_device(&cur);
  if (cur != h->device && emac_gpu_set_device(h->device)) return EMAC_ERR_DEVICE;
  rc = f(stream);
  if (cur >= 0 && cur != h->device) emac_gpu_set_device(cur);
  return rc;
}

int rows_sync(emac_handle *h) { return on_device(h, h->stream, emac_gpu_stream_sync); }
int rows_query(emac_handle *h) { return on_device(h, h->stream, emac_gpu_stream_query); }

/* whether a stream is the current device's */
static int stream_here(void *stream) {
  int dev, cur;
  if (emac_gpu_stream_device(stream, &dev)) return EMAC_ERR_ARG;
  return emac_gpu_get_device(&cur) || dev != cur ? EMAC_ERR_ARG : 0;
}

int rows_set_stream(emac_handle *h, void *stream) {
  const int rc = h->rows->anywhere ? 0 : on_device(h, stream, stream_here);
  if (rc) return rc;
  if (h->started && rows_sync(h)) return EMAC_ERR_DEVICE;
  h->started = 0;
  if (h->own_stream && h->stream) emac_gpu_stream_destroy(h->stream);
  h->stream = stream;
  h->own_stream = 0;
  h->rows->stream_set = 1;
  return 0;
}

int rows_start(emac_handle *h) {
  struct emac_rows *w = h->rows;
  const ext_mpi_amd_act_grad *r = &w->d.agrad;
  int rc, cur = -1;
  if ((rc = rows_stream(h))) return rc;
  emac_gpu_get_device(&cur);
  if (cur != h->device && emac_gpu_set_device(h->device)) return EMAC_ERR_DEVICE;
  switch (w->what) {
  case ROWS_NORM: rc = emac_gpu_layernorm(&w->d.norm, h->stream); break;
  case ROWS_NORM_GRAD: rc = emac_gpu_layernorm_grad(&w->d.grad, (float *)w->ws, h->stream); break;
  case ROWS_ACT: rc = emac_gpu_act(&w->d.act, h->stream); break;
  case ROWS_ACT_GRAD: rc = emac_gpu_act_grad(&w->d.agrad, h->stream); break;
  case ROWS_RESTORE8:
    rc = emac_gpu_restore8(r->rows, r->cols, r->dtype, r->qa, r->q_stride, r->sa, r->da, r->da_stride, h->stream);
    break;
  default: rc = EMAC_ERR_ARG;
  }
  if (cur >= 0 && cur != h->device) emac_gpu_set_device(cur);
  if (!rc) h->started = 1;
  return rc;
}

void rows_free(emac_handle *h) {
  if (!h->rows) return;
  if (h->started) rows_sync(h); /* the default stream too */
  emac_gpu_free(h->rows->ws);
  free(h->rows);
  h->rows = NULL;
}
