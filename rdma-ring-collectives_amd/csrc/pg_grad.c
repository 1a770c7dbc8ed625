/*
 * pg_grad.c -- pg_grad_clip (include/pg_ext.h): clip by the norm of gradients
 * that are spread over the ranks of a group.
 *
 * The local sum of squares and the clip are kernels (pgk_grad_*); between them
 * the ranks' sums meet in one pg_all_reduce of two doubles, the second of which
 * says how many ranks cannot go on.  A rank whose arguments are refused or
 * whose own sum fails takes part in it all the same, so the call fails on every
 * rank and nobody waits for a rank that has left.  What fails behind the
 * all-reduce (the upload of the sum, the clip) fails on that rank alone.
 */
#include <math.h>
#include <stdio.h>
#include <string.h>

#include "pg_impl.h"
#include "pgk_impl.h"

/* Memory that a kernel on `device` can read and write: that device's, or managed. */
static int on_device(const void *p, int device) {
  hipPointerAttribute_t a;
  memset(&a, 0, sizeof(a));
  if (hipPointerGetAttributes(&a, p) != hipSuccess) {
    (void)hipGetLastError();
    return 0;
  }
  return (a.type == hipMemoryTypeDevice && a.device == device) || a.type == hipMemoryTypeManaged || a.isManaged;
}

/* 0 when the handle's device is the current one, which the workspace is allocated on, and every tensor is
 * its memory (a kernel that read anything else would fault); -1 with the error set. */
static int check_device(int device, void *const *outs, const void *const *grads, const size_t *ns, int k) {
  int current = -1;
  PG_CHECK_HIP(hipGetDevice(&current));
  if (current != device) {
    pg_set_error("pg_grad_clip: the current device is %d, the handle's %d", current, device);
    return -1;
  }
  for (int j = 0; j < k; ++j) {
    if (!ns[j]) continue;
    const int grad = on_device(grads[j], device);
    if (grad && (outs[j] == grads[j] || on_device(outs[j], device))) continue;
    pg_set_error("pg_grad_clip: %s %d is not device memory of device %d", grad ? "output" : "gradient", j, device);
    return -1;
  }
  return 0;
}

/* This rank's sum of squares into *sum; 0, or -1 with the error set. */
static int local_sum(struct pg_impl *im, const void *const *grads, int dt, const size_t *ns, int k, double *sum) {
  if (pg_wait_producers(im, 0) || pg_ensure(&im->gwork, &im->gwork_cap, PGK_GRAD_WORK_BYTES + sizeof(double)))
    return -1;
  double *dsum = (double *)((char *)im->gwork + PGK_GRAD_WORK_BYTES);
  if (pgk_grad_sumsq(grads, ns, k, dt, dsum, im->gwork, (void *)im->red)) {
    pg_set_error("pg_grad_clip: %s", pgk_last_error());
    return -1;
  }
  PG_CHECK_HIP(hipMemcpyAsync(sum, dsum, sizeof(*sum), hipMemcpyDeviceToHost, im->red));
  return pg_stream_wait(im->red);
}

int pg_grad_clip(void *const *outs, int out_dt, const void *const *grads, int dt, const size_t *ns, int k,
                 double scale, double max_norm, double *norm, void *pg_handle) {
  struct pg *pg = (struct pg *)pg_handle;
  if (!pg) { pg_set_error("pg_grad_clip: NULL handle"); return -1; }
  struct pg_impl *im = (struct pg_impl *)pg->impl;
  if (!im) { pg_set_error("pg_grad_clip: closed handle"); return -1; }

  double sums[2] = {0.0, 0.0};                    /* sum of squares, ranks that failed */
  int bad = pgk_grad_clip_check(outs, out_dt, grads, dt, ns, k, scale, max_norm);
  if (bad) pg_set_error("pg_grad_clip: %s", pgk_last_error());
  else bad = check_device(pg->device, outs, grads, ns, k) || local_sum(im, grads, dt, ns, k, &sums[0]);
  if (bad) { sums[0] = 0.0; sums[1] = 1.0; }
  if (pg->world_size > 1) {
    char mine[256];
    snprintf(mine, sizeof(mine), "%s", bad ? pg_last_error() : "");
    if (pg_all_reduce(sums, sums, 2, DT_DOUBLE, OP_SUM, pg_handle)) return -1;
    if (bad) { pg_set_error("%s", mine); return -1; }
    if (sums[1] != 0.0) {
      pg_set_error("pg_grad_clip: %d of %d ranks could not take part", (int)sums[1], pg->world_size);
      return -1;
    }
  } else if (bad) {
    return -1;
  }

  double *dsum = (double *)((char *)im->gwork + PGK_GRAD_WORK_BYTES);       /* holds this rank's sum */
  if (pg->world_size > 1) PG_CHECK_HIP(hipMemcpyAsync(dsum, sums, sizeof(double), hipMemcpyHostToDevice, im->red));
  int rc = pgk_grad_clip(outs, out_dt, grads, dt, ns, k, dsum, 1, scale, max_norm, NULL, (void *)im->red);
  if (rc) pg_set_error("pg_grad_clip: %s", pgk_last_error());
  if (pg_stream_wait(im->red) || rc) return -1;
  if (norm) *norm = fabs(scale) * sqrt(sums[0]);
  return 0;
}
