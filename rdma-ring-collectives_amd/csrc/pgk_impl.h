/* pgk_impl.h -- what the files of libpg_amd.so share behind include/pgk.h (not installed). */
#ifndef PGK_IMPL_H
#define PGK_IMPL_H

#include <stddef.h>

#ifdef __cplusplus
extern "C" {
#endif

/* The calling thread's message behind pgk_last_error() (pgk_reduce.hip). */
void pgk_set_err(const char *fmt, ...) __attribute__((format(printf, 1, 2)));

/* Compute units of the current device, asked for once per device (pgk_reduce.hip). */
int pgk_cu_count(void);

/* The checks that pgk_grad_clip makes of these arguments; 0, or -1 with the message set (pgk_grad.hip). */
int pgk_grad_clip_check(void *const *outs, int out_dt, const void *const *grads, int dt, const size_t *ns, int k,
                        double scale, double max_norm);

#ifdef __cplusplus
}
#endif
#endif /* PGK_IMPL_H */
