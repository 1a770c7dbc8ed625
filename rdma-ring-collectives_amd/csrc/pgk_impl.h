// pgk_impl.h -- what the kernel files of libpg_amd.so share (not installed).
#ifndef PGK_IMPL_H
#define PGK_IMPL_H

// The calling thread's message behind pgk_last_error() (pgk_reduce.hip).
void pgk_set_err(const char* fmt, ...) __attribute__((format(printf, 1, 2)));

// Compute units of the current device, asked for once per device (pgk_reduce.hip).
int pgk_cu_count();

#endif  // PGK_IMPL_H
