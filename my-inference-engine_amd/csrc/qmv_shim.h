/*
 * What the library's host files share: the calling thread's error message, the
 * selected device and counted device allocations.
 */
#ifndef QMV_SHIM_H
#define QMV_SHIM_H

#include <hip/hip_runtime.h>
#include <stddef.h>

namespace qmv {

void shim_error(const char *text); /* qmv_last_error() of this thread */
int shim_device();                 /* qmv_set_device's */
hipError_t shim_malloc(void **p, size_t bytes);

} // namespace qmv

#endif
