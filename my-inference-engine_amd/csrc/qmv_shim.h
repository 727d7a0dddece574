/*
 * What the library's host files share: the calling thread's error message, the
 * selected device and the streams' workspaces.
 */
#ifndef QMV_SHIM_H
#define QMV_SHIM_H

#include <hip/hip_runtime.h>
#include <stddef.h>

#include <mutex>

namespace qmv {

void set_error(const char *fmt, ...);         /* qmv_last_error() of this thread */
bool hip_ok(hipError_t e, const char *what);  /* or the error message */

/* Byte ranges that share a byte. */
bool overlap(const void *a, size_t abytes, const void *b, size_t bbytes);

int shim_device(); /* qmv_set_device's */

/* Scratch of at least `bytes` in the workspace of a stream of the current
 * device, which is locked until the lock goes; 0 with a message where it cannot
 * grow. A buffer that is replaced is kept: a graph captured
 * earlier on the stream may still use it. */
int shim_scratch(int device, hipStream_t stream, size_t bytes, unsigned char **data, std::unique_lock<std::mutex> *lock);

} // namespace qmv

#define HIP_TRY(expr)                              \
    do {                                           \
        if (!qmv::hip_ok((expr), #expr)) return 0; \
    } while (0)

#endif
