// What the entry points outside shim.hip share with it: the library's
// initialisation, its device and the sticky error.
#pragma once

#include <hip/hip_runtime.h>

namespace exq {

// Initialises the library where needed; false (sticky error) when that fails
// or the calling thread's current device is not the library's.
bool lib_ready(const char *what);
// Records the sticky error (the first one stays).
void lib_error(int code, const char *fmt, ...) __attribute__((format(printf, 2, 3)));
bool lib_hip(hipError_t e, const char *what);

}  // namespace exq
