// Error text of the C entry points: one thread-local message, read with kamd_hip_last_error().
#pragma once
#include <hip/hip_runtime.h>

#define KAMD_HIDDEN __attribute__((visibility("hidden")))

// 0 if `e` is hipSuccess; otherwise the message becomes "<what>: <error>" and the result is -1
KAMD_HIDDEN int kamd_check(hipError_t e, const char* what);
// sets the message and returns -1
KAMD_HIDDEN int kamd_fail(const char* fmt, ...) __attribute__((format(printf, 1, 2)));
