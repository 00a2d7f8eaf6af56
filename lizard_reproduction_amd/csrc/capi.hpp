// Status and message of the C entry points (capi.hip, mixer_capi.hip).
#pragma once
#include <hip/hip_runtime.h>

namespace lz {
// Sets the calling thread's message (lz_last_error) and returns code.
int fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
// 0 and no message for hipSuccess, else the error's code and message.
int hip_status(hipError_t e, const char* what);
}  // namespace lz
