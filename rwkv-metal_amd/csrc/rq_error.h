// rq_error.h -- the thread-local error text behind rq_last_error() and the
// argument checks every C entry point makes before a launch.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace rq {

// Records the message and returns `code`; ok() clears it and returns RQ_OK.
int fail(int code, const char* fmt, ...);
int ok();
int launch_status(hipError_t e, const char* what);

inline bool valid_dt(int d) { return d >= 0 && d <= 2; }
inline bool aligned16(const void* p) { return ((uintptr_t)p & 15u) == 0; }

}  // namespace rq
