// Error plumbing of the sources beside glvoc.hip: messages go to the buffer that
// glv_last_error() returns (thread-local, 512 bytes, owned by glvoc.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>

#include "../../include/glvoc.h"

namespace glv {

constexpr int kErrorBytes = 512;

inline int report(int code, const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(const_cast<char*>(glv_last_error()), kErrorBytes, fmt, ap);
    va_end(ap);
    return code;
}

inline int launch_status(const char* what) {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? GLV_OK : report(GLV_ERR_HIP, "%s: launch failed: %s", what, hipGetErrorString(e));
}

// A launch counts its threads in 32 bits.
inline bool too_large(int64_t blocks, int threads) { return blocks * threads > UINT32_MAX; }

inline bool float_type(int type) { return type == GLV_F32 || type == GLV_BF16 || type == GLV_F16; }

}  // namespace glv
