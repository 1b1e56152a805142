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

// Launches `kernel` and reports that launch's own error: an earlier one, of another library's call that its caller has
// dealt with, stays in hipGetLastError() and is none of this call's.
template <typename... P, typename... A>
int launch(const char* what, void (*kernel)(P...), dim3 grid, dim3 block, size_t lds, hipStream_t stream, A... args) {
    static_assert(sizeof...(P) == sizeof...(A), "an argument for every parameter");
    return [&](P... values) {
        void* pointers[] = {const_cast<void*>(static_cast<const void*>(&values))...};
        const hipError_t e = hipLaunchKernel(reinterpret_cast<const void*>(kernel), grid, block, pointers, lds, stream);
        if (e == hipSuccess) return (int)GLV_OK;
        (void)hipGetLastError();  // it is reported here, and not once more by whoever looks next
        return report(GLV_ERR_HIP, "%s: launch failed: %s", what, hipGetErrorString(e));
    }(args...);
}

// A launch counts its threads in 32 bits.
inline bool too_large(int64_t blocks, int threads) { return blocks * threads > UINT32_MAX; }

inline bool float_type(int type) { return type == GLV_F32 || type == GLV_BF16 || type == GLV_F16; }

}  // namespace glv
