// Element types of the MXFP4 and block kernels: conversions to and from float, and vectors of
// eight elements read or written at the element's own alignment (gfx950 serves a 16-byte access
// at any address, so a row of odd length costs no scalar path).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace glv {

typedef __bf16 bf16;
typedef _Float16 f16;
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef f16 f16x2 __attribute__((ext_vector_type(2)));

template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Eight {
    T v[8];
};

// elements [0, valid) of p, zeros behind them; valid may be negative or beyond 8
template <typename T>
__device__ inline Eight<T> load_eight(const T* p, int valid) {
    Eight<T> r;
    if (valid >= 8) {
        r = *reinterpret_cast<const Eight<T>*>(p);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) r.v[i] = i < valid ? p[i] : T(0);
    }
    return r;
}

template <typename T>
__device__ inline void store_eight(T* p, const Eight<T>& r, int valid) {
    if (valid >= 8) {
        *reinterpret_cast<Eight<T>*>(p) = r;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < valid) p[i] = r.v[i];
    }
}

}  // namespace glv
