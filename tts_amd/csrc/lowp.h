// Element types of the MXFP4 and block kernels: conversions to and from float, and vectors of
// eight elements read or written at the element's own alignment (gfx950 serves a 16-byte access
// at any address, so a row of odd length costs no scalar path).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

namespace glv {

typedef __bf16 bf16;
typedef _Float16 f16;
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef f16 f16x2 __attribute__((ext_vector_type(2)));

template <typename T, int N>
struct Pack {
    T v[N];
};
template <typename T>
using Eight = Pack<T, 8>;

typedef int i32x4_at2 __attribute__((ext_vector_type(4), aligned(2)));
typedef int i32x4_at4 __attribute__((ext_vector_type(4), aligned(4)));
template <typename T>
using Unaligned = std::conditional_t<sizeof(T) == 2, i32x4_at2, i32x4_at4>;
template <typename T>
__device__ inline i32x4 load_16(const T* p) {
    return *reinterpret_cast<const Unaligned<T>*>(p);
}
template <typename T>
__device__ inline void store_16(T* p, i32x4 v) {
    *reinterpret_cast<Unaligned<T>*>(p) = v;
}

// v moved down by `by` elements (0 .. N), zeros from above
template <typename T, int N>
__device__ inline Pack<T, N> moved_down(const Pack<T, N>& v, int by) {
    constexpr int kWords = sizeof(v) / 4;
    struct Words {
        uint32_t w[2 * kWords];
    } x = {};
    __builtin_memcpy(x.w, &v, sizeof(v));
#pragma unroll
    for (int bit = N; bit >= 1; bit >>= 1) {
        const int bytes = bit * sizeof(T);
        if (by & bit) {
#pragma unroll
            for (int i = 0; i < kWords; ++i)
                x.w[i] = bytes >= 4 ? x.w[i + bytes / 4] : __builtin_amdgcn_alignbit(x.w[i + 1], x.w[i], 16);
        }
    }
    Pack<T, N> r;
    __builtin_memcpy(&r, x.w, sizeof(r));
    return r;
}

// Columns [col, col + N) of a row of `cols`, zeros behind the last, in two halves so that many loads can
// be under way before the first is used: fetch_pack reads, without branches, a piece that reaches over
// the end as the row's last N; place_pack moves it into place.  NARROW: rows of fewer than N, a kernel
// of its own wherever the others would carry its loads along.
template <bool NARROW, int N, typename T>
__device__ inline Pack<T, N> fetch_pack(const T* row, int col, int cols) {
    Pack<T, N> r;
    if constexpr (NARROW) {
#pragma unroll
        for (int i = 0; i < N; ++i) r.v[i] = row[min(i, cols - 1)];
    } else {
        const T* p = row + min(col, cols - N);
        constexpr int kEach = 16 / sizeof(T);
#pragma unroll
        for (int i = 0; i < N; i += kEach) {
            const i32x4 part = load_16(p + i);
            __builtin_memcpy(r.v + i, &part, 16);
        }
    }
    return r;
}
template <bool NARROW, int N, typename T>
__device__ inline Pack<T, N> place_pack(const Pack<T, N>& v, int col, int cols) {
    if constexpr (NARROW) {
        Pack<T, N> r;
#pragma unroll
        for (int i = 0; i < N; ++i) r.v[i] = col + i < cols ? v.v[i] : T(0);
        return r;
    } else {
        return col + N <= cols ? v : moved_down(v, min(col - (cols - N), N));
    }
}
template <typename T, int N>
__device__ inline void store_pack(T* p, const Pack<T, N>& r, int valid) {
    if (valid >= N) {
        constexpr int kEach = 16 / sizeof(T);
#pragma unroll
        for (int i = 0; i < N; i += kEach) {
            i32x4 part;
            __builtin_memcpy(&part, r.v + i, 16);
            store_16(p + i, part);
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
        if (i < valid) p[i] = r.v[i];
}

}  // namespace glv
