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
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef f16 f16x2 __attribute__((ext_vector_type(2)));

template <typename T>
struct Eight {
    T v[8];
};

// 16 bytes at the alignment of a T, in one access
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

// v moved down by `by` elements (0 .. 8), zeros from above
template <typename T>
__device__ inline Eight<T> moved_down(const Eight<T>& v, int by) {
    constexpr int kWords = sizeof(Eight<T>) / 4;
    struct Words {
        uint32_t w[kWords + 8];
    } x = {};
    __builtin_memcpy(x.w, &v, sizeof(v));
#pragma unroll
    for (int bit = 8; bit >= 1; bit >>= 1) {
        const int bytes = bit * sizeof(T);
        if (by & bit) {
#pragma unroll
            for (int i = 0; i < kWords; ++i)
                x.w[i] = bytes >= 4 ? x.w[i + bytes / 4] : __builtin_amdgcn_alignbit(x.w[i + 1], x.w[i], 16);
        }
    }
    Eight<T> r;
    __builtin_memcpy(&r, x.w, sizeof(r));
    return r;
}

// Columns [col, col + 8) of a row of `cols`, zeros behind the last, in two halves so that many loads can
// be under way before the first is used: fetch_eight reads, without branches, a piece that reaches
// over the end as the row's last eight; place_eight moves it into place.  NARROW: rows of fewer than
// eight, a kernel of its own wherever the others would carry its eight loads along.
template <bool NARROW, typename T>
__device__ inline Eight<T> fetch_eight(const T* row, int col, int cols) {
    Eight<T> r;
    if constexpr (NARROW) {
#pragma unroll
        for (int i = 0; i < 8; ++i) r.v[i] = row[min(i, cols - 1)];
    } else {
        const T* p = row + min(col, cols - 8);
        if constexpr (sizeof(T) == 2) {
            r = __builtin_bit_cast(Eight<T>, load_16(p));
        } else {
            const i32x4 a = load_16(p), b = load_16(p + 4);
            r = __builtin_bit_cast(Eight<T>, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
        }
    }
    return r;
}
template <bool NARROW, typename T>
__device__ inline Eight<T> place_eight(const Eight<T>& v, int col, int cols) {
    if constexpr (NARROW) {
        Eight<T> r;
#pragma unroll
        for (int i = 0; i < 8; ++i) r.v[i] = col + i < cols ? v.v[i] : T(0);
        return r;
    } else {
        return col + 8 <= cols ? v : moved_down(v, min(col - (cols - 8), 8));
    }
}
template <bool NARROW, typename T>
__device__ inline Eight<T> load_eight(const T* row, int col, int cols) {
    return place_eight<NARROW>(fetch_eight<NARROW>(row, col, cols), col, cols);
}

template <typename T>
__device__ inline void store_eight(T* p, const Eight<T>& r, int valid) {
    if (valid >= 8) {
        if constexpr (sizeof(T) == 2) {
            store_16(p, __builtin_bit_cast(i32x4, r));
        } else {
            const i32x8 v = __builtin_bit_cast(i32x8, r);
            store_16(p, __builtin_shufflevector(v, v, 0, 1, 2, 3));
            store_16(p + 4, __builtin_shufflevector(v, v, 4, 5, 6, 7));
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (i < valid) p[i] = r.v[i];
}

}  // namespace glv
