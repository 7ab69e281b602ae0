#pragma once
// Element types and 16-byte rows of the packed-sequence operators
// (gat_norm.hip, gat_embedding.hip, gat_packed.hip).
//
// Every operator reads and writes float32, bfloat16 or float16 rows and computes
// in float32.  A row is walked in 16-byte vectors whatever its first element's
// alignment: with `phase` = elements between the 16-byte boundary at or before
// the row's start and the row's start, vector i of the row holds columns
// [i * VEC - phase, (i + 1) * VEC - phase).  Vectors that lie inside the row are
// one load; the two that may stick out of it are read element by element, so
// nothing outside the row is touched.

#include "gat_common.h"

namespace {

typedef __bf16 bf16;
typedef _Float16 f16;

template <typename T>
struct Vec16 {
    static constexpr int N = 16 / (int)sizeof(T);
    typedef T type __attribute__((ext_vector_type(N)));
};

// v[0..N) = row[col0 .. col0 + N), zero outside [0, cols).  `whole`: the vector's
// address is 16-byte aligned when it lies inside the row.
template <typename T>
__device__ __forceinline__ typename Vec16<T>::type load_vec(const T* row, int col0, int cols,
                                                            bool whole) {
    constexpr int N = Vec16<T>::N;
    typename Vec16<T>::type v;
    if (whole && col0 >= 0 && col0 + N <= cols) {
        v = *reinterpret_cast<const typename Vec16<T>::type*>(row + col0);
    } else {
        v = typename Vec16<T>::type{};
        if (col0 < cols && col0 + N > 0) {
#pragma unroll
            for (int e = 0; e < N; ++e) {  // no branch between the loads: one wait for all
                const int c = col0 + e;
                const T x = row[c < 0 ? 0 : c < cols ? c : cols - 1];
                v[e] = c >= 0 && c < cols ? x : (T)0.f;
            }
        }
    }
    return v;
}

template <typename T>
__device__ __forceinline__ void store_vec(T* row, int col0, int cols, bool whole,
                                          typename Vec16<T>::type v) {
    constexpr int N = Vec16<T>::N;
    if (whole && col0 >= 0 && col0 + N <= cols) {
        *reinterpret_cast<typename Vec16<T>::type*>(row + col0) = v;
    } else if (col0 < cols && col0 + N > 0) {
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const int c = col0 + e;
            if (c >= 0 && c < cols) row[c] = v[e];
        }
    }
}

// Sum over the aligned group of W lanes that this one is in, given to all of them: no LDS
// round trip (DPP within 16 lanes, then the lane-half swaps).
template <int W>
__device__ __forceinline__ float lanes_sum(float v) {
    v = group_sum16(v, W);
    if constexpr (W >= 32) {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    if constexpr (W >= 64) {
        const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    return v;
}

// elements from the 16-byte boundary at or before p to p
template <typename T>
__host__ __device__ inline int phase_of(const T* p) {
    return (int)((reinterpret_cast<uintptr_t>(p) & 15) / sizeof(T));
}

inline bool known_dtype(int dtype) {
    return dtype == GAT_F32 || dtype == GAT_BF16 || dtype == GAT_F16;
}
inline size_t dtype_size(int dtype) { return dtype == GAT_F32 ? 4 : 2; }

// Whether the addresses p + k * stride fall on multiples of the element size.
inline bool element_aligned(const void* p, int dtype) {
    return (reinterpret_cast<uintptr_t>(p) & (dtype_size(dtype) - 1)) == 0;
}

}  // namespace
