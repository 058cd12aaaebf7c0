// Element types of the kernels that take fp32, bf16 or fp16 tensors: vector loads and stores through fp32 registers.
#pragma once
#include "common.h"

// type codes of the C-ABI
#define SV_F32 0
#define SV_BF16 1
#define SV_F16 2

__host__ __device__ constexpr int sv_elem_size(int type) { return type == SV_F32 ? 4 : 2; }

// N elements as one vector, at any address that an element may have: the hardware's 8 and 16-byte loads and stores need no more,
// so that odd widths and distances of rows take vectors too (there and back, against vectors that need aligned rows: dropout of
// 65536 x 2047 bf16 257 us instead of 564, lookup of 100000 x 333 bf16 83 instead of 197)
template <typename T, int N>
struct SvVec {
    typedef T type __attribute__((ext_vector_type(N), aligned(sizeof(T))));
};

template <int N, typename T>
__device__ __forceinline__ void sv_load(const T* __restrict__ p, float* v) {
    const typename SvVec<T, N>::type x = *reinterpret_cast<const typename SvVec<T, N>::type*>(p);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = (float)x[i];
}
// one rounding to the element type (nearest even; NaN stays NaN)
template <int N, typename T>
__device__ __forceinline__ void sv_store(T* __restrict__ p, const float* v) {
    typename SvVec<T, N>::type x;
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = (T)v[i];
    *reinterpret_cast<typename SvVec<T, N>::type*>(p) = x;
}

// widest vector of `most` elements or fewer for rows of n; `exact`: that divides n (else the last vector of a row reaches back over
// the one before)
inline int sv_vec_for(int most, int n, bool exact) {
    int v = most;
    while (v > 1 && (v > n || (exact && n % v != 0))) v >>= 1;
    return v;
}

// calls f(T{}) with the element type of a code
template <typename F>
inline void sv_by_type(int type, F f) {
    if (type == SV_F32) f(float{});
    else if (type == SV_BF16) f(__bf16{});
    else f(_Float16{});
}
