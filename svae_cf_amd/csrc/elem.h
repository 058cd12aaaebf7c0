// Element types of the kernels that take fp32, bf16 or fp16 tensors: vector loads and stores through fp32 registers.
#pragma once
#include "common.h"

// type codes of the C-ABI
#define SV_F32 0
#define SV_BF16 1
#define SV_F16 2

__host__ __device__ constexpr int sv_elem_size(int type) { return type == SV_F32 ? 4 : 2; }

// N elements as one vector; alignment as far as a single load goes (16 bytes)
template <typename T, int N>
struct SvVec {
    static constexpr int bytes = N * (int)sizeof(T) < 16 ? N * (int)sizeof(T) : 16;
    typedef T type __attribute__((ext_vector_type(N), aligned(bytes)));
};
template <typename T>
struct SvVec<T, 1> {
    static constexpr int bytes = (int)sizeof(T);
    typedef T type __attribute__((ext_vector_type(1)));
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

// widest vector of `most` elements or fewer that base addresses, row strides and the row length allow
inline int sv_vec_for(int most, int n, const void* p, long long ldp, int size_p, const void* q, long long ldq, int size_q) {
    for (int v = most; v > 1; v >>= 1) {
        const long long bp = v * size_p < 16 ? v * size_p : 16, bq = v * size_q < 16 ? v * size_q : 16;
        if (n % v == 0 && (unsigned long long)p % bp == 0 && ldp * size_p % bp == 0 && (unsigned long long)q % bq == 0 && ldq * size_q % bq == 0)
            return v;
    }
    return 1;
}

// calls f(T{}) with the element type of a code
template <typename F>
inline void sv_by_type(int type, F f) {
    if (type == SV_F32) f(float{});
    else if (type == SV_BF16) f(__bf16{});
    else f(_Float16{});
}
