// Elements of one of three types (HGQ_TYPE_*) as fp32 values, several per access.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/hgq_hip.h"

namespace hgq {

// 16 bytes of elements.  Rows of odd lengths begin at any multiple of the element's size: the accesses ask for no more (global memory takes
// them at any address; what a wavefront reads is contiguous, so the lines it touches are the same).
template <typename T>
struct Vec {
    static constexpr int N = 16 / sizeof(T);
    T v[N];
};

template <typename T>
__device__ __forceinline__ Vec<T> load_vec(const T *p) {
    Vec<T> r;
    __builtin_memcpy(&r, p, sizeof(r));
    return r;
}

template <typename T>
__device__ __forceinline__ void store_vec(T *p, const Vec<T> &r) {
    __builtin_memcpy(p, &r, sizeof(r));
}

// the first `n` elements of a row's last access (`fill` behind them)
template <typename T>
__device__ __forceinline__ Vec<T> load_part(const T *p, int n, T fill) {
    Vec<T> r;
#pragma unroll
    for (int e = 0; e < Vec<T>::N; ++e) r.v[e] = e < n ? p[e] : fill;
    return r;
}

template <typename T>
__device__ __forceinline__ void store_part(T *p, const Vec<T> &r, int n) {
#pragma unroll
    for (int e = 0; e < Vec<T>::N; ++e)
        if (e < n) p[e] = r.v[e];
}

// sums and maxima over teams of `width` neighbouring lanes (a power of two up to 64), the same to all of them
template <typename V>
__device__ __forceinline__ V team_sum(V v, int width) {
    for (int d = width >> 1; d; d >>= 1) v += __shfl_xor(v, d);
    return v;
}

__device__ __forceinline__ float team_max(float v, int width) {
    for (int d = width >> 1; d; d >>= 1) v = fmaxf(v, __shfl_xor(v, d));
    return v;
}

}  // namespace hgq
