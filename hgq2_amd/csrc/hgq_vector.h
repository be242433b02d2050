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

typedef uint32_t __attribute__((ext_vector_type(4))) u32x4;

template <int ALIGN>
struct WordsAt;
template <>
struct WordsAt<2> {
    typedef uint32_t __attribute__((ext_vector_type(4), aligned(2))) Type;
};
template <>
struct WordsAt<4> {
    typedef uint32_t __attribute__((ext_vector_type(4), aligned(4))) Type;
};

// THROUGH: past the cache, for what is larger than it
template <typename T, bool THROUGH = false>
__device__ __forceinline__ Vec<T> load_vec(const T *p) {
    using Words = typename WordsAt<sizeof(T)>::Type;
    const Words w = THROUGH ? __builtin_nontemporal_load((const Words *)p) : *(const Words *)p;
    return __builtin_bit_cast(Vec<T>, (u32x4)w);
}

template <typename T, bool THROUGH = false>
__device__ __forceinline__ void store_vec(T *p, const Vec<T> &r) {
    using Words = typename WordsAt<sizeof(T)>::Type;
    const Words w = __builtin_bit_cast(u32x4, r);
    if (THROUGH) __builtin_nontemporal_store(w, (Words *)p);
    else *(Words *)p = w;
}

// the words of an access as they arrive (kept as such until they are used: elements of 16 bits taken apart across a branch are waited for there)
template <typename T, bool THROUGH = false>
__device__ __forceinline__ u32x4 load_words(const T *p) {
    using Words = typename WordsAt<sizeof(T)>::Type;
    return THROUGH ? __builtin_nontemporal_load((const Words *)p) : *(const Words *)p;
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

// Sums and maxima over teams of `width` neighbouring lanes (a power of two up to 64), the same to all of them.  Lanes exchange in registers: through LDS
// (ds_bpermute, what a shuffle becomes) the sums of a row in sixteen wavefronts take longer than the row.  STEP 1 and 2 exchange lanes of a quad, 4 and 8 mirror 8 and 16 lanes
// (whose halves hold one value each by then), 16 and 32 swap rows and halves of the wavefront.
template <int STEP>
__device__ __forceinline__ uint32_t other_lane(uint32_t v) {
    if (STEP == 16 || STEP == 32) {
        const auto both = STEP == 16 ? __builtin_amdgcn_permlane16_swap(v, v, false, false) : __builtin_amdgcn_permlane32_swap(v, v, false, false);
        return (__lane_id() & STEP) ? both[0] : both[1];
    }
    constexpr int control = STEP == 1 ? 0xB1 : STEP == 2 ? 0x4E : STEP == 4 ? 0x141 : 0x140;
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, control, 0xf, 0xf, true);
}

template <int STEP>
__device__ __forceinline__ float other(float v) {
    return __uint_as_float(other_lane<STEP>(__float_as_uint(v)));
}

template <int STEP>
__device__ __forceinline__ double other(double v) {
    return __hiloint2double((int)other_lane<STEP>((uint32_t)__double2hiint(v)), (int)other_lane<STEP>((uint32_t)__double2loint(v)));
}

template <typename V, typename F>
__device__ __forceinline__ V team_fold(V v, int width, F f) {
    if (width > 1) v = f(v, other<1>(v));
    if (width > 2) v = f(v, other<2>(v));
    if (width > 4) v = f(v, other<4>(v));
    if (width > 8) v = f(v, other<8>(v));
    if (width > 16) v = f(v, other<16>(v));
    if (width > 32) v = f(v, other<32>(v));
    return v;
}

template <typename V>
__device__ __forceinline__ V team_sum(V v, int width) {
    return team_fold(v, width, [](V a, V b) { return a + b; });
}

__device__ __forceinline__ float team_max(float v, int width) {
    return team_fold(v, width, [](float a, float b) { return fmaxf(a, b); });
}

}  // namespace hgq
