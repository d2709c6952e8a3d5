// Element types of the patch-network operators: conversion to and from float.
#pragma once

#include "gs_common.h"

namespace gs {

using f16 = _Float16;
using bf16 = __bf16;

// Reads convert exactly; writes round to nearest even once, from a float.
template <typename T>
__device__ __forceinline__ float to_float(T v) { return (float)v; }
template <typename T>
__device__ __forceinline__ T from_float(float v) { return (T)v; }

inline bool element_type(int32_t t) { return t == GS_F32 || t == GS_F16 || t == GS_BF16; }

// Calls f with a value of the element type that `type` names.
template <typename F>
inline int with_element(int32_t type, F f) {
    switch (type) {
        case GS_F32: return f(float{});
        case GS_F16: return f(f16{});
        default: return f(bf16{});
    }
}

// v of the lane that differs in the bits of a pattern, within 16 lanes.
template <int PATTERN>
__device__ __forceinline__ float dpp(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(
                                         0, __builtin_bit_cast(int, v), PATTERN, 0xf, 0xf, true));
}

// f over LANES (16 or 64) neighbouring lanes' values, in each: quad permutations, the
// mirrors of 8 and of 16 lanes, then exchanges of 16 and of 32 lanes.  No LDS.
template <int LANES, typename F>
__device__ __forceinline__ float lane_reduce(float v, F f) {
    static_assert(LANES == 16 || LANES == 64, "a row of lanes or a wave");
    v = f(v, dpp<0xb1>(v));
    v = f(v, dpp<0x4e>(v));
    v = f(v, dpp<0x141>(v));
    v = f(v, dpp<0x140>(v));
    if constexpr (LANES == 64) {
        uint32_t u = __builtin_bit_cast(uint32_t, v);
        const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
        v = f(__builtin_bit_cast(float, (uint32_t)a[0]), __builtin_bit_cast(float, (uint32_t)a[1]));
        u = __builtin_bit_cast(uint32_t, v);
        const auto b = __builtin_amdgcn_permlane32_swap(u, u, false, false);
        v = f(__builtin_bit_cast(float, (uint32_t)b[0]), __builtin_bit_cast(float, (uint32_t)b[1]));
    }
    return v;
}

template <int LANES>
__device__ __forceinline__ float lane_sum(float v) {
    return lane_reduce<LANES>(v, [](float a, float b) { return a + b; });
}
__device__ __forceinline__ float wave_sum(float v) { return lane_sum<kWave>(v); }
__device__ __forceinline__ float wave_max(float v) {
    return lane_reduce<kWave>(v, [](float a, float b) { return fmaxf(a, b); });
}

// N neighbouring elements, read or written as one access, which on this target may begin at
// any element.
template <typename T, int N>
struct Pack {
    typedef T aligned_type __attribute__((ext_vector_type(N)));
    typedef aligned_type type __attribute__((aligned(sizeof(T))));
};
template <typename T>
struct Pack<T, 1> {
    typedef T type;
};
template <typename T, int N>
__device__ __forceinline__ void load_floats(const T *p, float *v) {
    const auto x = *(const typename Pack<T, N>::type *)p;
    if constexpr (N == 1)
        v[0] = to_float(x);
    else
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = to_float((T)x[i]);
}
template <typename T, int N>
__device__ __forceinline__ void store_floats(T *p, const float *v) {
    typename Pack<T, N>::type x;
    if constexpr (N == 1)
        x = from_float<T>(v[0]);
    else
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = from_float<T>(v[i]);
    *(typename Pack<T, N>::type *)p = x;
}

// The same of the first n, where there are not N.  WHOLE: there are N or none.
template <bool WHOLE, typename T, int N>
__device__ __forceinline__ void load_first(const T *p, float *v, int n, float rest) {
    if (WHOLE ? n > 0 : n >= N) {
        load_floats<T, N>(p, v);
    } else if constexpr (WHOLE) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = rest;
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = i < n ? to_float(p[i]) : rest;
    }
}
template <bool WHOLE, typename T, int N>
__device__ __forceinline__ void store_first(T *p, const float *v, int n) {
    if (WHOLE ? n > 0 : n >= N) {
        store_floats<T, N>(p, v);
    } else if constexpr (!WHOLE) {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i < n) p[i] = from_float<T>(v[i]);
    }
}

}  // namespace gs
