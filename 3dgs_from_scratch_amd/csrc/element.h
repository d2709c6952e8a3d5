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
inline int element_size(int32_t t) { return t == GS_F32 ? 4 : 2; }

// Calls f with a value of the element type that `type` names.
template <typename F>
inline int with_element(int32_t type, F f) {
    switch (type) {
        case GS_F32: return f(float{});
        case GS_F16: return f(f16{});
        default: return f(bf16{});
    }
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int o = kWave / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, kWave);
    return v;
}

}  // namespace gs
