// elem.hip.h — loads and stores of f32, f16 and bf16 elements as f32. Every
// conversion to 16 bits rounds to nearest, ties to even.
//
// SPDX-License-Identifier: MIT
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

template <class T>
struct __attribute__((aligned(4 * sizeof(T)))) Elem4 {
    T e[4];
};

// Four consecutive elements; VEC: one aligned load or store.
template <bool VEC, class T>
static __device__ __forceinline__ void load4(const T *p, float *v) {
    if constexpr (VEC) {
        const Elem4<T> x = *(const Elem4<T> *)p;
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = (float)x.e[i];
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = (float)p[i];
    }
}

template <bool VEC, class T>
static __device__ __forceinline__ void store4(T *p, const float *v) {
    if constexpr (VEC) {
        Elem4<T> x;
#pragma unroll
        for (int i = 0; i < 4; i++) x.e[i] = (T)v[i];
        *(Elem4<T> *)p = x;
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) p[i] = (T)v[i];
    }
}
