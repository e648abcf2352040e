// Shared by the tensor operators (dropout.hip, norm.hip, linear*.hip): element types, wide loads that ask for no alignment
// beyond an element's, rounding, activations.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include "../../include/ivae_amd.h"

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

template <typename T> struct Wide;                     // elements of one 16-byte load
template <> struct Wide<float> { static constexpr int N = 4; };
template <> struct Wide<bf16_t> { static constexpr int N = 8; };
template <> struct Wide<f16_t> { static constexpr int N = 8; };

// 16 bytes at an address that is a multiple of the element's size only: gfx950 serves a misaligned global_load_dwordx4 (at the
// price of the cache lines that it touches), so rows of odd width need no loads of single elements.
template <typename T> struct __attribute__((packed, aligned(sizeof(T)))) Vec { T e[Wide<T>::N]; };

template <typename T> __device__ __forceinline__ float to_f(T v) { return (float)v; }
template <typename T> __device__ __forceinline__ T from_f(float v) { return (T)v; }    // rounds to nearest even

template <typename T, int N> __device__ __forceinline__ void load_wide(const T* p, float (&out)[N]) {
    static_assert(N == Wide<T>::N, "one 16-byte load");
    const Vec<T> v = *reinterpret_cast<const Vec<T>*>(p);
#pragma unroll
    for (int j = 0; j < N; ++j) out[j] = to_f(v.e[j]);
}
template <typename T, int N> __device__ __forceinline__ void store_wide(T* p, const float (&in)[N]) {
    static_assert(N == Wide<T>::N, "one 16-byte store");
    Vec<T> v;
#pragma unroll
    for (int j = 0; j < N; ++j) v.e[j] = from_f<T>(in[j]);
    *reinterpret_cast<Vec<T>*>(p) = v;
}
// the first `n` (0 < n < N) of them
template <typename T, int N> __device__ __forceinline__ void load_part(const T* p, int n, float (&out)[N]) {
#pragma unroll
    for (int j = 0; j < N; ++j) out[j] = j < n ? to_f(p[j]) : 0.f;
}
template <typename T, int N> __device__ __forceinline__ void store_part(T* p, int n, const float (&in)[N]) {
#pragma unroll
    for (int j = 0; j < N; ++j)
        if (j < n) p[j] = from_f<T>(in[j]);
}
template <typename T, int N> __device__ __forceinline__ void load_some(const T* p, int n, float (&out)[N]) {
    if (n >= N) load_wide<T>(p, out);
    else load_part<T>(p, n, out);
}
template <typename T, int N> __device__ __forceinline__ void store_some(T* p, int n, const float (&in)[N]) {
    if (n >= N) store_wide<T>(p, in);
    else store_part<T>(p, n, in);
}

static inline size_t dtype_size(int dt) { return dt == IVAE_F32 ? 4 : 2; }
