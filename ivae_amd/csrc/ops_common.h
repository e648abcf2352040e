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
// `past`: past the caches
template <typename T, int N> __device__ __forceinline__ void store_wide(T* p, const float (&in)[N], bool past = false) {
    static_assert(N == Wide<T>::N, "one 16-byte store");
    Vec<T> v;
#pragma unroll
    for (int j = 0; j < N; ++j) v.e[j] = from_f<T>(in[j]);
    typedef uint32_t u4 __attribute__((ext_vector_type(4), aligned(2)));
    if (past) {
        asm volatile("");                                // (without these, both stores become one that goes through the caches)
        __builtin_nontemporal_store(__builtin_bit_cast(u4, v), reinterpret_cast<u4*>(p));
        asm volatile("");
    } else *reinterpret_cast<Vec<T>*>(p) = v;
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
template <typename T, int N> __device__ __forceinline__ void store_some(T* p, int n, const float (&in)[N], bool past = false) {
    if (n >= N) store_wide<T>(p, in, past);
    else store_part<T>(p, n, in);
}

// Elementwise results from 96 MB on are stored past the caches: together with its operands such a tensor does not stay in the 256 MB cache
// for its reader anyway, and then leaves the operands there.  (layer_norm, dropout with residual and both gradients, one after the other,
// us, through | past the caches: tensors of 32 MB 78 | 83, 64 MB 136 | 143, 128 MB bf16 295 | 258, 128 MB fp32 273 | 242, 256 MB 582 | 532.)
static inline bool past_caches(double elements, int dt) { return elements * (dt == IVAE_F32 ? 4 : 2) >= 96 * 1048576.0; }

static inline size_t dtype_size(int dt) { return dt == IVAE_F32 ? 4 : 2; }
