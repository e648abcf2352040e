// Arguments and element functions shared by the kernels of the linear operator (linear*.hip).
#pragma once
#include "ops_common.h"

struct LinArgs {
    const void* x; const void* w; const void* b; const void* res;
    void* y; float* pre;                   // forward; pre: or null, the pre-activations in 32 bits for the backward pass
    const void* dy; const float* cpre;     // backward
    void* dx; void* dw; void* db;
    int64_t M, ldx, ldr, lddy;
    int K, N;
    int act;
    float slope;
    float* part;                           // partial sums of a split reduction
};

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef bf16_t bf16x8 __attribute__((ext_vector_type(8)));
typedef f16_t f16x8 __attribute__((ext_vector_type(8)));

// Activations of 16-bit results from the hardware's exp2 and reciprocal (1 unit in the last place of 32 bits each): relative errors of a
// few 2^-24, and for each factor exp(-x) x 2^-23 more (2^-16 at gelu's smallest bf16 results), next to half steps of 2^-12 and 2^-9 relative to
// the result; an epilogue of 128 values a lane costs a third of what the exact forms do.
__device__ __forceinline__ float fast_exp(float x) { return __builtin_amdgcn_exp2f(x * 1.4426950408889634f); }
__device__ __forceinline__ float fast_sigmoid(float s) { return __builtin_amdgcn_rcpf(1.f + fast_exp(-s)); }
__device__ __forceinline__ float fast_tanh(float s) {
    const float a = fabsf(s), q = s * s;
    const float near = s * (1.f + q * (-1.f / 3.f + q * (2.f / 15.f - q * (17.f / 315.f))));          // Taylor: 2e-10 at 0.1
    const float far = copysignf(1.f - 2.f * __builtin_amdgcn_rcpf(1.f + fast_exp(2.f * a)), s);
    return a < 0.1f ? near : far;
}
// 1 + erf(s / sqrt 2) (twice the normal distribution): erfc(a) exp(a^2) = t P(t), t = 1 / (1 + 0.42 a), P fitted to the least relative error
// over 0 <= a <= 9.6, 1.8e-7, so that what is left of the tail below 0 keeps its digits; in 32 bits 5e-7 near 0, 8e-6 at the end, from exp
__device__ __forceinline__ float fast_cdf2(float s) {
    const float a = fabsf(s) * 0.70710678118654752f, t = __builtin_amdgcn_rcpf(1.f + 0.42f * a);
    const float p = 0.23682660f + t * (0.23955022f + t * (0.19494417f + t * (0.26803513f + t * (-0.12920924f + t * (0.43926111f + t * (-0.31944717f +
                    t * 0.070038993f))))));
    const float tail = t * p * fast_exp(-a * a);
    return s < 0.f ? tail : 2.f - tail;
}
template <typename T>
__device__ __forceinline__ float lin_act(int act, float slope, float s) {
    constexpr bool fast = sizeof(T) == 2;
    switch (act) {
        case IVAE_ACT_LRELU: return s > 0.f ? s : slope * s;
        case IVAE_ACT_XTANH: return (fast ? fast_tanh(s) : tanhf(s)) + slope * s;
        case IVAE_ACT_SIGMOID: return fast ? fast_sigmoid(s) : 1.f / (1.f + expf(-s));
        case IVAE_ACT_GELU: return 0.5f * s * (fast ? fast_cdf2(s) : erfcf(s * -0.70710678118654752f));     // (1 + erf would cancel below 0)
        case IVAE_ACT_SILU: return fast ? s * fast_sigmoid(s) : s / (1.f + expf(-s));
        default: return s;
    }
}
// sigmoid'(s) = e / (1 + e)^2, e = exp(-s), for s >= 0 (it is even): sigmoid (1 - sigmoid) would lose the digits of what is left of 1
template <bool FAST> __device__ __forceinline__ float logistic_slope(float s) {
    const float e = FAST ? fast_exp(-s) : expf(-s), r = FAST ? __builtin_amdgcn_rcpf(1.f + e) : 1.f / (1.f + e);
    return e * r * r;
}
template <typename T>
__device__ __forceinline__ float lin_act_slope(int act, float slope, float s) {
    constexpr bool fast = sizeof(T) == 2;
    switch (act) {
        case IVAE_ACT_LRELU: return s > 0.f ? 1.f : slope;
        case IVAE_ACT_XTANH: return 4.f * logistic_slope<fast>(2.f * fabsf(s)) + slope;          // 1 - tanh^2
        case IVAE_ACT_SIGMOID: return logistic_slope<fast>(fabsf(s));
        case IVAE_ACT_GELU:
            return 0.5f * (fast ? fast_cdf2(s) : erfcf(s * -0.70710678118654752f)) +
                   s * (fast ? fast_exp(-0.5f * s * s) : expf(-0.5f * s * s)) * 0.39894228040143268f;
        case IVAE_ACT_SILU: { const float t = fast ? fast_sigmoid(s) : 1.f / (1.f + expf(-s)); return t * (1.f + s * (1.f - t)); }
        default: return 1.f;
    }
}

// over N values, the switch outside of the loop over them
template <typename T, int N> __device__ __forceinline__ void lin_act_all(int act, float slope, float (&v)[N]) {
    switch (act) {
#define EACH(ID) case ID: _Pragma("unroll") for (int e = 0; e < N; ++e) v[e] = lin_act<T>(ID, slope, v[e]); break;
        EACH(IVAE_ACT_LRELU) EACH(IVAE_ACT_XTANH) EACH(IVAE_ACT_SIGMOID) EACH(IVAE_ACT_GELU) EACH(IVAE_ACT_SILU)
#undef EACH
    }
}
// v *= act'(s)
template <typename T, int N> __device__ __forceinline__ void lin_act_slope_all(int act, float slope, const float (&s)[N], float (&v)[N]) {
    switch (act) {
#define EACH(ID) case ID: _Pragma("unroll") for (int e = 0; e < N; ++e) v[e] *= lin_act_slope<T>(ID, slope, s[e]); break;
        EACH(IVAE_ACT_LRELU) EACH(IVAE_ACT_XTANH) EACH(IVAE_ACT_SIGMOID) EACH(IVAE_ACT_GELU) EACH(IVAE_ACT_SILU)
#undef EACH
    }
}

// 8 neighbouring values as they lie in memory, `n` of them inside the matrix
template <typename T> struct Raw8 {
    Vec<T> v[8 / Wide<T>::N];
    __device__ __forceinline__ void load(const T* p, int n) {
        constexpr int N = Wide<T>::N;
#pragma unroll
        for (int h = 0; h < 8 / N; ++h) {
            if (n >= (h + 1) * N) v[h] = *(const Vec<T>*)(p + h * N);
            else
#pragma unroll
                for (int j = 0; j < N; ++j) v[h].e[j] = n > h * N + j ? p[h * N + j] : (T)0.f;
        }
    }
    __device__ __forceinline__ float at(int e) const { return to_f(v[e / Wide<T>::N].e[e % Wide<T>::N]); }
};
template <typename T> __device__ __forceinline__ void store8(T* p, int n, const float (&v)[8]) {
    constexpr int N = Wide<T>::N;
#pragma unroll
    for (int h = 0; h < 8 / N; ++h) {
        float u[N];
#pragma unroll
        for (int j = 0; j < N; ++j) u[j] = v[h * N + j];
        store_some<T>(p + h * N, n - h * N, u);
    }
}

// What follows the sums of 8 neighbouring results (bias included, n of them inside the matrix, the first at element `at` of y).
template <typename T>
__device__ __forceinline__ void forward_store8(const LinArgs& A, int64_t at, int n, float (&v)[8], const Raw8<T>* res) {
    if (A.pre && n) store8(A.pre + at, n, v);
    lin_act_all<T>(A.act, A.slope, v);
    if (res)
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += res->at(e);
    if (n) store8((T*)A.y + at, n, v);
}
// what follows the sum of one result
template <typename T>
__device__ __forceinline__ void forward_store(const LinArgs& A, int64_t m, int n, float s) {
    if (A.b) s += to_f(((const T*)A.b)[n]);
    if (A.pre) A.pre[m * A.N + n] = s;
    s = lin_act<T>(A.act, A.slope, s);
    if (A.res) s += to_f(((const T*)A.res)[m * A.ldr + n]);
    ((T*)A.y)[m * A.N + n] = from_f<T>(s);
}

hipError_t linear_small_forward(const LinArgs& A, int dtype, hipStream_t st);
hipError_t linear_small_backward(const LinArgs& A, int dtype, hipStream_t st);
size_t linear_small_ws(const LinArgs& A, bool backward);
void linear_small_splits(const LinArgs& A, bool backward, int32_t* splits);     // two of them: y or dx, dw

// sums of split parts: kx, kw of them where there are two or more, kb where there is one (db is not written before the join)
struct LinParts { const float* x; const float* w; const float* b; int kx, kw, kb; };
hipError_t linear_join_forward(const LinArgs& A, int splits, int dtype, hipStream_t st);
hipError_t linear_join_backward(const LinArgs& A, const LinParts& J, int dtype, hipStream_t st);
