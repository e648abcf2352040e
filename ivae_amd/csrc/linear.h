// Arguments and element functions shared by the kernels of the linear operator (linear*.hip).
#pragma once
#include "ops_common.h"

struct LinArgs {
    const void* x; const void* w; const void* b; const void* res;
    void* y; void* pre;                    // forward
    const void* dy; const void* cpre;      // backward
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

// What the forward pass keeps of the pre-activation s for the backward pass's act'(s): 32 bits, but for bf16 operands fp16 --
// act' is a function of moderate s, where fp16 has 3 bits more than the gradients around it.  |s| beyond fp16's range is clamped
// (act' has reached its limit there) and a positive s never becomes 0, so lrelu's side is kept.  (For fp16 operands fp16 would
// add an error as large as that of rounding a gradient: x 1.5 together where 32 bits stay at x 1.41.)
template <typename T> struct Pre { typedef float t; };
template <> struct Pre<bf16_t> { typedef f16_t t; };
__device__ __forceinline__ float pre_pack(float s, float) { return s; }
__device__ __forceinline__ f16_t pre_pack(float s, f16_t) {
    if (s != s) return (f16_t)s;
    const f16_t h = (f16_t)fminf(fmaxf(s, -65504.f), 65504.f);
    return s > 0.f && h == (f16_t)0.f ? (f16_t)5.9604645e-8f : h;
}

__device__ __forceinline__ float lin_act(int act, float slope, float s) {
    switch (act) {
        case IVAE_ACT_LRELU: return s > 0.f ? s : slope * s;
        case IVAE_ACT_XTANH: return tanhf(s) + slope * s;
        case IVAE_ACT_SIGMOID: return 1.f / (1.f + expf(-s));
        case IVAE_ACT_GELU: return 0.5f * s * (1.f + erff(s * 0.70710678118654752f));
        case IVAE_ACT_SILU: return s / (1.f + expf(-s));
        default: return s;
    }
}
__device__ __forceinline__ float lin_act_slope(int act, float slope, float s) {
    switch (act) {
        case IVAE_ACT_LRELU: return s > 0.f ? 1.f : slope;
        case IVAE_ACT_XTANH: { const float t = tanhf(s); return (1.f - t * t) + slope; }
        case IVAE_ACT_SIGMOID: { const float t = 1.f / (1.f + expf(-s)); return t * (1.f - t); }
        case IVAE_ACT_GELU:
            return 0.5f * (1.f + erff(s * 0.70710678118654752f)) + s * expf(-0.5f * s * s) * 0.39894228040143268f;
        case IVAE_ACT_SILU: { const float t = 1.f / (1.f + expf(-s)); return t * (1.f + s * (1.f - t)); }
        default: return 1.f;
    }
}

hipError_t linear_small_forward(const LinArgs& A, int dtype, hipStream_t st);
hipError_t linear_small_backward(const LinArgs& A, int dtype, hipStream_t st);
size_t linear_small_ws(const LinArgs& A, bool backward);
