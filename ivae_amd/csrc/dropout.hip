// Dropout whose mask is never stored:  y_e = residual_e + (keep_e ? x_e / (1 - p) : 0).
//
// keep_e = (word e % 4 of Philox4x32-10(counter = (e / 4, offset), key = seed)) >= floor(p * 2^32)   [Salmon et al. 2011].
// The draw depends on the element's number, the seed and the offset alone, so the backward pass calls the same kernel with the
// same three and gets the same mask, whatever the launch geometry.  A dropped element is not read into the result: NaN and
// infinities in dropped places leave no trace.
#include "kernels.h"
#include "ops_common.h"

struct DropArgs {
    const void* x;
    const void* residual;      // or null
    void* y;
    int64_t n;
    uint32_t thr;
    int all;                   // p = 1: nothing is kept
    float scale;
    uint32_t k0, k1;
    uint64_t offset;
    const int64_t* offset_dev; // or null; added to offset
    bool past;                 // y is stored past the caches
};

// high and low half of a * m from ONE wide multiply (v_mad_u64_u32)
__device__ __forceinline__ void mulhilo(uint32_t a, uint32_t m, uint32_t& hi, uint32_t& lo) {
    const uint64_t p = (uint64_t)a * m;
    hi = (uint32_t)(p >> 32);
    lo = (uint32_t)p;
}
__device__ __forceinline__ void philox(uint64_t q, uint64_t offset, uint32_t k0, uint32_t k1, uint32_t (&out)[4]) {
    uint32_t c0 = (uint32_t)q, c1 = (uint32_t)(q >> 32), c2 = (uint32_t)offset, c3 = (uint32_t)(offset >> 32);
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        uint32_t h0, l0, h1, l1;
        mulhilo(c0, 0xD2511F53u, h0, l0);
        mulhilo(c2, 0xCD9E8D57u, h1, l1);
        c0 = h1 ^ c1 ^ k0;
        c1 = l1;
        c2 = h0 ^ c3 ^ k1;
        c3 = l0;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    out[0] = c0; out[1] = c1; out[2] = c2; out[3] = c3;
}

template <typename T>
__global__ __launch_bounds__(256) void k_dropout(DropArgs A) {
    constexpr int N = Wide<T>::N;
    const uint64_t offset = A.offset + (A.offset_dev ? (uint64_t)*A.offset_dev : 0ull);
    const int64_t chunks = (A.n + N - 1) / N;
    for (int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x; c < chunks; c += (int64_t)gridDim.x * 256) {
        const int64_t e = c * N;
        const int left = A.n - e < N ? (int)(A.n - e) : N;
        float x[N], r[N];
        load_some<T>((const T*)A.x + e, left, x);
        if (A.residual) load_some<T>((const T*)A.residual + e, left, r);
#pragma unroll
        for (int g = 0; g < N / 4; ++g) {
            uint32_t w[4];
            philox((uint64_t)(e / 4 + g), offset, A.k0, A.k1, w);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float v = !A.all && w[j] >= A.thr ? x[g * 4 + j] * A.scale : 0.f;
                x[g * 4 + j] = A.residual ? r[g * 4 + j] + v : v;
            }
        }
        store_some<T>((T*)A.y + e, left, x, A.past);
    }
}

hipError_t launch_dropout(int dtype, int64_t n, const void* x, const void* residual, void* y, double p, uint64_t seed, uint64_t offset,
                          const int64_t* offset_dev, hipStream_t st) {
    if (n == 0) return hipSuccess;
    DropArgs A;
    A.x = x; A.residual = residual; A.y = y; A.n = n;
    A.all = p >= 1.0;
    A.thr = A.all ? 0u : (uint32_t)(p * 4294967296.0);
    A.scale = A.all ? 0.f : (float)(1.0 / (1.0 - p));
    A.k0 = (uint32_t)seed; A.k1 = (uint32_t)(seed >> 32);
    A.offset = offset; A.offset_dev = offset_dev;
    A.past = past_caches((double)n, dtype);
    const int per = dtype == IVAE_F32 ? 4 : 8;
    int64_t blocks = ((n + per - 1) / per + 255) / 256;
    if (blocks > 8192) blocks = 8192;
    const dim3 g((unsigned)blocks), b(256);
    if (dtype == IVAE_F32) hipLaunchKernelGGL(k_dropout<float>, g, b, 0, st, A);
    else if (dtype == IVAE_BF16) hipLaunchKernelGGL(k_dropout<bf16_t>, g, b, 0, st, A);
    else hipLaunchKernelGGL(k_dropout<f16_t>, g, b, 0, st, A);
    return hipGetLastError();
}
