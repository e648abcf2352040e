// The forward product for few rows (single tokens, small batches): all of it is reading the weight once.
//
// A block takes 16 NF rows of the weight, its 8 waves the summed index in 8 runs; a wave loads its part of the weight from memory
// straight into the registers of the matrix instruction (first operand: 16 weight rows; second: 16 rows of x, MF of them), U loads in
// flight before the first product waits.  No LDS but for the sum over the waves.  With few weight rows the summed index is split over
// blocks too, and the parts are added in order by the join of the small kernel.
#include "kernels.h"
#include "linear_rows.h"

static constexpr int WAVES = 8;

template <typename T> struct Frag { typedef T t __attribute__((ext_vector_type(8))); static constexpr int K = 32; };
template <> struct Frag<float> { typedef f32x4 t; static constexpr int K = 16; };      // K: of the summed index, that 64 lanes' 16 bytes cover

__device__ __forceinline__ f32x4 mma(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 mma(f16x8 a, f16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 mma(f32x4 a, f32x4 b, f32x4 c) {                       // (the same order of the summed index on both sides)
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
    return c;
}
// 16 bytes of a row from k on, zeros from `end` on or where the row does not exist
template <typename T> __device__ __forceinline__ typename Frag<T>::t fetch(const T* row, int k, int end, bool live) {
    constexpr int N = Wide<T>::N;
    typename Frag<T>::t v;
    if (live && k + N <= end) {
        const Vec<T> u = *(const Vec<T>*)(row + k);
        __builtin_memcpy(&v, &u, sizeof(v));
    } else
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = live && k + e < end ? row[k + e] : (T)0.f;
    return v;
}

template <typename T, int MF, int NF>
__global__ __launch_bounds__(WAVES * 64) void k_linear_rows(LinArgs A, int len, int splits) {
    constexpr int FK = Frag<T>::K, N = Wide<T>::N, U = MF + NF <= 3 ? 8 : MF + NF <= 5 ? 4 : 2;
    __shared__ float sums[WAVES][MF * 16][NF * 16 + 1];
    const int l = threadIdx.x % 64, wave = threadIdx.x / 64, i = l % 16, g = l / 16;
    const int n0 = blockIdx.x * (16 * NF), split = blockIdx.y;
    const int ka = split * len, kb = ka + len < A.K ? ka + len : A.K;
    const int run = ((kb - ka + WAVES - 1) / WAVES + FK - 1) / FK * FK;
    const int k0 = ka + wave * run, k1 = k0 + run < kb ? k0 + run : kb;
    const T* x[MF];
    const T* w[NF];
    bool lx[MF], lw[NF];
#pragma unroll
    for (int m = 0; m < MF; ++m) {
        lx[m] = m * 16 + i < A.M;
        x[m] = (const T*)A.x + (lx[m] ? m * 16 + i : 0) * A.ldx;
    }
#pragma unroll
    for (int n = 0; n < NF; ++n) {
        lw[n] = n0 + n * 16 + i < A.N;
        w[n] = (const T*)A.w + (int64_t)(lw[n] ? n0 + n * 16 + i : 0) * A.K;
    }
    f32x4 acc[MF][NF];
#pragma unroll
    for (int m = 0; m < MF; ++m)
#pragma unroll
        for (int n = 0; n < NF; ++n) acc[m][n] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int k = k0; k < k1; k += U * FK) {
        typename Frag<T>::t fx[U][MF], fw[U][NF];
        if (k + U * FK <= k1) {             // (wave-uniform: no lane ends inside)
#pragma unroll
            for (int u = 0; u < U; ++u) {
#pragma unroll
                for (int n = 0; n < NF; ++n) {
                    const Vec<T> v = *(const Vec<T>*)(w[n] + k + u * FK + g * N);
                    __builtin_memcpy(&fw[u][n], &v, sizeof(v));
                }
#pragma unroll
                for (int m = 0; m < MF; ++m) {
                    const Vec<T> v = *(const Vec<T>*)(x[m] + k + u * FK + g * N);
                    __builtin_memcpy(&fx[u][m], &v, sizeof(v));
                }
            }
        } else {
#pragma unroll
            for (int u = 0; u < U; ++u) {
#pragma unroll
                for (int n = 0; n < NF; ++n) fw[u][n] = fetch<T>(w[n], k + u * FK + g * N, k1, lw[n]);
#pragma unroll
                for (int m = 0; m < MF; ++m) fx[u][m] = fetch<T>(x[m], k + u * FK + g * N, k1, lx[m]);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int m = 0; m < MF; ++m)
#pragma unroll
                for (int n = 0; n < NF; ++n) acc[m][n] = mma(fw[u][n], fx[u][m], acc[m][n]);
    }
    // rows that do not exist repeated row 0: their results are not stored
#pragma unroll
    for (int m = 0; m < MF; ++m)
#pragma unroll
        for (int n = 0; n < NF; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) sums[wave][m * 16 + i][n * 16 + g * 4 + e] = acc[m][n][e];
    __syncthreads();
    for (int c = threadIdx.x; c < MF * 16 * NF * 16; c += WAVES * 64) {
        const int m = c / (NF * 16), n = c % (NF * 16);
        if (m >= A.M || n0 + n >= A.N) continue;
        float s = 0.f;
#pragma unroll
        for (int v = 0; v < WAVES; ++v) s += sums[v][m][n];
        if (splits > 1) A.part[((int64_t)split * A.M + m) * A.N + n0 + n] = s;
        else forward_store<T>(A, m, n0 + n, s);
    }
}

// Up to 64 rows, the most that a block's registers hold; fp32 up to 32 where blocks of 16 weight rows (below) read x too often for its slower
// matrix instructions (us, here | on 64 x 64 tiles: fp16 64 x 1024 x 1024 6.9 | 9.5, 64 x 2048 x 8192 14 | 22, 64 x 4096 x 4096 21 | 22, 64 x 8192 x
// 2048 24 | 22; fp32 32 x 4096 x 4096 29 | 31, 33 x 4096 x 4096 39 | 35, 64 x 4096 x 4096 46 | 31, 64 x 1024 x 1024 13 | 11, 64 x 200 x 200 6.7 | 11,
// 64 x 2048 x 8192 30 | 31)
bool rows_serve(const LinArgs& A, int dtype) { return A.M <= (dtype == IVAE_F32 && A.K >= 1024 && A.N <= 4096 ? 32 : 64); }
// 32 weight rows a block, which halves what is read of x, where blocks of 16 would be more than the chip has CUs (us, 16 | 32 weight rows: fp16
// 24 x 2048 x 4096 7.1 | 8.7, 24 x 2048 x 6000 12.5 | 9.6, 64 x 2048 x 4096 12.0 | 11.5, 64 x 2048 x 6000 22 | 14, 64 x 4096 x 16384 78 | 45; fp32
// 24 x 2048 x 4096 13.7 | 14.8, 24 x 2048 x 6000 25.9 | 21.3, 64 x 2048 x 8192 47 | 30); up to 16 rows read little of it
static int rows_nf(const LinArgs& A) { return A.M > 16 && A.N > 4096 ? 2 : 1; }
RowsPlan rows_plan(const LinArgs& A) {
    RowsPlan p;
    p.nf = rows_nf(A);
    const int blocks = (int)((A.N + 16 * p.nf - 1) / (16 * p.nf));
    int s = blocks < 256 ? 256 / blocks : 1;
    if (s > A.K / 1024) s = A.K / 1024;
    if (s < 1) s = 1;
    p.len = ((A.K + s - 1) / s + 255) / 256 * 256;
    p.splits = (A.K + p.len - 1) / p.len;
    return p;
}
size_t rows_ws(const LinArgs& A) {
    const RowsPlan p = rows_plan(A);
    return p.splits > 1 ? (size_t)p.splits * A.M * A.N * 4 : 0;
}
template <typename T> static void launch(const LinArgs& A, const RowsPlan& p, hipStream_t st) {
    const dim3 g((unsigned)((A.N + 16 * p.nf - 1) / (16 * p.nf)), p.splits), b(WAVES * 64);
    if (A.M <= 16) hipLaunchKernelGGL((k_linear_rows<T, 1, 1>), g, b, 0, st, A, p.len, p.splits);
    else if (A.M <= 32 && p.nf == 2) hipLaunchKernelGGL((k_linear_rows<T, 2, 2>), g, b, 0, st, A, p.len, p.splits);
    else if (A.M <= 32) hipLaunchKernelGGL((k_linear_rows<T, 2, 1>), g, b, 0, st, A, p.len, p.splits);
    else if (p.nf == 2) hipLaunchKernelGGL((k_linear_rows<T, 4, 2>), g, b, 0, st, A, p.len, p.splits);
    else hipLaunchKernelGGL((k_linear_rows<T, 4, 1>), g, b, 0, st, A, p.len, p.splits);
}
hipError_t linear_rows_forward(const LinArgs& A, int dtype, hipStream_t st) {
    const RowsPlan p = rows_plan(A);
    if (dtype == IVAE_F32) launch<float>(A, p, st);
    else if (dtype == IVAE_BF16) launch<bf16_t>(A, p, st);
    else launch<f16_t>(A, p, st);
    const hipError_t e = hipGetLastError();
    return e != hipSuccess ? e : linear_join_forward(A, p.splits, dtype, st);
}
