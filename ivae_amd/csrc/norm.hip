// Layer norm over the last dimension, forward and backward.
//   forward   y = (x - mean) r g + c,  r = 1 / sqrt(var + eps); (mean, r) of a row are kept for the backward pass
//   backward  xh = (x - mean) r, a = dy g:   dx = r (a - mean(a) - xh mean(a xh)) [+ residual],  dg = sum_rows dy xh,  dc = sum_rows dy
// Both are bound by memory: a row is read once, held in registers by the TPR threads that share it (16 elements each), and the
// variance is summed from the centred values in those registers, so it does not cancel.  All sums are in 32 bits and in a fixed order.
#include "kernels.h"
#include "ops_common.h"

static constexpr int EPT = 16;                 // elements a thread holds of a row
static constexpr int NORM_MAX_D = 1024 * EPT;  // wider rows are walked instead of held

struct NormArgs {
    const void* x; const void* dy; const void* w; const void* b; const void* residual;
    void* y; float* stats;                     // stats: (2, rows): mean, r
    const float* cstats;
    float* part;                               // backward: (blocks, 2, D) sums of dy xh and dy
    int64_t rows, ldx, lddy, ldr;
    int D, w_f32;
    float eps;
};

__device__ __forceinline__ float wload(const void* w, int w_f32, int i, bool half_is_bf16) {
    if (w_f32) return ((const float*)w)[i];
    return half_is_bf16 ? to_f(((const bf16_t*)w)[i]) : to_f(((const f16_t*)w)[i]);
}
template <typename T> struct IsBf16 { static constexpr bool v = false; };
template <> struct IsBf16<bf16_t> { static constexpr bool v = true; };

// sums of K values over the TPR threads that share a row; every thread of the block calls it together
template <int TPR, int K, int BLOCK>
__device__ __forceinline__ void row_sum(float (&v)[K], float* lds) {
#pragma unroll
    for (int o = (TPR < 64 ? TPR : 64) / 2; o > 0; o >>= 1)
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] += __shfl_xor(v[k], o);
    if constexpr (TPR > 64) {
        constexpr int NW = TPR / 64;
        const int wave = threadIdx.x / 64;
        __syncthreads();                       // the last use of lds is over
        if (threadIdx.x % 64 == 0)
#pragma unroll
            for (int k = 0; k < K; ++k) lds[wave * K + k] = v[k];
        __syncthreads();
        const int w0 = wave / NW * NW;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            float s = 0.f;
#pragma unroll
            for (int w = 0; w < NW; ++w) s += lds[(w0 + w) * K + k];
            v[k] = s;
        }
    }
}

template <typename T, int TPR>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void k_norm_fwd(NormArgs A) {
    constexpr int N = Wide<T>::N, C = EPT / N, BLOCK = TPR > 256 ? TPR : 256;
    __shared__ float lds[BLOCK / 64];
    const int t = threadIdx.x % TPR;
    for (int64_t r0 = (int64_t)blockIdx.x * (BLOCK / TPR); r0 < A.rows; r0 += (int64_t)gridDim.x * (BLOCK / TPR)) {
        const int64_t row = r0 + threadIdx.x / TPR;
        const bool live = row < A.rows;
        const T* x = (const T*)A.x + (live ? row : 0) * A.ldx;
        float v[C][N];
        float s[1] = {0.f};
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int e = (c * TPR + t) * N;
            if (live && e < A.D) load_some<T>(x + e, A.D - e, v[c]);
            else
#pragma unroll
                for (int j = 0; j < N; ++j) v[c][j] = 0.f;
#pragma unroll
            for (int j = 0; j < N; ++j) s[0] += v[c][j];
        }
        row_sum<TPR, 1, BLOCK>(s, lds);
        const float mean = s[0] / (float)A.D;
        float q[1] = {0.f};
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int e = (c * TPR + t) * N;
#pragma unroll
            for (int j = 0; j < N; ++j) {
                v[c][j] -= mean;
                if (e + j < A.D) q[0] += v[c][j] * v[c][j];
            }
        }
        row_sum<TPR, 1, BLOCK>(q, lds);
        const float r = 1.f / sqrtf(q[0] / (float)A.D + A.eps);
        if (!live) continue;                    // (after the row's last barrier)
        if (A.stats && t == 0) {
            A.stats[row] = mean;
            A.stats[A.rows + row] = r;
        }
        T* y = (T*)A.y + row * A.D;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int e = (c * TPR + t) * N;
            if (e >= A.D) break;
            float o[N];
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const int i = e + j < A.D ? e + j : A.D - 1;
                const float g = A.w ? wload(A.w, A.w_f32, i, IsBf16<T>::v) : 1.f, b = A.b ? wload(A.b, A.w_f32, i, IsBf16<T>::v) : 0.f;
                o[j] = v[c][j] * r * g + b;
            }
            store_some<T>(y + e, A.D - e, o);
        }
    }
}

// rows wider than the registers of a block: walked three times (the second and third time from the cache)
template <typename T>
__global__ __launch_bounds__(1024) void k_norm_fwd_wide(NormArgs A) {
    __shared__ float lds[16];
    for (int64_t row = blockIdx.x; row < A.rows; row += gridDim.x) {
        const T* x = (const T*)A.x + row * A.ldx;
        float s[1] = {0.f};
        for (int i = threadIdx.x; i < A.D; i += 1024) s[0] += to_f(x[i]);
        row_sum<1024, 1, 1024>(s, lds);
        const float mean = s[0] / (float)A.D;
        float q[1] = {0.f};
        for (int i = threadIdx.x; i < A.D; i += 1024) {
            const float d = to_f(x[i]) - mean;
            q[0] += d * d;
        }
        row_sum<1024, 1, 1024>(q, lds);
        const float r = 1.f / sqrtf(q[0] / (float)A.D + A.eps);
        if (A.stats && threadIdx.x == 0) {
            A.stats[row] = mean;
            A.stats[A.rows + row] = r;
        }
        T* y = (T*)A.y + row * A.D;
        for (int i = threadIdx.x; i < A.D; i += 1024) {
            const float g = A.w ? wload(A.w, A.w_f32, i, IsBf16<T>::v) : 1.f, b = A.b ? wload(A.b, A.w_f32, i, IsBf16<T>::v) : 0.f;
            y[i] = from_f<T>((to_f(x[i]) - mean) * r * g + b);
        }
    }
}

// dx, and each block's sums of dy xh and dy over the rows it walks (block, block + grid, ...)
template <typename T, int TPR>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void k_norm_bwd(NormArgs A) {
    constexpr int N = Wide<T>::N, C = EPT / N, BLOCK = TPR > 256 ? TPR : 256, RPB = BLOCK / TPR;
    __shared__ float lds[BLOCK / 64 * 2];
    __shared__ float fold[RPB > 1 ? TPR * EPT * 2 : 1];
    const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR;
    float g[C][N], dg[C][N], dc[C][N];
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int i = (c * TPR + t) * N + j;
            g[c][j] = i < A.D ? (A.w ? wload(A.w, A.w_f32, i, IsBf16<T>::v) : 1.f) : 0.f;
            dg[c][j] = dc[c][j] = 0.f;
        }
    const float inv = 1.f / (float)A.D;
    for (int64_t r0 = (int64_t)blockIdx.x * RPB; r0 < A.rows; r0 += (int64_t)gridDim.x * RPB) {
        const int64_t row = r0 + sub;
        const bool live = row < A.rows;
        const T* x = (const T*)A.x + (live ? row : 0) * A.ldx;
        const T* dy = (const T*)A.dy + (live ? row : 0) * A.lddy;
        const float mean = live ? A.cstats[row] : 0.f, r = live ? A.cstats[A.rows + row] : 0.f;
        float xh[C][N], d[C][N];
        float s[2] = {0.f, 0.f};
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int e = (c * TPR + t) * N;
            if (live && e < A.D) {
                load_some<T>(x + e, A.D - e, xh[c]);
                load_some<T>(dy + e, A.D - e, d[c]);
            } else
#pragma unroll
                for (int j = 0; j < N; ++j) xh[c][j] = d[c][j] = 0.f;
#pragma unroll
            for (int j = 0; j < N; ++j) {
                xh[c][j] = live && e + j < A.D ? (xh[c][j] - mean) * r : 0.f;
                dg[c][j] += d[c][j] * xh[c][j];
                dc[c][j] += d[c][j];
                d[c][j] *= g[c][j];
                s[0] += d[c][j];
                s[1] += d[c][j] * xh[c][j];
            }
        }
        row_sum<TPR, 2, BLOCK>(s, lds);
        if (live && A.y) {
            const float m1 = s[0] * inv, m2 = s[1] * inv;
            T* dx = (T*)A.y + row * A.D;
            const T* add = A.residual ? (const T*)A.residual + row * A.ldr : nullptr;
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const int e = (c * TPR + t) * N;
                if (e >= A.D) break;
                float o[N], q[N];
                if (add) load_some<T>(add + e, A.D - e, q);
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    o[j] = r * (d[c][j] - m1 - xh[c][j] * m2);
                    if (add) o[j] += q[j];
                }
                store_some<T>(dx + e, A.D - e, o);
            }
        }
    }
    if (!A.part) return;
    float* part = A.part + (int64_t)blockIdx.x * 2 * A.D;
    if constexpr (RPB > 1) {                    // the rows of a block meet in LDS, one after the other
        for (int s = 0; s < RPB; ++s) {
            if (sub == s)
#pragma unroll
                for (int c = 0; c < C; ++c)
#pragma unroll
                    for (int j = 0; j < N; ++j) {
                        const int i = (c * TPR + t) * N + j;
                        fold[i] = s ? fold[i] + dg[c][j] : dg[c][j];
                        fold[TPR * EPT + i] = s ? fold[TPR * EPT + i] + dc[c][j] : dc[c][j];
                    }
            __syncthreads();
        }
        for (int i = threadIdx.x; i < A.D; i += BLOCK) {
            part[i] = fold[i];
            part[A.D + i] = fold[TPR * EPT + i];
        }
    } else {
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const int i = (c * TPR + t) * N + j;
                if (i < A.D) {
                    part[i] = dg[c][j];
                    part[A.D + i] = dc[c][j];
                }
            }
    }
}

template <typename T>
__global__ __launch_bounds__(1024) void k_norm_bwd_wide(NormArgs A) {
    __shared__ float lds[32];
    for (int64_t row = blockIdx.x; row < A.rows; row += gridDim.x) {
        const T* x = (const T*)A.x + row * A.ldx;
        const T* dy = (const T*)A.dy + row * A.lddy;
        const float mean = A.cstats[row], r = A.cstats[A.rows + row];
        float s[2] = {0.f, 0.f};
        for (int i = threadIdx.x; i < A.D; i += 1024) {
            const float a = to_f(dy[i]) * (A.w ? wload(A.w, A.w_f32, i, IsBf16<T>::v) : 1.f);
            s[0] += a;
            s[1] += a * ((to_f(x[i]) - mean) * r);
        }
        row_sum<1024, 2, 1024>(s, lds);
        const float m1 = s[0] / (float)A.D, m2 = s[1] / (float)A.D;
        T* dx = (T*)A.y + row * A.D;
        for (int i = threadIdx.x; i < A.D; i += 1024) {
            const float a = to_f(dy[i]) * (A.w ? wload(A.w, A.w_f32, i, IsBf16<T>::v) : 1.f);
            float o = r * (a - m1 - (to_f(x[i]) - mean) * r * m2);
            if (A.residual) o += to_f(((const T*)A.residual)[row * A.ldr + i]);
            dx[i] = from_f<T>(o);
        }
    }
}
// column sums of wide rows: a block takes 64 columns and every gridDim.y-th row
template <typename T>
__global__ __launch_bounds__(256) void k_norm_cols_wide(NormArgs A) {
    __shared__ float fold[2][4][64];
    const int l = threadIdx.x % 64, w = threadIdx.x / 64, i = blockIdx.x * 64 + l;
    float dg = 0.f, dc = 0.f;
    if (i < A.D)
        for (int64_t row = (int64_t)blockIdx.y * 4 + w; row < A.rows; row += (int64_t)gridDim.y * 4) {
            const float d = to_f(((const T*)A.dy)[row * A.lddy + i]);
            dg += d * ((to_f(((const T*)A.x)[row * A.ldx + i]) - A.cstats[row]) * A.cstats[A.rows + row]);
            dc += d;
        }
    fold[0][w][l] = dg;
    fold[1][w][l] = dc;
    __syncthreads();
    if (w < 2 && i < A.D) A.part[((int64_t)blockIdx.y * 2 + w) * A.D + i] = fold[w][0][l] + fold[w][1][l] + fold[w][2][l] + fold[w][3][l];
}

// dg, dc from the blocks' sums: 32 columns a block, 32 interleaved walks over the blocks with eight loads in flight, joined in a fixed order
template <typename T>
__global__ __launch_bounds__(1024) void k_norm_join(const float* part, int blocks, int D, int w_f32, void* dg, void* dc) {
    __shared__ float fold[32][33];
    const int l = threadIdx.x % 32, w = threadIdx.x / 32, i = blockIdx.x * 32 + l;
    void* out = blockIdx.y ? dc : dg;
    if (!out) return;
    float s = 0.f;
    if (i < D) {
        const float* p = part + (int64_t)blockIdx.y * D + i;
        int b = w;
        for (; b + 7 * 32 < blocks; b += 8 * 32) {
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = p[(int64_t)(b + e * 32) * 2 * D];
#pragma unroll
            for (int e = 0; e < 8; ++e) s += v[e];
        }
        for (; b < blocks; b += 32) s += p[(int64_t)b * 2 * D];
    }
    fold[w][l] = s;
    __syncthreads();
    if (w >= 1) return;
    s = 0.f;
#pragma unroll
    for (int k = 0; k < 32; ++k) s += fold[k][l];
    if (i >= D) return;
    if (w_f32) ((float*)out)[i] = s;
    else ((T*)out)[i] = from_f<T>(s);
}

static unsigned wide_blocks(int64_t rows) { return (unsigned)(rows < 65536 ? rows : 65536); }
static int tpr_of(int D) { return D <= 16 * EPT ? 16 : D <= 64 * EPT ? 64 : D <= 256 * EPT ? 256 : 1024; }

// blocks of the backward pass = rows of `part`
static int norm_blocks(int64_t rows, int D) {
    if (rows == 0) return 0;
    if (D > NORM_MAX_D) return (int)(rows < 256 ? (rows + 3) / 4 : 64);
    const int tpr = tpr_of(D), block = tpr > 256 ? tpr : 256, rpb = block / tpr;
    const int64_t need = (rows + rpb - 1) / rpb, most = 512;
    return (int)(need < most ? need : most);
}
size_t norm_ws_bytes(int64_t rows, int D) { return (size_t)norm_blocks(rows, D) * 2 * D * sizeof(float); }

template <typename T>
static void norm_fwd(const NormArgs& A, hipStream_t st) {
    if (A.D > NORM_MAX_D) {
        hipLaunchKernelGGL(k_norm_fwd_wide<T>, dim3(wide_blocks(A.rows)), dim3(1024), 0, st, A);
        return;
    }
    const int tpr = tpr_of(A.D), block = tpr > 256 ? tpr : 256;
    const int64_t need = (A.rows + block / tpr - 1) / (block / tpr);
    const dim3 g((unsigned)(need < 65536 ? need : 65536)), b(block);
    if (tpr == 16) hipLaunchKernelGGL((k_norm_fwd<T, 16>), g, b, 0, st, A);
    else if (tpr == 64) hipLaunchKernelGGL((k_norm_fwd<T, 64>), g, b, 0, st, A);
    else if (tpr == 256) hipLaunchKernelGGL((k_norm_fwd<T, 256>), g, b, 0, st, A);
    else hipLaunchKernelGGL((k_norm_fwd<T, 1024>), g, b, 0, st, A);
}
hipError_t launch_layer_norm(const IvaeNorm& N, const void* x, const void* w, const void* b, void* y, float* stats, hipStream_t st) {
    if (N.rows == 0) return hipSuccess;
    NormArgs A = {};
    A.x = x; A.w = w; A.b = b; A.y = y; A.stats = stats;
    A.rows = N.rows; A.ldx = N.ldx; A.D = N.width; A.w_f32 = N.weight_f32 || N.dtype == IVAE_F32; A.eps = N.eps;
    if (N.dtype == IVAE_F32) norm_fwd<float>(A, st);
    else if (N.dtype == IVAE_BF16) norm_fwd<bf16_t>(A, st);
    else norm_fwd<f16_t>(A, st);
    return hipGetLastError();
}

template <typename T>
static void norm_bwd(const NormArgs& A, int blocks, void* dg, void* dc, hipStream_t st) {
    const dim3 g((unsigned)blocks);
    if (blocks > 0 && A.D > NORM_MAX_D) {
        if (A.y) hipLaunchKernelGGL(k_norm_bwd_wide<T>, dim3(wide_blocks(A.rows)), dim3(1024), 0, st, A);
        if (A.part) hipLaunchKernelGGL(k_norm_cols_wide<T>, dim3((A.D + 63) / 64, (unsigned)blocks), dim3(256), 0, st, A);
    } else if (blocks > 0) {
        const int tpr = tpr_of(A.D);
        if (tpr == 16) hipLaunchKernelGGL((k_norm_bwd<T, 16>), g, dim3(256), 0, st, A);
        else if (tpr == 64) hipLaunchKernelGGL((k_norm_bwd<T, 64>), g, dim3(256), 0, st, A);
        else if (tpr == 256) hipLaunchKernelGGL((k_norm_bwd<T, 256>), g, dim3(256), 0, st, A);
        else hipLaunchKernelGGL((k_norm_bwd<T, 1024>), g, dim3(1024), 0, st, A);
    }
    if (dg || dc) hipLaunchKernelGGL(k_norm_join<T>, dim3((A.D + 31) / 32, 2), dim3(1024), 0, st, A.part, blocks, A.D, A.w_f32, dg, dc);
}
hipError_t launch_layer_norm_backward(const IvaeNorm& N, const void* dy, const void* x, const float* stats, const void* w, const void* residual,
                                      void* dx, void* dg, void* dc, float* ws, hipStream_t st) {
    NormArgs A = {};
    A.x = x; A.dy = dy; A.w = w; A.residual = residual; A.y = dx; A.cstats = stats; A.part = dg || dc ? ws : nullptr;
    A.rows = N.rows; A.ldx = N.ldx; A.lddy = N.lddy; A.ldr = N.ld_residual; A.D = N.width; A.w_f32 = N.weight_f32 || N.dtype == IVAE_F32;
    const int blocks = norm_blocks(N.rows, N.width);
    if (N.dtype == IVAE_F32) norm_bwd<float>(A, blocks, dg, dc, st);
    else if (N.dtype == IVAE_BF16) norm_bwd<bf16_t>(A, blocks, dg, dc, st);
    else norm_bwd<f16_t>(A, blocks, dg, dc, st);
    return hipGetLastError();
}
