// Layer norm over the last dimension, forward and backward.
//   forward   y = (x - mean) r g + c,  r = 1 / sqrt(var + eps); (mean, r) of a row are kept for the backward pass
//   backward  xh = (x - mean) r, a = dy g:   dx = r (a - mean(a) - xh mean(a xh)) [+ residual],  dg = sum_rows dy xh,  dc = sum_rows dy
// Both are bound by memory: a row is read once, held in registers by the TPR threads that share it (E = 16 or 8 elements each), and the
// variance is summed from the centred values in those registers, so it does not cancel.  All sums are in 32 bits and in a fixed order.
#include "kernels.h"
#include "ops_common.h"

static constexpr int NORM_MAX_D = 1024 * 16;   // wider rows are walked instead of held

struct NormArgs {
    const void* x; const void* dy; const void* w; const void* b; const void* residual;
    void* y; float* stats;                     // stats: (2, rows): mean, r
    const float* cstats;
    float* part;                               // backward: (blocks, 2, D) sums of dy xh and dy
    void* dg; void* dc;                        // ... or, from one block, the gradients themselves
    int64_t rows, ldx, lddy, ldr;
    int D, w_f32;
    float eps;
    bool past;                                 // y is stored past the caches
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

// The thread's E elements of a row as they lie in memory: C groups of 16 bytes, the c-th at element (c TPR + t) N.  A group that the row
// ends in is loaded by elements (TAIL: the width is no multiple of N); what lies beyond the row is 0.
template <typename T, int TPR, int E, bool TAIL> struct Row {
    static constexpr int N = Wide<T>::N, C = E / N;
    Vec<T> v[C];
    __device__ __forceinline__ void load(const T* row, int t, int D, bool live) {
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int e = (c * TPR + t) * N;
#pragma unroll
            for (int j = 0; j < N; ++j) v[c].e[j] = (T)0.f;
            if (c * TPR * N >= D) continue;                     // (the same for all threads: groups that no row reaches)
            if (live && (TAIL ? e + N <= D : e < D)) v[c] = *(const Vec<T>*)(row + e);
            else if (TAIL && live && e < D)
#pragma unroll
                for (int j = 0; j < N; ++j)
                    if (e + j < D) v[c].e[j] = row[e + j];
        }
    }
};
template <typename T, int TPR, bool TAIL, int C, int N> __device__ __forceinline__ void store_row(T* row, int t, int D, const float (&o)[C][N], bool past) {
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int e = (c * TPR + t) * N;
        if (TAIL ? e + N <= D : e < D) store_wide<T>(row + e, o[c], past);
        else if (TAIL && e < D) store_part<T>(row + e, D - e, o[c]);
    }
}
// the thread's elements of the weight or the bias (null: `none`)
template <typename T, int TPR, bool TAIL, int C, int N>
__device__ __forceinline__ void load_weight(const void* w, int w_f32, int t, int D, float none, float (&o)[C][N]) {
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int e = (c * TPR + t) * N;
#pragma unroll
        for (int j = 0; j < N; ++j) o[c][j] = e + j < D ? none : 0.f;
        if (!w || e >= D) continue;
        if (TAIL && e + N > D) {
#pragma unroll
            for (int j = 0; j < N; ++j)
                if (e + j < D) o[c][j] = w_f32 ? ((const float*)w)[e + j] : to_f(((const T*)w)[e + j]);
        } else if (w_f32) {
#pragma unroll
            for (int h = 0; h < N; h += 4) {
                float u[4];
                load_wide<float>((const float*)w + e + h, u);
#pragma unroll
                for (int j = 0; j < 4; ++j) o[c][h + j] = u[j];
            }
        } else {
            load_wide<T>((const T*)w + e, o[c]);
        }
    }
}

// A block walks rows; the next row's loads are under way while a row is summed.
template <typename T, int TPR, int E, bool TAIL>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void k_norm_fwd(NormArgs A) {
    constexpr int N = Wide<T>::N, C = E / N, BLOCK = TPR > 256 ? TPR : 256, RPB = BLOCK / TPR;
    __shared__ float lds[BLOCK / 64];
    const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR;
    const int64_t step = (int64_t)gridDim.x * RPB;
    int64_t r0 = (int64_t)blockIdx.x * RPB;
    Row<T, TPR, E, TAIL> now, next;
    now.load((const T*)A.x + (r0 + sub < A.rows ? r0 + sub : 0) * A.ldx, t, A.D, r0 + sub < A.rows);
    float g[C][N], b[C][N];
    load_weight<T, TPR, TAIL>(A.w, A.w_f32, t, A.D, 1.f, g);
    load_weight<T, TPR, TAIL>(A.b, A.w_f32, t, A.D, 0.f, b);
    for (; r0 < A.rows; r0 += step) {
        const int64_t row = r0 + sub, ahead = row + step;
        const bool live = row < A.rows;
        if (r0 + step < A.rows) next.load((const T*)A.x + (ahead < A.rows ? ahead : 0) * A.ldx, t, A.D, ahead < A.rows);
        float v[C][N];
        float s[1] = {0.f};
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int j = 0; j < N; ++j) {
                v[c][j] = to_f(now.v[c].e[j]);
                s[0] += v[c][j];
            }
        row_sum<TPR, 1, BLOCK>(s, lds);
        const float mean = s[0] / (float)A.D;
        float q[1] = {0.f};
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int j = 0; j < N; ++j) {
                v[c][j] -= mean;
                if ((c * TPR + t) * N + (TAIL ? j : 0) < A.D) q[0] += v[c][j] * v[c][j];
            }
        row_sum<TPR, 1, BLOCK>(q, lds);
        const float r = 1.f / sqrtf(q[0] / (float)A.D + A.eps);
        now = next;
        if (!live) continue;                    // (after the row's last barrier)
        if (A.stats && t == 0) {
            A.stats[row] = mean;
            A.stats[A.rows + row] = r;
        }
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int j = 0; j < N; ++j) v[c][j] = v[c][j] * r * g[c][j] + b[c][j];
        store_row<T, TPR, TAIL>((T*)A.y + row * A.D, t, A.D, v, A.past);
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

// dx, and each block's sums of dy xh and dy over the rows it walks (block, block + grid, ...).  (1024 threads have 128 registers each:
// no room for the next row.)
template <typename T, int TPR, int E, bool TAIL>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void k_norm_bwd(NormArgs A) {
    constexpr int N = Wide<T>::N, C = E / N, BLOCK = TPR > 256 ? TPR : 256, RPB = BLOCK / TPR;
    constexpr bool AHEAD = TPR < 1024;
    __shared__ float lds[BLOCK / 64 * 2];
    __shared__ float fold[RPB > 1 ? TPR * E * 2 : 1];
    const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR;
    const float inv = 1.f / (float)A.D;
    const int64_t step = (int64_t)gridDim.x * RPB;
    int64_t r0 = (int64_t)blockIdx.x * RPB;
    Row<T, TPR, E, TAIL> x, dy, xn, dyn;
    float mean = 0.f, r = 0.f, mean_n = 0.f, r_n = 0.f;
    auto load = [&](Row<T, TPR, E, TAIL>& a, Row<T, TPR, E, TAIL>& b, float& m, float& rs, int64_t row) {
        const bool live = row < A.rows;
        const int64_t at = live ? row : 0;
        a.load((const T*)A.x + at * A.ldx, t, A.D, live);
        b.load((const T*)A.dy + at * A.lddy, t, A.D, live);
        m = live ? A.cstats[row] : 0.f;
        rs = live ? A.cstats[A.rows + row] : 0.f;
    };
    if (AHEAD) load(x, dy, mean, r, r0 + sub);
    float g[C][N], dg[C][N], dc[C][N];
    load_weight<T, TPR, TAIL>(A.w, A.w_f32, t, A.D, 1.f, g);
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
        for (int j = 0; j < N; ++j) dg[c][j] = dc[c][j] = 0.f;
    for (; r0 < A.rows; r0 += step) {
        const int64_t row = r0 + sub;
        const bool live = row < A.rows;
        if (!AHEAD) load(x, dy, mean, r, row);
        else if (r0 + step < A.rows) load(xn, dyn, mean_n, r_n, row + step);
        Row<T, TPR, E, TAIL> add;
        if (A.residual) add.load((const T*)A.residual + (live ? row : 0) * A.ldr, t, A.D, live);
        float xh[C][N], d[C][N];
        float s[2] = {0.f, 0.f};
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const bool in = live && (c * TPR + t) * N + (TAIL ? j : 0) < A.D;
                const float dv = to_f(dy.v[c].e[j]);
                xh[c][j] = in ? (to_f(x.v[c].e[j]) - mean) * r : 0.f;
                dg[c][j] += dv * xh[c][j];
                dc[c][j] += dv;
                d[c][j] = dv * g[c][j];
                s[0] += d[c][j];
                s[1] += d[c][j] * xh[c][j];
            }
        row_sum<TPR, 2, BLOCK>(s, lds);
        const float m1 = s[0] * inv, m2 = s[1] * inv, rr = r;
        if (AHEAD) x = xn, dy = dyn, mean = mean_n, r = r_n;
        if (!live || !A.y) continue;
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int j = 0; j < N; ++j) {
                d[c][j] = rr * (d[c][j] - m1 - xh[c][j] * m2);
                if (A.residual) d[c][j] += to_f(add.v[c].e[j]);
            }
        store_row<T, TPR, TAIL>((T*)A.y + row * A.D, t, A.D, d, A.past);
    }
    if (!A.part && !A.dg && !A.dc) return;
    auto put = [&](int i, float vg, float vc) {
        if (A.part) {
            float* part = A.part + (int64_t)blockIdx.x * 2 * A.D;
            part[i] = vg;
            part[A.D + i] = vc;
        } else if (A.w_f32) {
            if (A.dg) ((float*)A.dg)[i] = vg;
            if (A.dc) ((float*)A.dc)[i] = vc;
        } else {
            if (A.dg) ((T*)A.dg)[i] = from_f<T>(vg);
            if (A.dc) ((T*)A.dc)[i] = from_f<T>(vc);
        }
    };
    if constexpr (RPB > 1) {                    // the rows of a block meet in LDS, one after the other
        for (int s = 0; s < RPB; ++s) {
            if (sub == s)
#pragma unroll
                for (int c = 0; c < C; ++c)
#pragma unroll
                    for (int j = 0; j < N; ++j) {
                        const int i = (c * TPR + t) * N + j;
                        fold[i] = s ? fold[i] + dg[c][j] : dg[c][j];
                        fold[TPR * E + i] = s ? fold[TPR * E + i] + dc[c][j] : dc[c][j];
                    }
            __syncthreads();
        }
        for (int i = threadIdx.x; i < A.D; i += BLOCK) put(i, fold[i], fold[TPR * E + i]);
    } else {
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const int i = (c * TPR + t) * N + j;
                if (i < A.D) put(i, dg[c][j], dc[c][j]);
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
// Threads that share a row and elements that each holds: the fewest threads with 16 where there is enough to read (16384 x 2048 bf16: 24 us
// forward, 29 backward, against 27 and 38 with 8), and with 8 in small matrices and rows of ragged width, which wait for latencies (5003 x 1037
// fp32: 14 and 18 us against 16 and 22 with 16; 64 x 200: 3 and 4 against 3 and 7).
struct Share { int tpr, e; };
static Share share_of(int64_t rows, int D, bool tail) {
    if (D <= 4096 && (tail || rows * D <= 1 << 21)) return {D <= 512 ? 64 : D <= 2048 ? 256 : 512, 8};
    for (int t : {16, 64, 128, 256, 512})
        if (D <= t * 16) return {t, 16};
    return {1024, 16};
}
static bool tail_of(int D, int dtype) { return D % (dtype == IVAE_F32 ? 4 : 8) != 0; }
static int64_t groups_of(int64_t rows, int tpr, int64_t most) {     // blocks of RPB rows each, at most `most`
    const int rpb = tpr < 256 ? 256 / tpr : 1;
    const int64_t need = (rows + rpb - 1) / rpb;
    return need < most ? need : most;
}
// about as many blocks as the chip holds: each keeps the weight in registers, and in the backward pass its sums (us, forward / gradients, half as
// many | these | twice as many blocks: 16384 x 4096 bf16 48/100 | 42/83 | 43/105, 5003 x 1037 fp32 17/30 | 13/23 | 15/28, 65536 x 256 bf16 14/29 | 13/27 |
// 14/33, 2048 x 16384 bf16 37/91 | 36/91 | 31/121, 4096 x 8192 bf16 30/53 | 31/65 | 28/93)
static int fwd_blocks(int64_t rows, Share h) { return (int)groups_of(rows, h.tpr, h.tpr <= 256 ? 1280 : h.tpr == 512 ? 640 : 320); }
// blocks of the backward pass = rows of `part`.  Few rows are walked by one block, which needs neither a workspace nor a join
// (up to 24 x 128, 6 x 2048, 4 x 4096: 11.6 us a call with the host's part, 16 with them; the kernel takes up to 10 us instead of 4 and 2.5).
static const int WALK = 6;
static int norm_blocks(int64_t rows, int D, int dtype) {
    if (rows == 0) return 0;
    if (D > NORM_MAX_D) return (int)(rows < 256 ? (rows + 3) / 4 : 64);
    const Share h = share_of(rows, D, tail_of(D, dtype));
    if (rows * D <= 1 << 15 && groups_of(rows, h.tpr, WALK + 1) <= WALK) return 1;
    return (int)groups_of(rows, h.tpr, h.tpr <= 256 ? 768 : h.tpr == 512 ? 512 : 256);
}
static bool one_block(int blocks, int D) { return blocks == 1 && D <= NORM_MAX_D; }
size_t norm_ws_bytes(int64_t rows, int D, int dtype) {
    const int blocks = norm_blocks(rows, D, dtype);
    return one_block(blocks, D) ? 0 : (size_t)blocks * 2 * D * sizeof(float);
}

#define NORM_CASE(K, TPR, E) case TPR * 32 + E: hipLaunchKernelGGL((K<T, TPR, E, TAIL>), g, b, 0, st, A); break;
#define NORM_CASES(K)                                                                                                                       \
    switch (h.tpr * 32 + h.e) {                                                                                                             \
        NORM_CASE(K, 64, 8) NORM_CASE(K, 256, 8) NORM_CASE(K, 512, 8) NORM_CASE(K, 512, 16) NORM_CASE(K, 1024, 16)                          \
    }                                                                                                                                       \
    if constexpr (!TAIL)                                                                                                                    \
        switch (h.tpr * 32 + h.e) { NORM_CASE(K, 16, 16) NORM_CASE(K, 64, 16) NORM_CASE(K, 128, 16) NORM_CASE(K, 256, 16) }
template <typename T, bool TAIL>
static void norm_fwd(const NormArgs& A, hipStream_t st) {
    const Share h = share_of(A.rows, A.D, TAIL);
    const dim3 g((unsigned)fwd_blocks(A.rows, h)), b(h.tpr > 256 ? h.tpr : 256);
    NORM_CASES(k_norm_fwd)
}
template <typename T>
static void norm_fwd(const NormArgs& A, hipStream_t st) {
    if (A.D > NORM_MAX_D) hipLaunchKernelGGL(k_norm_fwd_wide<T>, dim3(wide_blocks(A.rows)), dim3(1024), 0, st, A);
    else if (A.D % Wide<T>::N) norm_fwd<T, true>(A, st);
    else norm_fwd<T, false>(A, st);
}
hipError_t launch_layer_norm(const IvaeNorm& N, const void* x, const void* w, const void* b, void* y, float* stats, hipStream_t st) {
    if (N.rows == 0) return hipSuccess;
    NormArgs A = {};
    A.x = x; A.w = w; A.b = b; A.y = y; A.stats = stats;
    A.rows = N.rows; A.ldx = N.ldx; A.D = N.width; A.w_f32 = N.weight_f32 || N.dtype == IVAE_F32; A.eps = N.eps;
    A.past = past_caches((double)N.rows * N.width, N.dtype);
    if (N.dtype == IVAE_F32) norm_fwd<float>(A, st);
    else if (N.dtype == IVAE_BF16) norm_fwd<bf16_t>(A, st);
    else norm_fwd<f16_t>(A, st);
    return hipGetLastError();
}

template <typename T, bool TAIL>
static void norm_bwd(const NormArgs& A, int blocks, hipStream_t st) {
    const Share h = share_of(A.rows, A.D, TAIL);
    const dim3 g((unsigned)blocks), b(h.tpr > 256 ? h.tpr : 256);
    NORM_CASES(k_norm_bwd)
}
template <typename T>
static void norm_bwd(const NormArgs& A, int blocks, void* dg, void* dc, hipStream_t st) {
    if (blocks > 0 && A.D > NORM_MAX_D) {
        if (A.y) hipLaunchKernelGGL(k_norm_bwd_wide<T>, dim3(wide_blocks(A.rows)), dim3(1024), 0, st, A);
        if (A.part) hipLaunchKernelGGL(k_norm_cols_wide<T>, dim3((A.D + 63) / 64, (unsigned)blocks), dim3(256), 0, st, A);
    } else if (blocks > 0) {
        if (A.D % Wide<T>::N) norm_bwd<T, true>(A, blocks, st);
        else norm_bwd<T, false>(A, blocks, st);
    }
    if ((dg || dc) && !one_block(blocks, A.D)) hipLaunchKernelGGL(k_norm_join<T>, dim3((A.D + 31) / 32, 2), dim3(1024), 0, st, A.part, blocks, A.D, A.w_f32, dg, dc);
}
hipError_t launch_layer_norm_backward(const IvaeNorm& N, const void* dy, const void* x, const float* stats, const void* w, const void* residual,
                                      void* dx, void* dg, void* dc, float* ws, hipStream_t st) {
    NormArgs A = {};
    A.x = x; A.dy = dy; A.w = w; A.residual = residual; A.y = dx; A.cstats = stats; A.part = dg || dc ? ws : nullptr;
    A.rows = N.rows; A.ldx = N.ldx; A.lddy = N.lddy; A.ldr = N.ld_residual; A.D = N.width; A.w_f32 = N.weight_f32 || N.dtype == IVAE_F32;
    A.past = past_caches((double)N.rows * N.width, N.dtype);
    const int blocks = norm_blocks(N.rows, N.width, N.dtype);
    if (one_block(blocks, A.D)) A.part = nullptr, A.dg = dg, A.dc = dc;
    if (N.dtype == IVAE_F32) norm_bwd<float>(A, blocks, dg, dc, st);
    else if (N.dtype == IVAE_BF16) norm_bwd<bf16_t>(A, blocks, dg, dc, st);
    else norm_bwd<f16_t>(A, blocks, dg, dc, st);
    return hipGetLastError();
}
