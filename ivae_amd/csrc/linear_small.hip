// The linear operator on 64 x 64 tiles staged through registers: any size, any row stride, any alignment, and in the backward pass
// one launch for dx, dw and db (the gradient of the pre-activation is formed while its tile is loaded and never stored).
//
// One tile product serves the three products.  P rows, Q columns, R summed over:
//   forward  P = m, Q = n, R = k     y[m,n]  = sum_k x[m,k] w[n,k]
//   dx       P = m, Q = k, R = n     dx[m,k] = sum_n ds[m,n] w[n,k]
//   dw       P = n, Q = k, R = m     dw[n,k] = sum_m ds[m,n] x[m,k]        (db[n] = sum_m ds[m,n] on the way)
// The Q operand is the matrix instruction's first one, so that a lane ends up with 4 neighbouring columns of one row.
// In the 16-bit types the gradient of the pre-activation, act'(s) dy, enters as the sum of two numbers of the type (the second is
// the first's rounding error), one more matrix instruction each: these sizes wait for memory and launches, and the products then
// have no rounding but their result's.
// A long sum over few tiles is split; the parts are written in 32 bits and added in order by k_linear_join.
#include "kernels.h"
#include "linear.h"

static constexpr int TP = 64, TQ = 64, TR = 32;

template <typename T> struct Lds { static constexpr int LD = TR + 8; };       // row stride in elements; rows stay 16-byte aligned
template <> struct Lds<float> { static constexpr int LD = TR + 4; };

enum { MODE_FWD, MODE_DX, MODE_DW };

struct LinSplit { int64_t tp, tq; int splits; int64_t len; };   // tiles along P and Q, parts of R, each `len` long (a multiple of TR)

// 8 neighbouring elements from (outer, inner) of a row-major matrix, zero outside [0, outers) x [0, inner_end)
template <typename T>
__device__ __forceinline__ void fetch8(const T* base, int64_t ld, int64_t outer, int64_t outers, int64_t inner, int64_t inner_end, float (&v)[8]) {
    const int64_t left = outer < outers ? inner_end - inner : 0;
    const T* p = base + outer * ld + inner;
    constexpr int N = Wide<T>::N;
#pragma unroll
    for (int h = 0; h < 8 / N; ++h) {
        float u[N];
        if (left >= (h + 1) * N) load_wide<T>(p + h * N, u);
        else
#pragma unroll
            for (int j = 0; j < N; ++j) u[j] = left > h * N + j ? to_f(p[h * N + j]) : 0.f;
#pragma unroll
        for (int j = 0; j < N; ++j) v[h * N + j] = u[j];
    }
}

// RC: the summed index is the contiguous one.  (i0, r0): the tile's corner.
template <typename T, bool RC>
__device__ __forceinline__ void fetch_tile(const T* base, int64_t ld, int64_t i0, int64_t i_end, int64_t r0, int64_t r_end, float (&v)[8]) {
    const int t = threadIdx.x;
    if (RC) fetch8<T>(base, ld, i0 + t / 4, i_end, r0 + t % 4 * 8, r_end, v);
    else fetch8<T>(base, ld, r0 + t / 8, r_end, i0 + t % 8 * 8, i_end, v);
}
// ERR: what rounding to T leaves of them
template <typename T, bool RC, bool ERR = false>
__device__ __forceinline__ void put_tile(T* lds, const float (&u)[8]) {
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float r = to_f(from_f<T>(u[j]));
        v[j] = !ERR ? u[j] : fabsf(r) < __builtin_inff() ? u[j] - r : 0.f;       // (infinities and NaN are whole in the first number)
    }
    const int t = threadIdx.x;
    constexpr int LD = Lds<T>::LD;
    if (RC) {
#pragma unroll
        for (int j = 0; j < 8; ++j) lds[(t / 4) * LD + t % 4 * 8 + j] = from_f<T>(v[j]);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) lds[(t % 8 * 8 + j) * LD + t / 8] = from_f<T>(v[j]);
    }
}

__device__ __forceinline__ f32x4 mma32(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 mma32(f16x8 a, f16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
template <typename T> struct V8;
template <> struct V8<bf16_t> { typedef bf16x8 t; };
template <> struct V8<f16_t> { typedef f16x8 t; };

// one TR-long step of a wave's 32 x 32 part
template <typename T>
__device__ __forceinline__ void tile_mma(const T* lp, const T* lq, f32x4 (&acc)[2][2]) {
    typedef typename V8<T>::t v8;
    const int l = threadIdx.x % 64, w = threadIdx.x / 64, row = l % 16, r = l / 16 * 8;
    constexpr int LD = Lds<T>::LD;
    v8 p[2], q[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        p[i] = *(const v8*)(lp + (w / 2 * 32 + i * 16 + row) * LD + r);
        q[i] = *(const v8*)(lq + (w % 2 * 32 + i * 16 + row) * LD + r);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = mma32(q[j], p[i], acc[i][j]);
}
template <>
__device__ __forceinline__ void tile_mma<float>(const float* lp, const float* lq, f32x4 (&acc)[2][2]) {
    const int l = threadIdx.x % 64, w = threadIdx.x / 64, row = l % 16, r = l / 16 * 4;
    constexpr int LD = Lds<float>::LD;
#pragma unroll
    for (int b = 0; b < TR; b += 16) {
        f32x4 p[2], q[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            p[i] = *(const f32x4*)(lp + (w / 2 * 32 + i * 16 + row) * LD + b + r);
            q[i] = *(const f32x4*)(lq + (w % 2 * 32 + i * 16 + row) * LD + b + r);
        }
        // step e takes element e of each lane group's four: the same permutation of the summed index on both sides
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(q[j][e], p[i][e], acc[i][j], 0, 0, 0);
    }
}

template <typename T, int MODE>
__device__ __forceinline__ void tile_product(const LinArgs& A, const LinSplit& S, int64_t tile, float* part, float* part_db, T* lp, T* lq, T* le, float* lsum) {
    const int64_t split = tile / (S.tp * S.tq);
    tile -= split * S.tp * S.tq;
    const int64_t p0 = tile / S.tq * TP, q0 = tile % S.tq * TQ;
    const int64_t P = MODE == MODE_DW ? A.N : A.M, Q = MODE == MODE_FWD ? A.N : A.K, R = MODE == MODE_FWD ? A.K : MODE == MODE_DX ? A.N : A.M;
    const int64_t ra = split * S.len, rb = ra + S.len < R ? ra + S.len : R;
    const int t = threadIdx.x;
    const T* x = (const T*)A.x;
    const T* w = (const T*)A.w;
    const T* dy = (const T*)A.dy;
    typedef typename Pre<T>::t pre_t;
    const pre_t* pre = (const pre_t*)A.cpre;

    float vp[8], vq[8], sum[8] = {};
    auto fetch = [&](int64_t r0) {
        if constexpr (MODE == MODE_FWD) {
            fetch_tile<T, true>(x, A.ldx, p0, P, r0, rb, vp);
            fetch_tile<T, true>(w, A.K, q0, Q, r0, rb, vq);
        } else {
            constexpr bool RC = MODE == MODE_DX;
            fetch_tile<T, RC>(dy, A.lddy, p0, P, r0, rb, vp);
            if (A.act != IVAE_ACT_NONE) {
                float s[8];
                fetch_tile<pre_t, RC>(pre, A.N, p0, P, r0, rb, s);
#pragma unroll
                for (int j = 0; j < 8; ++j) vp[j] *= lin_act_slope<T>(A.act, A.slope, s[j]);
            }
            if (MODE == MODE_DW)
#pragma unroll
                for (int j = 0; j < 8; ++j) sum[j] += vp[j];
            if (MODE == MODE_DX) fetch_tile<T, false>(w, A.K, q0, Q, r0, rb, vq);
            else fetch_tile<T, false>(x, A.ldx, q0, Q, r0, rb, vq);
        }
    };
    f32x4 acc[2][2] = {};
    if (ra < rb) fetch(ra);
    for (int64_t r = ra; r < rb; r += TR) {
        __syncthreads();
        put_tile<T, MODE != MODE_DW>(lp, vp);
        put_tile<T, MODE == MODE_FWD>(lq, vq);
        const bool two = sizeof(T) == 2 && MODE != MODE_FWD && A.act != IVAE_ACT_NONE;
        if (two) put_tile<T, MODE != MODE_DW, true>(le, vp);
        __syncthreads();
        if (r + TR < rb) fetch(r + TR);
        tile_mma<T>(lp, lq, acc);
        if (two) tile_mma<T>(le, lq, acc);
    }
    const int l = t % 64, wv = t / 64;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int64_t p = p0 + wv / 2 * 32 + i * 16 + l % 16, q = q0 + wv % 2 * 32 + j * 16 + l / 16 * 4 + e;
                if (p >= P || q >= Q) continue;
                if (S.splits > 1) part[(split * P + p) * Q + q] = acc[i][j][e];
                else if (MODE == MODE_FWD) forward_store<T>(A, p, (int)q, acc[i][j][e]);
                else if (MODE == MODE_DX) ((T*)A.dx)[p * Q + q] = from_f<T>(acc[i][j][e]);
                else if (A.dw) ((T*)A.dw)[p * Q + q] = from_f<T>(acc[i][j][e]);
            }
    if (MODE == MODE_DW && A.db && q0 == 0) {       // thread t holds the sums of 8 columns over every 32nd row: 32 threads hold each column
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 8; ++j) lsum[(t / 8) * TP + t % 8 * 8 + j] = sum[j];
        __syncthreads();
        if (t < TP && p0 + t < P) {
            float s = 0.f;
            for (int i = 0; i < 32; ++i) s += lsum[i * TP + t];
            if (S.splits > 1) part_db[split * P + p0 + t] = s;
            else ((T*)A.db)[p0 + t] = from_f<T>(s);
        }
    }
    __syncthreads();                                // the tiles are free for the next round
}

template <typename T>
__global__ __launch_bounds__(256) void k_linear_fwd(LinArgs A, LinSplit S) {
    __shared__ __attribute__((aligned(16))) T lp[TP * Lds<T>::LD];
    __shared__ __attribute__((aligned(16))) T lq[TQ * Lds<T>::LD];
    const int64_t tiles = S.tp * S.tq * S.splits;
    for (int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) tile_product<T, MODE_FWD>(A, S, tile, A.part, nullptr, lp, lq, nullptr, nullptr);
}
template <typename T>
__global__ __launch_bounds__(256) void k_linear_bwd(LinArgs A, LinSplit X, LinSplit W, float* part_w, float* part_b) {
    __shared__ __attribute__((aligned(16))) T lp[TP * Lds<T>::LD];
    __shared__ __attribute__((aligned(16))) T lq[TQ * Lds<T>::LD];
    __shared__ __attribute__((aligned(16))) T le[sizeof(T) == 2 ? TP * Lds<T>::LD : 1];
    __shared__ float lsum[32 * TP];
    const int64_t nx = X.tp * X.tq * X.splits, tiles = nx + W.tp * W.tq * W.splits;
    for (int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
        if (tile < nx) tile_product<T, MODE_DX>(A, X, tile, A.part, nullptr, lp, lq, le, nullptr);
        else tile_product<T, MODE_DW>(A, W, tile - nx, part_w, part_b, lp, lq, le, lsum);
    }
}

__device__ __forceinline__ float join(const float* part, int splits, int64_t n, int64_t i) {
    float s = 0.f;
    for (int k = 0; k < splits; ++k) s += part[k * n + i];
    return s;
}
template <typename T>
__global__ __launch_bounds__(256) void k_linear_join_fwd(LinArgs A, int splits) {
    const int64_t n = A.M * A.N;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256)
        forward_store<T>(A, i / A.N, (int)(i % A.N), join(A.part, splits, n, i));
}
// db is a sum over up to hundreds of parts of a few thousand columns: its blocks (the first ones) take 64 columns each, four walks
// over the parts side by side, eight loads in flight
__device__ __forceinline__ float join_walk(const float* part, int k, int64_t n, int64_t i, int w) {
    float s = 0.f;
    int j = w;
    for (; j + 28 < k; j += 32) {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = part[(j + e * 4) * n + i];
#pragma unroll
        for (int e = 0; e < 8; ++e) s += v[e];
    }
    for (; j < k; j += 4) s += part[j * n + i];
    return s;
}
template <typename T>
__global__ __launch_bounds__(256) void k_linear_join_bwd(LinArgs A, LinParts J) {
    const int64_t nx = J.kx > 1 ? A.M * A.K : 0, nw = J.kw > 1 ? (int64_t)A.N * A.K : 0, nb = J.kb > 0 ? (A.N + 63) / 64 : 0;
    if (blockIdx.x < nb) {
        __shared__ float fold[4][64];
        const int l = threadIdx.x % 64, w = threadIdx.x / 64;
        const int64_t i = (int64_t)blockIdx.x * 64 + l;
        fold[w][l] = i < A.N ? join_walk(J.b, J.kb, A.N, i, w) : 0.f;
        __syncthreads();
        if (w == 0 && i < A.N) ((T*)A.db)[i] = from_f<T>((fold[0][l] + fold[1][l]) + (fold[2][l] + fold[3][l]));
        return;
    }
    for (int64_t i = (int64_t)(blockIdx.x - nb) * 256 + threadIdx.x; i < nx + nw; i += (int64_t)(gridDim.x - nb) * 256) {
        if (i < nx) ((T*)A.dx)[i] = from_f<T>(join(J.x, J.kx, nx, i));
        else ((T*)A.dw)[i - nx] = from_f<T>(join(J.w, J.kw, nw, i - nx));
    }
}

// The marked tiles of a large fp32 product: a block takes one of them in 64 x 64 parts.
template <int MODE>
__device__ __forceinline__ void mend(const LinArgs& A, const LinMarks& K, int64_t P, int64_t Q, int64_t R, int64_t b, float* lp, float* lq) {
    const int64_t tp = (P + K.tile_p - 1) / K.tile_p, tq = (Q + K.tile_q - 1) / K.tile_q;
    int marked = 0;
    for (int k = 0; k < K.splits; ++k) marked |= K.flags[k * tp * tq + b];
    if (!marked) return;
    const LinSplit S = {(P + TP - 1) / TP, (Q + TQ - 1) / TQ, 1, (R + TR - 1) / TR * TR};
    const int64_t i0 = b / tq * (K.tile_p / TP), j0 = b % tq * (K.tile_q / TQ);
    for (int64_t i = i0; i < i0 + K.tile_p / TP && i < S.tp; ++i)
        for (int64_t j = j0; j < j0 + K.tile_q / TQ && j < S.tq; ++j) tile_product<float, MODE>(A, S, i * S.tq + j, nullptr, nullptr, lp, lq, nullptr, nullptr);
}
__global__ __launch_bounds__(256) void k_linear_mend_fwd(LinArgs A, LinMarks y) {
    __shared__ __attribute__((aligned(16))) float lp[TP * Lds<float>::LD];
    __shared__ __attribute__((aligned(16))) float lq[TQ * Lds<float>::LD];
    mend<MODE_FWD>(A, y, A.M, A.N, A.K, blockIdx.x, lp, lq);
}
__global__ __launch_bounds__(256) void k_linear_mend_bwd(LinArgs A, LinMarks x, int64_t nx, LinMarks w) {
    __shared__ __attribute__((aligned(16))) float lp[TP * Lds<float>::LD];
    __shared__ __attribute__((aligned(16))) float lq[TQ * Lds<float>::LD];
    if (blockIdx.x < nx) mend<MODE_DX>(A, x, A.M, A.K, A.N, blockIdx.x, lp, lq);
    else mend<MODE_DW>(A, w, A.N, A.K, A.M, blockIdx.x - nx, lp, lq);
}

static LinSplit split_of(int64_t P, int64_t Q, int64_t R) {
    LinSplit S;
    S.tp = (P + TP - 1) / TP;
    S.tq = (Q + TQ - 1) / TQ;
    const int64_t tiles = S.tp * S.tq, most = R / 256;          // a part sums over 256 or more
    int64_t s = tiles > 0 && tiles < 256 ? 512 / tiles : 1;
    if (s > most) s = most;
    if (s > 64) s = 64;
    if (s < 1) s = 1;
    S.len = ((R + s - 1) / s + TR - 1) / TR * TR;
    if (S.len < TR) S.len = TR;
    S.splits = R > 0 ? (int)((R + S.len - 1) / S.len) : 1;
    return S;
}
struct BwdPlan { LinSplit X, W; int64_t off_w, off_b, floats; };
static BwdPlan plan_bwd(const LinArgs& A) {
    BwdPlan p;
    p.X = split_of(A.M, A.K, A.N);
    p.W = split_of(A.N, A.K, A.M);
    if (!A.dx) p.X.tp = 0;
    if (!A.dw) p.W.tq = A.db ? 1 : 0;                           // db alone: the first column of tiles sums it
    const int64_t nx = A.dx && p.X.splits > 1 ? p.X.splits * A.M * A.K : 0;
    const int64_t nw = p.W.tq && p.W.splits > 1 ? (int64_t)p.W.splits * A.N * A.K : 0;
    p.off_w = nx;
    p.off_b = nx + nw;
    p.floats = nx + nw + (nw ? (int64_t)p.W.splits * A.N : 0);
    return p;
}
size_t linear_small_ws(const LinArgs& A, bool backward) {
    if (!backward) {
        const LinSplit S = split_of(A.M, A.N, A.K);
        return S.splits > 1 ? (size_t)S.splits * A.M * A.N * 4 : 0;
    }
    return (size_t)plan_bwd(A).floats * 4;
}

static unsigned cap(int64_t blocks) { return (unsigned)(blocks < (1 << 20) ? blocks : 1 << 20); }

hipError_t linear_join_forward(const LinArgs& A, int splits, int dtype, hipStream_t st) {
    if (splits < 2) return hipSuccess;
    const dim3 g(cap((A.M * A.N + 255) / 256)), b(256);
    if (dtype == IVAE_F32) hipLaunchKernelGGL(k_linear_join_fwd<float>, g, b, 0, st, A, splits);
    else if (dtype == IVAE_BF16) hipLaunchKernelGGL(k_linear_join_fwd<bf16_t>, g, b, 0, st, A, splits);
    else hipLaunchKernelGGL(k_linear_join_fwd<f16_t>, g, b, 0, st, A, splits);
    return hipGetLastError();
}
hipError_t linear_join_backward(const LinArgs& A, const LinParts& J0, int dtype, hipStream_t st) {
    LinParts J = J0;
    if (!A.dx) J.kx = 0;
    if (!A.dw) J.kw = 0;
    if (!A.db) J.kb = 0;
    const int64_t n = (J.kx > 1 ? A.M * A.K : 0) + (J.kw > 1 ? (int64_t)A.N * A.K : 0);
    const unsigned blocks = cap((n + 255) / 256) + (J.kb > 0 ? (unsigned)((A.N + 63) / 64) : 0);
    if (blocks == 0) return hipSuccess;
    const dim3 g(blocks), b(256);
    if (dtype == IVAE_F32) hipLaunchKernelGGL(k_linear_join_bwd<float>, g, b, 0, st, A, J);
    else if (dtype == IVAE_BF16) hipLaunchKernelGGL(k_linear_join_bwd<bf16_t>, g, b, 0, st, A, J);
    else hipLaunchKernelGGL(k_linear_join_bwd<f16_t>, g, b, 0, st, A, J);
    return hipGetLastError();
}
static int64_t mend_tiles(int64_t P, int64_t Q, const LinMarks& K) { return ((P + K.tile_p - 1) / K.tile_p) * ((Q + K.tile_q - 1) / K.tile_q); }
hipError_t linear_mend_forward(const LinArgs& A, const LinMarks& y, hipStream_t st) {
    hipLaunchKernelGGL(k_linear_mend_fwd, dim3((unsigned)mend_tiles(A.M, A.N, y)), dim3(256), 0, st, A, y);
    return hipGetLastError();
}
hipError_t linear_mend_backward(const LinArgs& A, const LinMarks& x, const LinMarks& w, hipStream_t st) {
    const int64_t nx = A.dx ? mend_tiles(A.M, A.K, x) : 0, nw = A.dw ? mend_tiles(A.N, A.K, w) : 0;
    LinArgs B = A;
    B.db = nullptr;                                             // (its sums are fp32 already)
    if (nx + nw) hipLaunchKernelGGL(k_linear_mend_bwd, dim3((unsigned)(nx + nw)), dim3(256), 0, st, B, x, nx, w);
    return hipGetLastError();
}

template <typename T> static void fwd(const LinArgs& A, hipStream_t st) {
    const LinSplit S = split_of(A.M, A.N, A.K);
    hipLaunchKernelGGL(k_linear_fwd<T>, dim3(cap(S.tp * S.tq * S.splits)), dim3(256), 0, st, A, S);
}
hipError_t linear_small_forward(const LinArgs& A, int dtype, hipStream_t st) {
    if (dtype == IVAE_F32) fwd<float>(A, st);
    else if (dtype == IVAE_BF16) fwd<bf16_t>(A, st);
    else fwd<f16_t>(A, st);
    const hipError_t e = hipGetLastError();
    return e != hipSuccess ? e : linear_join_forward(A, split_of(A.M, A.N, A.K).splits, dtype, st);
}
template <typename T> static void bwd(const LinArgs& A, const BwdPlan& p, float* pw, float* pb, hipStream_t st) {
    const int64_t tiles = p.X.tp * p.X.tq * p.X.splits + p.W.tp * p.W.tq * p.W.splits;
    if (tiles) hipLaunchKernelGGL(k_linear_bwd<T>, dim3(cap(tiles)), dim3(256), 0, st, A, p.X, p.W, pw, pb);
}
hipError_t linear_small_backward(const LinArgs& A, int dtype, hipStream_t st) {
    const BwdPlan p = plan_bwd(A);
    float* pw = A.part ? A.part + p.off_w : nullptr;
    float* pb = A.part ? A.part + p.off_b : nullptr;
    if (dtype == IVAE_F32) bwd<float>(A, p, pw, pb, st);
    else if (dtype == IVAE_BF16) bwd<bf16_t>(A, p, pw, pb, st);
    else bwd<f16_t>(A, p, pw, pb, st);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    return linear_join_backward(A, {A.part, pw, pb, p.X.splits, p.W.splits, p.W.splits > 1 ? p.W.splits : 0}, dtype, st);
}
