// The 64 x 64 tile of a product, staged through registers: any size, any row stride, any alignment.
//
// One tile product serves the three products.  P rows, Q columns, R summed over:
//   forward  P = m, Q = n, R = k     y[m,n]  = sum_k x[m,k] w[n,k]
//   dx       P = m, Q = k, R = n     dx[m,k] = sum_n ds[m,n] w[n,k]
//   dw       P = n, Q = k, R = m     dw[n,k] = sum_m ds[m,n] x[m,k]        (db[n] = sum_m ds[m,n] on the way)
// The Q operand is the matrix instruction's first one, so that a lane ends up with 4 neighbouring columns of one row.
// T: of the tensors, C: of the products' operands, T or float.  With an activation the gradient of the pre-activation, act'(s) dy, is a
// number of 32 bits that the 16-bit types cannot hold (fp16 neither its range), so the backward pass then multiplies in fp32: these sizes
// wait for memory and launches, and the products have no rounding but their result's.  (fp16, gelu, gradients of 64 x 50 x 50 8.1 us,
// of 256 x 256 x 256 16.6 us; as two numbers of the type, which lose fp16's smallest and largest gradients and make a NaN where
// an infinity meets a second number of 0, 7.4 and 13.8 us.)
#pragma once
#include "linear.h"

// A step holds 64 of the summed index: with 32 there are twice the barriers, and each waits for a load's whole latency (fp16 1024 x 1024 x
// 1024, us: forward 22.6 with 32, 21.5 with 64; gradients 85 and 67).  The tiles lie in LDS as in memory, and dw's operands and dx's
// weight are turned by the LDS reads that transpose.  The sums leave through LDS as well, so that residual, output and saved values move 16
// bytes a thread along rows (forward 21.5 -> 19.2 us).
static constexpr int TP = 64, TQ = 64, TR = 64;

template <typename T> struct Lds { static constexpr int LD = TR + 8; };       // row stride in elements; rows stay 16-byte aligned
template <> struct Lds<float> { static constexpr int LD = TR + 4; };

enum { MODE_FWD, MODE_DX, MODE_DW };

struct LinSplit { int64_t tp, tq; int splits; int64_t len; };   // tiles along P and Q, parts of R, each `len` long

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

// A thread's 16 values of a tile, in two groups of 8 neighbours.  RC: the summed index is the contiguous one.  (i0, r0): the tile's corner.
template <typename T, bool RC>
__device__ __forceinline__ void fetch_tile(int t, const T* base, int64_t ld, int64_t i0, int64_t i_end, int64_t r0, int64_t r_end, float (&v)[2][8]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        if (RC) fetch8<T>(base, ld, i0 + t / 4, i_end, r0 + h * 32 + t % 4 * 8, r_end, v[h]);
        else fetch8<T>(base, ld, r0 + h * 32 + t / 8, r_end, i0 + t % 8 * 8, i_end, v[h]);
    }
}
// ... into LDS as they lie in memory, 16 bytes at a time: [row of the tile][summed index] (RC) or [summed index][column of the tile].
template <typename C, bool RC>
__device__ __forceinline__ void put_tile(int t, C* lds, const float (&u)[2][8]) {
    constexpr int LD = Lds<C>::LD;
    struct __attribute__((aligned(16))) V { C e[8]; };
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        V v;
#pragma unroll
        for (int j = 0; j < 8; ++j) v.e[j] = from_f<C>(u[h][j]);
        *(V*)(lds + (RC ? (t / 4) * LD + h * 32 + t % 4 * 8 : (h * 32 + t / 8) * LD + t % 8 * 8)) = v;
    }
}

__device__ __forceinline__ f32x4 mma32(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 mma32(f16x8 a, f16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
template <typename T> struct V8;
template <> struct V8<bf16_t> { typedef bf16x8 t; };
template <> struct V8<f16_t> { typedef f16x8 t; };

// A lane's part of a fragment of 16 rows or columns from `base`: 16-bit types 8 of the summed index from b + l / 16 * 8 on (out of [summed
// index][column] by two reads that transpose 4 x 16 values), fp32 4 from b + l / 16 * 4 on.
typedef short tile_s16x4 __attribute__((ext_vector_type(4)));
template <typename T, bool RC> __device__ __forceinline__ typename V8<T>::t fragment(int l, const T* lds, int base, int b) {
    constexpr int LD = Lds<T>::LD;
    const int i = l % 16, g = l / 16;
    if constexpr (RC) return *(const typename V8<T>::t*)(lds + (base + i) * LD + b + g * 8);
    else {
        typedef __attribute__((address_space(3))) tile_s16x4* p4;
        const T* at = lds + (b + g * 8 + i / 4) * LD + base + i % 4 * 4;
        const tile_s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((p4)at), hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((p4)(at + 4 * LD));
        typedef short s16x8 __attribute__((ext_vector_type(8)));
        const s16x8 v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        return __builtin_bit_cast(typename V8<T>::t, v);
    }
}
template <bool RC> __device__ __forceinline__ f32x4 fragment32(int l, const float* lds, int base, int b) {
    constexpr int LD = Lds<float>::LD;
    const int i = l % 16, g = l / 16;
    if constexpr (RC) return *(const f32x4*)(lds + (base + i) * LD + b + g * 4);
    else {
        const float* at = lds + (b + g * 4) * LD + base + i;
        return f32x4{at[0], at[LD], at[2 * LD], at[3 * LD]};
    }
}

// one TR-long step of a wave's 32 x 32 part
template <typename C, bool PRC, bool QRC>
__device__ __forceinline__ void tile_mma(int t, const C* lp, const C* lq, f32x4 (&acc)[2][2]) {
    const int l = t % 64, w = t / 64;
    if constexpr (sizeof(C) == 2) {
#pragma unroll
        for (int b = 0; b < TR; b += 32) {
            typename V8<C>::t p[2], q[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                p[i] = fragment<C, PRC>(l, lp, w / 2 * 32 + i * 16, b);
                q[i] = fragment<C, QRC>(l, lq, w % 2 * 32 + i * 16, b);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) acc[i][j] = mma32(q[j], p[i], acc[i][j]);
        }
    } else {
#pragma unroll
        for (int b = 0; b < TR; b += 16) {
            f32x4 p[2], q[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                p[i] = fragment32<PRC>(l, lp, w / 2 * 32 + i * 16, b);
                q[i] = fragment32<QRC>(l, lq, w % 2 * 32 + i * 16, b);
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
}

// The tile at (p0, q0), whole or (S.splits > 1) its part over a split of R.  256 threads, numbered t; several such groups of a block may run
// together if they all walk the same R.  A tile outside the matrix stores nothing.
template <typename T, typename C, int MODE>
__device__ __forceinline__ void tile_product(int t, const LinArgs& A, const LinSplit& S, int64_t split, int64_t p0, int64_t q0, float* part, float* part_db,
                                             char* smem) {
    C* lp = (C*)smem;
    C* lq = lp + TP * Lds<C>::LD;
    const int64_t P = MODE == MODE_DW ? A.N : A.M, Q = MODE == MODE_FWD ? A.N : A.K, R = MODE == MODE_FWD ? A.K : MODE == MODE_DX ? A.N : A.M;
    const int64_t ra = split * S.len, rb = ra + S.len < R ? ra + S.len : R;
    const T* x = (const T*)A.x;
    const T* w = (const T*)A.w;
    const T* dy = (const T*)A.dy;

    const bool product = MODE != MODE_DW || A.dw;   // (db alone: the column sums of ds; x may be null)
    float vp[2][8], vq[2][8], sum[8] = {};
    auto fetch = [&](int64_t r0) {
        if constexpr (MODE == MODE_FWD) {
            fetch_tile<T, true>(t, x, A.ldx, p0, P, r0, rb, vp);
            fetch_tile<T, true>(t, w, A.K, q0, Q, r0, rb, vq);
        } else {
            constexpr bool RC = MODE == MODE_DX;
            fetch_tile<T, RC>(t, dy, A.lddy, p0, P, r0, rb, vp);
            if (A.act != IVAE_ACT_NONE) {
                float s[2][8];
                fetch_tile<float, RC>(t, A.cpre, A.N, p0, P, r0, rb, s);
#pragma unroll
                for (int h = 0; h < 2; ++h) lin_act_slope_all<T>(A.act, A.slope, s[h], vp[h]);
            }
            if (MODE == MODE_DW)
#pragma unroll
                for (int j = 0; j < 8; ++j) sum[j] += vp[0][j] + vp[1][j];
            if (MODE == MODE_DX) fetch_tile<T, false>(t, w, A.K, q0, Q, r0, rb, vq);
            else if (product) fetch_tile<T, false>(t, x, A.ldx, q0, Q, r0, rb, vq);
        }
    };
    f32x4 acc[2][2] = {};
    if (ra < rb) fetch(ra);
    for (int64_t r = ra; r < rb; r += TR) {
        if (!product) {
            if (r + TR < rb) fetch(r + TR);
            continue;
        }
        __syncthreads();
        put_tile<C, MODE != MODE_DW>(t, lp, vp);
        put_tile<C, MODE == MODE_FWD>(t, lq, vq);
        __syncthreads();
        if (r + TR < rb) fetch(r + TR);
        tile_mma<C, MODE != MODE_DW, MODE == MODE_FWD>(t, lp, lq, acc);
    }
    // the sums go through LDS, so that what follows runs along rows, 8 columns a thread
    constexpr int LD = TQ + 4;
    float* sums = (float*)smem;
    const int l = t % 64, wv = t / 64;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) *(f32x4*)(sums + (wv / 2 * 32 + i * 16 + l % 16) * LD + wv % 2 * 32 + j * 16 + l / 16 * 4) = acc[i][j];
    const int64_t q = q0 + t % 8 * 8, left = Q - q;
    const int n = left >= 8 ? 8 : left > 0 ? (int)left : 0;
    const bool fwd = MODE == MODE_FWD && S.splits == 1;
    Raw8<T> bias, res[2];
    if (fwd) {
        if (A.b) bias.load((const T*)A.b + q, n);
        if (A.res)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int64_t p = p0 + h * 32 + t / 8;
                res[h].load((const T*)A.res + p * A.ldr + q, p < P ? n : 0);
            }
    }
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int64_t p = p0 + h * 32 + t / 8, at = p * Q + q;
        const int m = p < P ? n : 0;
        const float* from = sums + (h * 32 + t / 8) * LD + t % 8 * 8;
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = from[e] + (fwd && A.b ? bias.at(e) : 0.f);
        if (fwd) forward_store8<T>(A, at, m, v, A.res ? &res[h] : nullptr);
        else if (m && product) {
            if (S.splits > 1) store8(part + split * P * Q + at, m, v);
            else if (MODE == MODE_DX) store8((T*)A.dx + at, m, v);
            else store8((T*)A.dw + at, m, v);
        }
    }
    if (MODE == MODE_DW && A.db && q0 == 0) {       // thread t holds the sums of 8 columns over every 32nd row: 32 threads hold each column
        float* lsum = (float*)smem;
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
// LDS of one group of 256 threads: the tiles, then the sums
template <typename C> static constexpr int tile_lds() { return 2 * TP * Lds<C>::LD * (int)sizeof(C); }
static_assert(tile_lds<f16_t>() >= TP * (TQ + 4) * 4, "the sums fit");
