// The linear operator on 64 x 64 tiles staged through registers (linear_tile.h): any size, any row stride, any alignment, and in the backward
// pass one launch for dx, dw and db (the gradient of the pre-activation is formed while its tile is loaded and never stored).
// A long sum over few tiles is split; the parts are written in 32 bits and added in order by k_linear_join_*.
#include "kernels.h"
#include "linear_tile.h"

struct At { int64_t split, p0, q0; };
__device__ __forceinline__ At at_of(const LinSplit& S, int64_t b) {
    const int64_t split = b / (S.tp * S.tq), tile = b - split * S.tp * S.tq;
    return {split, tile / S.tq * TP, tile % S.tq * TQ};
}

template <typename T>
__global__ __launch_bounds__(256) void k_linear_fwd(LinArgs A, LinSplit S) {
    __shared__ __attribute__((aligned(16))) char smem[tile_lds<T>()];
    const int64_t tiles = S.tp * S.tq * S.splits;
    for (int64_t b = blockIdx.x; b < tiles; b += gridDim.x) {
        const At at = at_of(S, b);
        tile_product<T, T, MODE_FWD>(threadIdx.x, A, S, at.split, at.p0, at.q0, A.part, nullptr, smem);
    }
}
template <typename T, typename C>
__global__ __launch_bounds__(256) void k_linear_bwd(LinArgs A, LinSplit X, LinSplit W, float* part_w, float* part_b) {
    __shared__ __attribute__((aligned(16))) char smem[tile_lds<C>()];
    const int64_t nx = X.tp * X.tq * X.splits, tiles = nx + W.tp * W.tq * W.splits;
    for (int64_t b = blockIdx.x; b < tiles; b += gridDim.x) {
        const At at = b < nx ? at_of(X, b) : at_of(W, b - nx);
        if (b < nx) tile_product<T, C, MODE_DX>(threadIdx.x, A, X, at.split, at.p0, at.q0, A.part, nullptr, smem);
        else tile_product<T, C, MODE_DW>(threadIdx.x, A, W, at.split, at.p0, at.q0, part_w, part_b, smem);
    }
}

// 8 neighbouring sums of `splits` parts of n values, four parts under way at a time
__device__ __forceinline__ void join8(const float* part, int splits, int64_t n, int64_t i, int left, float (&v)[8]) {
    Raw8<float> u[4];
    u[0].load(part + i, left);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = u[0].at(e);
    int k = 1;
    if (left == 8)
        for (; k + 4 <= splits; k += 4) {
#pragma unroll
            for (int j = 0; j < 4; ++j) u[j].load(part + (k + j) * n + i, 8);
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] += u[j].at(e);
        }
    for (; k < splits; ++k) {
        u[0].load(part + k * n + i, left);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += u[0].at(e);
    }
}
template <typename T>
__global__ __launch_bounds__(256) void k_linear_join_fwd(LinArgs A, int splits) {
    const int64_t n = A.M * A.N, groups = (A.N + 7) / 8, all = A.M * groups;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) {
        const int64_t m = i / groups, q = (i - m * groups) * 8, at = m * A.N + q;
        const int left = A.N - q < 8 ? (int)(A.N - q) : 8;
        Raw8<T> r, b;
        if (A.res) r.load((const T*)A.res + m * A.ldr + q, left);
        float v[8];
        join8(A.part, splits, n, at, left, v);
        if (A.b) {
            b.load((const T*)A.b + q, left);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] += b.at(e);
        }
        forward_store8<T>(A, at, left, v, A.res ? &r : nullptr);
    }
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
    const int64_t gx = (nx + 7) / 8, gw = (nw + 7) / 8;
    for (int64_t g = (int64_t)(blockIdx.x - nb) * 256 + threadIdx.x; g < gx + gw; g += (int64_t)(gridDim.x - nb) * 256) {
        const bool x = g < gx;
        const int64_t n = x ? nx : nw, i = (x ? g : g - gx) * 8;
        const int left = n - i < 8 ? (int)(n - i) : 8;
        float v[8];
        join8(x ? J.x : J.w, x ? J.kx : J.kw, n, i, left, v);
        store8((T*)(x ? A.dx : A.dw) + i, left, v);
    }
}

// A part sums over 128 (two steps of a tile) or more, where R is `from` or more: in the backward pass a step takes 1.3 to 3.5 us (16 bits without
// an activation; fp32, xtanh), less in the forward pass, and a join takes 4 us and a launch.  Gradients of 1024 x 96 x 72 in fp32 with xtanh
// and their join: parts of 256 28 us, of 128 18 us; 300 x 300 x 300: one part 28 us, two 23 us; 256 rows: no difference,
// unless the other gradient is joined anyway.
static const int SPLIT_FORWARD = 512, SPLIT_BACKWARD = 257;
static LinSplit split_of(int64_t P, int64_t Q, int64_t R, int from) {
    LinSplit S;
    S.tp = (P + TP - 1) / TP;
    S.tq = (Q + TQ - 1) / TQ;
    const int64_t tiles = S.tp * S.tq;
    auto parts = [&](int64_t blocks, int64_t len) { return blocks / tiles < R / len ? blocks / tiles : R / len; };
    // up to one block a CU in parts of 128 or more, up to two in parts of 256 or more
    int64_t s = tiles == 0 || tiles >= 256 || R < from ? 1 : parts(256, 128) > parts(512, 256) ? parts(256, 128) : parts(512, 256);
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
    p.X = split_of(A.M, A.K, A.N, SPLIT_BACKWARD);
    p.W = split_of(A.N, A.K, A.M, SPLIT_BACKWARD);
    if (p.X.splits > 1 && A.dx) p.W = split_of(A.N, A.K, A.M, 0);
    else if (p.W.splits > 1 && A.dw) p.X = split_of(A.M, A.K, A.N, 0);
    if (!A.dx) p.X.tp = 0;
    if (!A.dw) p.W.tq = A.db ? 1 : 0;                           // db alone: the first column of tiles sums it
    const int64_t nx = A.dx && p.X.splits > 1 ? p.X.splits * A.M * A.K : 0;
    const bool split_w = p.W.tq && p.W.splits > 1;
    const int64_t nw = A.dw && split_w ? (int64_t)p.W.splits * A.N * A.K : 0;
    p.off_w = nx;
    p.off_b = nx + nw;
    p.floats = nx + nw + (split_w ? (int64_t)p.W.splits * A.N : 0);
    return p;
}
size_t linear_small_ws(const LinArgs& A, bool backward) {
    if (!backward) {
        const LinSplit S = split_of(A.M, A.N, A.K, SPLIT_FORWARD);
        return S.splits > 1 ? (size_t)S.splits * A.M * A.N * 4 : 0;
    }
    return (size_t)plan_bwd(A).floats * 4;
}

void linear_small_splits(const LinArgs& A, bool backward, int32_t* splits) {
    if (!backward) {
        splits[0] = split_of(A.M, A.N, A.K, SPLIT_FORWARD).splits;
        return;
    }
    const BwdPlan p = plan_bwd(A);
    splits[0] = p.X.splits;
    splits[1] = p.W.splits;
}

static unsigned cap(int64_t blocks) { return (unsigned)(blocks < (1 << 20) ? blocks : 1 << 20); }

hipError_t linear_join_forward(const LinArgs& A, int splits, int dtype, hipStream_t st) {
    if (splits < 2) return hipSuccess;
    const dim3 g(cap((A.M * ((A.N + 7) / 8) + 255) / 256)), b(256);
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
    const int64_t n = (J.kx > 1 ? (A.M * A.K + 7) / 8 : 0) + (J.kw > 1 ? ((int64_t)A.N * A.K + 7) / 8 : 0);
    const unsigned blocks = cap((n + 255) / 256) + (J.kb > 0 ? (unsigned)((A.N + 63) / 64) : 0);
    if (blocks == 0) return hipSuccess;
    const dim3 g(blocks), b(256);
    if (dtype == IVAE_F32) hipLaunchKernelGGL(k_linear_join_bwd<float>, g, b, 0, st, A, J);
    else if (dtype == IVAE_BF16) hipLaunchKernelGGL(k_linear_join_bwd<bf16_t>, g, b, 0, st, A, J);
    else hipLaunchKernelGGL(k_linear_join_bwd<f16_t>, g, b, 0, st, A, J);
    return hipGetLastError();
}
template <typename T> static void fwd(const LinArgs& A, hipStream_t st) {
    const LinSplit S = split_of(A.M, A.N, A.K, SPLIT_FORWARD);
    hipLaunchKernelGGL(k_linear_fwd<T>, dim3(cap(S.tp * S.tq * S.splits)), dim3(256), 0, st, A, S);
}
hipError_t linear_small_forward(const LinArgs& A, int dtype, hipStream_t st) {
    if (dtype == IVAE_F32) fwd<float>(A, st);
    else if (dtype == IVAE_BF16) fwd<bf16_t>(A, st);
    else fwd<f16_t>(A, st);
    const hipError_t e = hipGetLastError();
    return e != hipSuccess ? e : linear_join_forward(A, split_of(A.M, A.N, A.K, SPLIT_FORWARD).splits, dtype, st);
}
template <typename T> static void bwd(const LinArgs& A, const BwdPlan& p, float* pw, float* pb, hipStream_t st) {
    const int64_t tiles = p.X.tp * p.X.tq * p.X.splits + p.W.tp * p.W.tq * p.W.splits;
    if (tiles == 0) return;
    const dim3 g(cap(tiles)), b(256);
    if (A.act == IVAE_ACT_NONE) hipLaunchKernelGGL((k_linear_bwd<T, T>), g, b, 0, st, A, p.X, p.W, pw, pb);
    else hipLaunchKernelGGL((k_linear_bwd<T, float>), g, b, 0, st, A, p.X, p.W, pw, pb);
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
