// What a large product needs done to a matrix before it can be loaded 16 bytes at a time: rows brought to 16-byte boundaries,
// fp32 cut into three bf16 parts, and in the backward pass the gradient of the pre-activation, ds = act'(s) dy, for 16-bit types as
// two numbers of the type, with its column sums (db) taken on the way.  One read and one write of the matrix; a thread takes 8
// neighbouring values of every row that its group walks.
#include "kernels.h"
#include "linear_pack.h"

// x = x0 + x1 + x2, 8 bits each, cut off rather than rounded: every part has x's sign and the first never overflows.  Infinities and
// NaN are whole in the first part.  -> what is lost, as bits that are not 0: below 2^-110 x has bits under 2^-133, the smallest that bf16 holds.
__device__ __forceinline__ uint32_t cut(float x, bf16_t (&o)[3]) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    const bool finite = (u & 0x7f800000u) != 0x7f800000u;
    const uint32_t h0 = finite || (u & 0x007fffffu) == 0 ? u & 0xffff0000u : u | 0x00400000u;
    const float r1 = finite ? x - __builtin_bit_cast(float, h0 & 0xffff0000u) : 0.f;
    const uint32_t u1 = __builtin_bit_cast(uint32_t, r1) & 0xffff0000u;
    const float r2 = r1 - __builtin_bit_cast(float, u1);
    o[0] = __builtin_bit_cast(bf16_t, (uint16_t)(h0 >> 16));
    o[1] = __builtin_bit_cast(bf16_t, (uint16_t)(u1 >> 16));
    o[2] = __builtin_bit_cast(bf16_t, (uint16_t)(__builtin_bit_cast(uint32_t, r2) >> 16));
    return __builtin_bit_cast(uint32_t, r2) << 16;
}

// scale v = hi + lo / up, both of type T.  A finite value stays finite; infinities and NaN are whole in hi.
template <typename T> struct Largest { static constexpr float v = 65504.f; };
template <> struct Largest<bf16_t> { static constexpr float v = 3.3895313892515355e38f; };
template <typename T> __device__ __forceinline__ void halve(float v, float up, float& hi, float& lo) {
    hi = to_f(from_f<T>(v));
    if (fabsf(hi) == __builtin_inff() && fabsf(v) < __builtin_inff()) hi = copysignf(Largest<T>::v, v);
    lo = fabsf(hi) < __builtin_inff() ? (v - hi) * up : 0.f;
}

struct PackJobs { PackArgs job[3]; };
template <typename T>
__global__ __launch_bounds__(256) void k_pack(PackJobs J) {
    int block = blockIdx.x, k = 0;
    while (block >= J.job[k].blocks) block -= J.job[k++].blocks;
    const PackArgs& A = J.job[k];
    const int bx = block % A.blocks_x, by = block / A.blocks_x, rows_of_blocks = A.blocks / A.blocks_x;
    const int group = A.group;                          // threads that share a row of 8 * group values
    const int col = (bx * group + threadIdx.x % group) * 8, sub = threadIdx.x / group, subs = 256 / group;
    float sum[8] = {};
    uint32_t lost = 0, most = 0;
    const int left = A.cols - col;                      // <= 0: beyond the last value (the padding is zeros)
    for (int64_t r = (int64_t)by * subs + sub; r < A.rows && col < A.ldo; r += (int64_t)rows_of_blocks * subs) {
        float v[8], s[8];
        const T* p = (const T*)A.src + r * A.ld + col;
        constexpr int N = Wide<T>::N;
#pragma unroll
        for (int h = 0; h < 8 / N; ++h) {
            float u[N];
            if (left - h * N >= N) load_wide<T>(p + h * N, u);
            else load_part<T>(p + h * N, left - h * N, u);
#pragma unroll
            for (int j = 0; j < N; ++j) v[h * N + j] = u[j];
        }
        if (A.pre) {
            const float* q = A.pre + r * A.cols + col;
#pragma unroll
            for (int h = 0; h < 8; h += 4) {
                float u[4];
                if (left - h >= 4) load_wide<float>(q + h, u);
                else load_part<float>(q + h, left - h, u);
#pragma unroll
                for (int j = 0; j < 4; ++j) s[h + j] = u[j];
            }
            lin_act_slope_all<T>(A.act, A.slope, s, v);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) sum[j] += v[j];
        if (!A.out) continue;
        if constexpr (sizeof(T) == 2) {
            T* to = (T*)A.out + r * A.ldo + col;
            if (A.pair) {
                float lo[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) halve<T>(v[j] * A.scale, A.up, v[j], lo[j]);
                store_wide<T>(to + A.plane, lo);
            }
            store_wide<T>(to, v);
        } else {
            const int64_t at = (col / 32 * A.rows + r) * 32 + col % 32;
            if (A.flip != FLIP_NONE && ((A.flip == FLIP_ROWS ? (int)(r >> 5) : col >> 5) & 1))
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = -v[j];
            struct __attribute__((aligned(16))) V { bf16_t e[8]; } part[3];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                bf16_t o[3];
                lost |= cut(v[j], o);
                const uint32_t size = __builtin_bit_cast(uint32_t, v[j]) & 0x7fffffffu;
                if (size < 0x7f800000u && size > most) most = size;
#pragma unroll
                for (int k = 0; k < 3; ++k) part[k].e[j] = o[k];
            }
#pragma unroll
            for (int k = 0; k < 3; ++k) *(V*)((bf16_t*)A.out + k * A.plane + at) = part[k];
        }
    }
    if (sizeof(T) == 4 && A.out) {
        __shared__ uint32_t waves[4];
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) most = max(most, (uint32_t)__shfl_xor((int)most, o));
        if (threadIdx.x % 64 == 0) waves[threadIdx.x / 64] = most;
        const int any = __syncthreads_or(lost != 0);
        if (threadIdx.x == 0) A.range[block] = uint2{any ? 1u : 0u, max(max(waves[0], waves[1]), max(waves[2], waves[3]))};
    }
    if (!A.colsum) return;
    __shared__ float fold[256][9];
#pragma unroll
    for (int j = 0; j < 8; ++j) fold[threadIdx.x][j] = sum[j];
    __syncthreads();
    for (int i = threadIdx.x; i < group * 8; i += 256) {
        float s = 0.f;
        for (int k = 0; k < subs; ++k) s += fold[k * group + i / 8][i % 8];
        const int c = bx * group * 8 + i;
        if (c < A.cols) A.colsum[(int64_t)by * A.cols + c] = s;
    }
}

// threads that share a row, a power of two: their 8 values each cover it, or 512 values of it; fp32 128, four columns of the result
// (8192 x 2048 twice and 2048 x 2048, with ds: 70 us; one column 84 us, 16 columns 90 us)
static int group_of(int64_t width, int dtype) {
    if (dtype == IVAE_F32) return 16;
    int g = 1;
    while (g < 64 && g * 8 < width) g *= 2;
    return g;
}
// blocks along the rows: about 2048 blocks in all, and then more rows a thread; with column sums at most 256, whose sums are joined
int pack_row_blocks(int64_t rows, int64_t width, bool colsum, int dtype) {
    const int g = group_of(width, dtype);
    const int64_t strips = (width + g * 8 - 1) / (g * 8), subs = 256 / g;
    int64_t y = (rows + subs - 1) / subs, most = 2048 / strips;
    if (colsum && most > 256) most = 256;
    if (y > most) y = most;
    return (int)(y < 1 ? 1 : y);
}
int pack_blocks(int64_t rows, int64_t width, bool colsum, int dtype) {
    const int g = group_of(width, dtype);
    return (int)((width + g * 8 - 1) / (g * 8)) * pack_row_blocks(rows, width, colsum, dtype);
}
hipError_t launch_packs(const PackArgs* const* P, int n, int dtype, hipStream_t st) {
    PackJobs J = {};
    int jobs = 0, blocks = 0;
    for (int i = 0; i < n; ++i) {
        if (!P[i]) continue;
        PackArgs& A = J.job[jobs++] = *P[i];
        A.group = group_of(A.ldo, dtype);
        A.blocks_x = (int)((A.ldo + A.group * 8 - 1) / (A.group * 8));
        A.blocks = pack_blocks(A.rows, A.ldo, A.colsum != nullptr, dtype);
        blocks += A.blocks;
    }
    if (blocks == 0) return hipSuccess;
    const dim3 g((unsigned)blocks), b(256);
    if (dtype == IVAE_F32) hipLaunchKernelGGL(k_pack<float>, g, b, 0, st, J);
    else if (dtype == IVAE_BF16) hipLaunchKernelGGL(k_pack<bf16_t>, g, b, 0, st, J);
    else hipLaunchKernelGGL(k_pack<f16_t>, g, b, 0, st, J);
    return hipGetLastError();
}
