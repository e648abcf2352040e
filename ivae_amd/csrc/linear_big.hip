// Large products of the linear operator on the matrix cores.
//
// Operands go from memory straight into LDS (buffer_load ... lds, 16 bytes a lane) in two buffers or more: a step's loads are issued, spread
// over matrix instructions, once its buffer has been read, so that one barrier a step is enough.  An operand whose summed index runs along its rows
// is read from LDS 16 bytes a lane; one whose summed index runs down its rows (the weight in dx, both operands of dw) is read with
// ds_read_b64_tr_b16, which transposes 4 x 16 values on the way into the registers: no operand is ever transposed in memory.
// LDS rows cannot be padded (a load fills them in lane order), so the 16-byte groups of a row are permuted instead, by an XOR with
// bits of the row number that puts every 16 lanes (along) or every 8 groups of 32 bytes (down) on distinct banks.
//
// 16-bit types with an activation, backward: act'(s) dy has 32 bits and enters as a pair of numbers of the type, P = scale (first + low
// second), the whole sum over the second before the one over the first, in the same registers.  bf16: the second is what rounding left,
// times 2^7 (half of the first at most): off by 2^-16 of the value, or 2^-141 among the smallest.  fp16: values are divided by a bound of
// act', so that dy's range fits, and what rounding left is multiplied by 2^11: off by 2^-22 of the value, or 2^-36 times the bound among the
// smallest.  The products cost twice the time (8192 x 4096 x 4096 bf16, gelu: 446 -> 826 us); with one number the results had 1.4 times the
// error of their own rounding, and fp16 lost gradients of 1e-6 and those beyond 65504.  A second number of 0 makes a NaN of an infinity: tiles
// with a NaN are computed again in fp32, as below.
//
// fp32 (k_split_*): x = x0 + x1 + x2 with bf16 parts cut off after 8 bits each (exact from 2^-110 on), and x y = x0 y0 + x0 y1 + x1 y0 + x1 y1 + x0 y2 +
// x2 y0 up to 2^-23 |x y|: six products at 16 times the rate of the fp32 matrix instructions.  The running sum of the bf16 matrix
// instructions drifts downwards, by little but always the same way, and a column sum over such results would add that up; so every 32 of
// the summed index start from zero, smallest products first, and are added to the sum by fp32 additions that round to nearest.
// An infinity times a part that is 0 makes a NaN that fp32 would not: a tile with a NaN in it is computed again in fp32, from the
// tensors themselves.  So is one with a result of which the bits that smaller values lost can be more than 2^-25.
#include <type_traits>

#include "kernels.h"
#include "linear_big.h"
#include "linear_tile.h"

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) char* lds_ptr;

__device__ __forceinline__ f32x4 mma(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 mma(f16x8 a, f16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
template <typename E> struct E8;
template <> struct E8<bf16_t> { typedef bf16x8 t; };
template <> struct E8<f16_t> { typedef f16x8 t; };

__device__ const uint4 g_zeros = {0, 0, 0, 0};          // where lanes beyond the sum read

// One operand's tile of B rows (along) or B columns (down) and BR (64 or 32) of the summed index.  THREADS x 16 bytes a load.
template <int B, int BR, bool ALONG, bool COLUMNS, int THREADS>
struct Stage {
    static constexpr int BYTES = B * BR * 2, LOADS = BYTES / (THREADS * 16), PER_ROW = (ALONG ? BR : B) / 8;
    static_assert(!COLUMNS || BR == 32, "a step is one column");
    static_assert(BYTES % (THREADS * 16) == 0 && THREADS / PER_ROW % 16 == 0, "whole loads; the rows of one thread share a swizzle");
    uint32_t voff[LOADS];       // bytes from the tile's corner
    int row, col;               // of load 0, in elements; load j is j * (THREADS / PER_ROW) rows further
    const char* corner;
    int64_t step;               // bytes from one BR to the next

    static __device__ __forceinline__ int swizzle(int row) {
        if (ALONG) return BR == 64 ? row >> 1 & 7 : -(row >> 2) & 3;
        return ((row & 3) | (row >> 1 & 4)) << 1 & (PER_ROW - 1);          // (row >> 1 & 4 is bit 3 of the row, moved to bit 2)
    }

    __device__ __forceinline__ void init(const BigOperand& O, int64_t e0, int64_t r0) {
        const int t = threadIdx.x;
        row = t / PER_ROW;
        col = (t % PER_ROW ^ swizzle(row)) * 8;
        if (ALONG) {
            corner = (const char*)O.base + (COLUMNS ? (r0 / 32 * O.ld + e0) * 64 : (e0 * O.ld + r0) * 2);
            step = COLUMNS ? O.ld * 64 : BR * 2;
#pragma unroll
            for (int j = 0; j < LOADS; ++j) {
                int64_t e = row + j * (THREADS / PER_ROW);
                if (e0 + e >= O.extent) e = O.extent - 1 - e0;             // rows past the end repeat the last one; their results are not stored
                voff[j] = (uint32_t)(COLUMNS ? e * 64 + col * 2 : (e * O.ld + col) * 2);
            }
        } else {
            corner = (const char*)O.base + (COLUMNS ? (e0 / 32 * O.ld + r0) * 64 : (r0 * O.ld + e0) * 2);
            step = COLUMNS ? BR * 64 : (int64_t)BR * O.ld * 2;
            int64_t c = col;
            if (e0 + c >= O.extent) c = O.extent - 8 - e0;
#pragma unroll
            for (int j = 0; j < LOADS; ++j) {
                const int r = row + j * (THREADS / PER_ROW);
                voff[j] = (uint32_t)(COLUMNS ? (c / 32 * O.ld + r) * 64 + c % 32 * 2 : (r * O.ld + c) * 2);
            }
        }
    }
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    __device__ __forceinline__ u32x4 resource(int64_t advance) const {
        const uint64_t a = (uint64_t)(corner + advance);
        u32x4 r;
        r.x = __builtin_amdgcn_readfirstlane((uint32_t)a);
        r.y = __builtin_amdgcn_readfirstlane((uint32_t)(a >> 32)) & 0xffffu;
        r.z = 0xffffffffu;
        r.w = 0x00020000u;
        return r;
    }
    static __device__ __forceinline__ uint32_t wave_base(uint32_t lds) { return __builtin_amdgcn_readfirstlane(lds + threadIdx.x / 64 * 1024); }
    // (m0 is written without the compiler's knowledge, which takes no clobber of it: nothing that it makes of these kernels uses m0)
    __device__ __forceinline__ void load_one(int j, uint32_t base, u32x4 rsrc) const {
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(base + j * THREADS * 16), "v"(voff[j]), "s"(rsrc)
                     : "memory");
    }
    // all of BR lies inside the operand
    __device__ __forceinline__ void load_full(uint32_t lds, int64_t advance) const {
        const u32x4 rsrc = resource(advance);
        const uint32_t base = wave_base(lds);
#pragma unroll
        for (int j = 0; j < LOADS; ++j) load_one(j, base, rsrc);
    }
    // `left` of the summed index remain: what lies beyond reads zeros
    __device__ __forceinline__ void load_part(uint32_t lds, int64_t advance, int64_t left) const {
        const uint32_t base = __builtin_amdgcn_readfirstlane(lds + threadIdx.x / 64 * 1024);
#pragma unroll
        for (int j = 0; j < LOADS; ++j) {
            const bool in = ALONG ? col < left : row + j * (THREADS / PER_ROW) < left;
            const char* p = in ? corner + advance + voff[j] : (const char*)&g_zeros;
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(base + j * THREADS * 16), "v"(p) : "memory");
        }
    }
    // lane's address in the fragment of the 16 rows / columns from `base` (a multiple of 64) in the first 32 of the summed index
    static __device__ __forceinline__ int frag(int base) {
        const int l = threadIdx.x % 64, i = l % 16, g = l / 16;
        if (ALONG) return (base + i) * (BR * 2) + ((g ^ swizzle(i)) << 4);
        const int r = g * 8 + i / 4, c = base + i % 4 * 4;                 // the first four of a lane group's eight rows
        return r * (B * 2) + (((c >> 3) ^ swizzle(r)) << 4) + (c & 4) * 2;
    }
    // The i-th 16 from there on (i * 16 < 128), in the k-th 32, of the tile at `lds` (a multiple of 256): from(lds, first, k), then read(from, i,
    // k).  Along: 16 rows keep the swizzle, k flips bit 2 of the group.  Down: 16 columns are 2 groups, and i flips bits of the group like
    // the swizzle does; 32 rows keep it, and 4 rows too (bit 2 of the row is in no swizzle).  Steps of 32: k counts tiles that follow.
    static __device__ __forceinline__ uint32_t from(uint32_t lds, int first, int k) {
        uint32_t a = lds + (ALONG ? first ^ k << 6 : first);
        asm("" : "+v"(a));                      // one register that all reads share, what is constant goes into their offsets
        return a;
    }
    template <typename E> static __device__ __forceinline__ typename E8<E>::t read(uint32_t from, int i, int k) {
        if constexpr (ALONG) return *(const __attribute__((address_space(3))) typename E8<E>::t*)(uintptr_t)(from + i * 16 * BR * 2 + (BR == 32 ? k * BYTES : 0));
        else {
            typedef __attribute__((address_space(3))) s16x4* p4;
            const uint32_t at = (from ^ i << 5) + k * 32 * B * 2;
            const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((p4)(uintptr_t)at);
            const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((p4)(uintptr_t)(at + B * 8));
            typedef short s16x8 __attribute__((ext_vector_type(8)));
            const s16x8 v = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
            return __builtin_bit_cast(typename E8<E>::t, v);
        }
    }
};

// LDS of a block: `buffers` of a step, and in the end 128 rows of sums (4 words of padding keep a column off one bank)
static constexpr int big_lds(int buffers, int step_bytes, int btq) {
    return buffers * step_bytes > 128 * (btq + 4) * 4 ? buffers * step_bytes : 128 * (btq + 4) * 4;
}

// all but the last N loads into LDS have arrived (they are counted in the order of their issue), and all LDS reads
template <int N> __device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory"); }
__device__ __forceinline__ void block_barrier() {
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// Tiles in bands of 8 rows of tiles, neighbours in a band one after the other, and a contiguous run of them for each of the 8 dies
// (blocks go to the dies in turn): a die's cache then serves the few operand strips that its run shares.
// (Bands of 1 | 4 | 8 | 16: fp16 2048 x 8192 x 8192 gradients 485 | 443 | 446 | 451 us, fp32 8192 x 2048 x 2048 forward 339 | 338 | 347 | 351.)
struct Place { int64_t p0, q0, ra, rb; int split; };
template <int BTP, int BTQ> __device__ __forceinline__ Place place(const BigProduct& G, int b) {
    const int tp = (int)((G.p_end + BTP - 1) / BTP), tq = (int)((G.q_end + BTQ - 1) / BTQ), tiles = tp * tq, blocks = tiles * G.splits;
    const int per = blocks / 8, extra = blocks % 8, die = b % 8;
    b = die * per + (die < extra ? die : extra) + b / 8;
    Place r;
    r.split = b / tiles;
    b -= r.split * tiles;
    const int band = b / (8 * tq), in_band = b - band * 8 * tq, rows = tp - band * 8 < 8 ? tp - band * 8 : 8;
    const int ip = band * 8 + in_band % rows, iq = in_band / rows;
    r.p0 = (int64_t)ip * BTP;
    r.q0 = (int64_t)iq * BTQ;
    r.ra = r.split * G.len;
    r.rb = r.ra + G.len < G.R ? r.ra + G.len : G.R;
    return r;
}

// The residual of a tile on its way into the L2 cache while the last step is multiplied (with saved values, 8192 x 4096 x 4096 bf16: 283 -> 266
// us): 4 bytes of each 64 are loaded, into LDS `at` which nothing reads.
template <typename T, int BTP, int BTQ, int THREADS>
__device__ __forceinline__ void touch_residual(const BigProduct& G, const LinArgs& A, const Place& at0, uint32_t at) {
    constexpr int E = 64 / sizeof(T), PER_ROW = BTQ / E, LOADS = BTP * PER_ROW / THREADS;
    const uint32_t base = __builtin_amdgcn_readfirstlane(at + threadIdx.x / 64 * 256);
    int64_t q = at0.q0 + threadIdx.x % PER_ROW * E;
    // (4 bytes inside the row, of 64 columns at least: at the element, or where that lies off 4 bytes at the next one)
    constexpr int INSIDE = sizeof(T) == 2 ? 3 : 1;
    if (q > G.q_end - INSIDE) q = G.q_end - INSIDE;
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
        int64_t p = at0.p0 + threadIdx.x / PER_ROW + j * (THREADS / PER_ROW);
        if (p >= G.p_end) p = G.p_end - 1;
        const uintptr_t a = ((uintptr_t)((const T*)A.res + p * A.ldr + q) + 3) & ~(uintptr_t)3;
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(base), "v"(a) : "memory");
    }
}

// The sums go through LDS, up to 128 rows of the tile at a time, so that what follows runs along whole rows: 16-byte loads of the residual
// (two rows ahead of their use) and stores of the results, side by side, and one copy of the code for them.
template <typename T, int BTP, int BTQ, int WP, int WQ, int EPI, int FP, int FQ>
__device__ __forceinline__ void finish(const BigProduct& G, const LinArgs& A, const Place& at0, const f32x4 (&acc)[FP][FQ], float* sums) {
    constexpr int THREADS = WP * WQ * 64, ROWS = BTP < 128 ? BTP : 128, HALVES = BTP / ROWS, LD = BTQ + 4;
    constexpr int RW = 16 * FP / HALVES, STEP = THREADS / (BTQ / 8), ITERS = ROWS / STEP;          // RW rows of each row of waves
    static_assert(WP * RW == ROWS && FP % HALVES == 0 && ITERS * STEP == ROWS, "whole passes");
    const int wave = threadIdx.x / 64, l = threadIdx.x % 64, wq = wave % WQ * (BTQ / WQ);
    const int col = threadIdx.x % (BTQ / 8) * 8, row0 = threadIdx.x / (BTQ / 8);
    const int64_t Q = G.q_end, q = at0.q0 + col, left = Q - q;
    const int n = left >= 8 ? 8 : left > 0 ? (int)left : 0;
    const bool fwd = EPI == EPI_FWD && G.splits == 1, res = fwd && A.res;
    float bias[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (fwd && A.b) {
        Raw8<T> b;
        b.load((const T*)A.b + q, n);
#pragma unroll
        for (int e = 0; e < 8; ++e) bias[e] = b.at(e);
    }
#pragma unroll
    for (int h = 0; h < HALVES; ++h) {
        auto p_of = [&](int it) {
            const int row = row0 + it * STEP;
            return at0.p0 + (HALVES == 1 ? row : row / RW * (BTP / WP) + h * RW + row % RW);
        };
        auto load_res = [&](int it) {
            Raw8<T> r;
            const int64_t p = p_of(it);
            r.load((const T*)A.res + p * A.ldr + q, it < ITERS && p < G.p_end ? n : 0);
            return r;
        };
        Raw8<T> r0, r1;
        if (res) r0 = load_res(0), r1 = load_res(1);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < FP / HALVES; ++i)
#pragma unroll
            for (int j = 0; j < FQ; ++j)
                *(f32x4*)(sums + (wave / WQ * RW + i * 16 + l % 16) * LD + wq + j * 16 + l / 16 * 4) = acc[h * (FP / HALVES) + i][j];
        __syncthreads();
        if (EPI == EPI_FWD && h == 0) wait_loads<0>();          // (what touch_residual loads into LDS among them)
#pragma unroll 1
        for (int it = 0; it < ITERS; ++it) {
            Raw8<T> r2;
            if (res) r2 = load_res(it + 2);
            const int64_t p = p_of(it), at = p * Q + q;
            const float* from = sums + (row0 + it * STEP) * LD + col;
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = from[e] + bias[e];
            const int m = p < G.p_end ? n : 0;
            if (fwd) forward_store8<T>(A, at, m, v, res ? &r0 : nullptr);
            else if (m) {
                if (G.splits > 1) store8(G.part + (int64_t)at0.split * G.p_end * Q + at, m, v);
                else store8((T*)G.out + at, m, v);
            }
            r0 = r1;
            r1 = r2;
        }
    }
}

// Split fp32: cutting drops bits under 2^-133 of values below 2^-110, so a sum over R terms is off by at most R 2^-133 (the largest |P| and
// the largest |Q|).  Has a block that cut an operand seen such a value? (four blocks' answers under way at a time)
template <int THREADS> __device__ __forceinline__ uint32_t lost_bits(const BigOperand& O) {
    uint32_t lost = 0;
    for (int i = threadIdx.x; i < O.ranges; i += 4 * THREADS) {
        uint32_t v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = O.range[min(i + j * THREADS, O.ranges - 1)].x;
        lost |= v[0] | v[1] | v[2] | v[3];
    }
    return lost;
}
__device__ __forceinline__ float largest(const BigOperand& O) {             // by every wave for itself
    uint32_t most = 0;
    for (int i = threadIdx.x % 64; i < O.ranges; i += 64) most = max(most, O.range[i].y);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) most = max(most, (uint32_t)__shfl_xor((int)most, o));
    return __builtin_bit_cast(float, most);
}
// A tile with a NaN in it, or with a result of which lost bits can be more than 2^-25, is computed again in fp32 from the tensors, 64 x 64 at a
// time by every 256 threads.  -> whether it was.
template <typename T, int BTP, int BTQ, int THREADS, int MODE, int FP, int FQ>
__device__ __forceinline__ bool again_if_needed(const BigProduct& G, const LinArgs& A, const Place& at0, const f32x4 (&acc)[FP][FQ], char* smem) {
    constexpr bool CUT = sizeof(T) == 4;
    uint32_t lost = 0;
    if (CUT) lost = lost_bits<THREADS>(G.P) | lost_bits<THREADS>(G.Q);
    int nan = 0;
#pragma unroll
    for (int i = 0; i < FP; ++i)
#pragma unroll
        for (int j = 0; j < FQ; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) nan |= acc[i][j][e] != acc[i][j][e];
    if (!__syncthreads_or(nan | (int)lost)) return false;
    if (CUT) {
        const float scale = 0x1p-108f * (float)G.len, least = scale * largest(G.P) + scale * largest(G.Q);
#pragma unroll
        for (int i = 0; i < FP; ++i)
#pragma unroll
            for (int j = 0; j < FQ; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) nan |= fabsf(acc[i][j][e]) < least;
        if (!__syncthreads_or(nan)) return false;
    }
    constexpr int GROUPS = THREADS / 256, SUBS = (BTP / 64) * (BTQ / 64);
    static_assert(SUBS % GROUPS == 0, "the groups meet the same barriers");
    const LinSplit S = {0, 0, G.splits, G.len};
    LinArgs B = A;
    B.db = nullptr;                         // (its sums are fp32 already)
    const int group = threadIdx.x / 256;
    wait_loads<0>();
    __syncthreads();
    for (int u = group; u < SUBS; u += GROUPS)
        tile_product<T, float, MODE>(threadIdx.x % 256, B, S, at0.split, at0.p0 + u / (BTQ / 64) * 64, at0.q0 + u % (BTQ / 64) * 64, G.part, nullptr,
                                     smem + group * tile_lds<float>());
    return true;
}

// 16-bit types.  BT x BT tiles, WP x WQ waves, 64 of the summed index a step, BUFS buffers.
template <typename T, int BT, int WP, int WQ, int BUFS, bool PA, bool QA, int EPI>
__device__ __forceinline__ void big_tile(const BigProduct& G, const LinArgs& A, int block, char* smem) {
    constexpr int THREADS = WP * WQ * 64, FP = BT / WP / 16, FQ = BT / WQ / 16, BR = 64;
    typedef Stage<BT, BR, PA, false, THREADS> SP;
    typedef Stage<BT, BR, QA, false, THREADS> SQ;
    typedef typename E8<T>::t v8;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_ptr)smem;
    constexpr int BUF = SP::BYTES + SQ::BYTES, LOADS = SP::LOADS + SQ::LOADS;
    const Place at0 = place<BT, BT>(G, block);

    SP sp;
    SQ sq;
    sp.init(G.P, at0.p0, at0.ra);
    sq.init(G.Q, at0.q0, at0.ra);
    const int wave = threadIdx.x / 64;
    const int op = SP::frag(wave / WQ * (BT / WP)), oq = SP::BYTES + SQ::frag(wave % WQ * (BT / WQ));

    const int steps = (int)((at0.rb - at0.ra + BR - 1) / BR);
    auto load = [&](int s) {
        const uint32_t at = lds0 + s % BUFS * BUF;
        const int64_t r = at0.ra + (int64_t)s * BR, end = at0.rb;
        // a split ends at a multiple of BR or at R, so only R itself cuts a step short
        const int64_t lp = (end < G.R ? end : PA ? G.P.limit : G.R) - r, lq = (end < G.R ? end : QA ? G.Q.limit : G.R) - r;
        if (lp >= BR) sp.load_full(at, s * sp.step);
        else sp.load_part(at, s * sp.step, lp);
        if (lq >= BR) sq.load_full(at + SP::BYTES, s * sq.step);
        else sq.load_part(at + SP::BYTES, s * sq.step, lq);
    };
    v8 p0[FP], q0[FQ], p1[FP], q1[FQ];          // fragments of the first and the second 32 of a step
    struct From { uint32_t p, q; };
    auto from = [&](int s, int k) {
        const uint32_t at = lds0 + s % BUFS * BUF;
        return From{SP::from(at, op, k), SQ::from(at, oq, k)};
    };
    auto read_one = [&](v8 (&p)[FP], v8 (&q)[FQ], const From& f, int k, int i) {
        if (i < FQ) q[i] = SQ::template read<T>(f.q, i, k);
        else p[i - FQ] = SP::template read<T>(f.p, i - FQ, k);
    };
    auto read = [&](v8 (&p)[FP], v8 (&q)[FQ], int s, int k) {
        const From f = from(s, k);
#pragma unroll
        for (int i = 0; i < FP + FQ; ++i) read_one(p, q, f, k, i);
    };
    f32x4 acc[FP][FQ];
#pragma unroll
    for (int i = 0; i < FP; ++i)
#pragma unroll
        for (int j = 0; j < FQ; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    // 32 of the summed index multiplied, the next 32 read (k of step s) and, if `next` says so, step `fill` loaded.  Reads and loads stand between
    // the products, so that the matrix cores wait for neither's queue: with the loads of a step in a row the waves of a block stand
    // in front of the address unit together (8192 x 4096 x 4096 bf16, forward: loads in a row 224 us, between half of the products 209, between
    // all of them 202).
    auto half = [&](const v8 (&p)[FP], const v8 (&q)[FQ], v8 (&pn)[FP], v8 (&qn)[FQ], int s, int k, auto next, int fill) {
        constexpr bool LOAD = decltype(next)::value;
        constexpr int READS = FP + FQ, PER = (READS + FP - 3) / (FP - 2), PER_L = (LOADS + FP - 1) / FP;
        const From f = from(s, k);
        typename SP::u32x4 rp = {}, rq = {};
        uint32_t bp = 0, bq = 0;
        if (LOAD) {
            rp = sp.resource(fill * sp.step), rq = sq.resource(fill * sq.step);
            bp = SP::wave_base(lds0 + fill % BUFS * BUF), bq = SQ::wave_base(lds0 + fill % BUFS * BUF + SP::BYTES);
        }
#pragma unroll
        for (int i = 0; i < FP; ++i) {
            if (LOAD)
#pragma unroll
                for (int j = i * PER_L; j < (i + 1) * PER_L && j < LOADS; ++j) {
                    if (j < SP::LOADS) sp.load_one(j, bp, rp);
                    else sq.load_one(j - SP::LOADS, bq, rq);
                }
#pragma unroll
            for (int j = i * PER; j < (i + 1) * PER && j < READS; ++j) read_one(pn, qn, f, k, j);
#pragma unroll
            for (int j = 0; j < FQ; ++j) acc[i][j] = mma(q[j], p[i], acc[i][j]);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    auto multiply = [&](const v8 (&p)[FP], const v8 (&q)[FQ]) {
#pragma unroll
        for (int i = 0; i < FP; ++i)
#pragma unroll
            for (int j = 0; j < FQ; ++j) acc[i][j] = mma(q[j], p[i], acc[i][j]);
    };

    const bool touch = G.splits == 1 && A.res;
    auto scaled = [&](float by) {
#pragma unroll
        for (int i = 0; i < FP; ++i)
#pragma unroll
            for (int j = 0; j < FQ; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[i][j][e] *= by;
    };
    const bool pair = EPI == EPI_STORE && G.pair;
    if (pair) sp.corner += G.P.plane * 2;           // the second numbers first
#pragma unroll 1
    for (int pass = pair ? 2 : 1; pass > 0 && steps > 0; --pass) {
        if (pair && pass == 1) {
            wait_loads<0>();
            block_barrier();                        // all of the last step has been read
            sp.corner -= G.P.plane * 2;
            scaled(G.low);
        }
        for (int s = 0; s < BUFS && s < steps; ++s) load(s);
        if (steps >= BUFS) wait_loads<(BUFS - 1) * LOADS>();
        else wait_loads<0>();
        block_barrier();
        read(p0, q0, 0, 0);
        int s = 0;
        for (; s + BUFS + 1 < steps; ++s) {         // (step s + BUFS is not the last one, so it is whole)
            half(p0, q0, p1, q1, s, 1, std::false_type(), 0);
            wait_loads<(BUFS - 2) * LOADS>();
            block_barrier();                    // the next step's operands are in LDS, and all of this one's have been read
            half(p1, q1, p0, q0, s + 1, 0, std::true_type(), s + BUFS);
        }
        for (; s + 1 < steps; ++s) {
            half(p0, q0, p1, q1, s, 1, std::false_type(), 0);
            if (s + BUFS <= steps) wait_loads<(BUFS - 2) * LOADS>();
            else wait_loads<0>();
            block_barrier();
            if (s + BUFS < steps) load(s + BUFS);
            if (EPI == EPI_FWD && s + 2 == steps && touch) touch_residual<T, BT, BT, THREADS>(G, A, at0, lds0 + big_lds(BUFS, BUF, BT));
            half(p1, q1, p0, q0, s + 1, 0, std::false_type(), 0);
        }
        read(p1, q1, steps - 1, 1);
        multiply(p0, q0);
        multiply(p1, q1);
    }
    if (pair) {
        scaled(G.scale);
        if (again_if_needed<T, BT, BT, THREADS, PA ? MODE_DX : MODE_DW>(G, A, at0, acc, smem)) return;
    }
    finish<T, BT, BT, WP, WQ, EPI>(G, A, at0, acc, (float*)smem);
}

// fp32 in three bf16 parts.  BTP x BTQ tiles, 64 x 64 a wave, 32 of the summed index a step, all three parts of both operands in LDS:
// six products for each pair of fragments that is read.
template <int BTP, int BTQ, int BUFS, bool PA, bool QA, int EPI>
__device__ __forceinline__ void split_tile(const BigProduct& G, const LinArgs& A, int block, char* smem) {
    constexpr int WP = BTP / 64, WQ = BTQ / 64, THREADS = WP * WQ * 64, BR = 32;
    typedef Stage<BTP, BR, PA, true, THREADS> SP;
    typedef Stage<BTQ, BR, QA, true, THREADS> SQ;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_ptr)smem;
    constexpr int BUF = 3 * (SP::BYTES + SQ::BYTES), LOADS = 3 * (SP::LOADS + SQ::LOADS);
    const Place at0 = place<BTP, BTQ>(G, block);

    SP sp;
    SQ sq;
    sp.init(G.P, at0.p0, at0.ra);
    sq.init(G.Q, at0.q0, at0.ra);
    const int wave = threadIdx.x / 64, op = SP::frag(wave / WQ * 64), oq = 3 * SP::BYTES + SQ::frag(wave % WQ * 64);

    const int steps = (int)((at0.rb - at0.ra + BR - 1) / BR);
    auto load = [&](int s) {
        const uint32_t at = lds0 + s % BUFS * BUF;
        const int64_t r = at0.ra + (int64_t)s * BR, end = at0.rb;
        const int64_t lp = (end < G.R ? end : PA ? G.P.limit : G.R) - r, lq = (end < G.R ? end : QA ? G.Q.limit : G.R) - r;
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            const int64_t ap = k * G.P.plane * 2 + s * sp.step, aq = k * G.Q.plane * 2 + s * sq.step;
            if (lp >= BR) sp.load_full(at + k * SP::BYTES, ap);
            else sp.load_part(at + k * SP::BYTES, ap, lp);
            if (lq >= BR) sq.load_full(at + 3 * SP::BYTES + k * SQ::BYTES, aq);
            else sq.load_part(at + 3 * SP::BYTES + k * SQ::BYTES, aq, lq);
        }
    };

    f32x4 acc[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    bf16x8 p[3][4], q[2][3][2];                 // parts of the P fragments; parts of the Q fragments, two columns of tiles at a time
    auto read_p = [&](int s, int k) {
        const uint32_t from = SP::from(lds0 + s % BUFS * BUF, op, 0);
#pragma unroll
        for (int i = 0; i < 4; ++i) p[k][i] = SP::template read<bf16_t>(from, i, k);
    };
    auto read_q = [&](int s, int half) {
        const uint32_t from = SQ::from(lds0 + s % BUFS * BUF, oq, 0);
#pragma unroll
        for (int k = 0; k < 3; ++k)
#pragma unroll
            for (int j = 0; j < 2; ++j) q[half][k][j] = SQ::template read<bf16_t>(from, half * 2 + j, k);
    };
    f32x4 c[4][2];
    auto product = [&](int half, int kp, int kq, bool first) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) c[i][j] = mma(q[half][kq][j], p[kp][i], first ? f32x4{0.f, 0.f, 0.f, 0.f} : c[i][j]);
    };
    auto add = [&](int half, float sign) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[i][half * 2 + j][e] = __fmaf_rn(c[i][j][e], sign, acc[i][half * 2 + j][e]);
    };

    const bool touch = G.splits == 1 && A.res;
    if (steps > 0) {
        for (int s = 0; s < BUFS && s < steps; ++s) load(s);
        if (steps >= BUFS) wait_loads<(BUFS - 1) * LOADS>();
        else wait_loads<0>();
        block_barrier();
        read_p(0, 0), read_p(0, 1), read_p(0, 2), read_q(0, 0);
        auto first_half = [&](int s, float sign) {
            read_q(s, 1);
            product(0, 0, 2, true), product(0, 2, 0, false), product(0, 1, 1, false), product(0, 0, 1, false), product(0, 1, 0, false), product(0, 0, 0, false);
            add(0, sign);
            __builtin_amdgcn_sched_barrier(0);
        };
        float sign = 1.f;                       // (a split starts at a multiple of 64)
        // LOAD: step `fill` is loaded, piece by piece between the products.  The next step's P takes each part's registers as soon as its last
        // product is issued.
        auto second_half = [&](int s, float sign, auto what, int fill) {
            auto part = [&](int n, int kp, int kq) {          // the n-th of six products of the half
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (decltype(what)::value) {
#pragma unroll
                        for (int j = ((n * 4 + i) * LOADS + 23) / 24; j < ((n * 4 + i + 1) * LOADS + 23) / 24; ++j) {
                            const int k = j / (LOADS / 3), at = j % (LOADS / 3);
                            const uint32_t to = lds0 + fill % BUFS * BUF;
                            if (at < SP::LOADS) sp.load_one(at, SP::wave_base(to + k * SP::BYTES), sp.resource(k * G.P.plane * 2 + fill * sp.step));
                            else sq.load_one(at - SP::LOADS, SQ::wave_base(to + 3 * SP::BYTES + k * SQ::BYTES), sq.resource(k * G.Q.plane * 2 + fill * sq.step));
                        }
                    }
#pragma unroll
                    for (int j = 0; j < 2; ++j) c[i][j] = mma(q[1][kq][j], p[kp][i], n == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : c[i][j]);
                    if (decltype(what)::value) __builtin_amdgcn_sched_barrier(0);
                }
            };
            read_q(s + 1, 0);
            part(0, 0, 2), part(1, 2, 0);
            __builtin_amdgcn_sched_barrier(0);
            read_p(s + 1, 2);
            part(2, 1, 1), part(3, 1, 0);
            __builtin_amdgcn_sched_barrier(0);
            read_p(s + 1, 1);
            part(4, 0, 1), part(5, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
            read_p(s + 1, 0);
            add(1, sign);
        };
        int s = 0;
        for (; s + BUFS + 1 < steps; ++s) {         // (step s + BUFS is not the last one, so it is whole)
            first_half(s, sign);
            wait_loads<(BUFS - 2) * LOADS>();
            block_barrier();                    // the next step's operands are in LDS, and all of this one's have been read
            second_half(s, sign, std::true_type(), s + BUFS);
            sign = -sign;
        }
        for (; s + 1 < steps; ++s) {
            first_half(s, sign);
            if (s + BUFS <= steps) wait_loads<(BUFS - 2) * LOADS>();
            else wait_loads<0>();
            block_barrier();
            if (s + BUFS < steps) load(s + BUFS);
            if (EPI == EPI_FWD && s + 2 == steps && touch) touch_residual<float, BTP, BTQ, THREADS>(G, A, at0, lds0 + big_lds(BUFS, BUF, BTQ));
            second_half(s, sign, std::false_type(), 0);
            sign = -sign;
        }
        first_half(steps - 1, sign);
        product(1, 0, 2, true), product(1, 2, 0, false), product(1, 1, 1, false), product(1, 0, 1, false), product(1, 1, 0, false), product(1, 0, 0, false);
        add(1, sign);
    }

    if (again_if_needed<float, BTP, BTQ, THREADS, EPI == EPI_FWD ? MODE_FWD : PA ? MODE_DX : MODE_DW>(G, A, at0, acc, smem)) return;
    finish<float, BTP, BTQ, WP, WQ, EPI>(G, A, at0, acc, (float*)smem);
}

// One launch for both products of the backward pass: the first nx blocks are dx's.
template <typename T, int BT, int WP, int WQ, int BUFS>
__global__ __launch_bounds__(WP * WQ * 64, 2) void k_big_fwd(BigProduct G, LinArgs A) {
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    big_tile<T, BT, WP, WQ, BUFS, true, true, EPI_FWD>(G, A, blockIdx.x, smem);
}
template <typename T, int BT, int WP, int WQ, int BUFS>
__global__ __launch_bounds__(WP * WQ * 64, 2) void k_big_bwd(BigProduct X, int nx, BigProduct W, LinArgs A) {
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    if ((int)blockIdx.x < nx) big_tile<T, BT, WP, WQ, BUFS, true, false, EPI_STORE>(X, A, blockIdx.x, smem);
    else big_tile<T, BT, WP, WQ, BUFS, false, false, EPI_STORE>(W, A, blockIdx.x - nx, smem);
}
template <int BTP, int BTQ, int BUFS>
__global__ __launch_bounds__(BTP * BTQ / 64, 2) void k_split_fwd(BigProduct G, LinArgs A) {
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    split_tile<BTP, BTQ, BUFS, true, true, EPI_FWD>(G, A, blockIdx.x, smem);
}
template <int BTP, int BTQ, int BUFS>
__global__ __launch_bounds__(BTP * BTQ / 64, 2) void k_split_bwd(BigProduct X, int nx, BigProduct W, LinArgs A) {
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    if ((int)blockIdx.x < nx) split_tile<BTP, BTQ, BUFS, true, false, EPI_STORE>(X, A, blockIdx.x, smem);
    else split_tile<BTP, BTQ, BUFS, false, false, EPI_STORE>(W, A, blockIdx.x - nx, smem);
}

int64_t big_tiles(const BigProduct& B) { return ((B.p_end + B.tile_p - 1) / B.tile_p) * ((B.q_end + B.tile_q - 1) / B.tile_q); }
static int blocks_of(const BigProduct& B) { return (int)(big_tiles(B) * B.splits); }

template <typename F, typename... Args>
static hipError_t go(F fn, int bytes, int threads, SmemCache& cache, int blocks, hipStream_t st, Args... args) {
    const hipError_t e = set_smem((const void*)fn, bytes, cache);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(fn, dim3((unsigned)blocks), dim3(threads), bytes, st, args...);
    return hipGetLastError();
}
template <typename T, int BT, int WP, int WQ, int BUFS> struct Big16 {
    static constexpr int THREADS = WP * WQ * 64, LDS = big_lds(BUFS, 2 * BT * 64 * 2, BT) + THREADS * 4;
    static_assert(LDS >= THREADS / 256 * tile_lds<float>(), "a tile with a NaN is computed again here");
    static hipError_t fwd(const BigProduct& B, const LinArgs& A, hipStream_t st) {
        static SmemCache cache;
        return go(k_big_fwd<T, BT, WP, WQ, BUFS>, LDS, THREADS, cache, blocks_of(B), st, B, A);
    }
    static hipError_t bwd(const BigProduct& X, int nx, const BigProduct& W, int nw, const LinArgs& A, hipStream_t st) {
        static SmemCache cache;
        return go(k_big_bwd<T, BT, WP, WQ, BUFS>, LDS, THREADS, cache, nx + nw, st, X, nx, W, A);
    }
};
template <int BTP, int BTQ, int BUFS> struct Big32 {
    static constexpr int THREADS = BTP * BTQ / 64, LDS = big_lds(BUFS, 3 * (BTP + BTQ) * 32 * 2, BTQ) + THREADS * 4;
    static_assert(LDS >= THREADS / 256 * tile_lds<float>(), "a tile with a NaN is computed again here");
    static hipError_t fwd(const BigProduct& B, const LinArgs& A, hipStream_t st) {
        static SmemCache cache;
        return go(k_split_fwd<BTP, BTQ, BUFS>, LDS, THREADS, cache, blocks_of(B), st, B, A);
    }
    static hipError_t bwd(const BigProduct& X, int nx, const BigProduct& W, int nw, const LinArgs& A, hipStream_t st) {
        static SmemCache cache;
        return go(k_split_bwd<BTP, BTQ, BUFS>, LDS, THREADS, cache, nx + nw, st, X, nx, W, A);
    }
};
// 128 x 128 tiles of 16-bit types: up to one block a CU has four buffers (its loads are three steps ahead: such products wait for
// memory, not for the matrix cores), more have two, and two blocks share a CU.
template <typename T, typename... Args> static hipError_t fwd16(int blocks, int tile, Args... a) {
    if (tile == 256) return Big16<T, 256, 2, 4, 2>::fwd(a...);
    return blocks <= 256 ? Big16<T, 128, 2, 2, 4>::fwd(a...) : Big16<T, 128, 2, 2, 2>::fwd(a...);
}
template <typename T, typename... Args> static hipError_t bwd16(int blocks, int tile, Args... a) {
    if (tile == 256) return Big16<T, 256, 2, 4, 2>::bwd(a...);
    return blocks <= 256 ? Big16<T, 128, 2, 2, 4>::bwd(a...) : Big16<T, 128, 2, 2, 2>::bwd(a...);
}
hipError_t big_forward_launch(const BigProduct& B, const LinArgs& A, int dtype, hipStream_t st) {
    if (dtype == IVAE_F32) return B.tile_p == 256 ? Big32<256, 128, 2>::fwd(B, A, st) : Big32<128, 128, 3>::fwd(B, A, st);
    if (dtype == IVAE_BF16) return fwd16<bf16_t>(blocks_of(B), B.tile_p, B, A, st);
    return fwd16<f16_t>(blocks_of(B), B.tile_p, B, A, st);
}
hipError_t big_backward_launch(const BigProduct& X, const BigProduct& W, const LinArgs& A, int dtype, hipStream_t st) {
    const int nx = A.dx ? blocks_of(X) : 0, nw = A.dw ? blocks_of(W) : 0;
    if (nx + nw == 0) return hipSuccess;
    if (dtype == IVAE_F32) return X.tile_p == 256 ? Big32<256, 128, 2>::bwd(X, nx, W, nw, A, st) : Big32<128, 128, 3>::bwd(X, nx, W, nw, A, st);
    if (dtype == IVAE_BF16) return bwd16<bf16_t>(nx + nw, X.tile_p, X, nx, W, nw, A, st);
    return bwd16<f16_t>(nx + nw, X.tile_p, X, nx, W, nw, A, st);
}
