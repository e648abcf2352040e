// Dispatch of the linear operator (ivae_linear, ivae_linear_backward) to its kernels.
#include <math.h>

#include "kernels.h"
#include "linear_big.h"
#include "linear_pack.h"
#include "linear_rows.h"

static LinArgs lin_args(const IvaeLinear& L) {
    LinArgs A = {};
    A.M = L.rows; A.K = L.in_features; A.N = L.out_features;
    A.ldx = L.ldx; A.ldr = L.ld_residual; A.lddy = L.lddy;
    A.act = L.activation; A.slope = L.slope;
    return A;
}

// ---- large products -------------------------------------------------------------------------------------------------
static const int64_t BIG_MAX_LD = 1 << 21;              // 32-bit byte offsets inside a tile of 256 rows

static int64_t up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }
static int64_t tiles_of(const BigProduct& B, int tp, int tq) { return ((B.p_end + tp - 1) / tp) * ((B.q_end + tq - 1) / tq); }
// Tiles and splits of the products of one launch: the choice for which a simple model of its time is least.  A round of 256 blocks, one a
// CU, takes `start` us (those after the first `again` of it) and `per` ns for each of its summed index (fitted to products of one to four
// rounds: 16 bits, 256 x 256 and 128 x 128 tiles, the small ones two a CU; split fp32, 256 x 128 and 128 x 128); a pair's sum is twice as long; split sums cost a launch
// and are joined at 6 TB/s.  What it decides between (us, forward, 256-wide | 128-wide): fp16 4096 x 4096 x 4096 114 | 136,
// 4096 x 2048 x 2048 53 | 42, 8192 x 1024 x 1024 36 | 26; fp32 4096 x 1024 x 4096 197 | 216, 2048 x 2048 x 2048 118 | 109.
struct BigModel { int tile_p, tile_q; double start, again, per; };
static double big_time(BigProduct** B, int n, const BigModel& m, const int64_t* s) {
    double load = 0, longest = 0, join = 0;
    int64_t blocks = 0;
    for (int i = 0; i < n; ++i) {
        const int64_t tiles = tiles_of(*B[i], m.tile_p, m.tile_q) * s[i], len = (B[i]->R + s[i] - 1) / s[i] * (B[i]->pair ? 2 : 1);
        load += (double)tiles * (double)len;
        blocks += tiles;
        if ((double)len > longest) longest = (double)len;
        if (s[i] > 1) join += 4.0 + ((double)s[i] + 0.5) * (double)B[i]->p_end * (double)B[i]->q_end * 4 / 6e6;
    }
    const double rounds = (double)((blocks + 255) / 256), each = blocks ? rounds * load / (double)blocks : 0;
    return m.start * (1 + m.again * (rounds - 1)) + 1e-3 * m.per * (each > longest ? each : longest) + join;
}
static void big_geometry(BigProduct** B, int n, int dtype) {
    static const BigModel m16[2] = {{256, 256, 15.0, 0.3, 24.5}, {128, 128, 10.0, 0.1, 7.6}};
    static const BigModel m32[2] = {{256, 128, 20.0, 0.5, 72.0}, {128, 128, 14.0, 0.5, 41.0}};
    double best = 1e30;
    for (const BigModel& m : dtype == IVAE_F32 ? m32 : m16)
        for (int64_t s0 = 1; s0 <= 16; s0 *= 2)
            for (int64_t s1 = 1; s1 <= (n == 2 ? 16 : 1); s1 *= 2) {
                const int64_t s[2] = {s0, s1};
                if ((s0 > 1 && B[0]->R / s0 < 192) || (n == 2 && s1 > 1 && B[1]->R / s1 < 192)) continue;
                const double t = big_time(B, n, m, s);
                if (t >= best) continue;
                best = t;
                for (int i = 0; i < n; ++i) {
                    B[i]->tile_p = m.tile_p;
                    B[i]->tile_q = m.tile_q;
                    B[i]->len = up((B[i]->R + s[i] - 1) / s[i], 64);
                    B[i]->splits = (int)((B[i]->R + B[i]->len - 1) / B[i]->len);
                }
            }
}

struct Bytes {                                          // a workspace, handed out in pieces of 256 bytes
    char* base;
    size_t used;
    template <typename T> T* take(int64_t n) {
        T* p = (T*)(base ? base + used : nullptr);
        used += ((size_t)n * sizeof(T) + 255) / 256 * 256;
        return p;
    }
};

// (a job's blocks, with column sums or without)
static int max_ranges(int64_t rows, int64_t ldo) {
    const int a = pack_blocks(rows, ldo, false, IVAE_F32), b = pack_blocks(rows, ldo, true, IVAE_F32);
    return a > b ? a : b;
}
// A matrix as an operand: in place where its rows are 16-byte groups already, packed otherwise (fp32 always)
struct Packed { BigOperand O; PackArgs P; bool needed; };
static Packed pack_of(const void* src, int64_t rows, int cols, int64_t ld, int dtype, Bytes& ws, bool pair = false) {
    Packed r = {};
    r.needed = pair || dtype == IVAE_F32 || ld % 8 != 0 || cols % 8 != 0;
    if (!r.needed) {
        r.O = {src, ld, 0, 0, 0, false};
        r.P.ldo = cols;
        return r;
    }
    const int64_t ldo = up(cols, 64), plane = rows * ldo;           // (fp32: columns of 32, `rows` long each)
    void* out = ws.take<uint16_t>(plane * (dtype == IVAE_F32 ? 3 : pair ? 2 : 1));
    r.P.src = src; r.P.out = out; r.P.rows = rows; r.P.cols = cols; r.P.ld = ld; r.P.ldo = ldo; r.P.plane = plane; r.P.pair = pair;
    r.O = {out, dtype == IVAE_F32 ? rows : ldo, 0, 0, plane, false};
    if (dtype == IVAE_F32) r.P.range = ws.take<uint2>(max_ranges(rows, ldo));
    return r;
}
// rows are what the product has as rows or columns, the summed index runs along them / down the rows
static BigOperand along(const Packed& p, int64_t rows) {
    BigOperand o = p.O;
    o.along = true; o.extent = rows; o.limit = p.P.ldo;
    o.range = p.P.range;
    return o;
}
static BigOperand down(const Packed& p, int64_t rows) {
    BigOperand o = p.O;
    o.along = false; o.extent = p.P.ldo; o.limit = rows;
    o.range = p.P.range;
    return o;
}

static int ranges_of(const Packed& p, int dtype) { return dtype == IVAE_F32 ? pack_blocks(p.P.rows, p.P.ldo, p.P.colsum != nullptr, dtype) : 0; }

struct BigForward { Packed x, w; BigProduct B; size_t bytes; };
static BigForward plan_big_forward(const LinArgs& A, int dtype, void* ws) {
    BigForward f = {};
    Bytes m = {(char*)ws, 0};
    f.x = pack_of(A.x, A.M, A.K, A.ldx, dtype, m);
    f.w = pack_of(A.w, A.N, A.K, A.K, dtype, m);
    BigProduct& B = f.B;
    f.w.P.flip = FLIP_COLS;
    B.P = along(f.x, A.M);
    B.Q = along(f.w, A.N);
    B.p_end = A.M; B.q_end = A.N; B.R = A.K;
    BigProduct* one[1] = {&B};
    big_geometry(one, 1, dtype);
    if (B.splits > 1) B.part = m.take<float>(B.splits * A.M * A.N);
    f.bytes = m.used;
    return f;
}
static hipError_t big_forward(LinArgs A, int dtype, void* ws, hipStream_t st) {
    BigForward f = plan_big_forward(A, dtype, ws);
    hipError_t e = hipSuccess;
    f.B.P.ranges = ranges_of(f.x, dtype), f.B.Q.ranges = ranges_of(f.w, dtype);
    const PackArgs* packs[2] = {f.x.needed ? &f.x.P : nullptr, f.w.needed ? &f.w.P : nullptr};
    e = launch_packs(packs, 2, dtype, st);
    if (e == hipSuccess) e = big_forward_launch(f.B, A, dtype, st);
    A.part = f.B.part;
    if (e == hipSuccess) e = linear_join_forward(A, f.B.splits, dtype, st);
    return e;
}

// |act'(s)| <= 2^shift (0 at least).  fp16 pairs serve up to SHIFT_MAX: each more costs the smallest gradients a bit.
static const int SHIFT_MAX = 4;
static float slope_bound(int act, float slope) {
    switch (act) {
        case IVAE_ACT_LRELU: return fmaxf(1.f, fabsf(slope));
        case IVAE_ACT_XTANH: return fmaxf(fabsf(slope), fabsf(1.f + slope));
        case IVAE_ACT_GELU: return 1.13f;
        case IVAE_ACT_SILU: return 1.1f;
        default: return 1.f;
    }
}
static int slope_shift(int act, float slope) {
    const float c = slope_bound(act, slope);
    int e = 0;
    while (e < SHIFT_MAX && c > (float)(1 << e)) ++e;
    return e;
}
struct BigBackward { Packed ds, x, w; BigProduct X, W; float* colsum; int kb; size_t bytes; };
static BigBackward plan_big_backward(const LinArgs& A, int dtype, void* ws) {
    BigBackward f = {};
    Bytes m = {(char*)ws, 0};
    const bool pair = dtype != IVAE_F32 && A.act != IVAE_ACT_NONE;
    f.ds = pack_of(A.dy, A.M, A.N, A.lddy, dtype, m, pair);
    const int shift = dtype == IVAE_F16 ? slope_shift(A.act, A.slope) : 0;
    f.ds.P.scale = ldexpf(1.f, -shift); f.ds.P.up = dtype == IVAE_F16 ? 2048.f : 128.f;
    f.ds.P.pre = A.act != IVAE_ACT_NONE ? A.cpre : nullptr;
    f.ds.P.act = A.act; f.ds.P.slope = A.slope;
    if (!f.ds.needed) {                                 // dy itself; only its column sums are taken
        f.ds.P.src = A.dy; f.ds.P.rows = A.M; f.ds.P.cols = A.N; f.ds.P.ld = A.lddy; f.ds.P.ldo = A.N;
    }
    f.kb = pack_row_blocks(A.M, f.ds.P.ldo, true, dtype);
    f.colsum = m.take<float>((int64_t)f.kb * A.N);
    f.x = pack_of(A.x, A.M, A.K, A.ldx, dtype, m);
    f.w = pack_of(A.w, A.N, A.K, A.K, dtype, m);
    f.x.P.flip = f.w.P.flip = FLIP_ROWS;
    BigProduct& X = f.X;
    X.P = along(f.ds, A.M);
    X.Q = down(f.w, A.N);
    X.p_end = A.M; X.q_end = A.K; X.R = A.N;
    X.out = A.dx;
    BigProduct& W = f.W;
    W.P = down(f.ds, A.M);
    W.Q = down(f.x, A.M);
    W.p_end = A.N; W.q_end = A.K; W.R = A.M;
    W.out = A.dw;
    BigProduct* both[2] = {&X, &W};
    for (BigProduct* B : both) B->pair = pair, B->scale = ldexpf(1.f, shift), B->low = 1.f / f.ds.P.up;
    big_geometry(both, 2, dtype);
    for (BigProduct* B : both) {
        if (B->splits > 1) B->part = m.take<float>(B->splits * B->p_end * B->q_end);
    }
    f.bytes = m.used;
    return f;
}
static hipError_t big_backward(const LinArgs& A, int dtype, void* ws, hipStream_t st) {
    BigBackward f = plan_big_backward(A, dtype, ws);
    hipError_t e = hipSuccess;
    f.ds.P.colsum = A.db ? f.colsum : nullptr;
    f.X.P.ranges = f.W.P.ranges = ranges_of(f.ds, dtype);
    f.X.Q.ranges = ranges_of(f.w, dtype), f.W.Q.ranges = ranges_of(f.x, dtype);
    const PackArgs* packs[3] = {f.ds.needed || A.db ? &f.ds.P : nullptr, A.dx && f.w.needed ? &f.w.P : nullptr, A.dw && f.x.needed ? &f.x.P : nullptr};
    e = launch_packs(packs, 3, dtype, st);
    if (e == hipSuccess) e = big_backward_launch(f.X, f.W, A, dtype, st);
    if (e == hipSuccess) e = linear_join_backward(A, {f.X.part, f.W.part, f.colsum, f.X.splits, f.W.splits, f.kb}, dtype, st);
    return e;
}

// ---- which kernel -----------------------------------------------------------------------------------------------------
static bool aligned(const void* p) { return (uintptr_t)p % 16 == 0; }
// The large kernels from the size on from which they take less time, all their launches together (us, small | large):
//   16 bits, forward    256 x 2048 x 2048 20 | 23, 1024 x 1024 x 1024 18 | 14, 65 x 4096 x 4096 31 | 18, 2048 x 1024 x 1024 24 | 14
//                       odd sizes 701 x 701 x 701 16 | 17, 803 x 803 x 803 19 | 18, 1003 x 901 x 777 24 | 20, 65 x 4099 x 4099 51 | 35
//                       (but 129 x 2003 x 2003 20 | 28)
//   16 bits, backward   no activation 512 x 512 x 512 13 | 14, 1024 x 512 x 512 16 | 20, 1003 x 777 x 531 28 | 25, 768 x 768 x 768 24 | 17
//                       gelu (the small kernel in fp32, the large one in pairs) 512 x 512 x 512 20 | 22, 300 x 1001 x 777 34 | 23,
//                       1024 x 512 x 512 31 | 27, 1024 x 1024 x 1024 84 | 36
//   fp32, forward       1024 x 1024 x 1024 28 | 39, 2048 x 1024 x 1024 45 | 49, 1024 x 2048 x 1024 51 | 49, 300 x 4096 x 2048 81 | 75, 128 x
//                       4096 x 4096 49 | 68 (cutting the weight in three costs as much as a product with 128 rows)
//                       odd sizes 803 x 803 x 803 29 | 37, 1003 x 901 x 777 37 | 36, 1003 x 1001 x 1003 46 | 38
//   fp32, backward      512 x 512 x 512 25 | 27, 1024 x 512 x 512 36 | 30, 1024 x 1024 x 1024 96 | 47
// Forward, rows that do not start on 16 bytes cost the small kernel twice the loads, the large one only its packing.
static bool big_by_size(const LinArgs& A, int dtype, bool backward) {
    const int64_t lds[] = {A.ldx, A.lddy, A.K, A.N};
    for (int64_t ld : lds)
        if (ld > BIG_MAX_LD) return false;
    // (blocks are counted, and bytes inside a tile of fp32 columns offset, in 32 bits)
    if (A.M < 64 || A.N < 64 || A.K < 64 || A.M >= (dtype == IVAE_F32 ? 1 << 22 : 1 << 29)) return false;
    if (backward && dtype == IVAE_F16 && !(isfinite(A.slope) && slope_bound(A.act, A.slope) <= (float)(1 << SHIFT_MAX))) return false;
    const double flops = 2.0 * (double)A.M * (double)A.N * (double)A.K;
    const bool ragged = A.K % (dtype == IVAE_F32 ? 4 : 8) != 0;
    if (dtype == IVAE_F32) return backward ? flops >= 5e8 : flops >= (ragged ? 1.4e9 : 5e9) && A.M >= 256;
    if (backward) return flops >= (A.act == IVAE_ACT_NONE ? 8e8 : 3e8);
    return flops >= (ragged ? 1e9 : 2.1e9);
}
// a matrix that would be loaded in place has to start on 16 bytes
static bool big_in_place(const void* p, int64_t cols, int64_t ld, int dtype) { return dtype == IVAE_F32 || ld % 8 || cols % 8 || aligned(p); }

size_t linear_ws_bytes(const IvaeLinear& L, bool backward) {
    LinArgs A = lin_args(L);
    A.dx = A.dw = A.db = &A;           // the size serves a call that asks for all of them
    if (!backward && rows_serve(A, L.dtype)) return rows_ws(A);
    size_t n = linear_small_ws(A, backward);
    if (big_by_size(A, L.dtype, backward)) {
        const size_t big = backward ? plan_big_backward(A, L.dtype, nullptr).bytes : plan_big_forward(A, L.dtype, nullptr).bytes;
        if (big > n) n = big;
    }
    return n;
}
void linear_plan(const IvaeLinear& L, bool backward, int32_t (&out)[5]) {
    LinArgs A = lin_args(L);
    A.dx = A.dw = A.db = &A;
    if (!backward && rows_serve(A, L.dtype)) {
        const RowsPlan p = rows_plan(A);
        out[1] = 16 * p.nf;
        out[2] = p.splits;
    } else if (!big_by_size(A, L.dtype, backward)) {
        out[0] = 1;
        out[1] = 64;
        linear_small_splits(A, backward, out + 2);
    } else {
        out[0] = 2;
        const BigForward f = backward ? BigForward{} : plan_big_forward(A, L.dtype, nullptr);
        const BigBackward g = backward ? plan_big_backward(A, L.dtype, nullptr) : BigBackward{};
        const BigProduct& B = backward ? g.X : f.B;
        out[1] = B.tile_p;
        out[2] = B.splits;
        out[3] = backward ? g.W.splits : 0;
        out[4] = (int32_t)(big_tiles(B) * B.splits + (backward ? big_tiles(g.W) * g.W.splits : 0));
    }
}
hipError_t launch_linear(const IvaeLinear& L, const void* x, const void* w, const void* b, const void* residual, void* y, void* saved,
                         void* ws, hipStream_t st) {
    LinArgs A = lin_args(L);
    A.x = x; A.w = w; A.b = b; A.res = residual; A.y = y; A.pre = (float*)saved; A.part = (float*)ws;
    if (rows_serve(A, L.dtype)) return linear_rows_forward(A, L.dtype, st);
    if (big_by_size(A, L.dtype, false) && big_in_place(x, A.K, A.ldx, L.dtype) && big_in_place(w, A.K, A.K, L.dtype) && aligned(ws))
        return big_forward(A, L.dtype, ws, st);
    return linear_small_forward(A, L.dtype, st);
}
hipError_t launch_linear_backward(const IvaeLinear& L, const void* dy, const void* x, const void* w, const void* saved, void* dx, void* dw,
                                  void* db, void* ws, hipStream_t st) {
    LinArgs A = lin_args(L);
    A.x = x; A.w = w; A.dy = dy; A.cpre = (const float*)saved; A.dx = dx; A.dw = dw; A.db = db; A.part = (float*)ws;
    if (big_by_size(A, L.dtype, true) && (A.act != IVAE_ACT_NONE || big_in_place(dy, A.N, A.lddy, L.dtype)) && (!dw || big_in_place(x, A.K, A.ldx, L.dtype)) &&
        (!dx || big_in_place(w, A.K, A.K, L.dtype)) && aligned(ws))
        return big_backward(A, L.dtype, ws, st);
    return linear_small_backward(A, L.dtype, st);
}
