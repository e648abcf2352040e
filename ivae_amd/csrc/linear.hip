// Dispatch of the linear operator (ivae_linear, ivae_linear_backward) to its kernels.
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

static bool big_product(int64_t P, int64_t Q, int64_t R) {
    return P >= 64 && Q >= 64 && R >= 64 && 2.0 * (double)P * (double)Q * (double)R >= 5e8;
}
static int64_t tiles_of(const BigProduct& B, int tp, int tq) { return ((B.p_end + tp - 1) / tp) * ((B.q_end + tq - 1) / tq); }
static void big_geometry(BigProduct& B, int dtype) {
    const int wide = dtype == IVAE_F32 ? 128 : 256;
    const bool large = tiles_of(B, 256, wide) >= (dtype == IVAE_F32 ? 96 : 192);
    B.tile_p = large ? 256 : 128;
    B.tile_q = large ? wide : 128;
    const int64_t tiles = tiles_of(B, B.tile_p, B.tile_q);
    int64_t s = tiles < 256 ? (large ? 256 : 512) / tiles : 1;
    const int64_t most = B.R / 512;
    if (s > most) s = most;
    if (s > 32) s = 32;
    if (s < 1) s = 1;
    B.len = ((B.R + s - 1) / s + 63) / 64 * 64;
    B.splits = (int)((B.R + B.len - 1) / B.len);
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
static int64_t up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

// A matrix as an operand: in place where its rows are 16-byte groups already, packed otherwise (fp32 always)
struct Packed { BigOperand O; PackArgs P; bool needed; };
static Packed pack_of(const void* src, int64_t rows, int cols, int64_t ld, int dtype, Bytes& ws, bool must = false) {
    Packed r = {};
    r.needed = must || dtype == IVAE_F32 || ld % 8 != 0 || cols % 8 != 0;
    if (!r.needed) {
        r.O = {src, ld, 0, 0, 0, false};
        r.P.ldo = cols;
        return r;
    }
    const int64_t ldo = up(cols, 64), plane = rows * ldo;
    void* out = ws.take<uint16_t>(plane * (dtype == IVAE_F32 ? 3 : 1));
    r.P.src = src; r.P.out = out; r.P.rows = rows; r.P.cols = cols; r.P.ld = ld; r.P.ldo = ldo; r.P.plane = plane;
    r.O = {out, ldo, 0, 0, plane, false};
    return r;
}
// rows are what the product has as rows or columns, the summed index runs along them / down the rows
static BigOperand along(const Packed& p, int64_t rows) {
    BigOperand o = p.O;
    o.along = true; o.extent = rows; o.limit = p.P.ldo;
    return o;
}
static BigOperand down(const Packed& p, int64_t rows) {
    BigOperand o = p.O;
    o.along = false; o.extent = p.P.ldo; o.limit = rows;
    return o;
}

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
    B.epi = EPI_FWD;
    big_geometry(B, dtype);
    if (B.splits > 1) B.part = m.take<float>(B.splits * A.M * A.N);
    if (dtype == IVAE_F32) B.nan_seen = m.take<int>(big_tiles(B) * B.splits);
    f.bytes = m.used;
    return f;
}
static hipError_t big_forward(LinArgs A, int dtype, void* ws, hipStream_t st) {
    const BigForward f = plan_big_forward(A, dtype, ws);
    hipError_t e = hipSuccess;
    if (f.x.needed) e = launch_pack(f.x.P, dtype, st);
    if (e == hipSuccess && f.w.needed) e = launch_pack(f.w.P, dtype, st);
    if (e == hipSuccess) e = big_launch(f.B, A, dtype, st);
    A.part = f.B.part;
    if (e == hipSuccess) e = linear_join_forward(A, f.B.splits, dtype, st);
    if (e == hipSuccess && dtype == IVAE_F32) e = linear_mend_forward(A, {f.B.nan_seen, f.B.tile_p, f.B.tile_q, f.B.splits}, st);
    return e;
}

struct BigBackward { Packed ds, x, w; BigProduct X, W; float* colsum; int kb; size_t bytes; };
static BigBackward plan_big_backward(const LinArgs& A, int dtype, void* ws) {
    BigBackward f = {};
    Bytes m = {(char*)ws, 0};
    f.ds = pack_of(A.dy, A.M, A.N, A.lddy, dtype, m, A.act != IVAE_ACT_NONE);
    f.ds.P.pre = A.act != IVAE_ACT_NONE ? A.cpre : nullptr;
    f.ds.P.act = A.act; f.ds.P.slope = A.slope;
    if (!f.ds.needed) {                                 // dy itself; only its column sums are taken
        f.ds.P.src = A.dy; f.ds.P.rows = A.M; f.ds.P.cols = A.N; f.ds.P.ld = A.lddy; f.ds.P.ldo = A.N;
    }
    f.kb = pack_row_blocks(A.M, f.ds.P.ldo);
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
    for (BigProduct* B : both) {
        B->epi = EPI_STORE;
        big_geometry(*B, dtype);
        if (B->splits > 1) B->part = m.take<float>(B->splits * B->p_end * B->q_end);
        if (dtype == IVAE_F32) B->nan_seen = m.take<int>(big_tiles(*B) * B->splits);
    }
    f.bytes = m.used;
    return f;
}
static hipError_t big_backward(const LinArgs& A, int dtype, void* ws, hipStream_t st) {
    BigBackward f = plan_big_backward(A, dtype, ws);
    hipError_t e = hipSuccess;
    f.ds.P.colsum = A.db ? f.colsum : nullptr;
    if (f.ds.needed || A.db) e = launch_pack(f.ds.P, dtype, st);
    if (e == hipSuccess && A.dx && f.w.needed) e = launch_pack(f.w.P, dtype, st);
    if (e == hipSuccess && A.dw && f.x.needed) e = launch_pack(f.x.P, dtype, st);
    if (e == hipSuccess && A.dx) e = big_launch(f.X, A, dtype, st);
    if (e == hipSuccess && A.dw) e = big_launch(f.W, A, dtype, st);
    if (e == hipSuccess) e = linear_join_backward(A, {f.X.part, f.W.part, f.colsum, f.X.splits, f.W.splits, f.kb}, dtype, st);
    if (e == hipSuccess && dtype == IVAE_F32)
        e = linear_mend_backward(A, {f.X.nan_seen, f.X.tile_p, f.X.tile_q, f.X.splits}, {f.W.nan_seen, f.W.tile_p, f.W.tile_q, f.W.splits}, st);
    return e;
}

// ---- which kernel -----------------------------------------------------------------------------------------------------
static bool aligned(const void* p) { return (uintptr_t)p % 16 == 0; }
static bool big_by_size(const LinArgs& A, bool backward) {
    const int64_t lds[] = {A.ldx, A.lddy, A.K, A.N};
    for (int64_t ld : lds)
        if (ld > BIG_MAX_LD) return false;
    return big_product(A.M, A.N, A.K) && (!backward || A.M > 0);
}
// a matrix that would be loaded in place has to start on 16 bytes
static bool big_in_place(const void* p, int64_t cols, int64_t ld, int dtype) { return dtype == IVAE_F32 || ld % 8 || cols % 8 || aligned(p); }

size_t linear_ws_bytes(const IvaeLinear& L, bool backward) {
    LinArgs A = lin_args(L);
    A.dx = A.dw = A.db = &A;           // the size serves a call that asks for all of them
    if (!backward && A.M <= ROWS_MAX) return rows_ws(A);
    size_t n = linear_small_ws(A, backward);
    if (big_by_size(A, backward)) {
        const size_t big = backward ? plan_big_backward(A, L.dtype, nullptr).bytes : plan_big_forward(A, L.dtype, nullptr).bytes;
        if (big > n) n = big;
    }
    return n;
}
hipError_t launch_linear(const IvaeLinear& L, const void* x, const void* w, const void* b, const void* residual, void* y, void* saved,
                         void* ws, hipStream_t st) {
    LinArgs A = lin_args(L);
    A.x = x; A.w = w; A.b = b; A.res = residual; A.y = y; A.pre = saved; A.part = (float*)ws;
    if (A.M <= ROWS_MAX) return linear_rows_forward(A, L.dtype, st);
    if (big_by_size(A, false) && big_in_place(x, A.K, A.ldx, L.dtype) && big_in_place(w, A.K, A.K, L.dtype) && aligned(ws))
        return big_forward(A, L.dtype, ws, st);
    return linear_small_forward(A, L.dtype, st);
}
hipError_t launch_linear_backward(const IvaeLinear& L, const void* dy, const void* x, const void* w, const void* saved, void* dx, void* dw,
                                  void* db, void* ws, hipStream_t st) {
    LinArgs A = lin_args(L);
    A.x = x; A.w = w; A.dy = dy; A.cpre = saved; A.dx = dx; A.dw = dw; A.db = db; A.part = (float*)ws;
    if (big_by_size(A, true) && (A.act != IVAE_ACT_NONE || big_in_place(dy, A.N, A.lddy, L.dtype)) && (!dw || big_in_place(x, A.K, A.ldx, L.dtype)) &&
        (!dx || big_in_place(w, A.K, A.K, L.dtype)) && aligned(ws))
        return big_backward(A, L.dtype, ws, st);
    return linear_small_backward(A, L.dtype, st);
}
