// Dispatch of the linear operator (ivae_linear, ivae_linear_backward) to its kernels.
#include "kernels.h"
#include "linear.h"

static LinArgs lin_args(const IvaeLinear& L) {
    LinArgs A = {};
    A.M = L.rows; A.K = L.in_features; A.N = L.out_features;
    A.ldx = L.ldx; A.ldr = L.ld_residual; A.lddy = L.lddy;
    A.act = L.activation; A.slope = L.slope;
    return A;
}
size_t linear_ws_bytes(const IvaeLinear& L, bool backward) {
    LinArgs A = lin_args(L);
    A.dx = A.dw = A.db = &A;           // the size serves a call that asks for all of them
    return linear_small_ws(A, backward);
}
hipError_t launch_linear(const IvaeLinear& L, const void* x, const void* w, const void* b, const void* residual, void* y, void* saved,
                         void* ws, hipStream_t st) {
    LinArgs A = lin_args(L);
    A.x = x; A.w = w; A.b = b; A.res = residual; A.y = y; A.pre = saved; A.part = (float*)ws;
    return linear_small_forward(A, L.dtype, st);
}
hipError_t launch_linear_backward(const IvaeLinear& L, const void* dy, const void* x, const void* w, const void* saved, void* dx, void* dw,
                                  void* db, void* ws, hipStream_t st) {
    LinArgs A = lin_args(L);
    A.x = x; A.w = w; A.dy = dy; A.cpre = saved; A.dx = dx; A.dw = dw; A.db = db; A.part = (float*)ws;
    return linear_small_backward(A, L.dtype, st);
}
