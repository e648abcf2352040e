// Interface of the large-product kernels (linear_big.hip).
#pragma once
#include "linear.h"

// One operand of a product C[p][q] = sum_r P(p, r) Q(q, r), in memory as a row-major 16-bit matrix.
//   along = true:  (extent, R): the summed index runs along a row;   along = false: (R, extent): it runs down the rows
// Rows start at multiples of 16 bytes and hold whole 16-byte groups.  Split fp32 is stored in columns of 32 values, ld rows each
// (value (r, c) at (c / 32 * ld + r) * 32 + c % 32): what a step loads of a tile lies in one piece, or (down) in pieces of 2 KB, where
// rows of 64 bytes out of a row-major matrix would use half of each cache line.  `limit` is the end of the stored values along R (a multiple
// of 8 where `along`; values between R and limit are 0).  Split fp32: of every second 32 along R, Q has its sign turned.
// `plane`: elements between the three parts of split fp32 values, or the two numbers of a pair.  `range`: PackArgs' of split fp32.
struct BigOperand {
    const void* base;
    int64_t ld, extent, limit, plane;
    bool along;
    const uint2* range;
    int ranges;
};

enum { EPI_FWD, EPI_STORE };    // what follows the sums: forward_store's, or a store of the result type

struct BigProduct {
    BigOperand P, Q;
    int64_t p_end, q_end, R;    // size of C and of the sum
    void* out;                  // backward pass: (p_end, q_end) of the tensors' type
    float* part;                // split sums: (splits, p_end, q_end)
    int tile_p, tile_q;         // 16-bit types: 256 x 256 or 128 x 128; fp32: 256 x 128 or 128 x 128
    int splits;
    int64_t len;                // R of a split, a multiple of 64
    bool pair;                  // 16-bit types: P's values are scale (first + low second), two numbers of the type
    float scale, low;           // powers of two
};

int64_t big_tiles(const BigProduct& B);
// dtype: of the tensors (fp32: operands are split bf16).  The two products of a backward pass have tiles of one size.
hipError_t big_forward_launch(const BigProduct& B, const LinArgs& A, int dtype, hipStream_t st);
hipError_t big_backward_launch(const BigProduct& X, const BigProduct& W, const LinArgs& A, int dtype, hipStream_t st);
